"""Packed attention where V holds Inf or NaN: what a row sees stays in its result, what it does not see stays out, and neither takes long."""
import pytest
import torch

from kv4_ref import HALF

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def _cu(lens, dev):
    return torch.cumsum(torch.tensor([0] + list(lens)), 0).int().to(dev)


def _check_rows(got, q, k, v, past, picked, scale=128 ** -0.5):
    """Rows `picked` of one sequence behind `past` keys, in 64 bits: dims in which a visible V row is not finite are not finite, all others are within
    the bound of the packed tests (a rounding of the result, one of each p, the scores' cut-offs)."""
    dtype, group = q.dtype, q.shape[1] // k.shape[1]
    for h in range(q.shape[1]):
        kk, vv = k[:, h // group].double(), v[:, h // group].double()
        bad = torch.cummax((~vv.isfinite()).int(), 0).values.bool()          # [keys][dims]: at this key or before
        clean = vv.nan_to_num(0.0, 0.0, 0.0)
        qq, last = q[picked, h].double(), past + picked
        hidden = torch.arange(len(kk), device=q.device)[None] > last[:, None]
        p = torch.softmax((qq @ kk.T * scale).masked_fill(hidden, -float("inf")), -1)
        want, size = p @ clean, p @ clean.abs()
        d = 128 * 2.0 ** -23 * scale * (qq.abs() @ kk.abs().T).masked_fill(hidden, 0.0).amax(-1, keepdim=True) + 2.0 ** -20
        err, seen = (got[picked, h].double() - want).abs(), bad[last]
        assert torch.equal(~got[picked, h].isfinite(), seen), h
        bound = HALF[dtype] * want.abs() + (2 * d + 2 * HALF[dtype]) * size + 2.0 ** -24
        assert ((err <= bound) | seen).all(), h


def _time(call):
    call()
    times = []
    for _ in range(3):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        call()
        end.record()
        end.synchronize()
        times.append(start.elapsed_time(end))
    return min(times)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("heads,kv", [(8, 2), (3, 3)])
def test_a_value_early_in_a_prompt(ops, cuda, dtype, value, heads, kv):
    """NaN or Inf in key 5's V: nearly all rows see it.  They are not done again, the call takes about its usual time (ten times it at most; done again
    row by row it took hundreds)."""
    n = 4001
    g = torch.Generator(device=cuda).manual_seed(1)
    q, k, v = (torch.randn(n, x, 128, device=cuda, generator=g).to(dtype) for x in (heads, kv, kv))
    cu, ws = _cu([n], cuda), ops.Workspace()
    usual = _time(lambda: ops.attn_packed(q, k, v, cu, cu, ws))
    v[5, 1, 9] = v[5, 1, 127] = value
    picked = torch.tensor([0, 4, 5, 6, 31, 32, 127, 128, 255, 256, 257, 2000, 3999, 4000], device=cuda)
    got = ops.attn_packed(q, k, v, cu, cu, ws)
    ws.check()
    _check_rows(got, q, k, v, 0, picked)
    assert _time(lambda: ops.attn_packed(q, k, v, cu, cu, ws)) <= 10 * usual
    v[:, 0] = value                       # a prompt whose V is lost altogether
    assert _time(lambda: ops.attn_packed(q, k, v, cu, cu, ws)) <= 10 * usual
    got = ops.attn_packed(q, k, v, cu, cu, ws)
    ws.check()
    _check_rows(got, q, k, v, 0, picked)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv", [(8, 1), (2, 2)])
def test_values_seen_and_not_seen_at_once(ops, cuda, dtype, heads, kv):
    """Inf and NaN in other dims before and behind the rows of a block, behind a prefix, beside a healthy sequence."""
    past, n, other = 700, 600, 300
    g = torch.Generator(device=cuda).manual_seed(2)
    q = torch.randn(n + other, heads, 128, device=cuda, generator=g).to(dtype)
    k, v = (torch.randn(past + n + other, kv, 128, device=cuda, generator=g).to(dtype) for _ in range(2))
    for key, dim, value in ((3, 1, "nan"), (690, 2, "inf"), (past + 40, 1, "nan"), (past + 41, 64, "-inf"), (past + 200, 2, "nan"), (past + 300, 65, "inf"), (past + n - 1, 127, "nan"),
                            (past + 255, 3, "nan"), (past + 256, 4, "nan"), (past + 257, 5, "inf")):
        v[key, kv - 1, dim] = float(value)
    ws = ops.Workspace()
    got = ops.attn_packed(q, k, v, _cu([n, other], cuda), _cu([past + n, other], cuda), ws)
    ws.check()
    _check_rows(got[:n], q[:n], k[:past + n], v[:past + n], past, torch.arange(n, device=cuda))
    _check_rows(got[n:], q[n:], k[past + n:], v[past + n:], 0, torch.arange(other, device=cuda))


def test_sums_that_pass_fp32_are_done_again(ops, cuda):
    """bf16: key 200 has a score 7.9 powers of two above all others, so that P is 2^7.9 there, below the 8 that rescale; its V of 2^122 passes fp32
    as P V, the result does not."""
    n, heads, kv = 300, 4, 2
    g = torch.Generator(device=cuda).manual_seed(3)
    q, k = torch.zeros(n, heads, 128, device=cuda), torch.zeros(n, kv, 128, device=cuda)
    q[..., 0], k[200, :, 0] = 8.0, 7.75
    v = torch.randn(n, kv, 128, device=cuda, generator=g)
    v[200, :, 3], v[200, 0, 77] = 2.0 ** 122, -(2.0 ** 121)
    q, k, v = (t.bfloat16() for t in (q, k, v))
    ws = ops.Workspace()
    got = ops.attn_packed(q, k, v, _cu([n], cuda), _cu([n], cuda), ws)
    ws.check()
    _check_rows(got, q, k, v, 0, torch.arange(n, device=cuda))


def test_rows_done_again_for_seconds_are_waited_for(ops, cuda):
    """NaN in the last key of a sequence of 600000: its rows before are done again, 32 a warp, which takes longer than a wait for one tile may, while
    the CTA has the next block already.  Nothing gives up, and that block is whole."""
    n, long, rows, many = 25600, 600000, 200, 96
    g = torch.Generator(device=cuda).manual_seed(4)
    total = many * n + long
    q = torch.zeros(many * n + rows, 1, 128, device=cuda, dtype=torch.bfloat16)
    k = torch.zeros(total, 1, 128, device=cuda, dtype=torch.bfloat16)
    v = torch.randn(total, 1, 128, device=cuda, generator=g).bfloat16() + 0.5
    v[-1, 0, 3] = float("nan")
    ws = ops.Workspace()
    got = ops.attn_packed(q, k, v, _cu([n] * many + [rows], cuda), _cu([n] * many + [long], cuda), ws)
    ws.check()
    bad = got.isnan().nonzero().tolist()
    assert bad == [[many * n + rows - 1, 0, 3]]
    # scores are 0: every row is the mean of the V rows that it sees
    for a, c, nq, nk in [(b * n, b * n, n, n) for b in (0, 20, many - 1)] + [(many * n, many * n, rows, long)]:
        vv = v[c:c + nk, 0].double().nan_to_num(0.0)
        count = torch.arange(1, nk + 1, device=cuda, dtype=torch.float64)[:, None]
        want, size = (torch.cumsum(x, 0).div_(count)[nk - nq:] for x in (vv, vv.abs()))
        err = (got[a:a + nq, 0].double() - want).abs()
        assert ((err <= HALF[torch.bfloat16] * (want.abs() + 2 * size) + 2.0 ** -19 * size) | got[a:a + nq, 0].isnan()).all()


def test_out_in_the_place_of_an_input_is_refused(ops, cuda):
    """Rows that are done again read q after their result is stored, so it cannot go there."""
    g = torch.Generator(device=cuda).manual_seed(6)
    q, k, v = (torch.randn(40, x, 128, device=cuda, generator=g).half() for x in (4, 4, 4))
    ws, cu = ops.Workspace(), _cu([40], cuda)
    for out in (q, k, v, q.view(-1, 512)):
        with pytest.raises(ops.cabi.Qw3Error) as e:
            ops.attn_packed(q, k, v, cu, cu, ws, out=out)
        assert e.value.status == ops.cabi.QW3_ERR_ARG
    ops.attn_packed(q, k, v, cu, cu, ws, out=torch.empty_like(q))
    ws.check()
