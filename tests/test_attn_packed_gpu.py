"""Causal attention of packed sequences on the GPU against its definition in 64 bits."""
import pytest
import torch

from kv4_ref import HALF

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def _cu(lens, dev):
    return torch.cumsum(torch.tensor([0] + list(lens)), 0).int().to(dev)


def _rows(lens_q, lens_k, heads, kv, dtype, dev, seed, grow=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    q = torch.randn(sum(lens_q), heads, 128, device=dev, generator=g).to(dtype)
    k = torch.randn(sum(lens_k), kv, 128, device=dev, generator=g)
    k = (k * torch.linspace(1.0, grow, max(sum(lens_k), 1), device=dev)[:k.shape[0], None, None]).to(dtype)
    v = torch.randn(sum(lens_k), kv, 128, device=dev, generator=g).to(dtype)
    return q, k, v


def _check(got, q, k, v, lens_q, lens_k, scale=128 ** -0.5, rows=None):
    """Result and bound in 64 bits.  The kernel rounds the result once (half a step), each p to the type (half a step of p v), and holds the
    scores in fp32: 128 products summed by the tensor cores, which cut off what the accumulator cannot hold, change a score by at
    most 128 * 2^-23 of the sum of the products' sizes, typically far less; p and its sum change by that much, relatively, and
    by 2^-20 for the exponentials and the sums of p and p v."""
    dtype = q.dtype
    group = q.shape[1] // k.shape[1]
    a = c = 0
    for nq, nk in zip(lens_q, lens_k):
        pick = range(nq) if rows is None else sorted({r for r in rows if r < nq} | {nq - 1} if nq else ())
        pick = torch.tensor([r for r in pick], dtype=torch.long, device=q.device)
        if len(pick):
            last = nk - nq + pick
            for h in range(q.shape[1]):
                qq, kk, vv = q[a + pick, h].double(), k[c:c + nk, h // group].double(), v[c:c + nk, h // group].double()
                hidden = torch.arange(nk, device=q.device)[None] > last[:, None]
                s = (qq @ kk.T * scale).masked_fill(hidden, -float("inf"))
                p = torch.softmax(s, -1).masked_fill((last < 0)[:, None], 0.0)
                want, size = p @ vv, p @ vv.abs()
                d = 128 * 2.0 ** -23 * scale * (qq.abs() @ kk.abs().T).masked_fill(hidden, 0.0).amax(-1, keepdim=True) + 2.0 ** -20 if nk else 0
                err = (got[a + pick, h].double() - want).abs()
                bound = HALF[dtype] * want.abs() + (2 * d + 2 * HALF[dtype]) * size + 2.0 ** -24
                assert not err.isnan().any() and (err <= bound).all(), (nq, nk, h, (err / bound).max().item())
        a, c = a + nq, c + nk


LENS = [([1], [1]), ([1, 1, 1], [1, 64, 65]), ([0, 5, 0, 0, 31], [0, 5, 7, 0, 31]), ([63, 64, 65, 66], [63, 64, 65, 66]), ([127, 3, 129], [127, 3, 129]),
        ([255, 256, 257], [255, 256, 257]), ([100, 1, 40], [400, 333, 41]), ([600], [600]), ([10, 70, 5], [4, 1, 0]), ([2] * 70, [3] * 70)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 1), (6, 3), (3, 1), (16, 1), (32, 1)])
@pytest.mark.parametrize("lens", LENS)
def test_packed(ops, cuda, dtype, lens, heads, kv):
    """Lengths around a tile of keys, of rows and a block; prefixes; sequences without queries, without keys, with fewer keys than
    queries (rows that see none); groups of one head, of powers of two, of others."""
    q, k, v = _rows(*lens, heads, kv, dtype, cuda, seed=heads + len(lens[0]))
    ws = ops.Workspace()
    args = (q, k, v, _cu(lens[0], cuda), _cu(lens[1], cuda), ws)
    got = ops.attn_packed(*args)
    ws.check()
    _check(got, q, k, v, *lens)
    assert torch.equal(ops.attn_packed(*args), got)
    ws.check()


@pytest.mark.parametrize("dtype", TYPES)
def test_packed_long_and_ragged(ops, cuda, dtype):
    lens = [1, 1500, 0, 333, 64], [1, 1500, 0, 2100, 64]
    q, k, v = _rows(*lens, 12, 3, dtype, cuda, seed=5, grow=5.0)   # maxima that grow along the keys: sums are rescaled many times
    ws = ops.Workspace()
    got = ops.attn_packed(q, k, v, _cu(lens[0], cuda), _cu(lens[1], cuda), ws)
    ws.check()
    _check(got, q, k, v, *lens, rows=[0, 1, 31, 32, 33, 63, 64, 127, 128, 255, 256, 700, 1400])
    for scale in (1.0, 0.01):
        got = ops.attn_packed(q, k, v, _cu(lens[0], cuda), _cu(lens[1], cuda), ws, scale=scale)
        _check(got, q, k, v, *lens, scale=scale, rows=[0, 31, 256, 1400])
    ws.check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("gain", [1000.0, 15000.0])
def test_packed_large_scores(ops, cuda, dtype, gain):
    """Rows equal to one of their keys at sizes that fp16 can just hold: scores of 1e7 to 3e9.  The equal key wins by far."""
    n, heads = 300, 2
    g = torch.Generator(device=cuda).manual_seed(6)
    k = (torch.randn(n, heads, 128, device=cuda, generator=g).clamp(-4, 4) * gain).to(dtype)
    v = torch.randn(n, heads, 128, device=cuda, generator=g).to(dtype)
    key = torch.tensor([(37 * r) % (r + 1) for r in range(n)], device=cuda)
    ws = ops.Workspace()
    got = ops.attn_packed(k[key].contiguous(), k, v, _cu([n], cuda), _cu([n], cuda), ws)
    ws.check()
    assert torch.equal(got, v[key])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("inf"), float("nan"), -float("inf")])
def test_packed_nothing_that_a_row_does_not_see_reaches_it(ops, cuda, dtype, value):
    """Inf and NaN in other sequences, in keys behind a row of its own, and in rows of the buffers behind the last sequence."""
    lens = [70, 130, 40], [90, 130, 40]
    heads, kv, spare = 4, 2, 77
    q, k, v = _rows(*lens, heads, kv, dtype, cuda, seed=7)
    k, v, q = (torch.cat([t, torch.full((spare, t.shape[1], 128), value, dtype=dtype, device=cuda)]) for t in (k, v, q))
    ws = ops.Workspace()
    cu_q, cu_k = _cu(lens[0], cuda), _cu(lens[1], cuda)
    want = ops.attn_packed(q, k, v, cu_q, cu_k, ws, out=torch.full_like(q, 3.0))
    assert (want[240:] == 3.0).all()
    _check(want, q, k, v, *lens)
    at = 90 + 100   # key 100 of the second sequence, KV head 1
    k[at, 1, 5] = v[at, 1, 9] = value
    v[at, 1, 100] = value
    got = ops.attn_packed(q, k, v, cu_q, cu_k, ws, out=torch.full_like(q, 3.0))
    ws.check()
    same = torch.ones(240, heads, dtype=torch.bool, device=cuda)
    same[70 + 100:200, 2:] = False
    # a row before the key is done again in another order where its tile holds the key: the same within the bound
    assert torch.equal(got[:240][same.nonzero(as_tuple=True)].isnan().any(), torch.tensor(False, device=cuda))
    assert torch.equal(got[:70], want[:70]) and torch.equal(got[200:], want[200:]) and torch.equal(got[:, :2], want[:, :2])
    clean_k, clean_v = k.clone(), v.clone()
    clean_k[at, 1], clean_v[at, 1] = 0, 0
    before = slice(70, 170)
    _check(got[before], q[before], clean_k[90:190], clean_v[90:190], [100], [100])
    assert not got[170:200, 2:, [9, 100]].isfinite().any()


def test_packed_rows_that_are_parts_of_wider_ones(ops, cuda):
    """q, k and v as parts of one QKV product."""
    heads, kv, lens = 6, 2, [50, 3, 91]
    g = torch.Generator(device=cuda).manual_seed(8)
    qkv = torch.randn(sum(lens), (heads + 2 * kv) * 128 + 8, device=cuda, generator=g).half()
    q, k, v = qkv[:, :heads * 128], qkv[:, heads * 128:(heads + kv) * 128], qkv[:, (heads + kv) * 128:(heads + 2 * kv) * 128]
    ws = ops.Workspace()
    got = ops.attn_packed(q, k, v, _cu(lens, cuda), _cu(lens, cuda), ws)
    ws.check()
    _check(got, q.reshape(-1, heads, 128), k.reshape(-1, kv, 128), v.reshape(-1, kv, 128), lens, lens)


@pytest.mark.parametrize("cu_q,cu_k", [([0, 40, 30, 60], [0, 20, 40, 60]), ([0, 20, 40, 61], [0, 20, 40, 60]), ([-1, 20, 40, 60], [0, 20, 40, 60]), ([0, 20, 40, 60], [0, 20, 10, 60]),
                                       ([0, 20, 40, 60], [0, 20, 40, 2 ** 31 - 1])])
def test_packed_reports_sequences_outside_of_the_buffers(ops, cuda, cu_q, cu_k):
    q, k, v = _rows([60], [60], 4, 2, torch.float16, cuda, seed=9)
    ws = ops.Workspace()
    out = torch.full_like(q, 7.0)
    ops.attn_packed(q, k, v, *(torch.tensor(x, dtype=torch.int32, device=cuda) for x in (cu_q, cu_k)), ws, out=out)
    with pytest.raises(ops.cabi.Qw3Error) as e:
        ws.check()
    assert e.value.status == ops.cabi.QW3_ERR_RANGE
    for b in range(3):
        good = all(0 <= cu[b] <= cu[b + 1] <= 60 for cu in (cu_q, cu_k))
        if good and [cu_q, cu_k] != [[0, 40, 30, 60], [0, 20, 40, 60]]:
            n = cu_q[b + 1] - cu_q[b]
            s, t = slice(cu_q[b], cu_q[b + 1]), slice(cu_k[b], cu_k[b + 1])
            _check(out[s], q[s], k[t], v[t], [n], [cu_k[b + 1] - cu_k[b]])
    ws.check()


def test_packed_without_keys_or_rows(ops, cuda):
    q = torch.randn(5, 4, 128, device=cuda).half()
    none = torch.empty(0, 2, 128, dtype=torch.float16, device=cuda)
    ws = ops.Workspace()
    got = ops.attn_packed(q, none, none, _cu([2, 3], cuda), _cu([0, 0], cuda), ws)
    assert (got == 0).all()
    assert ops.attn_packed(q[:0], none, none, _cu([0], cuda), _cu([0], cuda), ws).shape == (0, 4, 128)
    out = torch.full_like(q, 2.0)
    assert (ops.attn_packed(q, none, none, _cu([], cuda), _cu([], cuda), ws, out=out) == 2.0).all()
    ws.check()


def test_packed_captured_and_replayed_with_other_lengths(ops, cuda):
    heads, kv = 4, 2
    q, k, v = _rows([300], [300], heads, kv, torch.bfloat16, cuda, seed=10)
    cu_q, cu_k = _cu([100, 0, 50], cuda), _cu([120, 0, 50], cuda)
    ws = ops.Workspace(pdl=True)
    out = torch.zeros_like(q)
    ops.attn_packed(q, k, v, cu_q, cu_k, ws, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attn_packed(q, k, v, cu_q, cu_k, ws, out=out)
    for lens in (([100, 0, 50], [120, 0, 50]), ([1, 200, 99], [1, 200, 99]), ([0, 0, 0], [0, 0, 0]), ([30, 30, 30], [100, 100, 100])):
        cu_q.copy_(_cu(lens[0], cuda))
        cu_k.copy_(_cu(lens[1], cuda))
        out.fill_(9.0)
        graph.replay()
        ws.check()
        _check(out, q, k, v, *lens)
        assert (out[sum(lens[0]):] == 9.0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_prompt_then_tokens_through_the_cache(ops, cuda, dtype):
    """Requests served as a program would: prompts packed (attention over the rotated rows themselves), the second chunk of one of them over its
    cached beginning, then single tokens, all slots from the GPU.  Each result against attention over the rows that the cache holds."""
    heads, kv, page, max_pos = 6, 2, 32, 400
    a = torch.arange(max_pos, dtype=torch.float64, device=cuda)[:, None] * 1e4 ** (-torch.arange(0, 128, 2, dtype=torch.float64, device=cuda) / 128)
    cos, sin = a.cos().float(), a.sin().float()
    g = torch.Generator(device=cuda).manual_seed(11)
    ws = ops.Workspace(pdl=True)
    cache = ops.Kv4Cache.alloc(40, page, kv, dtype, cuda)
    n_free = torch.tensor([40], dtype=torch.int32, device=cuda)
    free = torch.randperm(40, device=cuda, generator=g).int()
    table = torch.full((3, 14), -1, dtype=torch.int32, device=cuda)
    lens = torch.zeros(3, dtype=torch.int32, device=cuda)
    width = (heads + 2 * kv) * 128

    def slots_of(b, n):
        t = torch.arange(n, device=cuda)
        return (table[b].long()[t // page] * page + t % page).int()

    held = [0, 0, 0]
    for new in ([70, 1, 133], [5, 0, 200], [1, 1, 1], [1, 1, 1]):
        total = sum(new)
        qkv = torch.randn(total, width, device=cuda, generator=g).to(dtype)
        d_new = torch.tensor(new, dtype=torch.int32, device=cuda)
        cu, pos, slots, _, _ = ops.page_slots(lens, d_new, page, table, free, n_free, total, ws, kv_len=lens, n_free_out=n_free)
        q, k = ops.rope_kv4_append(qkv, cache, slots, pos, cos, sin, heads, ws)
        v = qkv[:, (heads + kv) * 128:].reshape(total, kv, 128)
        before, held = held, [x + n for x, n in zip(held, new)]
        assert lens.tolist() == held and cu.tolist() == [0] + torch.cumsum(torch.tensor(new), 0).tolist()
        if new == [1, 1, 1]:
            out = ops.attn_kv4_decode(q, cache, table, lens, ws)
            kr, vr = zip(*(ops.kv4_read(cache, slots_of(b, held[b]), ws) for b in range(3)))
            kr, vr = torch.cat(kr), torch.cat(vr)
            # rows read back carry half a step each on top of the bound
            for b in range(3):
                s = slice(sum(held[:b]), sum(held[:b + 1]))
                for h in range(heads):
                    kk, vv, qq = kr[s, h // 3].double(), vr[s, h // 3].double(), q[b, h].double()
                    p = torch.softmax(kk @ qq * 128 ** -0.5, 0)
                    d = 2 * HALF[dtype] * (kk.abs() @ qq.abs()).max() * 128 ** -0.5
                    assert ((out[b, h].double() - p @ vv).abs() <= HALF[dtype] * (p @ vv).abs() + (2 * d + 4 * 2.0 ** -11 + HALF[dtype]) * (p @ vv.abs())).all()
        else:
            # keys: the cached beginning, read back, and the new rows as they are
            ks, vs, at = [], [], 0
            for b in range(3):
                kr, vr = ops.kv4_read(cache, slots_of(b, before[b]), ws)
                ks += [kr, k[at:at + new[b]]]
                vs += [vr, v[at:at + new[b]]]
                at += new[b]
            kk, vv = torch.cat(ks), torch.cat(vs)
            out = ops.attn_packed(q, kk, vv, cu, _cu(held, cuda), ws)
            _check(out, q, kk, vv, new, held)
    ws.check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_packed_a_key_that_is_not_finite_reaches_every_row_that_sees_it(ops, cuda, dtype, value):
    """NaN or Inf in key i of sequence i, for every place in two tiles of keys (the exponentials of a tile are computed in two ways): the rows that
    see it are NaN, the ones before it are not."""
    n = 260
    lens = [n] * n
    g = torch.Generator(device=cuda).manual_seed(12)
    q = torch.randn(2 * n, 4, 128, device=cuda, generator=g).abs().to(dtype)
    k = torch.randn(n, n, 1, 128, device=cuda, generator=g).to(dtype)
    v = torch.randn(n * n, 1, 128, device=cuda, generator=g).to(dtype)
    i = torch.arange(n, device=cuda)
    k[i, i, 0, 7] = value
    ws = ops.Workspace()
    # two queries a sequence: its last rows, which see all keys but the last one, and all
    got = ops.attn_packed(q, k.flatten(0, 1), v, _cu([2] * n, cuda), _cu(lens, cuda), ws).view(n, 2, 4, 128)
    ws.check()
    bad = got.isnan().all(-1).all(-1)
    want = torch.ones(n, 2, dtype=torch.bool, device=cuda)
    want[n - 1, 0] = False
    assert torch.equal(bad, want) and got[n - 1, 0].isfinite().all()


def test_packed_many_sequences(ops, cuda):
    """More sequences than a CTA looks at in one step, of lengths that make blocks of every size."""
    lens = [(7 * b) % 19 for b in range(1500)]
    q, k, v = _rows(lens, lens, 2, 1, torch.float16, cuda, seed=13)
    ws = ops.Workspace()
    got = ops.attn_packed(q, k, v, _cu(lens, cuda), _cu(lens, cuda), ws)
    ws.check()
    _check(got, q, k, v, lens, lens)


def test_packed_on_two_streams_at_once(ops, cuda):
    lens = ([700, 3, 90], [900, 3, 90])
    q, k, v = _rows(*lens, 8, 2, torch.bfloat16, cuda, seed=31)
    cu = _cu(lens[0], cuda), _cu(lens[1], cuda)
    want = ops.attn_packed(q, k, v, *cu, ops.Workspace())
    torch.cuda.synchronize()
    streams, ws, got = [torch.cuda.Stream() for _ in range(2)], [ops.Workspace(pdl=True) for _ in range(2)], []
    for _ in range(8):
        for s, w in zip(streams, ws):
            with torch.cuda.stream(s):
                got.append(ops.attn_packed(q, k, v, *cu, w))
    torch.cuda.synchronize()
    for w in ws:
        w.check()
    assert all(torch.equal(x, want) for x in got)
    _check(want, q, k, v, *lens)
