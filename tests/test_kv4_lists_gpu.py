"""Decode attention over the paged 4-bit cache: rows that were never stored, long lists, lists cut between CTAs, the low terms of P."""
import ctypes as C

import pytest
import torch

import kv4_ref_gpu as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ---- rows that append left out ---------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv", [(4, 2), (6, 1)])
def test_rows_of_zero_bytes_are_zeros(ops, cuda, dtype, heads, kv):
    """A pool as alloc() makes it, in which some tokens that the lengths count were never stored: code, scale and minimum are 0, and so is the row,
    as kv4_read says.  One request has no stored row at all."""
    page, lens = 16, [50, 33, 20]
    cache = ops.Kv4Cache.alloc(12, page, kv, dtype, cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    table = torch.randperm(12, device=cuda, generator=g).int().view(3, 4)
    ws = ops.Workspace()
    angle = torch.arange(64, device=cuda, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(64, device=cuda, dtype=torch.float64) / 64)
    cos, sin = angle.cos().float(), angle.sin().float()
    for b in (0, 1):
        slots, pos = ref.slots_of(table[b], lens[b], page).int(), torch.arange(lens[b], device=cuda).int()
        pos[[3, 17, 18]] = 64          # outside of the tables: the token is left out
        slots[20:32] = -1
        qkv = torch.randn(lens[b], (heads + 2 * kv) * 128, device=cuda, generator=g).to(dtype)
        ops.rope_kv4_append(qkv, cache, slots, pos, cos, sin, heads, ws)
        with pytest.raises(ops.cabi.Qw3Error):
            ws.check()
    k, v = ops.kv4_read(cache, ref.slots_of(table[0], lens[0], page).int(), ws)
    assert (k[[3, 17, 18, 25]] == 0).all() and (v[[3, 17, 18, 25]] == 0).all() and (v[4] != 0).any()
    q = torch.randn(3, heads, 128, device=cuda, generator=g).to(dtype)
    for scale in (128 ** -0.5, 0.002):
        got = ops.attn_kv4_decode(q, cache, table, _i32(lens, cuda), ws, scale=scale)
        ws.check()
        ref.check_decode(got, q, cache, table, lens, scale)
    assert (got[2].abs() <= 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_scale_of_zero_leaves_the_minimum(ops, cuda, dtype):
    """Pairs of another producer: scale 0 for a row of one value, codes of any kind.  Attention takes a scale below the floor for the floor, which
    is up to 15 floors beside the definition; a NaN in the pair is NaN as before."""
    page, kv, heads, n = 16, 1, 2, 40
    cache = ops.Kv4Cache.alloc(4, page, kv, dtype, cuda)
    g = torch.Generator(device=cuda).manual_seed(2)
    slots = torch.randperm(64, device=cuda, generator=g)[:n].int()
    ws = ops.Workspace()
    ops.rope_kv4_append(torch.randn(n, (heads + 2 * kv) * 128, device=cuda, generator=g).to(dtype), cache, slots, None, None, None, heads, ws)
    q = torch.randn(1, heads, 128, device=cuda, generator=g).to(dtype)
    tiles = cache.pages.view(-1, 2176)
    bits = torch.randint(0, 256, (64,), device=cuda, generator=g).to(torch.uint8)
    for which, row, value in ((1, 5, 0.75), (1, 9, -2.0), (0, 5, 0.25), (1, 11, 0.0)):
        tile, r = tiles[row // 16], row % 16
        tile[1024 * which + 64 * r:1024 * which + 64 * r + 64] = bits
        tile[2048 + 64 * which + 4 * r:2048 + 64 * which + 4 * r + 4] = torch.tensor([0.0, value], dtype=dtype, device=cuda).view(torch.uint8)
    table = _i32([[0, 1, 2, 3]], cuda)
    got = ops.attn_kv4_decode(q, cache, table, _i32([64], cuda), ws)
    ws.check()
    want, bound = ref.decode(q[0], *ref.rows(cache, torch.arange(64, device=cuda)), 128 ** -0.5, 2.0 ** -11, dtype)
    assert ((got[0].double() - want).abs() <= ref.HALF[dtype] * want.abs() + bound + 15 * ref.FLOOR[dtype] + 2.0 ** -25).all()
    for pair in ([float("nan"), 1.0], [1.0, float("nan")]):
        tiles[0][2112 + 4 * 5:2112 + 4 * 6] = torch.tensor(pair, dtype=dtype, device=cuda).view(torch.uint8)
        assert ops.attn_kv4_decode(q, cache, table, _i32([64], cuda), ws).isnan().all()
    ws.check()


@pytest.mark.parametrize("scale", [3e38, -3e38, float("inf"), float("nan")])
def test_a_scale_that_passes_fp32_in_the_kernel_is_refused(ops, cuda, scale):
    cache, ws = ops.Kv4Cache.alloc(2, 16, 1, torch.float16, cuda), ops.Workspace()
    with pytest.raises(ops.cabi.Qw3Error) as e:
        ops.attn_kv4_decode(torch.zeros(1, 2, 128, dtype=torch.float16, device=cuda), cache, _i32([[0]], cuda), _i32([1], cuda), ws, scale=scale)
    assert e.value.status == ops.cabi.QW3_ERR_ARG


def test_append_refuses_a_reserved_field_that_is_not_zero(ops, cuda):
    cabi = ops.cabi
    cache, ws = ops.Kv4Cache.alloc(2, 16, 2, torch.float16, cuda), ops.Workspace()
    qkv, slots, q = torch.zeros(1, 8 * 128, dtype=torch.float16, device=cuda), _i32([3], cuda), torch.empty(1, 4, 128, dtype=torch.float16, device=cuda)
    for reserved, status in ((1, cabi.QW3_ERR_ARG), (-1, cabi.QW3_ERR_ARG), (0, cabi.QW3_OK)):
        a = cabi.Kv4AppendArgs(qkv.data_ptr(), 8 * 128, 1, 4, cabi.ROPE_HALVES, 0, reserved, slots.data_ptr(), None, None, None, 0, q.data_ptr(), None)
        assert cabi.lib().qw3_rope_kv4_append(cache.ref, C.byref(a), ws.h, ops._stream()) == status
    ws.check()


@pytest.mark.parametrize("heads,kv", [(4, 2), (6, 1)])
def test_bf16_q_whose_sum_passes_fp32(ops, cuda, heads, kv):
    """128 values of 2^126 and more of one sign: their sum, which the minimum of a K row is multiplied with, is not a number of fp32; the scores are."""
    dtype, n, page = torch.bfloat16, 90, 16
    g = torch.Generator(device=cuda).manual_seed(7)
    cache, ws = ops.Kv4Cache.alloc(6, page, kv, dtype, cuda), ops.Workspace()
    slots = torch.arange(n, device=cuda).int()
    ops.rope_kv4_append(torch.randn(n, (heads + 2 * kv) * 128, device=cuda, generator=g).to(dtype), cache, slots, None, None, None, heads, ws)
    q = ((1 + torch.rand(1, heads, 128, device=cuda, generator=g)) * 2.0 ** 126).to(dtype)
    q[:, 1] = -q[:, 1]
    assert q.float().sum(-1).isinf().all()
    table = torch.arange(6, device=cuda).int()[None]
    got = ops.attn_kv4_decode(q, cache, table, _i32([n], cuda), ws, scale=2.0 ** -126)
    ws.check()
    ref.check_decode(got, q, cache, table, [n], 2.0 ** -126)


# ---- long lists ------------------------------------------------------------------------------------------------------------------

def _pool(ops, cuda, dtype, kv, page, n_pages, seed):
    """A pool of stored rows; the V rows of a page share an offset of the page's own, so that no part of a list is like another."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    cache, ws = ops.Kv4Cache.alloc(n_pages, page, kv, dtype, cuda), ops.Workspace()
    n = n_pages * page
    qkv = torch.randn(n, 1 + 2 * kv, 128, device=cuda, generator=g)
    qkv[:, 1 + kv:] += torch.randn(n_pages, 1, kv, 128, device=cuda, generator=g).expand(-1, page, -1, -1).reshape(n, kv, 128)
    order = torch.randperm(n, device=cuda, generator=g)
    ops.rope_kv4_append(qkv.to(dtype)[order].flatten(1), cache, order.int(), None, None, None, 1, ws)
    ws.check()
    return cache, ws, g


def _check_and_see_parts(got, q, cache, table, lens, scale=128 ** -0.5):
    """check_decode, and that it would see a part of 8 chunks missing: without these 256 tokens the 64-bit result itself is outside of the bound."""
    ref.check_decode(got, q, cache, table, lens, scale)
    b = max(range(len(lens)), key=lambda i: lens[i])
    n, dtype = lens[b], cache.dtype
    slots = ref.slots_of(table[b], n, cache.page_size)
    want, bound = ref.decode(q[b], *ref.rows(cache, slots), scale, 2.0 ** -11, dtype)
    for at in (0, n // 2 // 32 * 32, n - 256):
        less, _ = ref.decode(q[b], *ref.rows(cache, torch.cat([slots[:at], slots[at + 256:]])), scale, 2.0 ** -11, dtype)
        seen = ((less - want).abs() > 2 * (ref.HALF[dtype] * want.abs() + bound + 2.0 ** -25)).any(-1)
        assert seen.all(), (at, seen)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,kv", [(5, 1), (8, 1), (12, 1), (17, 1), (14, 2), (3, 1)])
def test_lists_cut_between_ctas(ops, cuda, dtype, heads, kv):
    """Pairs of more than 32 chunks share CTAs with others and are joined: groups above four heads and above eight (two and three tiles of heads), rows of
    both types."""
    page, lens = 64, [5000, 40, 1100, 0, 2000, 33 * 32 + 1, 1]
    cache, ws, g = _pool(ops, cuda, dtype, kv, page, 61, seed=heads)
    table = torch.randint(0, 61, (len(lens), 80), device=cuda, generator=g).int()
    q = torch.randn(len(lens), heads, 128, device=cuda, generator=g).to(dtype)
    args = (q, cache, table, _i32(lens, cuda), ws)
    got = ops.attn_kv4_decode(*args)
    ws.check()
    _check_and_see_parts(got, q, cache, table, lens)
    assert torch.equal(ops.attn_kv4_decode(*args), got)
    ws.check()


@pytest.mark.parametrize("heads,kv,dtype", [(16, 4, torch.float16), (16, 4, torch.bfloat16), (32, 4, torch.float16), (48, 4, torch.bfloat16)])
def test_lists_of_more_chunks_than_a_warp_looks_up_at_once(ops, cuda, heads, kv, dtype):
    """60000 chunks and more, 135 a CTA and 33 a warp at least: the second look-up, sums that leave the accumulators, most pairs in several CTAs."""
    page, n_pages, lens = 64, 97, [40000 + 17 * b for b in range(12)]
    sms = torch.cuda.get_device_properties(cuda).multi_processor_count
    assert sum(-(-n // 32) for n in lens) * kv > 128 * 3 * sms
    cache, ws, g = _pool(ops, cuda, dtype, kv, page, n_pages, seed=heads + kv)
    table = torch.randint(0, n_pages, (len(lens), 40960 // page), device=cuda, generator=g).int()
    q = torch.randn(len(lens), heads, 128, device=cuda, generator=g).to(dtype)
    args = (q, cache, table, _i32(lens, cuda), ws)
    got = ops.attn_kv4_decode(*args)
    ws.check()
    _check_and_see_parts(got, q, cache, table, lens)
    assert torch.equal(ops.attn_kv4_decode(*args), got)
    ws.check()


@pytest.mark.parametrize("heads,kv", [(1, 1), (4, 2), (3, 1), (8, 2)])
def test_what_the_rounding_of_p_takes_off_is_added(ops, cuda, heads, kv):
    """fp16 rows, groups of four heads at most: P is two fp16 numbers.  Scores of some ten-thousandths, so that their own errors do not hide it, P near
    one another, so that nothing of their sums is cut off, and results that are small beside the values they come from.  With P as one fp16 number the errors are 4 to 10 times the bound."""
    dtype, page, lens, scale = torch.float16, 16, [3, 31, 100, 117], 0.0002
    cache, ws, g = _pool(ops, cuda, dtype, kv, page, 40, seed=20 + heads)
    table = torch.randperm(40, device=cuda, generator=g)[:32].int().view(4, 8)
    q = torch.randn(4, heads, 128, device=cuda, generator=g).to(dtype)
    got = ops.attn_kv4_decode(q, cache, table, _i32(lens, cuda), ws, scale=scale)
    ws.check()
    ref.check_decode(got, q, cache, table, lens, scale, p_round=2.0 ** -22, no_cuts=True)


# ---- append ----------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("pairs", [False, True])
def test_a_rotated_minimum_that_passes_fp16_reads_back_as_nan(ops, cuda, pairs):
    """Finite fp16 rows that a rotation takes below fp16: the stored minimum would be -Inf.  Above, the row's other values are held, and the largest code
    stands for what fp16 makes of it."""
    kv, heads, page = 1, 1, 16
    cache, ws = ops.Kv4Cache.alloc(1, page, kv, torch.float16, cuda), ops.Workspace()
    angle = torch.full((4, 64), torch.pi / 4, dtype=torch.float64, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(9)
    qkv = torch.randn(3, 3 * 128, device=cuda, generator=g).half()
    i, j = (10, 11) if pairs else (10, 74)
    for token, sign in ((0, -1), (1, 1)):
        qkv[token, 128 + i], qkv[token, 128 + j] = sign * 60000.0, sign * 60000.0
    _, k = ops.rope_kv4_append(qkv, cache, _i32([2, 3, 4], cuda), _i32([0, 1, 2], cuda), angle.cos().float(), angle.sin().float(), heads, ws, pairs=pairs)
    kr, vr = ops.kv4_read(cache, _i32([2, 3, 4], cuda), ws)
    ws.check()
    assert k[0, 0, j] == -float("inf") and k[1, 0, j] == float("inf") and k[2].isfinite().all()
    assert kr[0].isnan().all() and vr.isfinite().all() and kr[2].isfinite().all()
    # 84853 / 15: a step of 5660, and the sum of the largest code passes fp16
    keep = torch.arange(128, device=cuda) != j
    assert kr[1, 0, j] == float("inf") and ((kr[1, 0, keep].float() - k[1, 0, keep].float()).abs() <= 5660 / 2 + 4).all()
