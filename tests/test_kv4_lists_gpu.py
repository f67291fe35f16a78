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
    want, bound = ref.decode(q[0], *ref.rows(cache, torch.arange(64, device=cuda)), 128 ** -0.5, 2.0 ** -11)
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
