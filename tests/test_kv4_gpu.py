"""The paged 4-bit cache on the GPU: pages and slots, append, read, decode attention, against the plain restatement in kv4_ref.py."""
import ctypes as C
import random

import pytest
import torch

import kv4_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _tables(max_pos, rot, base=1e4):
    a = torch.arange(max_pos, dtype=torch.float64)[:, None] * base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return a.cos().float(), a.sin().float()


# ---- pages and slots -------------------------------------------------------------------------------------------------------------

def _plan(ctx, new, page, table, free, n_free):
    """Token by token: the first token of a block takes the top of the stack."""
    table, left, cu, pos, slots = [r[:] for r in table], n_free, [0], [], []
    for b, (c, n) in enumerate(zip(ctx, new)):
        for t in range(c, c + n):
            if t % page == 0:
                left -= 1
                table[b][t // page] = free[left]
            pos.append(t)
            slots.append(table[b][t // page] * page + t % page)
        cu.append(len(pos))
    return table, cu, pos, slots, left


@pytest.mark.parametrize("n,page,ctx_max,new_max,pad", [(1, 16, 0, 1, 0), (1, 128, 40, 1, 3), (7, 16, 100, 1, 1), (33, 48, 300, 70, 5), (513, 16, 64, 5, 0),
                                                        (1200, 32, 90, 3, 7), (3, 64, 5, 9000, 11), (5000, 16, 33, 2, 2)])
def test_page_slots(ops, cuda, n, page, ctx_max, new_max, pad):
    rng = random.Random(n * page)
    ctx = [rng.choice([0, page, rng.randint(0, ctx_max)]) for _ in range(n)]
    new = [rng.choice([0, 1, rng.randint(0, new_max)]) for _ in range(n)]
    have = [-(-c // page) for c in ctx]
    need = [-(-(c + x) // page) for c, x in zip(ctx, new)]
    width, spare = max(need) + 2, sum(need) - sum(have) + 4
    ids = list(range(sum(have) + spare))
    rng.shuffle(ids)
    table, at = [], 0
    for h in have:
        table.append(ids[at:at + h] + [-7] * (width - h))
        at += h
    free = ids[at:] + [-9, -9]
    wide = torch.full((n, width + 3), -5, dtype=torch.int32, device=cuda)   # a table that is part of a wider one
    d_table = wide[:, :width]
    d_table.copy_(_i32(table, cuda))
    ws = ops.Workspace()
    total = sum(new)
    want_table, cu, pos, slots, left = _plan(ctx, new, page, table, free, spare)
    d_ctx, d_free = _i32(ctx, cuda), _i32(free, cuda)
    # outputs of their own
    got = ops.page_slots(d_ctx, _i32(new, cuda), page, d_table, d_free, _i32([spare], cuda), total + pad, ws)
    ws.check()
    assert got[0].tolist() == cu and got[1].tolist() == pos + [0] * pad and got[2].tolist() == slots + [-1] * pad
    assert got[3].tolist() == [c + x for c, x in zip(ctx, new)] and got[4].tolist() == [left]
    assert d_table.tolist() == want_table and (wide[:, width:] == -5).all() and d_ctx.tolist() == ctx and d_free.tolist() == free
    # the inputs' own buffers
    d_table.copy_(_i32(table, cuda))
    n_free = _i32([spare], cuda)
    got = ops.page_slots(d_ctx, _i32(new, cuda), page, d_table, d_free, n_free, total + pad, ws, kv_len=d_ctx, n_free_out=n_free)
    ws.check()
    assert got[2].tolist() == slots + [-1] * pad and d_table.tolist() == want_table
    assert d_ctx.tolist() == [c + x for c, x in zip(ctx, new)] and n_free.tolist() == [left]


@pytest.mark.parametrize("what", ["negative", "table", "pages", "tokens", "count"])
@pytest.mark.parametrize("new0", [1, 5000])
def test_page_slots_leaves_all_as_it_was_where_it_cannot_serve(ops, cuda, what, new0):
    page, ctx, new = 16, [5, 0, 31], [new0, 3, 2]
    width, spare, room = 400, 320, new0 + 5
    if what == "negative":
        new[1] = -1
    elif what == "table":
        width = -(-(5 + new0) // 16) - 1 if new0 > 1 else 2
    elif what == "pages":
        spare = 1 if new0 == 1 else 300
    elif what == "tokens":
        room -= 1
    table = torch.full((3, width), -3, dtype=torch.int32, device=cuda)
    table[:, 0] = _i32([400, 401, 402], cuda)
    if what == "table":
        table[2, 1:2] = 403
    before = table.clone()
    if what == "table" and new0 == 1:
        new[2] = 2 * 16
        room += 30
    ws = ops.Workspace()
    n_free = _i32([spare if what != "count" else 321], cuda)
    got = ops.page_slots(_i32(ctx, cuda), _i32(new, cuda), page, table, _i32(list(range(320)), cuda), n_free, room, ws)
    with pytest.raises(ops.cabi.Qw3Error) as e:
        ws.check()
    assert e.value.status == ops.cabi.QW3_ERR_RANGE
    assert torch.equal(table, before) and got[4].tolist() == n_free.tolist() and got[3].tolist() == ctx
    assert got[0].tolist() == [0] * 4 and (got[2] == -1).all() and (got[1] == 0).all()
    ws.check()   # the failing check has cleared the word


# ---- append and read -------------------------------------------------------------------------------------------------------------

APPEND = [(1, 1, 1, 16, 128, 0, 0), (33, 32, 8, 16, 128, 2, 0), (5, 12, 2, 32, 64, 0, 64), (70, 4, 4, 48, 32, 1, 16), (3, 6, 2, 64, 16, 0, 0), (17, 5, 1, 128, 0, 3, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,page,rot,pad,extra", APPEND)
def test_append_and_read(ops, cuda, dtype, pairs, tokens, heads, kv, page, rot, pad, extra):
    """Every byte of the pool after an append equals the definition's; rows that no slot names keep theirs; rotated rows and rows read
    back are within half a step of the 64-bit results."""
    g = _gen(tokens + page)
    max_pos, width = 300, (heads + 2 * kv) * 128
    base = torch.randn(tokens, width + 24, generator=g) * torch.exp(torch.randn(tokens, 1, generator=g))
    base[0, heads * 128:] = 0.5                       # rows without a range
    if tokens > 2:
        base[1, -128 - 24:] *= 2.0 ** -16             # a row near the smallest numbers of fp16
        base[2, heads * 128:(heads + kv) * 128] *= 1000.0
    qkv = base.to(dtype)[:, 8:8 + width]              # rows further apart than they are long
    pos = torch.randint(0, max_pos, (tokens,), generator=g)
    pos[0], pos[-1] = 0, max_pos - 1
    n_pages = tokens // page + 3
    slots = torch.randperm(n_pages * page, generator=g)[:tokens]
    slots[tokens - pad:] = -1
    cos, sin = _tables(max_pos, rot) if rot else (None, None)
    pool = ref.Pool(n_pages, page, kv, dtype, extra)
    pages = pool.bytes.to(cuda)
    cache = ops.Kv4Cache(pages, page, kv, dtype)
    ws = ops.Workspace()
    dev = base.to(dtype).to(cuda)[:, 8:8 + width]
    q, k = ops.rope_kv4_append(dev, cache, _i32(slots.tolist(), cuda), _i32(pos.tolist(), cuda), cos.to(cuda) if rot else None, sin.to(cuda) if rot else None,
                               heads, ws, pairs=pairs)
    ws.check()
    x = qkv.float().view(tokens, heads + 2 * kv, 128)
    y = ref.rotate(x[:, :heads + kv], cos[pos], sin[pos], pairs) if rot else x[:, :heads + kv]
    assert torch.equal(q.cpu(), y[:, :heads].to(dtype)) and torch.equal(k.cpu(), y[:, heads:].to(dtype))
    n = tokens - pad
    pool.put_rows(slots[:n], y[:n, heads:], x[:n, heads + kv:])
    assert torch.equal(pages.cpu(), pool.bytes)
    # 64 bits: two products and a sum, each rounded in fp32, then half a step
    if rot:
        half = rot // 2
        ia = torch.arange(half) * (2 if pairs else 1)
        ib = ia + (1 if pairs else half)
        c, s = cos[pos].double()[:, None], sin[pos].double()[:, None]
        a, b = x[:, :heads, ia].double(), x[:, :heads, ib].double()
        tiny = torch.finfo(dtype).smallest_normal * 2 * ref.HALF[dtype]
        for idx, want, size in ((ia, a * c - b * s, (a * c).abs() + (b * s).abs()), (ib, b * c + a * s, (b * c).abs() + (a * s).abs())):
            assert ((q.cpu()[..., idx].double() - want).abs() <= (ref.HALF[dtype] + 2.0 ** -23) * want.abs() + 2.0 ** -23 * size + tiny).all()
    # read back: code * scale is exact, the sum is rounded in fp32 and then to the type
    kr, vr = ops.kv4_read(cache, _i32(slots.tolist(), cuda), ws)
    ws.check()
    assert (kr[n:] == 0).all() and (vr[n:] == 0).all()
    tiny = torch.finfo(dtype).smallest_normal * 2 * ref.HALF[dtype]
    for got, row, rows in zip((kr, vr), pool.rows(slots[:n]), (y[:n, heads:], x[:n, heads + kv:])):
        want = ref.value(*row)
        assert ((got[:n].cpu().double() - want).abs() <= (ref.HALF[dtype] + 2.0 ** -23) * want.abs() + 2.0 ** -23 * row[2].double().abs()[..., None] + tiny).all()
        # what 4 bits can hold: half a step, the rounding of the minimum, and what the rounding of the scale cuts off at the top
        lo, hi = rows.double().amin(-1, keepdim=True), rows.double().amax(-1, keepdim=True)
        step = row[1].double()[..., None]
        assert ((want - rows.double()).abs() <= step * (0.5 + 2.0 ** -20) + ref.HALF[dtype] * (1.01 * lo.abs() + 1.01 * (hi - lo)) + tiny * 8).all()


def test_append_without_the_rotated_k_and_empty_calls(ops, cuda):
    """Through the C entry point: no buffer for k; and calls without tokens, requests or new tokens, which do nothing."""
    cabi = ops.cabi
    L, ws, st = cabi.lib(), ops.Workspace(), ops._stream()
    qkv = torch.randn(3, 8 * 128, generator=_gen(16)).half().to(cuda)
    caches = [ops.Kv4Cache.alloc(2, 16, 2, torch.float16, cuda) for _ in range(2)]
    slots = _i32([4, 31, 0], cuda)
    want, _ = ops.rope_kv4_append(qkv, caches[0], slots, None, None, None, 4, ws)
    q = torch.zeros_like(want)
    a = cabi.Kv4AppendArgs(qkv.data_ptr(), 8 * 128, 3, 4, cabi.ROPE_HALVES, 0, 0, slots.data_ptr(), None, None, None, 0, q.data_ptr(), None)
    cabi.check(L.qw3_rope_kv4_append(caches[1].ref, C.byref(a), ws.h, st), "qw3_rope_kv4_append")
    assert torch.equal(q, want) and torch.equal(caches[0].pages, caches[1].pages)
    none = torch.empty(0, dtype=torch.int32, device=cuda)
    assert ops.rope_kv4_append(qkv[:0], caches[0], none, None, None, None, 4, ws)[0].shape == (0, 4, 128)
    assert ops.kv4_read(caches[0], none, ws)[1].shape == (0, 2, 128)
    assert ops.attn_kv4_decode(q[:0], caches[0], torch.empty(0, 1, dtype=torch.int32, device=cuda), none, ws).shape == (0, 4, 128)
    table = torch.full((2, 3), -1, dtype=torch.int32, device=cuda)
    got = ops.page_slots(_i32([0, 0], cuda), _i32([0, 0], cuda), 16, table, none, _i32([0], cuda), 0, ws)
    ws.check()
    assert got[0].tolist() == [0, 0, 0] and got[1].numel() == got[2].numel() == 0 and got[3].tolist() == [0, 0] and (table == -1).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_append_of_halfway_values_rounds_to_even(ops, cuda, dtype):
    """Rows 0, 0.5, 1, .. 15: scale 1, and every second value halfway between two codes."""
    row = torch.arange(128).float() % 31 / 2
    qkv = torch.stack([row] * 3).flatten()[None].to(dtype).to(cuda)
    cache = ops.Kv4Cache.alloc(1, 16, 1, dtype, cuda)
    ws = ops.Workspace()
    ops.rope_kv4_append(qkv, cache, _i32([3], cuda), None, None, None, 1, ws)
    k, v = ops.kv4_read(cache, _i32([3], cuda), ws)
    ws.check()
    assert torch.equal(k.cpu().flatten().float(), torch.round(row)) and torch.equal(k, v)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan"), 1e30])
def test_rows_that_are_not_finite_read_back_as_nan(ops, cuda, dtype, bad):
    """Inf, NaN, and in bf16 a range that no scale holds: that row is NaN, its neighbours are what they were."""
    if dtype == torch.float16 and bad == 1e30:
        bad = float("inf")
    g = _gen(3)
    qkv = torch.randn(2, (2 + 4) * 128, generator=g)
    plain = qkv.clone()
    qkv[0, 2 * 128 + 5] = bad              # K of KV head 0 of the first token
    qkv[1, (2 + 2 + 1) * 128 + 127] = bad  # V of KV head 1 of the second
    ws = ops.Workspace()
    out = []
    for x in (plain, qkv):
        cache = ops.Kv4Cache.alloc(2, 16, 2, dtype, cuda)
        ops.rope_kv4_append(x.to(dtype).to(cuda), cache, _i32([17, 2], cuda), None, None, None, 2, ws)
        out.append(torch.stack(ops.kv4_read(cache, _i32([17, 2], cuda), ws)))
    ws.check()
    want = out[0].clone()
    want[0, 0, 0] = want[1, 1, 1] = float("nan")
    assert torch.equal(out[1].isnan(), want.isnan()) and torch.equal(out[1].nan_to_num(0.0), want.nan_to_num(0.0))


def test_slots_and_positions_outside_are_left_out_and_reported(ops, cuda):
    cabi = ops.cabi
    cache = ops.Kv4Cache.alloc(3, 16, 2, torch.float16, cuda)
    cos, sin = (t.to(cuda) for t in _tables(20, 128))
    qkv = torch.randn(4, 8 * 128, generator=_gen(5)).half().to(cuda)
    ws = ops.Workspace()
    for slots, pos in (([1, 48, 2, 47], [0, 1, 2, 19]), ([1, 3, 2, 47], [0, 20, 2, 19]), ([1, 3, 2, 47], [0, -1, 2, 19]), ([1, 2 ** 31 - 1, 2, 47], [0, 1, 2, 19])):
        cache.pages.zero_()
        ops.rope_kv4_append(qkv, cache, _i32(slots, cuda), _i32(pos, cuda), cos, sin, 4, ws)
        with pytest.raises(cabi.Qw3Error) as e:
            ws.check()
        assert e.value.status == cabi.QW3_ERR_RANGE
        good = [s for i, s in enumerate(slots) if i != 1]
        k, v = ops.kv4_read(cache, _i32(list(range(48)), cuda), ws)
        ws.check()
        stored = (v != 0).any(-1).any(-1)
        assert stored.nonzero().flatten().tolist() == sorted(good)
    k, v = ops.kv4_read(cache, _i32([1, 48, -1, 47], cuda), ws)
    with pytest.raises(cabi.Qw3Error):
        ws.check()
    assert (v[1] == 0).all() and (v[2] == 0).all() and (v[0] != 0).any() and (v[3] != 0).any()


# ---- decode attention ------------------------------------------------------------------------------------------------------------

def _case(lens, heads, kv, page, dtype, seed, extra=0, spread=1.0):
    """Pool, table and q of requests with these lengths; pages in a random order, NaN bytes in every row that no request holds."""
    g = _gen(seed)
    blocks = [-(-n // page) for n in lens]
    n_pages, width = sum(blocks) + 2, max(blocks + [1]) + 1
    order = torch.randperm(n_pages, generator=g).tolist()
    pool = ref.Pool(n_pages, page, kv, dtype, extra)
    table, at, rows = [], 0, []
    for n, b in zip(lens, blocks):
        table.append(order[at:at + b] + [-1] * (width - b))
        at += b
        slots = torch.tensor([table[-1][t // page] * page + t % page for t in range(n)], dtype=torch.long)
        k = torch.randn(n, kv, 128, generator=g) * torch.exp(0.5 * torch.randn(kv, 128, generator=g)) + 0.3
        v = torch.randn(n, kv, 128, generator=g) * torch.exp(spread * torch.randn(n, kv, 1, generator=g))
        pool.put_rows(slots, k, v)
        rows.append(slots)
    q = torch.randn(len(lens), heads, 128, generator=g).to(dtype)
    return pool, table, rows, q


def _check(got, pool, rows, q, dtype, scale=128 ** -0.5):
    got = got.cpu().double()
    heads, kv = q.shape[1], pool.kv
    for b, slots in enumerate(rows):
        if len(slots) == 0:
            assert (got[b] == 0).all(), b
            continue
        k, v = pool.rows(slots)
        for h in range(heads):
            j = h // (heads // kv)
            want, bound = ref.decode(q[b, h], tuple(t[:, j] for t in k), tuple(t[:, j] for t in v), scale)
            err = (got[b, h] - want).abs()
            assert (err <= ref.HALF[dtype] * want.abs() + bound + 2.0 ** -24).all(), (b, h, (err / (bound + ref.HALF[dtype] * want.abs())).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,heads,kv,page", [
    ([1], 1, 1, 16), ([0, 1, 2, 15, 16, 17, 31, 32, 33], 4, 2, 16), ([100, 0, 0, 257], 8, 1, 32), ([129, 64], 6, 2, 48), ([63, 500], 5, 5, 64),
    ([200], 12, 1, 128), ([77, 300], 17, 1, 16), ([1100], 4, 1, 1024), ([0], 4, 4, 16), ([3] * 70, 2, 2, 16)])
def test_decode(ops, cuda, dtype, lens, heads, kv, page):
    """Lengths of none, one, and around a tile, a chunk and a page; groups of one head, of less than a fragment's eight, and of more."""
    pool, table, rows, q = _case(lens, heads, kv, page, dtype, seed=len(lens) + heads, extra=16)
    ws = ops.Workspace()
    cache = ops.Kv4Cache(pool.bytes.to(cuda), page, kv, dtype)
    args = (q.to(cuda), cache, _i32(table, cuda), _i32(lens, cuda), ws)
    got = ops.attn_kv4_decode(*args)
    ws.check()
    _check(got, pool, rows, q, dtype)
    assert torch.equal(ops.attn_kv4_decode(*args), got)   # counters are back at zero, and the order of sums does not change
    ws.check()


@pytest.mark.parametrize("dtype", TYPES)
def test_decode_with_scales_far_apart(ops, cuda, dtype):
    """V rows of sizes 2^-10 .. 2^10 around the others', tokens with nearly all of the weight among them."""
    lens, heads, kv, page = [150, 90], 4, 1, 16
    pool, table, rows, q = _case(lens, heads, kv, page, dtype, seed=8, spread=2.5)
    ws = ops.Workspace()
    for scale in (128 ** -0.5, 1.0, 0.001, -0.2):
        got = ops.attn_kv4_decode(q.to(cuda), ops.Kv4Cache(pool.bytes.to(cuda), page, kv, dtype), _i32(table, cuda), _i32(lens, cuda), ws, scale=scale)
        ws.check()
        _check(got, pool, rows, q, dtype, scale)


def test_decode_bf16_rows_outside_of_fp16(ops, cuda):
    """q, K and V of sizes that fp16 does not have."""
    dtype, lens, heads, kv, page = torch.bfloat16, [70], 2, 1, 16
    pool, table, rows, q = _case(lens, heads, kv, page, dtype, seed=9)
    for up_q, up_k, up_v in ((2.0 ** 30, 2.0 ** -30, 2.0 ** 40), (2.0 ** -60, 2.0 ** 59, 2.0 ** -50), (0.0, 1.0, 1.0)):
        p = ref.Pool(pool.bytes.shape[0], page, kv, dtype)
        g = _gen(10)
        p.put_rows(rows[0], torch.randn(70, 1, 128, generator=g) * up_k, torch.randn(70, 1, 128, generator=g) * up_v)
        x = (q.float() * up_q).to(dtype)
        ws = ops.Workspace()
        got = ops.attn_kv4_decode(x.to(cuda), ops.Kv4Cache(p.bytes.to(cuda), page, kv, dtype), _i32(table, cuda), _i32(lens, cuda), ws)
        ws.check()
        k, v = p.rows(rows[0])
        for h in range(heads):
            want, bound = ref.decode(x[0, h], tuple(t[:, 0] for t in k), tuple(t[:, 0] for t in v), 128 ** -0.5)
            assert ((got[0, h].cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + bound).all()


def test_decode_of_q_that_is_part_of_wider_rows(ops, cuda):
    pool, table, rows, q = _case([40, 55, 7], 4, 2, 16, torch.float16, seed=11)
    wide = torch.full((3, 6 * 128 + 8), float("nan"), dtype=torch.float16, device=cuda)
    part = wide[:, 128:5 * 128]
    part.copy_(q.view(3, -1))
    big = torch.full((3, 20), -1, dtype=torch.int32, device=cuda)
    tab = big[:, :len(table[0])]
    tab.copy_(_i32(table, cuda))
    ws = ops.Workspace()
    got = ops.attn_kv4_decode(part, ops.Kv4Cache(pool.bytes.to(cuda), 16, 2, torch.float16), tab, _i32([40, 55, 7], cuda), ws)
    ws.check()
    _check(got, pool, rows, q, torch.float16)


def test_decode_nan_stays_with_its_request_and_head(ops, cuda):
    """A poisoned K row of one KV head, a poisoned V row of another request's: all heads of that group of that request are NaN (for V: every dim
    of a NaN minimum), no other."""
    dtype, lens, heads, kv = torch.float16, [50, 64, 33], 6, 2
    pool, table, rows, q = _case(lens, heads, kv, 16, dtype, seed=12)
    nan = torch.tensor(float("nan"), dtype=dtype)
    c, s, m = pool.get(int(rows[0][20]), 1, 0)
    pool.put(int(rows[0][20]), 1, 0, c, s, nan)
    c, s, m = pool.get(int(rows[2][32]), 0, 1)
    pool.put(int(rows[2][32]), 0, 1, c, s, nan)
    ws = ops.Workspace()
    got = ops.attn_kv4_decode(q.to(cuda), ops.Kv4Cache(pool.bytes.to(cuda), 16, kv, dtype), _i32(table, cuda), _i32(lens, cuda), ws).isnan()
    ws.check()
    want = torch.zeros(3, 6, dtype=torch.bool)
    want[0, 3:] = True
    want[2, :3] = True
    assert torch.equal(got.all(-1).cpu(), want) and torch.equal(got.any(-1).cpu(), want)


def test_decode_reports_pages_and_lengths_outside(ops, cuda):
    cabi = ops.cabi
    lens, heads, kv = [40, 40, 40, 40], 2, 1
    pool, table, rows, q = _case(lens, heads, kv, 16, torch.float16, seed=13)
    cache = ops.Kv4Cache(pool.bytes.to(cuda), 16, kv, torch.float16)
    ws = ops.Workspace()
    for bad in (-1, pool.bytes.shape[0], 2 ** 31 - 1):
        t = [r[:] for r in table]
        t[1] = [bad] * len(t[1])
        got = ops.attn_kv4_decode(q.to(cuda), cache, _i32(t, cuda), _i32(lens, cuda), ws)
        with pytest.raises(cabi.Qw3Error) as e:
            ws.check()
        assert e.value.status == cabi.QW3_ERR_RANGE and (got[1] == 0).all()
        for b in (0, 2, 3):
            _check(got[b:b + 1], pool, rows[b:b + 1], q[b:b + 1], torch.float16)
    for bad in (-5, 1000, 2 ** 31 - 1):   # a length that the table does not hold: cut off at its end, where there are no pages
        got = ops.attn_kv4_decode(q.to(cuda), cache, _i32(table, cuda), _i32([40, bad, 40, 40], cuda), ws)
        with pytest.raises(cabi.Qw3Error) as e:
            ws.check()
        assert e.value.status == cabi.QW3_ERR_RANGE
        for b in (0, 2, 3):
            _check(got[b:b + 1], pool, rows[b:b + 1], q[b:b + 1], torch.float16)
    got = ops.attn_kv4_decode(q.to(cuda), cache, _i32(table, cuda), _i32(lens, cuda), ws)
    ws.check()
    _check(got, pool, rows, q, torch.float16)


def test_decode_long_requests_share_ctas_and_offsets_pass_32_bits(ops, cuda):
    """Two long requests and short ones between them in a pool of 9 GB: pairs cut by the borders of CTAs, page offsets beyond 2^33."""
    dtype, kv, heads, page = torch.float16, 2, 6, 64
    lens = [30011, 5, 0, 20000, 77]
    stride = 1 << 25                          # 32 MB from page to page: other layers' pages lie between
    blocks = [-(-n // page) for n in lens]
    n_pages = 270
    pages = torch.full((n_pages, stride), 255, dtype=torch.uint8, device=cuda)[:, :kv * page * 136]
    cache = ops.Kv4Cache(pages, page, kv, dtype)
    ws = ops.Workspace()
    g = torch.Generator(device=cuda).manual_seed(4)
    # rows repeat with the pages: a block's page is its index modulo the pool's, which tests the addresses and keeps the reference small
    table = torch.stack([(torch.arange(max(blocks), device=cuda) * 7 + 31 * b) % n_pages for b in range(len(lens))]).int()
    n = n_pages * page
    qkv = torch.randn(n, 3 * kv * 128, device=cuda, generator=g).half()
    slots = torch.arange(n, device=cuda, dtype=torch.int32)
    ops.rope_kv4_append(qkv, cache, slots, None, None, None, kv, ws)
    k, v = ops.kv4_read(cache, slots, ws)
    q = torch.randn(len(lens), heads, 128, device=cuda, generator=g).half()
    got = ops.attn_kv4_decode(q, cache, table, _i32(lens, cuda), ws)
    again = ops.attn_kv4_decode(q, cache, table, _i32(lens, cuda), ws)
    ws.check()
    assert torch.equal(got, again)
    for b, m in enumerate(lens):
        t = torch.arange(m, device=cuda)
        at = table[b].long()[t // page] * page + t % page
        for h in range(heads):
            if m == 0:
                assert (got[b] == 0).all()
                continue
            kk, vv = k[at, h // 3].double(), v[at, h // 3].double()
            p = torch.softmax(kk @ q[b, h].double() * 128 ** -0.5, 0)
            want, size = p @ vv, p @ vv.abs()
            # rows are read back in fp16: half a step on each k q and each v on top of the bound of kv4_ref.decode (scores of a few units)
            d_score = (2.0 ** -11 * (kk.abs() @ q[b, h].double().abs()).max() * 128 ** -0.5)
            assert ((got[b, h].double() - want).abs() <= 2.0 ** -11 * want.abs() + (2 * d_score + 2.0 ** -9) * size).all()


def test_decode_two_streams_two_workspaces(ops, cuda):
    pool, table, rows, q = _case([700, 3, 90], 8, 2, 32, torch.bfloat16, seed=14)
    cache = ops.Kv4Cache(pool.bytes.to(cuda), 32, 2, torch.bfloat16)
    d_q, d_t, d_l = q.to(cuda), _i32(table, cuda), _i32([700, 3, 90], cuda)
    want = ops.attn_kv4_decode(d_q, cache, d_t, d_l, ops.Workspace())
    torch.cuda.synchronize()
    streams, ws, got = [torch.cuda.Stream() for _ in range(2)], [ops.Workspace(pdl=True) for _ in range(2)], [[], []]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.attn_kv4_decode(d_q, cache, d_t, d_l, ws[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for r in got for x in r)
    _check(want, pool, rows, q, torch.bfloat16)


def test_decode_step_captured_in_a_graph(ops, cuda):
    """Slots, append and attention of a batch as one captured step, lengths and stack updated in place, replayed token after token; a
    request that is idle (a padded batch) keeps its cache and gets the attention of its old tokens."""
    dtype, heads, kv, page, steps = torch.float16, 4, 2, 16, 20
    n, max_pos = 3, 64
    cos, sin = _tables(max_pos, 128)
    d_cos, d_sin = cos.to(cuda), sin.to(cuda)
    n_pages = 16
    pool = ref.Pool(n_pages, page, kv, dtype)
    cache = ops.Kv4Cache(pool.bytes.to(cuda), page, kv, dtype)
    ws = ops.Workspace(pdl=True)
    lens, new = _i32([0, 0, 0], cuda), _i32([1, 1, 0], cuda)
    table, free, n_free = torch.full((n, 6), -1, dtype=torch.int32, device=cuda), _i32(list(range(n_pages)), cuda), _i32([n_pages], cuda)
    qkv = torch.zeros(n, 8 * 128, dtype=dtype, device=cuda)

    def step():
        _, pos, slots, _, _ = ops.page_slots(lens, new, page, table, free, n_free, n, ws, kv_len=lens, n_free_out=n_free)
        q, _ = ops.rope_kv4_append(qkv, cache, slots, pos, d_cos, d_sin, heads, ws)
        return q, ops.attn_kv4_decode(q, cache, table, lens, ws)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    lens.zero_(); n_free.fill_(n_pages); table.fill_(-1)
    cache.pages.copy_(pool.bytes)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        q_out, out = step()
    lens.zero_(); n_free.fill_(n_pages); table.fill_(-1)
    g = _gen(15)
    held = [[], [], []]
    for t in range(steps):
        active = [1, int(t % 3 != 1), int(t == 4)]
        x = torch.randn(n, 8 * 128, generator=g).to(dtype)
        order = [b for b in range(n) if active[b]]      # rows of the step: the active requests in order, padding behind
        rows = x.clone()
        new.copy_(_i32(active, cuda))
        qkv.copy_(rows)
        graph.replay()
        torch.cuda.synchronize()
        y = ref.rotate(x.view(n, 8, 128)[:, :6], *(tab[torch.tensor([len(held[b]) for b in order] + [0] * (n - len(order)))] for tab in (cos, sin)), False)
        assert torch.equal(q_out.cpu(), y[:, :4].to(dtype))
        for i, b in enumerate(order):
            held[b].append((y[i, 4:6], x.view(n, 8, 128)[i, 6:]))
        tab = table.tolist()
        slots = [[tab[b][i // page] * page + i % page for i in range(len(held[b]))] for b in range(n)]
        for i, b in enumerate(order):
            pool.put_rows([slots[b][-1]], held[b][-1][0][None], held[b][-1][1][None])
        _check(out, pool, slots, q_out.cpu(), dtype)
    ws.check()
    assert torch.equal(cache.pages.cpu(), pool.bytes)
    assert lens.tolist() == [len(h) for h in held] and n_free.item() == n_pages - sum(-(-len(h) // page) for h in held)


# ---- the widest calls, and one workspace in turn ---------------------------------------------------------------------------------

@pytest.mark.parametrize("n,page,ctx_max,new_max,pad", [(16384, 16, 20, 1, 9), (16384, 64, 3, 2, 0)])
def test_page_slots_of_the_most_requests(ops, cuda, n, page, ctx_max, new_max, pad):
    test_page_slots(ops, cuda, n, page, ctx_max, new_max, pad)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,page,rot,pad,extra", [(2, 97, 3, 16, 128, 0, 0), (5, 96, 48, 32, 64, 1, 0), (1, 94, 1, 16, 0, 0, 0), (3, 300, 4, 16, 128, 0, 32),
                                                                (301, 95, 1, 16, 128, 2, 0)])
def test_append_in_slices_of_rows(ops, cuda, dtype, pairs, tokens, heads, kv, page, rot, pad, extra):
    """Tokens of 96 rows and more: slices of different sizes, some without rows of k or v."""
    test_append_and_read(ops, cuda, dtype, pairs, tokens, heads, kv, page, rot, pad, extra)


@pytest.mark.parametrize("dtype", TYPES)
def test_the_same_slot_read_many_times(ops, cuda, dtype):
    pool = ref.Pool(3, 16, 2, dtype)
    g = _gen(21)
    pool.put_rows(list(range(48)), torch.randn(48, 2, 128, generator=g), torch.randn(48, 2, 128, generator=g))
    cache, ws = ops.Kv4Cache(pool.bytes.to(cuda), 16, 2, dtype), ops.Workspace()
    slots = [5, 5, 47, -1, 5, 0, 47, 0] * 9
    once_k, once_v = ops.kv4_read(cache, _i32(list(range(48)), cuda), ws)
    k, v = ops.kv4_read(cache, _i32(slots, cuda), ws)
    ws.check()
    for i, s in enumerate(slots):
        assert torch.equal(k[i], once_k[s] if s >= 0 else torch.zeros_like(k[i])) and torch.equal(v[i], once_v[s] if s >= 0 else torch.zeros_like(v[i]))


def test_two_graphs_share_a_workspace_in_turn(ops, cuda):
    """Decode leaves its counters as it found them, so the graphs may alternate on a stream, packed attention of the same workspace between them."""
    heads, kv, page, dtype = 8, 2, 32, torch.float16
    ws, calls = ops.Workspace(pdl=True), []
    for lens, seed in (([2100, 0, 33], 5), ([1, 40, 3000], 6)):
        pool, table, rows, q = _case(lens, heads, kv, page, dtype, seed=seed)
        d_cache, d_q, d_t, d_l = ops.Kv4Cache(pool.bytes.to(cuda), page, kv, dtype), q.to(cuda), _i32(table, cuda), _i32(lens, cuda)
        want = ops.attn_kv4_decode(d_q, d_cache, d_t, d_l, ops.Workspace())
        torch.cuda.synchronize()
        ops.attn_kv4_decode(d_q, d_cache, d_t, d_l, ws)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.attn_kv4_decode(d_q, d_cache, d_t, d_l, ws)
        calls.append((graph, out, want, d_cache, d_q, d_t, d_l))
    g = torch.Generator(device=cuda).manual_seed(2)
    x = [torch.randn(300, h, 128, device=cuda, generator=g).half() for h in (heads, kv, kv)]
    cu = _i32([0, 100, 300], cuda)
    packed = ops.attn_packed(*x, cu, cu, ops.Workspace())
    for _ in range(6):
        for graph, out, want, *_ in calls:
            out.fill_(7.0)
            graph.replay()
            assert torch.equal(ops.attn_packed(*x, cu, cu, ws), packed)
            assert torch.equal(out, want)
    ws.check()
