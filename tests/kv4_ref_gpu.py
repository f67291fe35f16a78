"""Attention over the paged 4-bit cache in 64 bits on the GPU, from the bytes of the pool, for lists too long for the row-by-row restatement."""
import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # largest relative error of a rounding: finfo.eps / 2
FLOOR = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -60}
D = 128


def rows(cache, slots):
    """(codes, scale, minimum) of K and of V for the slots, in 64 bits: [slots][kv][128], [slots][kv][1], [slots][kv][1]."""
    p, kv = cache.page_size, cache.kv_heads
    slots = slots.long()
    page, tile, row = slots // p, slots % p // 16, slots % 16
    at = (torch.arange(kv, device=slots.device)[None] * (p // 16) + tile[:, None]) * 2176     # byte of the tile in its page
    out = []
    for which in (0, 1):
        b = cache.pages[page[:, None, None], (at + 1024 * which + 64 * row[:, None])[..., None] + torch.arange(64, device=slots.device)]
        pair = cache.pages[page[:, None, None], (at + 2048 + 64 * which + 4 * row[:, None])[..., None] + torch.arange(4, device=slots.device)]
        pair = pair.contiguous().view(cache.dtype).double()
        out.append((torch.stack([b % 16, b // 16], -1).flatten(-2).double(), pair[..., :1], pair[..., 1:]))
    return out


def slots_of(table_row, n, page):
    t = torch.arange(n, device=table_row.device)
    return table_row.long()[t // page] * page + t % page


def decode(q, k, v, scale, p_round):
    """q [heads][128] over k, v of rows(): the result [heads][128] and the bound of the kernel's error beside the rounding of the result.

    Scores: sums in fp32 of 128 products with the codes and of the minimum times the sum of q; the tensor cores cut off at 2^-23 of the partial
    sums, eight times, and the roundings are 2^-24: 2^-20 of the sum of the terms' sizes.  With the logarithm of V's scale added, half of the last place of
    that, and 2^-21 for the logarithm and the exponential.  All of this changes P, and with it numerator and denominator.
    P in the products with (code - 8): 2^-11 where it is one fp16 number, 2^-22 where the remainder of at most 2^-11 is a second one (11 bits
    again), and where it is below fp16's normal numbers half of their step, 2^-25, while the largest P is 2^8 at least: 2^-33 of the largest term a token.
    Sums of P code, P 8 and P (minimum + 8 scale): a warp's accumulators take 16 chunks at most, of 32 tokens, every fourth of the
    list, two products of two steps each a chunk, each of which cuts off 2^-23; then some roundings of 2^-24, and one for each part of
    the list, which has 8 chunks at least."""
    heads, kv = q.shape[0], k[0].shape[1]
    n = k[0].shape[0]
    q = q.double().view(kv, heads // kv, D)
    (kc, ks, km), (vc, vs, vm) = ([t.transpose(0, 1) for t in x] for x in (k, v))     # [kv][n][..]
    s = scale * ((q @ kc.transpose(1, 2)) * ks.transpose(1, 2) + q.sum(-1, keepdim=True) * km.transpose(1, 2))
    p = torch.softmax(s, -1)
    value = vs * vc + vm
    want, mean, size = p @ value, p @ value.abs(), p @ (vs * (vc + 8) + (vm + 8 * vs).abs())
    terms = abs(scale) * ((q.abs() @ kc.transpose(1, 2)) * ks.transpose(1, 2) + q.abs().sum(-1, keepdim=True) * km.abs().transpose(1, 2))
    floor = vs.clamp(min=2.0 ** -60)
    d_score = 2.0 ** -20 * terms.amax(-1, keepdim=True) + 2.0 ** -24 * (s.abs().amax(-1, keepdim=True) + floor.log().abs().amax()) + 2.0 ** -21
    weight = p * vs.transpose(1, 2)
    cuts = 4 * min(16, 1 + n // 128) + 8 + n / 512
    bound = 2 * d_score * mean + p_round * (p @ (vs * (vc - 8).abs())) + 8 * n * 2.0 ** -33 * weight.amax(-1, keepdim=True) + cuts * 2.0 ** -23 * size
    return want.reshape(heads, D), bound.reshape(heads, D)


def check_decode(got, q, cache, table, lens, scale=D ** -0.5, p_round=None):
    """Every output against the 64-bit one: one rounding of the result to its type, the bound of decode(), half of fp16's smallest number."""
    dtype, kv = cache.dtype, cache.kv_heads
    if p_round is None:
        p_round = 2.0 ** -22 if dtype == torch.float16 and q.shape[1] // kv <= 4 else 2.0 ** -11
    for b, n in enumerate(lens):
        if n == 0:
            assert (got[b] == 0).all(), b
            continue
        want, bound = decode(q[b], *rows(cache, slots_of(table[b], n, cache.page_size)), scale, p_round)
        ratio = (got[b].double() - want).abs() / (HALF[dtype] * want.abs() + bound + 2.0 ** -25)
        assert not ratio.isnan().any() and (ratio <= 1).all(), (b, n, ratio.max().item())
