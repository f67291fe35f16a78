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


# A product of the tensor cores: 16 terms and the accumulator are brought to the exponent of the largest and each is cut off 2^-23 below it (M. Fasi
# et al., Numerical behavior of NVIDIA tensor cores, 2021).  The exponent of a term is that of its operands as they are encoded, and a code in the low
# bits of a half is a subnormal number, 2^-14 times code / 1024 (code / 64 four bits further up): in units of the code the cut-off is at 2^-23 of
# 1024 (64) times the other operand, or of the accumulator if that is larger.
CUT = 17 * 2.0 ** -23


def _score_errors(q, kc, ks, km, scale, dtype):
    """Largest error of the scores s = scale (ks sum code q + km sum q) as the kernel sums them.  q [kv][g][128], kc [kv][n][128]: [kv][g][n].

    Byte i of a row holds dims 2i and 2i + 1; lane t of four has 16 bytes, and step j of four takes four of them in all lanes: even dims in one accumulator,
    odd ones, whose codes lie four bits further up, in another.  The sum of q: pairs of dims one after the other in a lane, then the four lanes."""
    out = torch.empty(q.shape[0], q.shape[1], kc.shape[1], dtype=torch.float64, device=q.device)
    up = torch.tensor([1024.0, 64.0], dtype=torch.float64, device=q.device)
    for h in range(q.shape[1]):
        p = (kc * q[:, h:h + 1]).view(*kc.shape[:2], 4, 4, 4, 2)              # [kv][n][t][j][..][even, odd]
        after = p.sum((2, 4)).cumsum(2)                                       # [kv][n][j][even, odd]
        before = torch.cat([torch.zeros_like(after[:, :, :1]), after[:, :, :-1]], 2)
        least = 2.0 ** -14 if dtype == torch.float16 else 0.0                 # the exponent that smaller q are encoded with
        terms = up * q[:, h].abs().clamp(min=least).view(-1, 1, 4, 4, 4, 2).amax((2, 4))
        largest = torch.maximum(terms, torch.maximum(before.abs(), after.abs()))
        code = CUT * largest.sum((2, 3)) + 2.0 ** -23 * after[:, :, -1].abs().sum(-1)
        pairs = q[:, h].view(-1, 4, 16, 2).sum(-1)
        one = pairs.cumsum(-1)
        q_sum = 2.0 ** -24 * (pairs.abs().sum((1, 2)) + one.abs().sum((1, 2)) + 2 * one[..., -1].abs().sum(-1))
        dot, total = after[:, :, -1].sum(-1), q[:, h].sum(-1)[:, None]
        out[:, h] = abs(scale) * (ks * code + km.abs() * q_sum[:, None] + 2.0 ** -22 * ((ks * dot).abs() + (km * total).abs()))
    return out


def decode(q, k, v, scale, p_round, dtype, warp_chunks=40, no_cuts=False):
    """q [heads][128] over k, v of rows(): the result [heads][128] and the bound of the kernel's error beside the rounding of the result.

    Scores: _score_errors, and 2^-23 of a score and of the logarithm of V's scale for the roundings of their sum and of its difference from the maximum;
    2^-21 for the logarithm and the exponential.  All of this changes P, and with it numerator and denominator.
    P in the products with (code - 8): 2^-11 where it is one fp16 number, 2^-22 where the remainder of at most 2^-11 is a second one (11 bits
    again), and where it is below fp16's normal numbers half of their step, 2^-25, while the largest P is 2^8 at least: 2^-33 of the largest term a token.
    Sums of P code and P 8, one product a tile of 16 tokens each: CUT of 1024 times the tile's largest P (2^-14 at least), and of the accumulator, which
    holds 16 chunks of 32 tokens at most, every fourth of the list.  no_cuts: P within a factor of 8 and 32 tokens an accumulator, where nothing is cut
    off: a term has 15 bits from a place 20 below its encoded exponent upwards, and the sum 24 bits; the second numbers of P are cut off 2^-11 below.
    Sums of P and of P (minimum + 8 scale) over a scale's reciprocal in fp32: four additions a chunk in a lane, at most `warp_chunks` of them, some
    roundings more, and one for each part of the list, which has 8 chunks at least."""
    heads, kv = q.shape[0], k[0].shape[1]
    n = k[0].shape[0]
    q = q.double().view(kv, heads // kv, D)
    (kc, ks, km), (vc, vs, vm) = ([t.transpose(0, 1) for t in x] for x in (k, v))     # [kv][n][..]
    s = scale * ((q @ kc.transpose(1, 2)) * ks.transpose(1, 2) + q.sum(-1, keepdim=True) * km.transpose(1, 2))
    p = torch.softmax(s, -1)
    value = vs * vc + vm
    want, code_part, least_part = p @ value, p @ (vs * (vc + 8)), p @ (vm + 8 * vs).abs()
    d = _score_errors(q, kc, ks[..., 0], km[..., 0], scale, dtype) + 2.0 ** -23 * (s.abs() + vs[..., 0].clamp(min=2.0 ** -60).log().abs()[:, None]) + 2.0 ** -21
    chunks = min(warp_chunks, 1 + n // 128)
    added = (4 * chunks + 8 + n / 256) * 2.0 ** -24
    weight = p * vs.transpose(1, 2)
    top = weight.amax(-1, keepdim=True)
    tiles = torch.nn.functional.pad(weight, (0, -n % 16)).unflatten(-1, (-1, 16)).amax(-1)
    cuts = 2 * 1024 * CUT * torch.maximum(tiles, 2.0 ** -22 * top).sum(-1, keepdim=True) + CUT * 2 * min(16, chunks) * code_part
    if no_cuts:
        assert chunks == 1 and (top <= 8 * weight.amin(-1, keepdim=True)).all()
        cuts = 2.0 ** -11 * cuts
    pd = p * d
    bound = (pd @ value.abs() + pd.sum(-1, keepdim=True) * want.abs()                                # P: numerator, denominator
             + p_round * (p @ (vs * (vc - 8).abs())) + 8 * n * 2.0 ** -33 * top                      # its rounding in the products
             + cuts + added * (code_part + least_part + want.abs()))                                 # sums
    return want.reshape(heads, D), 1.01 * bound.reshape(heads, D)


def check_decode(got, q, cache, table, lens, scale=D ** -0.5, p_round=None, no_cuts=False):
    """Every output against the 64-bit one: one rounding of the result to its type, the bound of decode(), half of fp16's smallest number."""
    dtype, kv = cache.dtype, cache.kv_heads
    if p_round is None:
        p_round = 2.0 ** -22 if dtype == torch.float16 and q.shape[1] // kv <= 4 else 2.0 ** -11
    for b, n in enumerate(lens):
        if n == 0:
            assert (got[b] == 0).all(), b
            continue
        want, bound = decode(q[b], *rows(cache, slots_of(table[b], n, cache.page_size)), scale, p_round, dtype, no_cuts=no_cuts)
        ratio = (got[b].double() - want).abs() / (HALF[dtype] * want.abs() + bound + 2.0 ** -25)
        assert not ratio.isnan().any() and (ratio <= 1).all(), (b, n, ratio.max().item())
