"""Plain restatement of the paged 4-bit cache in 64 bits (torch on the CPU), from the definition in include/qw3_cabi.h."""
import torch

FLOOR = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -60}
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # largest relative error of a rounding: finfo.eps / 2


def quantise(x, dtype):
    """fp32 rows [..., 128] -> codes int64 [..., 128], scale and minimum [...] in dtype; each step in fp32 as defined."""
    x = x.float()
    lo, hi = x.amin(-1), x.amax(-1)
    m = lo.to(dtype)
    s = ((hi - m.float()) / torch.full_like(lo, 15.0)).to(dtype)
    s = torch.maximum(s.float(), torch.tensor(FLOOR[dtype])).to(dtype)
    c = torch.round((x - m.float()[..., None]) / s.float()[..., None]).clamp(0, 15)
    return c.long(), s, m


def value(codes, s, m):
    return codes.double() * s.double()[..., None] + m.double()[..., None]


class Pool:
    """Bytes of a pool and the accessors of its rows.  Everything that is never stored holds 0xff: codes of 15, pairs of NaN."""

    def __init__(self, n_pages, page, kv, dtype, extra=0):
        self.page, self.kv, self.dtype = page, kv, dtype
        self.bytes = torch.full((n_pages, kv * page * 136 + extra), 255, dtype=torch.uint8)

    def _at(self, slot, head):
        p, r = slot // self.page, slot % self.page
        return self.bytes[p], (head * (self.page // 16) + r // 16) * 2176, r % 16

    def put(self, slot, head, which, codes, s, m):
        row, tile, r = self._at(slot, head)
        c = codes.to(torch.uint8)
        row[tile + 1024 * which + 64 * r:tile + 1024 * which + 64 * r + 64] = c[0::2] | (c[1::2] << 4)
        row[tile + 2048 + 64 * which + 4 * r:tile + 2048 + 64 * which + 4 * r + 4] = torch.stack([s, m]).view(torch.uint8)

    def get(self, slot, head, which):
        row, tile, r = self._at(slot, head)
        b = row[tile + 1024 * which + 64 * r:][:64].long()
        pair = row[tile + 2048 + 64 * which + 4 * r:][:4].clone().view(self.dtype)
        return torch.stack([b % 16, b // 16], -1).flatten(), pair[0], pair[1]

    def put_rows(self, slots, k, v):
        """k, v [tokens][kv][128] fp32 into the slots."""
        for which, x in ((0, k), (1, v)):
            c, s, m = quantise(x, self.dtype)
            for i, slot in enumerate(slots):
                for h in range(self.kv):
                    self.put(int(slot), h, which, c[i, h], s[i, h], m[i, h])

    def rows(self, slots):
        """(codes, scale, minimum) of K and of V for the slots: [tokens][kv]..."""
        out = []
        for which in (0, 1):
            got = [[self.get(int(s), h, which) for h in range(self.kv)] for s in slots]
            out.append(tuple(torch.stack([torch.stack([r[i] for r in row]) for row in got]) for i in range(3)))
        return out


def rotate(x, cos, sin, pairs):
    """x [tokens][heads][128] in fp32, each product and sum rounded; cos, sin [tokens][rot / 2]."""
    x = x.float()
    half = cos.shape[1]
    c, s = cos[:, None], sin[:, None]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if pairs else (x[..., :half], x[..., half:2 * half])
    ya, yb = a * c - b * s, b * c + a * s
    y = x.clone()
    if pairs:
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = ya, yb
    else:
        y[..., :half], y[..., half:2 * half] = ya, yb
    return y


def decode(q, k, v, scale):
    """One head's attention in 64 bits over cached rows k = (codes, s, m), v: the result, and the bound of the kernel's error.

    The kernel rounds once to q's type (half a step), P to fp16 (2^-11, on every p v), and holds the rest in fp32: scores are sums of
    128 products with the codes and of m times the sum of q (2^-20 of the sum of the terms' sizes covers 130 roundings and cut-offs of
    2^-24 and 2^-23 that fall on partial sums), which changes p by that much relatively, and so numerator and denominator; the sums of
    p code and p m, each far larger than their sum, by 2^-20 of their sizes."""
    q = q.double()
    kc, ks, km = (t.double() for t in k)
    vc, vs, vm = (t.double() for t in v)
    s = scale * (ks * (kc @ q) + km * q.sum())
    p = torch.softmax(s, 0)
    out = (p[:, None] * (vs[:, None] * vc + vm[:, None])).sum(0)
    d_score = 2.0 ** -20 * (abs(scale) * (ks * (kc @ q.abs()) + km.abs() * q.abs().sum())).max() + 2.0 ** -21
    size = (p[:, None] * (vs[:, None] * vc + vm.abs()[:, None])).sum(0)
    mean = (p[:, None] * (vs[:, None] * vc + vm[:, None]).abs()).sum(0)
    return out, 2 * d_score * mean + 2.0 ** -11 * 2 * mean + 2.0 ** -20 * size
