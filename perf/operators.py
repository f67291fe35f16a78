"""What the operators for serving a batch of requests from a paged 4-bit KV cache are measured on.

  page_slots       hands the pages of a pool to requests that grow, on the GPU, and lists the cache slot of every new token
  rope_kv4_append  rotates the rows of a QKV product, quantises K and V to 4 bits and stores them in their slots
  kv4_read         the rows of given slots as dense K and V rows (a cached prefix that a prompt attends to)
  attn_kv4_decode  attention of one new token a request over its pages
  attn_packed      causal attention of packed prompts of different lengths, heads grouped over KV heads

A cache row is one token's K or V of one KV head: 128 codes of 4 bits (byte i: dim 2i in the low nibble), a scale and a minimum in the
rows' type; the value it stands for is code * scale + minimum.  16 tokens of a KV head lie together in 2176 bytes: K codes, V codes, K
(scale, minimum) pairs, V pairs; a page is [kv_heads][page / 16] of these.

Sizes are those of the repository's configurations (32 heads of 128 dims, a KV head for each, 40960 positions), the same with grouped
heads, and generic ones.
"""
import importlib
import math
import random

import torch

PACKAGE = "cuda-kernel-qwen3-8b-awq_b200"
own = False

D = 128
TILE_BYTES = 2176                      # 16 tokens of a KV head
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
SCALE_FLOOR = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -60}


def _ops():
    return importlib.import_module(PACKAGE + ".ops")


# ---- what is measured ----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of a handful of requests: one new token each; what a call costs
        {"name": "slots 7 single", "op": "slots", "requests": 7, "ctx": 2000, "new": 1, "page": 16, "spread": 1},
        # a mixed step: 250 requests, some with a chunk of a prompt, some idle
        {"name": "slots 250 mixed", "op": "slots", "requests": 250, "ctx": 8000, "new": 500, "page": 64, "spread": 2},
        # a decode step of 33 requests, two rows of padding, halves rotated
        {"name": "append 33 single", "op": "append", "tokens": 33, "heads": 32, "kv": 8, "type": "fp16", "pairs": False, "rot": 128, "page": 16,
         "run": 1, "pad": 2},
        # a document's prompt, a KV head for each head, pairs rotated as the reference does
        {"name": "append 4001 pairs", "op": "append", "tokens": 4001, "heads": 32, "kv": 32, "type": "bf16", "pairs": True, "rot": 128, "page": 64,
         "run": 4001, "pad": 0},
        # the cached prefix of a short chat, part by part of small pages
        {"name": "read 517", "op": "read", "tokens": 517, "kv": 8, "type": "fp16", "page": 16},
        # the cached prefix of a long document
        {"name": "read 30011", "op": "read", "tokens": 30011, "kv": 8, "type": "bf16", "page": 64},
        # one request of the benchmark's context length, as many KV heads as heads
        {"name": "decode 1x517", "op": "decode", "requests": 1, "lo": 517, "hi": 517, "heads": 32, "kv": 32, "type": "fp16", "page": 16, "spread": 1},
        # a batch of requests of very different lengths, one of them empty (a padded batch)
        {"name": "decode 37 ragged", "op": "decode", "requests": 37, "lo": 0, "hi": 9000, "heads": 32, "kv": 8, "type": "bf16", "page": 32,
         "spread": 2},
        # long documents up to the model's last position
        {"name": "decode 48 long", "op": "decode", "requests": 48, "lo": 20000, "hi": 40960, "heads": 32, "kv": 8, "type": "fp16", "page": 64,
         "spread": 3},
        # a few short prompts together
        {"name": "packed 5 short", "op": "packed", "seqs": 5, "lo": 1, "hi": 150, "prefix": 0, "heads": 32, "kv": 32, "type": "fp16", "spread": 1},
        # a document's prompt, grouped heads
        {"name": "packed 4001", "op": "packed", "seqs": 1, "lo": 4001, "hi": 4001, "prefix": 0, "heads": 32, "kv": 8, "type": "bf16", "spread": 2},
        # prompts of all lengths, each behind a cached prefix
        {"name": "packed 11 prefixed", "op": "packed", "seqs": 11, "lo": 3, "hi": 3000, "prefix": 2000, "heads": 32, "kv": 8, "type": "fp16", "spread": 3},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["slots", "append", "read", "decode", "decode", "packed", "packed"])
    heads, kv = rng.choice([(32, 8), (32, 32), (32, 8), (28, 4), (12, 2), (16, 1), (40, 8), (64, 8), (4, 4), (6, 2)])
    kind, page, spread = rng.choice(["fp16", "bf16"]), rng.choice([16, 32, 64, 128]), rng.randint(1, 10 ** 6)
    if op == "slots":
        return {"op": op, "requests": _log_int(rng, 1, 512), "ctx": _log_int(rng, 1, 16000), "new": _log_int(rng, 1, 500), "page": page, "spread": spread}
    if op == "append":
        tokens = _log_int(rng, 1, 4001 * 96 // (heads + 2 * kv))
        return {"op": op, "tokens": tokens, "heads": heads, "kv": kv, "type": kind, "pairs": rng.random() < 0.5, "rot": rng.choice([128, 128, 64, 32]),
                "page": page, "run": rng.choice([1, max(1, tokens // 3), tokens]), "pad": rng.choice([0, 0, 1, 3])}
    if op == "read":
        return {"op": op, "tokens": _log_int(rng, 1, 30011 * 8 // kv), "kv": kv, "type": kind, "page": page}
    if op == "decode":
        requests = _log_int(rng, 1, 128)
        hi = _log_int(rng, 1, min(40960, 48 * 30000 * 8 // (requests * max(kv, heads // 4))))
        return {"op": op, "requests": requests, "lo": rng.choice([0, hi // 2, hi]), "hi": hi, "heads": heads, "kv": kv, "type": kind, "page": page,
                "spread": spread}
    seqs = _log_int(rng, 1, 24)
    hi = max(1, min(_log_int(rng, 1, 4001), int(4000 * math.sqrt(32 / (heads * seqs)))))
    return {"op": op, "seqs": seqs, "lo": rng.choice([0, hi // 2, hi]), "hi": hi, "prefix": rng.choice([0, 0, hi // 2]), "heads": heads, "kv": kv,
            "type": kind, "spread": spread}


# ---- lengths, a function of the case alone -------------------------------------------------------------------------------------

def _lengths(case):
    """(context, new) lengths for slots, context lengths for decode, (query, key) lengths for packed."""
    rng = random.Random(case["spread"])
    if case["op"] == "slots":
        ctx = [rng.randint(0, case["ctx"]) for _ in range(case["requests"])]
        if case["new"] == 1:
            return ctx, [1] * case["requests"]
        return ctx, [rng.choice([0, 1, 1, rng.randint(1, case["new"])]) for _ in range(case["requests"])]
    n = case["requests"] if case["op"] == "decode" else case["seqs"]
    lens = [rng.randint(case["lo"], case["hi"]) for _ in range(n)]
    lens[0] = case["hi"]
    if n > 2:
        lens[n // 2] = case["lo"]
    if case["op"] == "decode":
        return lens
    return lens, [x + (rng.randint(0, case["prefix"]) if case["prefix"] else 0) for x in lens]


def work(case):
    op = case["op"]
    if op == "slots":
        ctx, new = _lengths(case)
        p = case["page"]
        pages = sum((c + x + p - 1) // p - (c + p - 1) // p for c, x in zip(ctx, new))
        return {"bytes": 16 * len(ctx) + 8 * sum(new) + 8 * pages, "flops": 0}
    if op == "append":   # rows in; q and k rows out; the cache rows, and the values they stand for
        t, h, kv = case["tokens"], case["heads"], case["kv"]
        return {"bytes": t * (256 * (h + 2 * kv) + 256 * (h + kv) + 136 * kv + 512 * kv + 4 * case["rot"] + 8),
                "flops": t * (3 * case["rot"] * (h + kv) + 5 * 256 * kv)}
    if op == "read":
        return {"bytes": case["tokens"] * (4 + case["kv"] * (136 + 512)), "flops": 512 * case["tokens"] * case["kv"]}
    if op == "decode":
        n = sum(_lengths(case))
        return {"bytes": 136 * case["kv"] * n + 512 * case["heads"] * case["requests"], "flops": 4 * D * case["heads"] * n}
    q, k = _lengths(case)
    pairs = sum(a * b - a * (a - 1) // 2 for a, b in zip(q, k))
    return {"bytes": 512 * (case["heads"] * sum(q) + case["kv"] * sum(k)), "flops": 4 * D * case["heads"] * pairs}


# ---- inputs --------------------------------------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _int(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _parts(pages, kv, page):
    """Views of the pages [n][kv][page / 16][16][...]: codes of K and V (64 bytes a row), (scale, minimum) of K and V (4 bytes a row)."""
    body = pages.view(pages.shape[0], kv, page // 16, TILE_BYTES)
    cut = lambda a, b, n: body[..., a:b].unflatten(-1, (16, n))
    return cut(0, 1024, 64), cut(1024, 2048, 64), cut(2048, 2112, 4), cut(2112, 2176, 4)


def _quantise(x, dtype):
    """fp32 rows [..., 128] -> packed codes uint8 [..., 64], (scale, minimum) in dtype [..., 2]."""
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    m = lo.to(dtype)
    # division by a tensor: by a number torch multiplies with its reciprocal, and then values halfway between two codes go astray
    s = ((hi - m.float()) / torch.full_like(lo, 15.0)).to(dtype).clamp(min=SCALE_FLOOR[dtype])
    c = torch.round((x - m.float()) / s.float()).clamp(0, 15).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.cat([s, m], -1)


def _codes(packed):
    return torch.stack([packed & 15, packed >> 4], -1).flatten(-2)


def _rows(g, n, kv, dtype):
    """K and V rows as a model's projections give them: K with channels of their own size and offset, V smaller."""
    k = torch.randn(n, kv, D, device="cuda", generator=g)
    c = torch.Generator(device="cuda")
    c.manual_seed(7)
    size = torch.exp(0.5 * torch.randn(kv, D, device="cuda", generator=c))
    k = k * size + 0.5 * torch.randn(kv, D, device="cuda", generator=c) * size
    return k, 0.5 * torch.randn(n, kv, D, device="cuda", generator=g)


def _filled_pages(g, n_pages, page, kv, dtype):
    """A pool whose every row is a quantised row."""
    pages = torch.empty(n_pages, kv * page * 136, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 19) // (page * kv))
    for a in range(0, n_pages, step):
        part = pages[a:a + step]
        views = _parts(part, kv, page)
        n = part.shape[0]
        for x, codes, pair in zip(_rows(g, n * page, kv, dtype), views[:2], views[2:]):
            q, sm = _quantise(x, dtype)
            codes.copy_(q.view(n, page // 16, 16, kv, 64).permute(0, 3, 1, 2, 4))
            pair.copy_(sm.view(torch.uint8).view(n, page // 16, 16, kv, 4).permute(0, 3, 1, 2, 4))
    return pages


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    st = {"case": case, "op": op}
    if op == "slots":
        ctx, new = _lengths(case)
        p = case["page"]
        have = [(c + p - 1) // p for c in ctx]
        need = [(c + x + p - 1) // p for c, x in zip(ctx, new)]
        width, used, spare = max(max(need), 1) + 3, sum(have), sum(need) - sum(have) + 11
        ids = torch.randperm(used + spare, device="cuda", generator=g).int()
        table = torch.full((len(ctx), width), -1, dtype=torch.int32, device="cuda")
        own_col = torch.arange(width, device="cuda")[None] < _int(have)[:, None]
        table[own_col] = ids[:used]
        st.update(ctx=_int(ctx), new=_int(new), table=table, free=ids[used:].contiguous(), n_free=_int([spare]), total=sum(new) + 5)
    elif op in ("append", "read"):
        dtype, p, kv, t = TYPES[case["type"]], case["page"], case["kv"], case["tokens"]
        run = case.get("run", t)
        starts = range(0, t, run)
        blocks = [(min(run, t - a) + 2 * p - 2) // p for a in starts]   # each run may start inside a page
        n_pages = sum(blocks) + 3
        order = torch.randperm(n_pages, device="cuda", generator=g)
        slots, at = [], 0
        first = torch.randint(0, p, (len(blocks),), generator=torch.Generator().manual_seed(seed)).tolist()
        if op == "read":
            first = [0] * len(blocks)
        if run == 1:   # single tokens: one page each
            slots = order[:t] * p + torch.tensor(first, device="cuda")
        else:
            for i, a in enumerate(starts):
                off = first[i] + torch.arange(min(run, t - a), device="cuda")
                slots.append(order[at + off // p] * p + off % p)
                at += blocks[i]
            slots = torch.cat(slots)
        st["slots"] = slots.int()
        if op == "read":
            st["pages"] = _filled_pages(g, n_pages, p, kv, dtype)
        else:
            heads, rot, max_pos = case["heads"], case["rot"], 40960
            base = torch.randint(0, max_pos - run, (len(blocks),), device="cuda", generator=g)
            st["pos"] = (base[:, None] + torch.arange(run, device="cuda")).flatten()[:t].int()
            if case["pad"]:
                st["slots"][-case["pad"]:] = -1
            k, v = _rows(g, t, kv, dtype)
            q = torch.randn(t, heads * D, device="cuda", generator=g)
            st["qkv"] = torch.cat([q, k.flatten(1), v.flatten(1)], 1).to(dtype)
            angle = torch.arange(max_pos, device="cuda", dtype=torch.float64)[:, None] * 1e6 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
            st.update(cos=angle.cos().float(), sin=angle.sin().float())
            st["pages"] = torch.zeros(n_pages, kv * p * 136, dtype=torch.uint8, device="cuda")
    elif op == "decode":
        dtype, p, kv, lens = TYPES[case["type"]], case["page"], case["kv"], _lengths(case)
        blocks = [(n + p - 1) // p for n in lens]
        n_pages = sum(blocks) + 1
        order = torch.randperm(n_pages, device="cuda", generator=g).int()
        table = torch.full((len(lens), max(max(blocks), 1)), -1, dtype=torch.int32, device="cuda")
        table[torch.arange(table.shape[1], device="cuda")[None] < _int(blocks)[:, None]] = order[:sum(blocks)]
        st.update(pages=_filled_pages(g, n_pages, p, kv, dtype), table=table, lens=_int(lens), longest=max(lens), host_lens=lens,
                  q=torch.randn(len(lens), case["heads"], D, device="cuda", generator=g).to(dtype))
    else:
        dtype, kv = TYPES[case["type"]], case["kv"]
        lq, lk = _lengths(case)
        k, v = _rows(g, sum(lk), kv, dtype)
        st.update(q=torch.randn(sum(lq), case["heads"], D, device="cuda", generator=g).to(dtype), k=k.to(dtype), v=v.to(dtype), lq=lq, lk=lk)
        for name, lens in (("cu_q", lq), ("cu_k", lk)):
            st[name] = torch.cat([_int([0]), torch.cumsum(_int(lens), 0).int()])
    if own:
        _handles(st)
    return st


def _handles(st):
    """What a user's program keeps: the workspace of its stream and the handle of its cache."""
    if "ws" not in st:
        ops = _ops()
        st["ws"] = ops.Workspace()
        if "pages" in st:
            case = st["case"]
            st["cache"] = ops.Kv4Cache(st["pages"], case["page"], case["kv"], TYPES[case["type"]])


# ---- one pass ------------------------------------------------------------------------------------------------------------------

def run(st):
    if own:
        _handles(st)
        return _OWN[st["op"]](st)
    return _PLAIN[st["op"]](st)


def _own_slots(st):
    cu, pos, slots, kv_len, n_free = _ops().page_slots(st["ctx"], st["new"], st["case"]["page"], st["table"], st["free"], st["n_free"], st["total"], st["ws"])
    return st["table"], cu, pos, slots, kv_len, n_free


def _own_append(st):
    ops, case = _ops(), st["case"]
    q, k = ops.rope_kv4_append(st["qkv"], st["cache"], st["slots"], st["pos"], st["cos"], st["sin"], case["heads"], st["ws"], pairs=case["pairs"])
    return (q, k) + tuple(ops.kv4_read(st["cache"], st["slots"], st["ws"]))


def _own_read(st):
    return _ops().kv4_read(st["cache"], st["slots"], st["ws"])


def _own_decode(st):
    return _ops().attn_kv4_decode(st["q"], st["cache"], st["table"], st["lens"], st["ws"])


def _own_packed(st):
    return _ops().attn_packed(st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], st["ws"])


_OWN = {"slots": _own_slots, "append": _own_append, "read": _own_read, "decode": _own_decode, "packed": _own_packed}


def _plain_slots(st):
    ctx, new, p, table = st["ctx"], st["new"], st["case"]["page"], st["table"]
    kv_len = ctx + new
    have, need = (ctx + p - 1) // p, (kv_len + p - 1) // p
    ends = torch.cumsum(need - have, 0).int()
    col = torch.arange(table.shape[1], device="cuda", dtype=torch.int32)[None]
    at = st["n_free"] - 1 - ((ends - (need - have))[:, None] + col - have[:, None])
    fresh = (col >= have[:, None]) & (col < need[:, None])
    table.copy_(torch.where(fresh, st["free"][at.clamp(0, st["free"].numel() - 1)], table))
    cu = torch.cat([torch.zeros_like(ctx[:1]), torch.cumsum(new, 0).int()])
    i = torch.arange(st["total"], device="cuda", dtype=torch.int32)
    b = (torch.searchsorted(cu, i, right=True) - 1).clamp(max=ctx.numel() - 1)
    real = i < cu[-1]
    pos = torch.where(real, ctx[b] + i - cu[b], 0)
    slots = torch.where(real, table[b, pos // p] * p + pos % p, -1)
    return table, cu, pos, slots, kv_len, st["n_free"] - ends[-1:]


def _rotate(x, cos, sin, pairs):
    """x [rows][heads][128]; cos, sin [rows][1][rot / 2]."""
    half = cos.shape[-1]
    r, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (r[..., 0::2], r[..., 1::2]) if pairs else (r[..., :half], r[..., half:])
    y = (a * cos - b * sin, b * cos + a * sin)
    y = torch.stack(y, -1).flatten(-2) if pairs else torch.cat(y, -1)
    return torch.cat([y, rest], -1)


def _value(packed, pair, dtype):
    sm = pair.view(dtype).float()
    return _codes(packed).float() * sm[..., :1] + sm[..., 1:]


def _plain_append(st):
    case = st["case"]
    dtype, p, kv, heads = TYPES[case["type"]], case["page"], case["kv"], case["heads"]
    x = st["qkv"].float().unflatten(1, (heads + 2 * kv, D))
    cos, sin = (t[st["pos"]][:, None] for t in (st["cos"], st["sin"]))
    q, k, v = _rotate(x[:, :heads], cos, sin, case["pairs"]), _rotate(x[:, heads:heads + kv], cos, sin, case["pairs"]), x[:, heads + kv:]
    n = case["tokens"] - case["pad"]
    slot = st["slots"][:n].long()
    page, tile, row = slot // p, slot % p // 16, slot % 16
    views = _parts(st["pages"], kv, p)
    head = torch.arange(kv, device="cuda")[None]
    out = []
    for rows, codes, pair in zip((k, v), views[:2], views[2:]):
        packed, sm = _quantise(rows[:n], dtype)
        sm = sm.view(torch.uint8)
        codes[page[:, None], head, tile[:, None], row[:, None]] = packed
        pair[page[:, None], head, tile[:, None], row[:, None]] = sm
        value = torch.zeros(rows.shape, dtype=dtype, device="cuda")
        value[:n] = _value(packed, sm, dtype).to(dtype)
        out.append(value)
    return q.to(dtype), k.to(dtype), out[0], out[1]


def _plain_read(st):
    case = st["case"]
    dtype, p = TYPES[case["type"]], case["page"]
    slot = st["slots"].long()
    kc, vc, ks, vs = (t[slot // p, :, slot % p // 16, slot % 16] for t in _parts(st["pages"], case["kv"], p))
    return _value(kc, ks, dtype).to(dtype), _value(vc, vs, dtype).to(dtype)


def _plain_decode(st):
    case = st["case"]
    dtype, p, kv, heads = TYPES[case["type"]], case["page"], case["kv"], case["heads"]
    views = _parts(st["pages"], kv, p)
    out = torch.zeros_like(st["q"])
    for b, n in enumerate(st["host_lens"]):
        if n == 0:
            continue
        ids = st["table"][b, :(n + p - 1) // p].long()
        kc, vc, ks, vs = (t[ids].transpose(0, 1).flatten(1, 3)[:, :n] for t in views)       # [kv][n][...]
        q = st["q"][b].float().view(kv, heads // kv, D)
        s = q @ _value(kc, ks.contiguous(), dtype).transpose(1, 2) * D ** -0.5
        e = torch.exp(s - s.amax(-1, keepdim=True))
        o = e @ _value(vc, vs.contiguous(), dtype) / e.sum(-1, keepdim=True)
        out[b] = o.view(heads, D).to(dtype)
    return out


def _plain_packed(st):
    case = st["case"]
    dtype, kv, heads = TYPES[case["type"]], case["kv"], case["heads"]
    out = torch.zeros_like(st["q"])
    a = c = 0
    for nq, nk in zip(st["lq"], st["lk"]):
        if nq:
            q = st["q"][a:a + nq].float().view(nq, kv, heads // kv, D).permute(1, 2, 0, 3)
            k, v = (t[c:c + nk].float().permute(1, 0, 2) for t in (st["k"], st["v"]))
            seen = torch.arange(nk, device="cuda")[None] <= torch.arange(nk - nq, nk, device="cuda")[:, None]
            for h in range(kv):
                s = (q[h] @ k[h].T * D ** -0.5).masked_fill(~seen, -math.inf)
                e = torch.exp(s - s.amax(-1, keepdim=True))
                o = e @ v[h] / e.sum(-1, keepdim=True)
                out[a:a + nq, h * (heads // kv):(h + 1) * (heads // kv)] = o.transpose(0, 1).to(dtype)
        a, c = a + nq, c + nk
    return out


_PLAIN = {"slots": _plain_slots, "append": _plain_append, "read": _plain_read, "decode": _plain_decode, "packed": _plain_packed}


# ---- the same from the definitions in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"slots": _exact_slots, "append": _exact_append, "read": _exact_read, "decode": _exact_decode, "packed": _exact_packed}[case["op"]](case, st)


def _exact_slots(case, st):
    p = case["page"]
    ctx, new = _lengths(case)
    table, free, left = st["table"].tolist(), st["free"].tolist(), st["n_free"].item()
    cu, pos, slots = [0], [], []
    for b, (c, n) in enumerate(zip(ctx, new)):
        for t in range(c, c + n):
            if t % p == 0:                      # the first token of a block takes the top of the stack
                left -= 1
                table[b][t // p] = free[left]
            pos.append(t)
            slots.append(table[b][t // p] * p + t % p)
        cu.append(len(pos))
    more = st["total"] - len(pos)
    return _int(table), _int(cu), _int(pos + [0] * more), _int(slots + [-1] * more), _int([c + n for c, n in zip(ctx, new)]), _int([left])


def _exact_append(case, st):
    dtype, kv, heads, half, t = TYPES[case["type"]], case["kv"], case["heads"], case["rot"] // 2, case["tokens"]
    x = st["qkv"].double().view(t, heads + 2 * kv, D)
    at = st["pos"].long()
    angle = torch.complex(st["cos"][at].double(), st["sin"][at].double())[:, None]
    first = torch.arange(half, device="cuda") * (2 if case["pairs"] else 1)
    second = first + (1 if case["pairs"] else half)
    y = x[:, :heads + kv].clone()
    turned = torch.complex(y[..., first], y[..., second]) * angle
    y[..., first], y[..., second] = turned.real, turned.imag
    values = []
    for rows in (y[:, heads:], x[:, heads + kv:]):
        m = rows.min(-1, keepdim=True).values.to(dtype).double()
        s = ((rows.max(-1, keepdim=True).values - m) / 15).to(dtype).double().clamp_min(SCALE_FLOOR[dtype])
        value = ((rows - m) / s).round().clamp(0, 15) * s + m
        value[t - case["pad"]:] = 0
        values.append(value)
    return y[:, :heads], y[:, heads:], values[0], values[1]


def _exact_cache(case, st, slot):
    """Values of the K and V rows of the slots, [slots][kv][128] in 64 bits, from the bytes."""
    p, kv, dtype = case["page"], case["kv"], TYPES[case["type"]]
    tiles = st["pages"].view(-1, TILE_BYTES)
    tile = ((slot // p)[:, None] * kv + torch.arange(kv, device="cuda")) * (p // 16) + (slot % p // 16)[:, None]
    row = (slot % 16)[:, None, None]
    out = []
    for which in (0, 1):
        byte = tiles[tile[..., None], 1024 * which + 64 * row + torch.arange(64, device="cuda")]
        pair = tiles[tile[..., None], 2048 + 64 * which + 4 * row + torch.arange(4, device="cuda")].view(dtype).double()
        code = torch.empty(*byte.shape[:2], D, dtype=torch.float64, device="cuda")
        code[..., 0::2], code[..., 1::2] = (byte % 16).double(), (byte // 16).double()
        out.append(code * pair[..., :1] + pair[..., 1:])
    return out


def _exact_read(case, st):
    return tuple(_exact_cache(case, st, st["slots"].long()))


def _exact_decode(case, st):
    kv, heads, p = case["kv"], case["heads"], case["page"]
    out = torch.zeros(case["requests"], heads, D, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        t = torch.arange(n, device="cuda")
        slot = st["table"][b].long()[t // p] * p + t % p
        if n:
            k, v = _exact_cache(case, st, slot)
            q = st["q"][b].double().view(kv, heads // kv, D)
            weight = torch.softmax(torch.einsum("kgd,nkd->kgn", q, k) / math.sqrt(D), -1)
            out[b] = torch.einsum("kgn,nkd->kgd", weight, v).reshape(heads, D)
    return out


def _exact_packed(case, st):
    heads, kv = case["heads"], case["kv"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    cq, ck = st["cu_q"].tolist(), st["cu_k"].tolist()
    for i in range(case["seqs"]):
        q, k, v = st["q"][cq[i]:cq[i + 1]].double(), st["k"][ck[i]:ck[i + 1]].double(), st["v"][ck[i]:ck[i + 1]].double()
        for h in range(heads):
            g = h // (heads // kv)
            for a in range(0, len(q), 1024):
                last = len(k) - len(q) + torch.arange(a, min(a + 1024, len(q)), device="cuda")
                keys = int(len(k) - len(q) + min(a + 1024, len(q)))
                s = (q[a:a + 1024, h] @ k[:keys, g].T) / math.sqrt(D)
                s[torch.arange(keys, device="cuda") > last[:, None]] = -math.inf
                out[cq[i] + a:cq[i] + min(a + 1024, len(q)), h] = torch.softmax(s, -1) @ v[:keys, g]
    return out
