"""Per-operator entry points of the C ABI on torch CUDA tensors.

torch is used for device memory and streams only; every operator runs in libqw3awq.so.  fp16
tensors are torch.float16; packed weights are torch.uint8.
"""
import ctypes as C

import torch

from . import cabi


def _stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


class Workspace:
    """Of the device that is current when it is made."""

    def __init__(self, pdl=False):
        self.h = C.c_void_p()
        self.device = torch.cuda.current_device()
        cabi.check(cabi.lib().qw3_ws_create(C.byref(self.h)), "qw3_ws_create")
        cabi.check(cabi.lib().qw3_ws_set_pdl(self.h, int(pdl)), "qw3_ws_set_pdl")

    def check(self):
        """Waits for the current stream of the workspace's device, whichever is current, and raises what its operators reported."""
        with torch.cuda.device(self.device):
            cabi.check(cabi.lib().qw3_ws_check(self.h, _stream()), "qw3_ws_check")

    def close(self):
        if self.h.value:
            cabi.lib().qw3_ws_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class W4Linear:
    """One AWQ matrix in the on-disk layout, resident on the GPU (AWQWeight without d_dq)."""

    def __init__(self, packed, scale, zp, out_dim, in_dim, zp_integral=True):
        self.packed, self.scale, self.zp = packed, scale, zp   # keep the tensors alive
        self.out_dim, self.in_dim = out_dim, in_dim
        self.h = C.c_void_p()
        cabi.check(cabi.lib().qw3_w4_create(_ptr(packed), _ptr(scale), _ptr(zp), scale.numel(), out_dim, in_dim,
                                            int(zp_integral), C.byref(self.h)), "qw3_w4_create")

    def close(self):
        if self.h.value:
            cabi.lib().qw3_w4_destroy(self.h)
            self.h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


def dequant_w4(packed, scale, zp, rows, cols):
    out = torch.empty((rows, cols), dtype=torch.float16, device=packed.device)
    cabi.check(cabi.lib().qw3_dequant_w4(_ptr(packed), _ptr(scale), _ptr(zp), scale.numel(), rows, cols, _ptr(out), _stream()),
               "qw3_dequant_w4")
    return out


def gemv_args(x, epilogue=cabi.EPI_STORE, y=None, gamma=None, eps=1e-6, k_cache=None, v_cache=None, cos=None, sin=None,
              heads=0, max_pos=0, d_pos=None, pos=0, d_token=None, logits_f32=None):
    a = cabi.GemvArgs()
    a.d_x, a.d_gamma, a.eps, a.epilogue, a.d_y = _ptr(x), _ptr(gamma), eps, epilogue, _ptr(y)
    a.d_k_cache, a.d_v_cache, a.d_cos, a.d_sin = _ptr(k_cache), _ptr(v_cache), _ptr(cos), _ptr(sin)
    a.heads, a.head_dim, a.max_pos, a.d_pos, a.pos = heads, 128, max_pos, _ptr(d_pos), pos
    a.d_token, a.d_logits_f32 = _ptr(d_token), _ptr(logits_f32)
    return a


def gemv_w4a16(w, ws, args):
    cabi.check(cabi.lib().qw3_gemv_w4a16(w.h, C.byref(args), ws.h, _stream()), "qw3_gemv_w4a16")


def gemm_w4a16(w, ws, x, y):
    cabi.check(cabi.lib().qw3_gemm_w4a16(w.h, _ptr(x), x.shape[0], _ptr(y), ws.h, _stream()), "qw3_gemm_w4a16")


def gemm_w4a16_epilogue(w, ws, x, y, epilogue):
    cabi.check(cabi.lib().qw3_gemm_w4a16_epilogue(w.h, _ptr(x), x.shape[0], _ptr(y), ws.h, epilogue, _stream()), "qw3_gemm_w4a16_epilogue")


def rmsnorm(x, gamma, eps=1e-6):
    out = torch.empty_like(x)
    cabi.check(cabi.lib().qw3_rmsnorm(_ptr(x), _ptr(gamma), x.numel(), eps, _ptr(out), _stream()), "qw3_rmsnorm")
    return out


def rope_kv_append(qkv, q_out, k_cache, v_cache, cos, sin, heads, max_pos, pos, d_pos=None):
    cabi.check(cabi.lib().qw3_rope_kv_append(_ptr(qkv), _ptr(q_out), _ptr(k_cache), _ptr(v_cache), _ptr(cos), _ptr(sin),
                                             heads, 128, max_pos, _ptr(d_pos), pos, _stream()), "qw3_rope_kv_append")


def attn_decode(q, k_cache, v_cache, heads, max_pos, pos, ws, d_pos=None):
    ctx = torch.empty(heads * 128, dtype=torch.float16, device=q.device)
    cabi.check(cabi.lib().qw3_attn_decode(_ptr(q), _ptr(k_cache), _ptr(v_cache), heads, 128, max_pos, _ptr(d_pos), pos,
                                          _ptr(ctx), ws.h, _stream()), "qw3_attn_decode")
    return ctx


def attn_prefill(qkv, k_cache, v_cache, heads, max_pos, pos0, rows):
    """Causal attention of a block of prompt rows (qkv: [rows][3 * heads * 128], q already rotated)."""
    ctx = torch.empty(rows, heads * 128, dtype=torch.float16, device=qkv.device)
    cabi.check(cabi.lib().qw3_attn_prefill(_ptr(qkv), _ptr(k_cache), _ptr(v_cache), heads, 128, max_pos, pos0, rows, _ptr(ctx),
                                           _stream()), "qw3_attn_prefill")
    return ctx


def embed_gather_w4(packed, scale, zp, hidden, vocab, token, d_token=None):
    out = torch.empty(hidden, dtype=torch.float16, device=packed.device)
    cabi.check(cabi.lib().qw3_embed_gather_w4(_ptr(packed), _ptr(scale), _ptr(zp), scale.numel(), hidden, vocab,
                                              _ptr(d_token), token, _ptr(out), _stream()), "qw3_embed_gather_w4")
    return out


def argmax_f16(logits, ws):
    tok = torch.zeros(1, dtype=torch.int32, device=logits.device)
    cabi.check(cabi.lib().qw3_argmax_f16(_ptr(logits), logits.numel(), _ptr(tok), ws.h, _stream()), "qw3_argmax_f16")
    return tok


# ---- paged 4-bit KV cache: many requests, heads grouped over KV heads, fp16 or bf16 rows ----------------------------------------
# Tensors may live on any CUDA device (all of a call, and its workspace, on the same one); the call goes to that device's current
# stream.  What the device finds out of range is left out and reported by Workspace.check().

_I32 = torch.int32
_DTYPES = {torch.float16: cabi.F16, torch.bfloat16: cabi.BF16}


def _want(cond, message):
    if not cond:
        raise ValueError(message)


def _rows128(t, heads, what, device, dtype):
    """Rows of `heads` x 128 values, the heads of a token together: [tokens][heads][128], or [tokens][heads * 128] where heads is given."""
    shape, stride = t.shape, t.stride()
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{what}: {dtype} on {device} expected")
    if len(shape) == 3:
        n = shape[1]
        if shape[2] != 128 or stride[2] != 1 or (n > 1 and stride[1] != 128):
            raise ValueError(f"{what}: [tokens][heads][128] expected, the heads of a token together")
    else:
        if len(shape) != 2 or shape[1] % 128 or stride[1] != 1:
            raise ValueError(f"{what}: [tokens][heads * 128] expected")
        n = shape[1] // 128
    if heads is not None and n != heads:
        raise ValueError(f"{what}: {heads} heads expected, not {n}")
    return n, (stride[0] if shape[0] > 1 else n * 128)


def _ints(t, n, what, device):
    if t.dtype is _I32 and t.device == device and t.shape == (n,) and t.is_contiguous():
        return t.data_ptr()
    raise ValueError(f"{what}: contiguous int32 [{n}] on {device} expected")


def _table(t, rows, device):
    shape = t.shape
    if t.dtype != torch.int32 or t.device != device or len(shape) != 2 or shape[0] != rows or shape[1] == 0 or (shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"block_table: int32 [{rows}][blocks] on {device} expected")
    return t.stride(0) if rows > 1 else shape[1]


# The private functions take less of a call's time than the public ones; a build of torch without CUDA has none of them.
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda index: torch.cuda.current_stream(index).cuda_stream)


def _on(device, name, *args):
    """Calls entry point `name` on the device's current stream."""
    index = device.index
    if index is None or device.type != "cuda":
        raise ValueError(f"{name}: CUDA tensors expected")
    if index == _current_device():
        status = getattr(cabi.lib(), name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = getattr(cabi.lib(), name)(*args, _raw_stream(index))
    if status:
        cabi.check(status, name)


def _scale(scale):
    """As the C ABI takes it: fp32, 0 for 1 / sqrt(128).  A number that fp32 rounds to 0 must not become that."""
    if scale is None:
        return 0.0
    _want(C.c_float(scale).value != 0, "scale: 0 in fp32 is not a scale")
    return scale


class Kv4Cache:
    """A pool of pages of 4-bit K and V rows of one layer.  pages: uint8 [n_pages][page_bytes] (rows may be further apart, as where the
    pages of several layers are interleaved), page_bytes = kv_heads * page_size * 136."""

    def __init__(self, pages, page_size, kv_heads, dtype):
        _want(pages.dtype == torch.uint8 and pages.dim() == 2 and pages.shape[0] > 0 and pages.stride(1) == 1, "pages: uint8 [n_pages][bytes] expected")
        _want(dtype in _DTYPES, "dtype: torch.float16 or torch.bfloat16 expected")
        _want(page_size >= 16 and page_size % 16 == 0 and kv_heads > 0, "page_size: a multiple of 16 expected, and kv_heads above 0")
        _want(pages.shape[1] >= kv_heads * page_size * 136, f"pages: {kv_heads * page_size * 136} bytes a page expected")
        self.pages, self.page_size, self.kv_heads, self.dtype = pages, page_size, kv_heads, dtype
        stride = pages.stride(0) if pages.shape[0] > 1 else kv_heads * page_size * 136
        self.device = pages.device
        self.pool = cabi.Kv4Pool(pages.data_ptr(), pages.shape[0], stride, page_size, kv_heads, 128, _DTYPES[dtype])
        self.ref = C.byref(self.pool)

    @classmethod
    def alloc(cls, n_pages, page_size, kv_heads, dtype=torch.float16, device="cuda"):
        return cls(torch.zeros(n_pages, kv_heads * page_size * 136, dtype=torch.uint8, device=device), page_size, kv_heads, dtype)


def page_slots(ctx_len, new_len, page_size, block_table, free_pages, n_free, max_tokens, ws, kv_len=None, n_free_out=None):
    """Pages for new_len[b] more tokens of each request, taken from the top of the stack free_pages[: n_free].  Updates block_table; returns
    (cu, pos, slots, kv_len, n_free_out): new tokens before each request, position and slot of each new token (0 and -1 behind the last),
    the new lengths and what is left of the stack.  kv_len=ctx_len and n_free_out=n_free update those in place."""
    dev, n = ctx_len.device, ctx_len.shape[0]
    d_ctx = _ints(ctx_len, n, "ctx_len", dev)
    d_new = _ints(new_len, n, "new_len", dev)
    capacity = free_pages.numel()
    d_free = _ints(free_pages, capacity, "free_pages", dev)
    d_n_free = _ints(n_free, 1, "n_free", dev)
    stride = _table(block_table, n, dev)
    if not 0 <= max_tokens < 2 ** 31:
        raise ValueError("max_tokens: out of range")
    cu, pos, slots, own_len, own_free = ctx_len.new_empty(2 * n + 2 + 2 * max_tokens).split_with_sizes((n + 1, max_tokens, max_tokens, n, 1))
    kv_len = own_len if kv_len is None else kv_len
    n_free_out = own_free if n_free_out is None else n_free_out
    a = cabi.PageArgs(d_ctx, d_new, n, page_size, block_table.data_ptr(), stride, block_table.shape[1], capacity, d_free, d_n_free,
                      _ints(n_free_out, 1, "n_free_out", dev), cu.data_ptr(), _ints(kv_len, n, "kv_len", dev), pos.data_ptr(), slots.data_ptr(), max_tokens)
    _on(dev, "qw3_page_slots", C.byref(a), ws.h)
    return cu, pos, slots, kv_len, n_free_out


def rope_kv4_append(qkv, cache, slots, pos, cos, sin, heads, ws, pairs=False):
    """Rotates q and k of the rows qkv = [tokens][(heads + 2 kv_heads) * 128] by the angles of cos, sin = fp32 [max_pos][rot_dim / 2] (None: not
    at all) at pos, and stores k and v in 4 bits in their slots, which differ (below 0: not stored).  Returns the rotated q [tokens][heads][128] and
    k [tokens][kv_heads][128].  pairs: dims 2i and 2i + 1 turn together, as in rope_kv_append; else i and i + rot_dim / 2."""
    dev, kv, dtype = qkv.device, cache.kv_heads, cache.dtype
    _want(cache.device == dev, "qkv and the cache's pages: one device expected")
    _, stride = _rows128(qkv, heads + 2 * kv, "qkv", dev, dtype)
    tokens = qkv.shape[0]
    d_slots = _ints(slots, tokens, "slots", dev)
    rot, max_pos, d_pos, d_cos, d_sin = 0, 0, None, None, None
    if cos is not None:
        d_pos = _ints(pos, tokens, "pos", dev)
        for t, what in ((cos, "cos"), (sin, "sin")):
            _want(t is not None and t.dtype == torch.float32 and t.device == dev and t.dim() == 2 and t.is_contiguous() and t.shape == cos.shape,
                  f"{what}: contiguous float32 [max_pos][rot_dim / 2] on {dev} expected")
        max_pos, rot = cos.shape
        rot *= 2
        _want(max_pos > 0 and rot > 0, "cos: [max_pos][rot_dim / 2] expected")
        d_cos, d_sin = cos.data_ptr(), sin.data_ptr()
    q, k = qkv.new_empty((tokens, heads, 128)), qkv.new_empty((tokens, kv, 128))
    a = cabi.Kv4AppendArgs(qkv.data_ptr(), stride, tokens, heads, cabi.ROPE_PAIRS if pairs else cabi.ROPE_HALVES, rot, 0, d_slots, d_pos, d_cos, d_sin, max_pos,
                           q.data_ptr(), k.data_ptr())
    _on(dev, "qw3_rope_kv4_append", cache.ref, C.byref(a), ws.h)
    return q, k


def kv4_read(cache, slots, ws):
    """The rows of the slots as dense K and V, [tokens][kv_heads][128] each; zeros for a slot below 0."""
    dev = cache.device
    tokens = slots.numel()
    d_slots = _ints(slots, tokens, "slots", dev)
    k = torch.empty((tokens, cache.kv_heads, 128), dtype=cache.dtype, device=dev)
    v = torch.empty_like(k)
    _on(dev, "qw3_kv4_read", cache.ref, d_slots, tokens, k.data_ptr(), v.data_ptr(), ws.h)
    return k, v


def attn_kv4_decode(q, cache, block_table, kv_len, ws, scale=None):
    """Attention of one token a request, q = [requests][heads][128] after rotation, over the request's kv_len tokens in the cache; a row of
    zeros where there are none.  scale: of the scores, 1 / sqrt(128) by default."""
    dev, dtype = q.device, cache.dtype
    _want(cache.device == dev, "q and the cache's pages: one device expected")
    scale = _scale(scale)
    heads, stride = _rows128(q, None, "q", dev, dtype)
    n = q.shape[0]
    d_len = _ints(kv_len, n, "kv_len", dev)
    table_stride = _table(block_table, n, dev)
    out = torch.empty_like(q) if q.dim() == 3 and q.is_contiguous() else q.new_empty((n, heads, 128))
    a = cabi.AttnKv4Args(q.data_ptr(), stride, n, heads, block_table.data_ptr(), table_stride, block_table.shape[1], scale, d_len, out.data_ptr())
    _on(dev, "qw3_attn_kv4_decode", cache.ref, C.byref(a), ws.h)
    return out


def attn_packed(q, k, v, cu_q, cu_k, ws, scale=None, out=None):
    """Causal attention of packed sequences: q [q_rows][heads][128], k and v [k_rows][kv_heads][128] (rows may be further apart), sequence b in
    rows cu_q[b] .. cu_q[b + 1] of q and cu_k[b] .. cu_k[b + 1] of k and v.  Its queries are its last rows: row i of nq sees keys
    0 .. nk - nq + i, a row that sees none is zeros.  Rows behind the last sequence are left as they were (undefined in a new `out`).
    `out` must not share memory with q, k or v."""
    dev, dtype = q.device, q.dtype
    _want(dtype in _DTYPES, "q: torch.float16 or torch.bfloat16 expected")
    _want(scale is None or scale > 0, "scale: above 0 expected")
    scale = _scale(scale)
    heads, q_stride = _rows128(q, None, "q", dev, dtype)
    kv, k_stride = _rows128(k, None, "k", dev, dtype)
    _, v_stride = _rows128(v, kv, "v", dev, dtype)
    _want(v.shape[0] == k.shape[0], "k and v: the same number of rows expected")
    n = cu_q.numel() - 1
    _want(n >= 0, "cu_q: [sequences + 1] expected")
    d_cu_q, d_cu_k = _ints(cu_q, n + 1, "cu_q", dev), _ints(cu_k, n + 1, "cu_k", dev)
    if out is None:
        out = torch.empty_like(q) if q.dim() == 3 and q.is_contiguous() else q.new_empty((q.shape[0], heads, 128))
    else:
        _want(out.device == dev and out.dtype == dtype and out.is_contiguous() and out.numel() == q.shape[0] * heads * 128,
              "out: contiguous [q_rows][heads][128] expected")
    a = cabi.AttnPackedArgs(q.data_ptr(), q_stride, k.data_ptr(), k_stride, v.data_ptr(), v_stride, q.shape[0], k.shape[0], d_cu_q, d_cu_k, n,
                            heads, kv, 128, _DTYPES[dtype], scale, out.data_ptr())
    _on(dev, "qw3_attn_packed", C.byref(a), ws.h)
    return out
