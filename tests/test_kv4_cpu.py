"""Refusals of the operators of the paged 4-bit cache, which need no GPU, and the layout of their argument blocks."""
import ctypes as C
import importlib
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PTR = 4096   # an address that is never read: every call below is refused before


@pytest.mark.parametrize("struct,cls", [("Qw3Kv4Pool", "Kv4Pool"), ("Qw3PageArgs", "PageArgs"), ("Qw3Kv4AppendArgs", "Kv4AppendArgs"), ("Qw3AttnKv4Args", "AttnKv4Args"),
                                        ("Qw3AttnPackedArgs", "AttnPackedArgs")])
def test_argument_blocks_match_the_header(pkg, struct, cls):
    header = open(os.path.join(ROOT, "include", "qw3_cabi.h")).read()
    body = header[header.index("typedef struct %s {" % struct):header.index("} %s;" % struct)]
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    types = {"int32_t": C.c_int32, "int64_t": C.c_int64, "float": C.c_float}
    want = [(m[2], C.c_void_p if m[1] else types[m[0]]) for m in re.findall(r"^\s*(?:const\s+)?(void|int32_t|int64_t|float)\s*(\*?)\s+([a-z_0-9]+);", body, re.M)]
    assert want == list(getattr(pkg.cabi, cls)._fields_) and len(want) >= 7


def _pool(cabi, **kw):
    d = dict(d_pages=PTR, n_pages=4, page_stride=2 * 16 * 136, page_size=16, kv_heads=2, head_dim=128, dtype=0)
    d.update(kw)
    return cabi.Kv4Pool(*d.values())


BAD_POOLS = [dict(d_pages=None), dict(d_pages=PTR + 8), dict(n_pages=0), dict(n_pages=2 ** 31), dict(page_stride=2 * 16 * 136 - 16), dict(page_stride=2 * 16 * 136 + 8),
             dict(page_size=24), dict(page_size=0), dict(page_size=2048, page_stride=1 << 30), dict(kv_heads=0), dict(kv_heads=-1), dict(head_dim=64), dict(dtype=2), dict(dtype=-1)]


@pytest.mark.parametrize("bad", BAD_POOLS)
def test_bad_pools_are_refused(pkg, bad):
    cabi = pkg.cabi
    L = cabi.lib()
    ws = C.c_void_p(PTR)
    pool = _pool(cabi, **bad)
    app = cabi.Kv4AppendArgs(PTR, 1024, 1, 4, 0, 0, 0, PTR, None, None, None, 0, PTR, None)
    att = cabi.AttnKv4Args(PTR, 512, 1, 4, PTR, 4, 4, 0.0, PTR, PTR)
    assert L.qw3_rope_kv4_append(C.byref(pool), C.byref(app), ws, None) == cabi.QW3_ERR_ARG
    assert b"qw3_rope_kv4_append" in L.qw3_last_error()
    assert L.qw3_kv4_read(C.byref(pool), PTR, 1, PTR, PTR, ws, None) == cabi.QW3_ERR_ARG
    assert L.qw3_attn_kv4_decode(C.byref(pool), C.byref(att), ws, None) == cabi.QW3_ERR_ARG


def test_null_arguments_are_refused(pkg):
    cabi = pkg.cabi
    L = cabi.lib()
    pool = _pool(cabi)
    app, att, pages = cabi.Kv4AppendArgs(), cabi.AttnKv4Args(), cabi.PageArgs()
    for rc in (L.qw3_rope_kv4_append(None, C.byref(app), None, None), L.qw3_rope_kv4_append(C.byref(pool), None, None, None),
               L.qw3_rope_kv4_append(C.byref(pool), C.byref(app), None, None), L.qw3_kv4_read(None, None, 1, None, None, None, None),
               L.qw3_kv4_read(C.byref(pool), PTR, 1, PTR, PTR, None, None), L.qw3_attn_kv4_decode(C.byref(pool), C.byref(att), None, None),
               L.qw3_attn_kv4_decode(None, C.byref(att), None, None), L.qw3_page_slots(None, None, None), L.qw3_page_slots(C.byref(pages), None, None),
               L.qw3_page_slots(C.byref(pages), PTR, None)):
        assert rc == cabi.QW3_ERR_ARG


@pytest.mark.parametrize("field,value", [("d_ctx_len", None), ("d_free", None), ("d_cu", None), ("d_slot", None), ("n_req", 0), ("n_req", 16385), ("page_size", 8),
                                         ("page_size", 1040), ("max_blocks", 0), ("max_blocks", 2 ** 31 - 1), ("table_stride", 3), ("free_capacity", -1),
                                         ("max_tokens", -1), ("max_tokens", 2 ** 31 - 1)])
def test_page_slots_refuses(pkg, field, value):
    cabi = pkg.cabi
    a = cabi.PageArgs(PTR, PTR, 2, 16, PTR, 4, 4, 10, PTR, PTR, PTR, PTR, PTR, PTR, PTR, 9)
    setattr(a, field, value)
    assert cabi.lib().qw3_page_slots(C.byref(a), PTR, None) == cabi.QW3_ERR_ARG
    assert b"qw3_page_slots" in cabi.lib().qw3_last_error()


@pytest.fixture
def ops(pkg):
    return importlib.import_module("qw3awq_b200.ops")


class _Ws:
    h = C.c_void_p(PTR)


def test_python_checks_name_what_is_wrong(ops):
    f16, i32, u8 = torch.float16, torch.int32, torch.uint8
    pages = torch.zeros(2, 2 * 16 * 136, dtype=u8)
    for bad, page, kv, dtype in ((pages.int(), 16, 2, f16), (pages[0], 16, 2, f16), (pages, 16, 3, f16), (pages, 20, 1, f16), (pages, 16, 2, torch.float32), (pages.t(), 16, 2, f16),
                                 (pages[:0], 16, 2, f16), (pages, 16, 0, f16)):
        with pytest.raises(ValueError):
            ops.Kv4Cache(bad, page, kv, dtype)
    cache = ops.Kv4Cache(pages, 16, 2, f16)
    q, table, lens = torch.zeros(3, 4, 128, dtype=f16), torch.zeros(3, 2, dtype=i32), torch.zeros(3, dtype=i32)
    for args in ((q.float(), cache, table, lens), (q[..., :64], cache, table, lens), (q, cache, table[:2], lens), (q, cache, table.long(), lens), (q, cache, table, lens[:2]),
                 (q, cache, table, lens.long()), (q.transpose(0, 1), cache, table, lens), (q, cache, table.t().contiguous().t(), lens), (q, cache, table, lens)):   # the last: not on a GPU
        with pytest.raises(ValueError):
            ops.attn_kv4_decode(*args, _Ws())
    with pytest.raises(ValueError):
        ops.attn_kv4_decode(q, cache, table, lens, _Ws(), scale=0)
    qkv, slots, cos = torch.zeros(3, 8 * 128, dtype=f16), torch.zeros(3, dtype=i32), torch.zeros(9, 64)
    for args in ((qkv[:, :-128], cache, slots, slots, cos, cos, 4), (qkv, cache, slots[:2], slots, cos, cos, 4), (qkv, cache, slots, slots, cos.half(), cos.half(), 4),
                 (qkv, cache, slots, slots, cos, cos[:, :32], 4), (qkv, cache, slots, slots.long(), cos, cos, 4), (qkv.bfloat16(), cache, slots, slots, cos, cos, 4),
                 (qkv, cache, slots, slots, cos, cos, 4)):
        with pytest.raises(ValueError):
            ops.rope_kv4_append(*args, _Ws())
    for s in (slots.long(), slots[None], torch.zeros(6, dtype=i32)[::2], slots):
        with pytest.raises(ValueError):
            ops.kv4_read(cache, s, _Ws())
    one = torch.zeros(1, dtype=i32)
    for args in ((lens, lens[:2], 16, table, lens, one, 4), (lens, lens, 16, table, lens.long(), one, 4), (lens, lens, 16, table, lens, lens, 4), (lens, lens, 16, table, lens, one, -1),
                 (lens, lens, 16, table[:2], lens, one, 4), (lens, lens, 16, table, lens, one, 4)):
        with pytest.raises(ValueError):
            ops.page_slots(*args, _Ws())


def _packed(cabi, **kw):
    a = cabi.AttnPackedArgs(PTR, 512, PTR, 256, PTR, 256, 10, 10, PTR, PTR, 1, 4, 2, 128, 0, 0.0, PTR)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad", [dict(d_q=None), dict(d_k=None), dict(d_v=None), dict(d_out=None), dict(d_cu_q=None), dict(d_cu_k=None), dict(d_q=PTR + 8), dict(d_v=PTR + 2),
                                 dict(d_out=PTR + 4), dict(q_stride=504), dict(q_stride=516), dict(k_stride=128), dict(v_stride=260), dict(q_rows=-1), dict(k_rows=2 ** 31),
                                 dict(n_seq=-1), dict(heads=5), dict(heads=0), dict(kv_heads=0), dict(head_dim=64), dict(dtype=3), dict(scale=-1.0), dict(scale=float("nan")),
                                 dict(scale=float("inf"))])
def test_packed_attention_refuses(pkg, bad):
    cabi = pkg.cabi
    assert cabi.lib().qw3_attn_packed(C.byref(_packed(cabi, **bad)), PTR, None) == cabi.QW3_ERR_ARG
    assert b"qw3_attn_packed" in cabi.lib().qw3_last_error()
    assert cabi.lib().qw3_attn_packed(None, PTR, None) == cabi.QW3_ERR_ARG
    assert cabi.lib().qw3_attn_packed(C.byref(_packed(cabi)), None, None) == cabi.QW3_ERR_ARG
    assert cabi.lib().qw3_attn_packed(C.byref(_packed(cabi, n_seq=0)), PTR, None) == cabi.QW3_OK


def test_packed_attention_python_checks(ops):
    q, k, cu = torch.zeros(5, 4, 128).half(), torch.zeros(7, 2, 128).half(), torch.zeros(3, dtype=torch.int32)
    for args in ((q.float(), k.float(), k.float(), cu, cu), (q, k.bfloat16(), k, cu, cu), (q, k, k[:6], cu, cu), (q, k, k[:, :1], cu, cu), (q, k, k, cu[:2], cu),
                 (q, k, k, cu.long(), cu), (q, k, k, cu[:0], cu), (q[..., :64], k, k, cu, cu), (q, k, k, cu, cu)):   # the last: not on a GPU
        with pytest.raises(ValueError):
            ops.attn_packed(*args, _Ws())
    with pytest.raises(ValueError):
        ops.attn_packed(q, k, k, cu, cu, _Ws(), scale=-1.0)
    with pytest.raises(ValueError):
        ops.attn_packed(q, k, k, cu, cu, _Ws(), out=torch.zeros(5, 4, 128))
