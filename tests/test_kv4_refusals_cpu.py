"""Refusals of the batch server's operators that need no GPU, beside those of test_kv4_cpu.py."""
import ctypes as C

import pytest
import torch

PTR = 1 << 20   # an address that is never read: every call below is refused before


def _packed(cabi, **kw):
    a = cabi.AttnPackedArgs(PTR, 512, 2 * PTR, 256, 3 * PTR, 256, 10, 12, PTR, PTR, 1, 4, 2, 128, 0, 0.0, 4 * PTR)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


# q: 10 rows of 1024 bytes; k, v: 12 rows of 512 bytes; out: 10240 bytes
@pytest.mark.parametrize("kw", [dict(d_out=PTR), dict(d_out=PTR + 10 * 1024 - 32), dict(d_out=PTR - 10240 + 32), dict(d_out=2 * PTR), dict(d_out=2 * PTR + 12 * 512 - 32),
                                dict(d_out=3 * PTR - 10240 + 32), dict(d_out=3 * PTR + 32),
                                dict(d_out=PTR + 1024, q_stride=768), dict(d_out=PTR + 9 * 16384 + 992, q_stride=8192), dict(d_out=PTR + 16384 - 10240 + 32, q_stride=8192),
                                dict(d_out=2 * PTR + 8192 + 480, k_stride=4096, k_rows=2), dict(d_k=4 * PTR, d_v=4 * PTR + 512, k_stride=512, v_stride=512)])
def test_out_that_overlaps_an_input_is_refused(pkg, kw):
    cabi = pkg.cabi
    assert cabi.lib().qw3_attn_packed(C.byref(_packed(cabi, **kw)), PTR, None) == cabi.QW3_ERR_ARG
    assert b"overlap" in cabi.lib().qw3_last_error()


@pytest.mark.parametrize("kw", [dict(), dict(d_out=PTR + 10 * 1024), dict(d_out=PTR - 10240), dict(d_out=2 * PTR + 12 * 512), dict(d_out=3 * PTR - 10240),
                                dict(d_out=PTR + 1024, q_stride=8192), dict(d_out=PTR + 16384 - 10240, q_stride=8192), dict(d_out=PTR + 8192 * 20, q_stride=8192),
                                dict(d_out=2 * PTR + 512, k_stride=8192), dict(k_rows=0, d_k=None, d_v=None, k_stride=0, v_stride=0)])
def test_out_beside_and_between_the_rows_is_not(pkg, kw):
    """These pass the checks of arguments; without a GPU the call ends there."""
    if torch.cuda.is_available():
        pytest.skip("the addresses are none")
    cabi = pkg.cabi
    assert cabi.lib().qw3_attn_packed(C.byref(_packed(cabi, **kw)), PTR, None) == cabi.QW3_ERR_CUDA


def test_the_operators_import_without_torchs_private_functions(pkg, monkeypatch):
    """As in a build of torch without CUDA: the module loads, and its calls refuse tensors of the CPU."""
    import importlib.util
    import sys

    cabi = pkg.cabi
    for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
        if hasattr(torch._C, name):
            monkeypatch.delattr(torch._C, name)
    path = importlib.util.find_spec("qw3awq_b200.ops").origin
    spec = importlib.util.spec_from_file_location("qw3awq_b200._ops_again", path)
    ops = importlib.util.module_from_spec(spec)
    monkeypatch.setitem(sys.modules, spec.name, ops)
    spec.loader.exec_module(ops)
    cache = ops.Kv4Cache(torch.zeros(2, 2 * 16 * 136, dtype=torch.uint8), 16, 2, torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.kv4_read(cache, torch.zeros(3, dtype=torch.int32), type("Ws", (), {"h": C.c_void_p(PTR)}))
    assert ops.cabi is cabi


@pytest.fixture
def ops(pkg):
    import importlib
    return importlib.import_module("qw3awq_b200.ops")


@pytest.mark.parametrize("scale", [1e-46, -1e-50, 5e-324, 0.0, -0.0])
def test_a_scale_that_is_zero_in_fp32_does_not_become_the_usual_one(ops, scale):
    cache = ops.Kv4Cache(torch.zeros(2, 2 * 16 * 136, dtype=torch.uint8), 16, 2, torch.float16)
    q, ints = torch.zeros(3, 4, 128, dtype=torch.float16), torch.zeros(3, dtype=torch.int32)
    ws = type("Ws", (), {"h": C.c_void_p(PTR)})
    with pytest.raises(ValueError, match="scale"):
        ops.attn_kv4_decode(q, cache, ints[:, None], ints, ws, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        ops.attn_packed(q, q, q, ints, ints, ws, scale=scale)
    # the smallest number of fp32 passes, and the next check is that of the device
    with pytest.raises(ValueError, match="CUDA"):
        ops.attn_packed(q, q, q, ints, ints, ws, scale=1.4e-45)


@pytest.mark.parametrize("scale", [3e38, float("inf"), float("nan")])
def test_a_scale_that_passes_fp32_in_the_kernel_is_refused(pkg, scale):
    cabi = pkg.cabi
    assert cabi.lib().qw3_attn_packed(C.byref(_packed(cabi, scale=scale)), PTR, None) == cabi.QW3_ERR_ARG
    assert b"scale" in cabi.lib().qw3_last_error()


def test_a_workspace_is_checked_on_its_own_device(ops, monkeypatch):
    """The operators go to the device of their tensors; so does the check, from a program whose current device is another one."""
    import contextlib

    current, calls = [1], []

    @contextlib.contextmanager
    def device(index):
        before, current[0] = current[0], index
        yield
        current[0] = before

    class Lib:
        def qw3_ws_create(self, h):
            return 0

        def qw3_ws_set_pdl(self, h, pdl):
            return 0

        def qw3_ws_check(self, h, stream):
            calls.append((current[0], stream.value))
            return 0

    monkeypatch.setattr(ops.cabi, "lib", Lib)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: type("Stream", (), {"cuda_stream": 100 + current[0]}))
    ws = ops.Workspace()
    current[0] = 0
    ws.check()
    assert calls == [(1, 101)] and current == [0]
