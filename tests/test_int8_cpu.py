"""8-bit integer operators without a GPU: argument checks that never reach a device."""
import ctypes
import os

import pytest
import torch

os.environ.setdefault("VMOE_NO_VLLM", "1")


def _lib():
    from sm120_moe_bench_b200 import _lib
    return _lib.lib


def _buf(n=4096):
    return (ctypes.c_char * n)()


def test_quantize_checks():
    lib, keep = _lib(), _buf()
    b = ctypes.addressof(keep) & ~15

    def quantize(x=b, xs=16, dtype=0, rows=4, K=16, T=0, rp=None, q=b, qs=16, s=b):
        return lib.vmoe_int8_quantize(x, xs, dtype, rows, K, T, rp, None, q, qs, s, None)

    assert quantize(rows=0) == 0
    assert quantize(rows=-1) == 2 and quantize(K=-1) == 2 and quantize(dtype=3) == 2 and quantize(xs=-1) == 2 and quantize(qs=15) == 2
    assert quantize(rp=b, T=0) == 2 and quantize(rp=b, T=17) == 2
    assert quantize(x=None) == 1 and quantize(q=None) == 1 and quantize(s=None) == 1
    assert quantize(x=b + 1) == 3 and quantize(dtype=2, x=b + 2) == 3


def test_matmul_checks():
    lib, keep = _lib(), _buf()
    b = ctypes.addressof(keep) & ~15

    def matmul(a=b, sa=b, M=4, w=b, sw=b, N=8, K=16, E=1, off=None, out=b, os_=8, dtype=0, ast=16, wst=16, est=0):
        return lib.vmoe_int8_matmul(a, ast, sa, M, w, wst, est, sw, N, K, E, off, 0, 0, out, os_, dtype, None)

    assert matmul(M=0) == 0
    assert matmul(M=-1) == 2 and matmul(N=0) == 2 and matmul(K=-1) == 2 and matmul(E=0) == 2 and matmul(dtype=3) == 2
    assert matmul(E=2) == 2                               # several experts need their offsets
    assert matmul(ast=-1) == 2 and matmul(wst=-1) == 2 and matmul(est=-1) == 2 and matmul(os_=7) == 2
    assert matmul(K=131072) == 8 and matmul(E=65536, off=b) == 8
    for name in ("a", "sa", "w", "sw", "out"):
        assert matmul(**{name: None}) == 1, name
    assert matmul(out=b + 1) == 3 and matmul(dtype=2, out=b + 2) == 3


def test_host_tensors_are_refused():
    import sm120_moe_bench_b200 as vm
    with pytest.raises(ValueError, match="CUDA tensor"):
        vm.Int8Rows(torch.zeros(4, 16, dtype=torch.int8), torch.zeros(4))
    with pytest.raises(ValueError, match="CUDA tensor"):
        vm.quantize_int8(torch.zeros(4, 16))
    with pytest.raises(ValueError, match="gradient"):
        vm.quantize_int8(torch.zeros(4, 16, requires_grad=True))
