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
        return lib.vmoe_int8_matmul(a, ast, sa, M, w, wst, est, sw, N, K, E, off, 0, 0, out, os_, dtype, None, 0, None)

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


def test_linear_and_experts_checks():
    lib, keep = _lib(), _buf()
    b = ctypes.addressof(keep) & ~15
    assert lib.vmoe_int8_linear_scratch_bytes(0, 64) == 0 and lib.vmoe_int8_linear_scratch_bytes(3, 131072) == 0
    assert lib.vmoe_int8_linear_scratch_bytes(9, 100) >= 9 * 112 + 36

    def linear(x=b, xs=16, dtype=0, M=16, w=b, ws=16, sw=b, N=8, K=16, out=b, os_=8, to=0, scratch=b, bytes_=4096):
        return lib.vmoe_int8_linear(x, xs, dtype, M, w, ws, sw, N, K, 0, out, os_, to, scratch, bytes_, None)

    assert linear(M=0) == 0
    assert linear(dtype=3) == 2 and linear(xs=-1) == 2 and linear(M=-1) == 2 and linear(N=0) == 2 and linear(os_=7) == 2 and linear(K=131072) == 8
    assert linear(x=None) == 1 and linear(w=None) == 1 and linear(sw=None) == 1 and linear(out=None) == 1
    assert linear(x=b + 1) == 3 and linear(scratch=b + 8) == 3
    assert linear(scratch=None) == 4 and linear(bytes_=16) == 4

    assert lib.vmoe_int8_pack_bytes(0, 8, 20, 1) == 0 and lib.vmoe_int8_pack_bytes(3, 8, 20, 2) >= 3 * 32 + 2 * 8 * 32

    size = lib.vmoe_int8_experts_scratch_bytes
    assert size(4, 17, 8, 64, 32, 0) == 0 and size(4, 2, 8193, 64, 32, 0) == 0 and size(2 ** 28, 16, 8, 64, 32, 0) == 0
    assert size(64, 10, 512, 4096, 1024, 0) >= 640 * 4096 * 4
    assert size(64, 10, 512, 4096, 1024, 1) >= size(64, 10, 512, 4096, 1024, 0) + 512 * 2048 * 4096

    def experts(x=b, dtype=0, M=4, T=2, E=4, K=32, N=16, ids=b, wt=b, w13=b, s13=b, w2=b, s2=b, out=b, scratch=b, bytes_=1 << 40):
        return lib.vmoe_int8_experts(x, K, dtype, M, T, E, K, N, ids, wt, None, 0, w13, K, 2 * N * K, s13, w2, N, N * K, s2, out, K, 0,
                                     scratch, bytes_, None)

    assert experts(M=0) == 0
    assert experts(dtype=3) == 2 and experts(M=-1) == 2 and experts(K=0) == 2 and experts(N=0) == 2 and experts(E=0) == 2
    assert experts(K=131072) == 8 and experts(T=17) == 8 and experts(E=8193) == 8
    for name in ("x", "ids", "wt", "w13", "s13", "w2", "s2", "out"):
        assert experts(**{name: None}) == 1, name
    assert experts(scratch=None) == 4 and experts(bytes_=64) == 4 and experts(scratch=b + 8) == 3


def test_wait_limit_checks():
    lib = _lib()
    assert lib.vmoe_int8_set_wait_limit(-1) == 2
    assert lib.vmoe_int8_set_wait_limit(10 ** 6) == 0     # what it is from the start


def test_few_rows_rule():
    one = _lib().vmoe_int8_one_launch
    assert one(0, 64, 64, 16) == 0 and one(1, 0, 64, 16) == 0 and one(1, 64, 0, 16) == 0 and one(1, 64, 64, 0) == 0 and one(9, 64, 64, 16) == 0
    # the codes have to fit 64 KB, whatever the alignment
    for align in (16, 4, 1):
        assert one(8, 16, 8192, align) == (align < 16) and one(8, 16, 8193, align) == 0 and one(4, 16, 16385, align) == 0 and one(1, 16, 65537, align) == 0
    # a row more, or a channel more, never makes it the better kernel
    for align in (16, 4, 1):
        for K in (16, 256, 1024, 2048, 4096, 8192):
            for N in (8, 512, 4096, 8192, 16384, 32768, 131072):
                got = [one(M, N, K, align) for M in range(1, 9)]
                assert got == sorted(got, reverse=True)
                assert all(one(M, 2 * N, K, align) <= got[M - 1] for M in range(1, 9))
    assert [one(M, 131072, 1024, 16) for M in (1, 2, 4, 8)] == [0, 0, 0, 0] and one(1, 131072, 4096, 16) == 1 and one(4, 131072, 4096, 16) == 0
    assert [one(M, 2048, 4096, 16) for M in (1, 2, 4, 8)] == [1, 1, 1, 1] and one(1, 4096, 4095, 1) == 0 and one(4, 64, 128, 1) == 1


def test_python_agrees_with_the_few_row_rule():
    from sm120_moe_bench_b200.int8 import _one_launch
    one = _lib().vmoe_int8_one_launch
    for M in range(0, 11):
        for K in (0, 1, 15, 16, 255, 1000, 1024, 2047, 2048, 4095, 4096, 8191, 8192, 8193, 16384, 65537):
            for n in (1, 2, 60, 255, 256, 257, 1024, 2048, 4096, 8192, 8193, 16384, 131072):
                for address, pitch in ((512, (K + 15) // 16 * 16), (512, K), (516, K + 4 - K % 4), (513, K)):
                    want = one(M, n, K, 16 | (address | pitch) & 15)
                    assert _one_launch(M, n, K, address, max(pitch, 1)) == bool(want) or M == 0, (M, n, K, address, pitch)
    assert not _one_launch(2, 64, 64, 512, 32) and _one_launch(2, 1, 64, 512, 1)       # rows that overlap; one row has no pitch
