"""Token sort without a GPU: argument checks of the C entry points and of the torch functions, none of which reach a device."""
import copy
import ctypes
import os
import pickle

import pytest
import torch

os.environ.setdefault("VMOE_NO_VLLM", "1")


def _lib():
    from sm120_moe_bench_b200 import _lib
    return _lib.lib


def _buf(n=4096):
    return (ctypes.c_char * n)()          # host memory: a call that got past its checks would not be made here


def test_plan_checks():
    lib, b = _lib(), ctypes.addressof(_buf())
    plan = lambda M, T, E, ids=b, off=b, rp=b, pr=b, emap=None, n=0, ws=None, bytes_=0: \
        lib.vmoe_plan_tokens(ids, emap, n, M, T, E, off, rp, pr, ws, bytes_, None)
    assert plan(-1, 2, 4) == 2 and plan(4, 0, 4) == 2 and plan(4, 2, 0) == 2
    assert plan(4, 17, 32) == 8 and plan(4, 2, 8193) == 8 and plan(2 ** 31 - 1, 16, 4) == 8 and plan(2 ** 27, 16, 4) == 8
    assert plan(4, 2, 4, ids=None) == 1 and plan(4, 2, 4, off=None) == 1 and plan(4, 2, 4, rp=None) == 1 and plan(4, 2, 4, pr=None) == 1
    assert plan(4, 2, 4, emap=b, n=-1) == 2
    need = lib.vmoe_plan_scratch_bytes
    assert need(64, 10, 512) == 0 and need(512, 8, 512) == 0 and need(4097, 1, 8) == 5 * 8 * 4 and need(2 ** 20, 16, 4) == 148 * 4 * 4
    assert need(-1, 2, 4) == 0
    assert plan(4097, 1, 8) == 4 and plan(4097, 1, 8, ws=b, bytes_=159) == 4


def test_sort_checks():
    lib, b = _lib(), ctypes.addressof(_buf())

    def sort(M=4, T=2, E=4, K=8, dtype=0, x=b, xs=8, off=b, rp=b, rows=b, rs=8):
        return lib.vmoe_sort_tokens(x, xs, dtype, M, T, E, K, off, rp, 1, rows, rs, None)

    assert sort(M=0) == 0 and sort(K=0) == 0                       # nothing to do
    assert sort(M=-1) == 2 and sort(T=0) == 2 and sort(K=-1) == 2 and sort(dtype=3) == 2 and sort(dtype=-1) == 2
    assert sort(T=17) == 8 and sort(E=8193) == 8
    assert sort(rs=7) == 2 and sort(xs=-1) == 2
    for name in ("x", "off", "rp", "rows"):
        assert sort(**{name: None}) == 1, name
    assert sort(x=b + 1) == 3 and sort(dtype=2, rows=b + 2) == 3    # not a multiple of the element


def test_unsort_checks():
    lib, b = _lib(), ctypes.addressof(_buf())

    def unsort(M=4, T=2, K=8, dtype=0, rows=b, rs=8, rp=b, out=b, os_=8, to=None):
        return lib.vmoe_unsort_tokens(rows, rs, dtype, M, T, K, rp, None, out, os_, dtype if to is None else to, None)

    assert unsort(M=0) == 0 and unsort(K=0) == 0
    assert unsort(M=-1) == 2 and unsort(dtype=7) == 2 and unsort(os_=7) == 2 and unsort(rs=-1) == 2 and unsort(T=17) == 8
    for name in ("rows", "rp", "out"):
        assert unsort(**{name: None}) == 1, name
    assert unsort(out=b + 1) == 3 and unsort(dtype=2, rows=b + 2) == 3
    assert unsort(to=1) == 2 and unsort(to=2) == 2 and unsort(dtype=2, to=3) == 2      # only f32 rows change their type

    def grad(M=4, T=2, E=4, K=8, dy=b, ds=8, rows=b, rs=8, off=b, rp=b, drows=b, gs=8, dw=b):
        return lib.vmoe_unsort_tokens_grad(dy, ds, rows, rs, 0, M, T, E, K, off, rp, None, drows, gs, dw, None)

    assert grad(M=0) == 0 and grad(drows=None, dw=None) == 0
    assert grad(dy=None) == 1 and grad(off=None) == 1 and grad(rp=None) == 1 and grad(rows=None) == 1
    assert grad(ds=-1) == 2 and grad(rs=-1) == 2 and grad(gs=7) == 2 and grad(T=17) == 8 and grad(dy=b + 1) == 3


def test_host_tensors_are_refused():
    import sm120_moe_bench_b200 as vm
    ids = torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        vm.plan_tokens(ids, 4)
    z = lambda *n: torch.zeros(*n, dtype=torch.int32)
    for bad in ((z(4), z(4, 2), z(8), 4), (z(5), z(4, 2), z(7), 4), (z(5).long(), z(4, 2), z(8), 4), (z(5), z(2, 4).t(), z(8), 4)):
        with pytest.raises(ValueError):
            vm.TokenPlan(*bad)
    plan = vm.TokenPlan(torch.zeros(5, dtype=torch.int32), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), 4)
    assert (plan.tokens, plan.topk, plan.rows) == (4, 2, 8)
    for twin in (copy.deepcopy(plan), pickle.loads(pickle.dumps(plan))):
        assert twin.expert_offsets.data_ptr() != plan.expert_offsets.data_ptr()
        assert twin._offsets_ptr == twin.expert_offsets.data_ptr() and twin._rows_ptr == twin.row_of_pair.data_ptr()
    with pytest.raises(ValueError, match="CUDA tensor"):
        vm.sort_tokens(torch.zeros(4, 8), plan)
    with pytest.raises(ValueError, match="CUDA tensor"):
        vm.unsort_tokens(torch.zeros(8, 8), plan)


def test_shared_memory_is_found():
    from sm120_moe_bench_b200.token_sort import overlap

    buf = torch.zeros(4096, dtype=torch.uint8)
    g = torch.Generator().manual_seed(1)

    def view():
        dtype = (torch.int8, torch.bfloat16, torch.float32)[int(torch.randint(3, (1,), generator=g))]
        flat = buf.view(dtype)
        rows, cols, pitch, at = (int(torch.randint(n, (1,), generator=g)) for n in (5, 7, 14, 60))
        return flat.as_strided((rows, cols), (pitch, 1), at)

    def touched(t):
        size = t.element_size()
        first = [t.storage_offset() + r * t.stride(0) + c for r in range(t.shape[0]) for c in range(t.shape[1])]
        return {size * e + b for e in first for b in range(size)}

    met = apart = 0
    for _ in range(3000):
        a, b = view(), view()
        if touched(a) & touched(b):
            met += 1
            assert overlap(a, b) and overlap(b, a)
        elif not overlap(a, b):
            apart += 1
            assert not overlap(b, a)
    assert met > 300 and apart > 300
    # side by side in one buffer, below one another, and columns that meet
    wide = torch.zeros(9, 20)
    assert not overlap(wide[:, :8], wide[:, 8:]) and not overlap(wide[:5, 8:], wide[:, :8]) and not overlap(wide[:4], wide[4:])
    assert not overlap(wide[:, :0], wide) and not overlap(wide[3:4, :8], wide[:, 8:12])
    assert overlap(wide[:, :8], wide[:, 7:]) and overlap(wide[:5], wide[4:]) and overlap(wide, wide[8, 19:])
    assert overlap(torch.zeros(1, 4).expand(5, 4), wide) is False


def test_forward_mode_tangents_are_seen():
    from torch.autograd import forward_ad
    from sm120_moe_bench_b200.token_sort import has_tangent

    x = torch.ones(3)
    assert not has_tangent(x)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(3))
        assert has_tangent(dual) and has_tangent(None, x, dual * 2) and not has_tangent(x, None) and not dual.requires_grad
        with torch.no_grad():                             # forward mode does not mind
            assert has_tangent(dual)
    assert not has_tangent(dual)


def test_tracing_is_seen():
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode
    from torch.utils.flop_counter import FlopCounterMode
    from sm120_moe_bench_b200.token_sort import launch, traced

    x, seen = torch.ones(3), []

    def f(t):
        seen.append(traced())
        return t + 1

    class Plain(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    f(x)
    with Plain(), FlopCounterMode(display=False):
        f(x)
    assert seen == [False, False]                         # modes that only watch are no hindrance
    seen.clear()
    torch.jit.trace(f, x, check_trace=False)
    for mode in ("real", "fake", "symbolic"):
        for pre in (False, True):
            make_fx(f, tracing_mode=mode, pre_dispatch=pre)(x)
    with Plain():
        make_fx(f)(x)
    make_fx(torch.func.functionalize(f))(x)
    assert len(seen) >= 9 and all(seen)
    assert not traced()
    with pytest.raises(RuntimeError, match="cannot be traced"):
        make_fx(lambda t: launch(torch.device("cuda", 0), "f", lambda *a: 0) or t)(x)
