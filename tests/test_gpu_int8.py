"""8-bit integer rows, their products and the expert layer on them, against the definitions in 64 bits.

Codes and scales are equal: 127 x / max|x| in 64 bits has no other nearest integer than the exact quotient, and f32's
quotient by 127 is the 64-bit one rounded.  A product is an exact integer that meets three f32 roundings (to f32, times the
row's scale, times the channel's): 3 * 2^-24 of its value, 4 to have a whole one for the products of those errors, and half a
step of the output type."""
import os

import pytest
import torch

os.environ.setdefault("VMOE_NO_VLLM", "1")
pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def half_step(dtype, value):
    return torch.finfo(dtype).eps / 2 * value.abs() * (1 + 2.0 ** -18) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)


def codes64(x):
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    return torch.where(top > 0, torch.round(127 * x / top), 0.0), (top / 127).float()[..., 0]


def random_rows(vm, shape, seed, pitch=None):
    """Codes over the whole range, -128 included, with rows `pitch` bytes apart, and scales."""
    K = shape[-1]
    q = torch.randint(-128, 128, (*shape[:-1], pitch or K), generator=gen(seed), device="cuda", dtype=torch.int8)[..., :K]
    return vm.Int8Rows(q, (0.5 + torch.rand(shape[:-1], generator=gen(seed + 1), device="cuda")) / 1000)


def exact_product(a, w, offsets=None):
    if offsets is None:
        return (a.q.double() @ w.q.double().T) * a.scale.double()[:, None] * w.scale.double()
    y = torch.zeros(a.q.shape[0], w.q.shape[1], dtype=torch.float64, device="cuda")
    o = offsets.tolist()
    for e in range(w.q.shape[0]):
        r = slice(o[e], o[e + 1])
        y[r] = (a.q[r].double() @ w.q[e].double().T) * a.scale.double()[r, None] * w.scale[e].double()
    return y


def check_product(y, want):
    assert bool(((y.double() - want).abs() <= 4 * 2.0 ** -24 * want.abs() + half_step(y.dtype, want)).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 4096), (7, 33), (64, 1024), (129, 1000), (33, 1021), (20, 7168), (9, 2), (3, 20000)])
def test_quantize(M, K, dtype):
    import sm120_moe_bench_b200 as vm
    x = torch.randn(M, K, generator=gen(1), device="cuda").to(dtype)
    r = vm.quantize_int8(x)
    q, s = codes64(x)
    assert torch.equal(r.q.double(), q) and torch.equal(r.scale, s)
    assert r.q.stride(0) % 16 == 0
    wide = torch.randn(M + 1, 2 * K + 1, generator=gen(2), device="cuda").to(dtype)
    for v in (wide[:M, 1:K + 1], wide[1:, K:2 * K], wide[:1, :K].expand(M, K)):
        q, s = codes64(v)
        r = vm.quantize_int8(v)
        assert torch.equal(r.q.double(), q) and torch.equal(r.scale, s)


def test_quantize_borders_and_extremes():
    import sm120_moe_bench_b200 as vm
    # every border between two codes, exactly: x = (k + 1/2) * 2 with max 254
    x = torch.cat([torch.arange(-253, 254, 2, device="cuda").float(), torch.tensor([254.0], device="cuda")])[None]
    for scale in (1.0, 2.0 ** -20, 2.0 ** 100, 2.0 ** -130):
        for dtype in (torch.float32, torch.bfloat16):
            v = (x * scale).to(dtype)
            q, s = codes64(v)
            r = vm.quantize_int8(v)
            assert torch.equal(r.q.double(), q) and torch.equal(r.scale, s)
    # next to the borders in f32
    v = torch.stack([torch.nextafter(x[0], torch.full_like(x[0], d)) for d in (float("inf"), float("-inf"))])
    v[:, -1] = 254.0
    q, s = codes64(v)
    r = vm.quantize_int8(v)
    assert torch.equal(r.q.double(), q) and torch.equal(r.scale, s)
    for dtype in DTYPES:
        big = torch.finfo(dtype).max
        v = torch.zeros(6, 40, dtype=dtype, device="cuda")
        v[1, 3], v[1, 4] = big, -big / 2
        v[2, 0] = float("inf")
        v[3, 39] = float("nan")
        v[4, 7] = torch.finfo(dtype).tiny
        v[5] = -big
        r = vm.quantize_int8(v)
        fine = torch.tensor([0, 1, 4, 5], device="cuda")
        q, s = codes64(v[fine])
        assert torch.equal(r.q[fine].double(), q) and torch.equal(r.scale[fine], s)
        assert bool(r.scale[2:4].isnan().all()) and torch.count_nonzero(r.q[2:4]) == 0
        w = random_rows(vm, (5, 40), 3)
        y = vm.int8_matmul(r, w, out_dtype=torch.float32)
        assert bool(y[2:4].isnan().all()) and not bool(y[fine].isnan().any()) and torch.count_nonzero(y[0]) == 0


def test_quantize_sorted_equals_sorted_quantized():
    import sm120_moe_bench_b200 as vm
    for K in (64, 1021, 4096):
        x = torch.randn(40, K, generator=gen(4), device="cuda").bfloat16()
        ids = torch.randint(-1, 6, (40, 3), generator=gen(5), device="cuda", dtype=torch.int32)
        plan = vm.plan_tokens(ids, 6)
        kept = int(plan.expert_offsets[-1])
        r, one = vm.quantize_int8(x, plan), vm.quantize_int8(x)
        tok = (plan.pair_of_row[:kept] // 3).long()
        assert torch.equal(r.q[:kept], one.q[tok]) and torch.equal(r.scale[:kept], one.scale[tok])


def test_quantize_weights_of_several_experts():
    import sm120_moe_bench_b200 as vm
    w = torch.randn(3, 10, 50, generator=gen(6), device="cuda")
    r = vm.quantize_int8(w)
    q, s = codes64(w)
    assert r.q.shape == w.shape and torch.equal(r.q.double(), q) and torch.equal(r.scale, s)
    assert bool(((r.dequantize() - w).abs() <= s[..., None] * (0.5 + 2.0 ** -16)).all())


SIZES = [(1, 1, 1), (1, 2048, 4096), (1, 7, 16), (2, 130, 48), (3, 64, 4096), (5, 1000, 272), (8, 512, 1024), (9, 300, 640), (16, 4096, 1024),
         (17, 129, 160), (33, 255, 4096), (48, 4096, 4096), (64, 100, 2048), (65, 1235, 1008), (128, 257, 512), (129, 128, 128), (200, 1024, 96),
         (256, 256, 256), (333, 1235, 1008), (1000, 700, 2064), (2049, 513, 1024)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", SIZES)
def test_product(M, N, K, dtype):
    import sm120_moe_bench_b200 as vm
    a, w = random_rows(vm, (M, K), 7), random_rows(vm, (N, K), 9)
    check_product(vm.int8_matmul(a, w, out_dtype=dtype), exact_product(a, w))


@pytest.mark.parametrize("M,N,K,pa,pw", [(1, 70, 1000, 1000, 1000), (1, 64, 1001, 1001, 1001), (6, 129, 37, 37, 37), (40, 200, 1000, 1000, 1000),
                                         (333, 1235, 1000, 1000, 1000), (300, 300, 1021, 1021, 1021), (300, 300, 1021, 1024, 1021),
                                         (300, 300, 1021, 1021, 1040), (64, 96, 500, 512, 528), (1, 96, 500, 512, 528), (20, 33, 3, 16, 16),
                                         (150, 33, 1, 1, 1)])
def test_product_of_unaligned_rows(M, N, K, pa, pw):
    import sm120_moe_bench_b200 as vm
    a, w = random_rows(vm, (M, K), 11, pa), random_rows(vm, (N, K), 13, pw)
    want = exact_product(a, w)
    check_product(vm.int8_matmul(a, w), want)
    out = torch.full((M + 1, N + 9), 3.0, device="cuda")
    vm.int8_matmul(a, w, out=out[:M, 5:N + 5])
    check_product(out[:M, 5:N + 5], want)
    assert bool((out[M] == 3).all()) and bool((out[:, :5] == 3).all()) and bool((out[:, N + 5:] == 3).all())
    odd = vm.Int8Rows(torch.randint(-128, 128, (M * K + 1,), generator=gen(15), device="cuda", dtype=torch.int8)[1:].view(M, K), a.scale)
    check_product(vm.int8_matmul(odd, w), exact_product(odd, w))


@pytest.mark.parametrize("M", [1, 2, 3, 8])
@pytest.mark.parametrize("K", [1, 5, 127, 1001, 4098, 9001])
def test_few_rows_of_any_alignment(M, K):
    import sm120_moe_bench_b200 as vm
    for skew in range(5):
        q = torch.randint(-128, 128, (61 * (K + skew) + skew,), generator=gen(64 + skew), device="cuda", dtype=torch.int8)
        w = vm.Int8Rows(q[skew:].view(61, K + skew)[:, :K], torch.rand(61, generator=gen(65), device="cuda"))
        a = random_rows(vm, (M, K), 66)
        check_product(vm.int8_matmul(a, w, out_dtype=torch.float32), exact_product(a, w))
        half = vm.Int8Rows(w.q[:60], w.scale[:60])
        check_swiglu(vm.int8_matmul(a, half, swiglu=True, out_dtype=torch.float32), exact_product(a, half), 30)
        x = torch.randn(M, K, generator=gen(67), device="cuda").half()
        assert torch.equal(vm.int8_linear(x, w), vm.int8_matmul(vm.quantize_int8(x), w, out_dtype=torch.float16))


def test_broadcast_rows():
    import sm120_moe_bench_b200 as vm
    for M in (3, 40):
        a, w = random_rows(vm, (1, 64), 68), random_rows(vm, (1, 64), 70)
        many = vm.Int8Rows(a.q.expand(M, 64), a.scale.expand(M).contiguous())
        wide = vm.Int8Rows(w.q.expand(50, 64), w.scale.expand(50).contiguous())
        for l, r in ((many, wide), (many, random_rows(vm, (50, 64), 72)), (random_rows(vm, (M, 64), 74), wide)):
            check_product(vm.int8_matmul(l, r, out_dtype=torch.float32), exact_product(l, r))
        x = torch.randn(M, 64, generator=gen(76), device="cuda")
        check_product(vm.int8_linear(x, wide), exact_product(vm.quantize_int8(x), wide))
        nothing = vm.Int8Rows(torch.zeros(7, 0, dtype=torch.int8, device="cuda"), torch.ones(7, device="cuda"))
        assert torch.equal(vm.int8_linear(torch.zeros(M, 0, device="cuda"), nothing), torch.zeros(M, 7, device="cuda"))


def test_expert_layer_with_unaligned_weights():
    import sm120_moe_bench_b200 as vm
    E, K, N, T = 3, 200, 72, 2
    w13, w2 = random_rows(vm, (E, 2 * N, K), 77, K + 3), random_rows(vm, (E, K, N), 79, N + 1)
    a13 = vm.Int8Rows(torch.nn.functional.pad(w13.q, (0, 8))[..., :K], w13.scale)
    a2 = vm.Int8Rows(torch.nn.functional.pad(w2.q, (0, 8))[..., :N], w2.scale)
    for M in (2, 12, 30, 200):
        x = torch.randn(M, K, generator=gen(81), device="cuda").bfloat16()
        ids = torch.randint(0, E, (M, T), generator=gen(82), device="cuda", dtype=torch.int32)
        wt = torch.rand(M, T, generator=gen(83), device="cuda")
        assert torch.equal(vm.int8_experts(x, w13, w2, ids, wt), vm.int8_experts(x, a13, a2, ids, wt))


def test_product_at_the_ends_of_the_integers():
    import sm120_moe_bench_b200 as vm
    for M in (1, 20, 140):
        for K in (131071, 65536):
            a = vm.Int8Rows(torch.full((M, K), -128, dtype=torch.int8, device="cuda"), torch.ones(M, device="cuda"))
            w = vm.Int8Rows(torch.full((17, K), -128, dtype=torch.int8, device="cuda"), torch.ones(17, device="cuda"))
            assert bool((vm.int8_matmul(a, w, out_dtype=torch.float32) == float(torch.tensor(16384.0 * K))).all())
    a = vm.Int8Rows(torch.zeros(5, 0, dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda"))
    w = vm.Int8Rows(torch.zeros(3, 0, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda"))
    assert torch.equal(vm.int8_matmul(a, w), torch.zeros(5, 3, dtype=torch.bfloat16, device="cuda"))
    a = random_rows(vm, (0, 64), 16)
    assert vm.int8_matmul(a, random_rows(vm, (9, 64), 17)).shape == (0, 9)


def silu64(x):
    return x / (1 + torch.exp(-x))


def check_swiglu(y, gu, N):
    """gate and up carry 4 * 2^-24 each.  silu has a slope of at most 1.1 and its own error: expf and the sum 4 * 2^-24 of the
    denominator, the quotient 2^-24; a gate below -87 is flushed to less than 1e-30.  16 * 2^-24 * (|gate| + |silu|) |up| covers them."""
    gate, up = gu[:, :N], gu[:, N:]
    want = silu64(gate) * up
    tol = 16 * 2.0 ** -24 * (gate.abs() + silu64(gate).abs()) * up.abs() + 1e-30 * up.abs()
    assert bool(((y.double() - want).abs() <= tol + half_step(y.dtype, want)).all())


@pytest.mark.parametrize("M,N,K", [(1, 40, 100), (1, 1024, 4096), (4, 300, 512), (20, 128, 1024), (70, 200, 272), (300, 513, 640)])
def test_swiglu(M, N, K):
    import sm120_moe_bench_b200 as vm
    a, w = random_rows(vm, (M, K), 18), random_rows(vm, (2 * N, K), 20)
    gu = exact_product(a, w)
    check_swiglu(vm.int8_matmul(a, w, swiglu=True, out_dtype=torch.float32), gu, N)
    check_swiglu(vm.int8_matmul(a, w, swiglu=True), gu, N)


@pytest.mark.parametrize("M,T,E,N,K,drop", [(1, 1, 1, 64, 128, False), (1, 10, 512, 256, 256, False), (64, 10, 512, 128, 256, False),
                                            (7, 3, 5, 100, 272, True), (50, 2, 4, 513, 640, True), (130, 4, 6, 256, 512, True), (40, 8, 64, 96, 1021, True),
                                            (600, 2, 3, 200, 1024, True), (1000, 4, 64, 384, 256, False), (300, 16, 16, 130, 96, False)])
def test_grouped_product(M, T, E, N, K, drop):
    import sm120_moe_bench_b200 as vm
    ids = torch.randint(-1 if drop else 0, E, (M, T), generator=gen(22), device="cuda", dtype=torch.int32)
    if E > 2:
        ids[ids == 1] = 2                                 # an expert without rows, another with twice as many
    plan = vm.plan_tokens(ids, E)
    a, w = random_rows(vm, (M * T, K), 23), random_rows(vm, (E, 2 * N, K), 25)
    want = exact_product(a, w, plan.expert_offsets)
    kept = int(plan.expert_offsets[-1])
    y = vm.int8_matmul(a, w, plan, out_dtype=torch.float32)
    check_product(y, want)                                # rows behind the last kept one are zero
    gu = want[:kept]
    check_swiglu(vm.int8_matmul(a, w, plan, swiglu=True, out_dtype=torch.float32)[:kept], gu, N)
    out = torch.full((M * T, 2 * N), 9.0, dtype=torch.float16, device="cuda")
    vm.int8_matmul(a, w, plan, out=out)
    check_product(out[:kept], want[:kept])
    assert bool((out[kept:] == 9).all())


def test_grouped_product_with_strided_experts():
    import sm120_moe_bench_b200 as vm
    E, N, K = 4, 72, 160
    big = torch.randint(-128, 128, (E, N + 8, K + 32), generator=gen(27), device="cuda", dtype=torch.int8)
    w = vm.Int8Rows(big[:, :N, :K], torch.rand(E, N, generator=gen(28), device="cuda"))
    for M in (6, 400):
        plan = vm.plan_tokens(torch.randint(0, E, (M, 2), generator=gen(29), device="cuda", dtype=torch.int32), E)
        a = random_rows(vm, (2 * M, K), 30)
        check_product(vm.int8_matmul(a, w, plan, out_dtype=torch.float32), exact_product(a, w, plan.expert_offsets))
        same = vm.Int8Rows(w.q[:1].expand(E, N, K), w.scale)     # one matrix for every expert
        check_product(vm.int8_matmul(a, same, plan, out_dtype=torch.float32), exact_product(a, same, plan.expert_offsets))


def test_a_row_does_not_depend_on_the_batch():
    import sm120_moe_bench_b200 as vm
    a, w = random_rows(vm, (700, 512), 31), random_rows(vm, (400, 512), 33)
    full = vm.int8_matmul(a, w)
    for rows in (1, 2, 5, 17, 100, 300):
        part = vm.Int8Rows(a.q[:rows], a.scale[:rows])
        assert torch.equal(vm.int8_matmul(part, w), full[:rows])
    half = random_rows(vm, (800, 512), 35)
    h = vm.int8_matmul(a, half, swiglu=True, out_dtype=torch.float32)
    for rows in (1, 3, 40, 300):
        assert torch.equal(vm.int8_matmul(vm.Int8Rows(a.q[:rows], a.scale[:rows]), half, swiglu=True, out_dtype=torch.float32), h[:rows])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", [(1, 2048, 4096), (1, 100, 1000), (2, 60, 72), (5, 333, 4096), (48, 512, 1021), (400, 300, 520)])
def test_linear_equals_its_parts(M, N, K, dtype):
    import sm120_moe_bench_b200 as vm
    x, w = torch.randn(M, K, generator=gen(36), device="cuda").to(dtype), random_rows(vm, (2 * N, K), 37)
    assert torch.equal(vm.int8_linear(x, w), vm.int8_matmul(vm.quantize_int8(x), w, out_dtype=dtype))
    assert torch.equal(vm.int8_linear(x, w, swiglu=True), vm.int8_matmul(vm.quantize_int8(x), w, swiglu=True, out_dtype=dtype))
    out = torch.empty(M, 2 * N + 3, dtype=dtype, device="cuda")[:, 1:2 * N + 1]
    assert torch.equal(vm.int8_linear(x, w, out=out), vm.int8_linear(x, w))
    wide = torch.randn(M, K + 5, generator=gen(39), device="cuda").to(dtype)
    assert torch.equal(vm.int8_linear(wide[:, 3:K + 3], w), vm.int8_linear(wide[:, 3:K + 3].contiguous(), w))
    x[M // 2, K // 2] = float("nan")
    y = vm.int8_linear(x, w)
    assert bool(y[M // 2].isnan().all()) and int(y.isnan().any(1).sum()) == 1


def experts64(vm, x, w13, w2, plan, weights):
    """The layer in 64 bits, and how far a correct f32 evaluation may be: a code of the activations whose quotient lies within
    2^-12 of a border may be the next one (f32 is off by less than 2^-16 of a quotient of at most 127, and of its row's largest),
    and the rest carries 64 * 2^-24 of the sum of magnitudes."""
    M, T = plan.row_of_pair.shape
    N = w2.q.shape[-1]
    y = torch.zeros(M, x.shape[1], dtype=torch.float64, device="cuda")
    tol, mag = torch.zeros_like(y), torch.zeros_like(y)
    q, s = codes64(x)
    o = plan.expert_offsets.tolist()
    for e in range(w13.q.shape[0]):
        if o[e + 1] == o[e]:
            continue
        pair = plan.pair_of_row[o[e]:o[e + 1]].long()
        tok, wt = pair // T, weights.reshape(-1)[pair].double()[:, None]
        gu = (q[tok] @ w13.q[e].double().T) * s[tok].double()[:, None] * w13.scale[e].double()
        h = silu64(gu[:, :N]) * gu[:, N:]
        top = h.abs().amax(1, keepdim=True)
        quot = torch.where(top > 0, 127 * h / top, 0.0)
        hq, near = torch.round(quot), ((quot - torch.floor(quot) - 0.5).abs() < 2.0 ** -12).double()
        w2e = w2.q[e].double().T * w2.scale[e].double()
        y.index_add_(0, tok, wt * ((hq @ w2e) * (top / 127)))
        tol.index_add_(0, tok, wt.abs() * ((near @ w2e.abs()) * (top / 127)))
        mag.index_add_(0, tok, wt.abs() * ((hq.abs() @ w2e.abs()) * (top / 127)))
    return y, tol + 64 * 2.0 ** -24 * mag


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,T,E,K,N,local", [(1, 2, 4, 64, 32, 4), (1, 10, 64, 1024, 512, 64), (6, 2, 8, 1024, 512, 8), (64, 10, 32, 512, 256, 32),
                                             (33, 3, 7, 1000, 300, 7), (40, 8, 64, 256, 128, 8), (300, 4, 8, 512, 256, 8), (500, 2, 3, 1040, 528, 2)])
def test_expert_layer(M, T, E, K, N, local, dtype):
    import sm120_moe_bench_b200 as vm
    x = torch.randn(M, K, generator=gen(40), device="cuda").to(dtype)
    top, ids = torch.topk(torch.randn(M, E, generator=gen(41), device="cuda"), T, dim=1)
    weights, ids, emap = torch.softmax(top, 1), ids.int(), None
    if local < E:
        emap = torch.full((E,), -1, dtype=torch.int32, device="cuda")
        emap[1:1 + local] = torch.arange(local, device="cuda", dtype=torch.int32)
    w13 = vm.quantize_int8(torch.randn(local, 2 * N, K, generator=gen(42), device="cuda") / K ** 0.5)
    w2 = vm.quantize_int8(torch.randn(local, K, N, generator=gen(43), device="cuda") / N ** 0.5)
    y = vm.int8_experts(x, w13, w2, ids, weights, emap)
    plan = vm.plan_tokens(ids, local, emap)
    want, tol = experts64(vm, x, w13, w2, plan, weights)
    assert y.dtype == dtype and bool(((y.double() - want).abs() <= tol + half_step(dtype, want)).all())
    # the same through the public operators one by one
    h = vm.int8_matmul(vm.quantize_int8(x, plan), w13, plan, swiglu=True, out_dtype=torch.float32)
    rows = vm.int8_matmul(vm.quantize_int8(h), w2, plan, out_dtype=torch.float32)
    assert torch.equal(y, vm.unsort_tokens(rows, plan, weights).to(dtype))
    assert torch.equal(y, vm.int8_experts(x, w13, w2, ids, weights, emap))


def test_expert_layer_without_kept_pairs_or_tokens():
    import sm120_moe_bench_b200 as vm
    w13, w2 = random_rows(vm, (4, 64, 128), 44), random_rows(vm, (4, 128, 32), 46)
    x = torch.randn(5, 128, device="cuda").bfloat16()
    none = torch.full((5, 2), -1, dtype=torch.int32, device="cuda")
    assert torch.count_nonzero(vm.int8_experts(x, w13, w2, none, torch.ones(5, 2, device="cuda"))) == 0
    y = vm.int8_experts(x[:0], w13, w2, none[:0], torch.ones(0, 2, device="cuda"))
    assert y.shape == (0, 128)
    twice = torch.full((5, 2), 3, dtype=torch.int32, device="cuda")        # the same expert twice
    half = torch.full((5, 2), 0.5, device="cuda")
    once = vm.int8_experts(x, w13, w2, twice[:, :1].contiguous(), torch.ones(5, 1, device="cuda"))
    assert torch.equal(vm.int8_experts(x, w13, w2, twice, half), once)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,T,E,K,N,map_len", [(1, 1, 1, 1, 1, 0), (3, 16, 8192, 20, 8, 0), (64, 16, 300, 40, 24, 0), (1024, 1, 5, 33, 16, 0),
                                               (1025, 1, 5, 33, 16, 0), (93, 11, 40, 130, 16, 70), (94, 11, 40, 130, 16, 70),
                                               (7, 3, 257, 9000, 16, 0), (512, 2, 256, 64, 32, 300)])
def test_expert_layer_of_any_ids_equals_its_parts(M, T, E, K, N, map_len, dtype):
    """Ids that repeat within a token, lie outside the experts or the map; empty and all-zero rows; both sides of 1024 pairs,
    where the rows are planned another way; rows apart."""
    import sm120_moe_bench_b200 as vm
    x = torch.randn(M, K + 3, generator=gen(60), device="cuda").to(dtype)[:, :K]
    x[M // 2] = 0
    ids = torch.randint(-2, (map_len or E) + 2, (M, T), generator=gen(61), device="cuda", dtype=torch.int32)
    if T > 1:
        ids[:, 1] = ids[:, 0]
    emap = None
    if map_len:
        emap = torch.randint(-1, E + 1, (map_len,), generator=gen(62), device="cuda", dtype=torch.int32)
    weights = torch.randn(M, T, generator=gen(63), device="cuda")
    w13, w2 = random_rows(vm, (E, 2 * N, K), 64), random_rows(vm, (E, K, N), 66)
    y = vm.int8_experts(x, w13, w2, ids, weights, emap)
    plan = vm.plan_tokens(ids, E, emap)
    h = vm.int8_matmul(vm.quantize_int8(x, plan), w13, plan, swiglu=True, out_dtype=torch.float32)
    rows = vm.int8_matmul(vm.quantize_int8(h), w2, plan, out_dtype=torch.float32)
    kept = (plan.row_of_pair >= 0).any(1)
    assert torch.equal(y, vm.unsort_tokens(rows, plan, weights).to(dtype)) and torch.count_nonzero(y[~kept]) == 0
    assert bool(y.isfinite().all()) or dtype == torch.float16
    x[0, 0] = float("nan")
    bad = vm.int8_experts(x, w13, w2, ids, weights, emap)
    assert torch.equal(bad[1:], y[1:]) and bool(bad[0].isnan().all()) == bool(kept[0])


def test_side_stream_and_graph():
    import sm120_moe_bench_b200 as vm
    M, T, E, K, N = 24, 3, 8, 512, 256
    w13, w2 = random_rows(vm, (E, 2 * N, K), 48), random_rows(vm, (E, K, N), 50)
    lin = [random_rows(vm, (n, K), 52) for n in (64, 640)]
    x = torch.randn(M, K, generator=gen(54), device="cuda").bfloat16()
    ids = torch.randint(0, E, (M, T), generator=gen(55), device="cuda", dtype=torch.int32)
    weights = torch.rand(M, T, generator=gen(56), device="cuda")

    def everything():
        return [vm.int8_experts(x, w13, w2, ids, weights)] + [vm.int8_linear(x[:m], w) for w in lin for m in (1, 9, M)]

    want = everything()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = everything()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(side, want))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    got = []
    for g in graphs:
        with torch.cuda.graph(g):
            got.append(everything())
    for seed in (57, 58):
        x.copy_(torch.randn(M, K, generator=gen(seed), device="cuda"))
        ids.copy_(torch.randint(0, E, (M, T), generator=gen(seed + 9), device="cuda", dtype=torch.int32))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for g, st in zip(graphs, streams):                # both at once
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        want = everything()
        for out in got:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals():
    import sm120_moe_bench_b200 as vm
    q, s = torch.zeros(6, 32, dtype=torch.int8, device="cuda"), torch.ones(6, device="cuda")
    for bad in ((q.short(), s), (q, s[:5]), (q, s.double()), (q, s.cpu()), (q[0], s), (q.t().contiguous().t(), s),
                (torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), s[:1]), (q, torch.ones(12, device="cuda")[::2])):
        with pytest.raises(ValueError):
            vm.Int8Rows(*bad)
    a, w, we = vm.Int8Rows(q, s), vm.Int8Rows(q[:4], s[:4]), vm.Int8Rows(q.view(2, 3, 32), s.view(2, 3))
    plan = vm.plan_tokens(torch.zeros(3, 2, dtype=torch.int32, device="cuda"), 2)
    for call in (lambda: vm.int8_matmul(we, w), lambda: vm.int8_matmul(a, we), lambda: vm.int8_matmul(a, w, plan),
                 lambda: vm.int8_matmul(vm.Int8Rows(q[:5], s[:5]), we, plan), lambda: vm.int8_matmul(a, we, plan, swiglu=True),
                 lambda: vm.int8_matmul(a, vm.Int8Rows(q[:, :16], s)), lambda: vm.int8_matmul(a, w, out_dtype=torch.float64),
                 lambda: vm.int8_matmul(a, vm.Int8Rows(q[:0], s[:0])),
                 lambda: vm.int8_matmul(a, w, out=torch.empty(6, 5, device="cuda")), lambda: vm.int8_matmul(a, w, out=torch.empty(5, 4, device="cuda")),
                 lambda: vm.int8_matmul(a, w, out=torch.empty(6, 4)), lambda: vm.int8_matmul(a, w, out=torch.empty(1, 4, device="cuda").expand(6, 4)),
                 lambda: vm.int8_linear(torch.zeros(6, 32, device="cuda", requires_grad=True), w),
                 lambda: vm.int8_linear(torch.zeros(6, 31, device="cuda"), w), lambda: vm.int8_linear(torch.zeros(6, 32, device="cuda").double(), w),
                 lambda: vm.int8_linear(torch.zeros(6, 32, device="cuda"), w, out=torch.empty(6, 4, device="cuda").half()),
                 lambda: vm.quantize_int8(torch.zeros(2, 131072, device="cuda")), lambda: vm.quantize_int8(torch.zeros(4, 32, device="cuda"), plan),
                 lambda: vm.quantize_int8(torch.zeros(2, 3, 32, device="cuda"), plan),
                 lambda: vm.quantize_int8(torch.zeros(2, 32, 3, device="cuda").transpose(1, 2))):
        with pytest.raises(ValueError):
            call()
    x, ids, wt = torch.zeros(3, 32, device="cuda"), torch.zeros(3, 2, dtype=torch.int32, device="cuda"), torch.ones(3, 2, device="cuda")
    w13, w2 = random_rows(vm, (2, 32, 32), 60), random_rows(vm, (2, 32, 16), 62)
    for call in (lambda: vm.int8_experts(x, w13, w13, ids, wt), lambda: vm.int8_experts(x, w2, w2, ids, wt), lambda: vm.int8_experts(x[:2], w13, w2, ids, wt),
                 lambda: vm.int8_experts(x, w13, w2, ids, wt.half()), lambda: vm.int8_experts(x, w13, w2, ids.long(), wt),
                 lambda: vm.int8_experts(x, a, w2, ids, wt), lambda: vm.int8_experts(x.clone().requires_grad_(), w13, w2, ids, wt)):
        with pytest.raises(ValueError):
            call()
    with torch.no_grad():
        vm.int8_experts(x.clone().requires_grad_(), w13, w2, ids, wt)


@pytest.mark.parametrize("M", [1, 4, 9, 300])
def test_out_over_an_operand_is_refused(M):
    """Up to a few rows every block quantises them all for itself, while others already write out: x could be read overwritten."""
    import sm120_moe_bench_b200 as vm
    x, w = torch.randn(M, 64, generator=gen(90), device="cuda"), random_rows(vm, (64, 64), 91)
    with pytest.raises(ValueError, match="shares memory with x"):
        vm.int8_linear(x, w, out=x)
    a = random_rows(vm, (M, 64), 93)
    for out, name in ((a.q.view(torch.float32), "a"), (a.scale[:, None], "a's scales"), (w.scale[None], "w's scales"),
                      (w.q.view(torch.float32)[:1], "w")):
        n = out.shape[1]
        if out.shape[0] != M:
            continue
        with pytest.raises(ValueError, match=f"shares memory with {name}"):
            vm.int8_matmul(a, vm.Int8Rows(w.q[:n], w.scale[:n]), out=out)
    wide = torch.zeros(M, 128, device="cuda")
    wide[:, :64] = x
    vm.int8_linear(wide[:, :64], w, out=wide[:, 64:])     # columns side by side
    assert torch.equal(wide[:, :64], x) and torch.equal(wide[:, 64:], vm.int8_linear(x, w))


@pytest.mark.parametrize("M", [1, 2, 4, 8])
@pytest.mark.parametrize("K", [1, 15, 16, 17, 31, 1000, 1001, 4095, 4097, 4111, 8191])
def test_few_rows_of_aligned_weights_with_a_ragged_end(M, K):
    """Weights whose rows start on 16-byte boundaries and do not end on one: the last bytes are read one by one, nothing behind them."""
    import sm120_moe_bench_b200 as vm
    pitch = (K + 15) // 16 * 16
    for N in (1, 2, 60, 5000):
        a = random_rows(vm, (M, K), 94)
        store = torch.randint(-128, 128, (N * pitch + 16,), generator=gen(95), device="cuda", dtype=torch.int8)
        w = vm.Int8Rows(store[:N * pitch].view(N, pitch)[:, :K], torch.rand(N, generator=gen(96), device="cuda"))
        y = vm.int8_matmul(a, w, out_dtype=torch.float32)
        check_product(y, exact_product(a, w))
        store.view(-1)[N * pitch:] = 99
        for r in range(0, N, 7):
            store[r * pitch + K:(r + 1) * pitch] = 99     # what lies behind a row counts for nothing
        assert torch.equal(vm.int8_matmul(a, w, out_dtype=torch.float32), y)
        if N % 2 == 0:
            check_swiglu(vm.int8_matmul(a, w, swiglu=True, out_dtype=torch.float32), exact_product(a, w), N // 2)
        x = torch.randn(M, K, generator=gen(97), device="cuda").bfloat16()
        assert torch.equal(vm.int8_linear(x, w), vm.int8_matmul(vm.quantize_int8(x), w))


@pytest.mark.parametrize("M,N,K,E", [(20, 300, 2048, 0), (48, 512, 4096, 0), (129, 640, 256, 0), (700, 1024, 4096, 0), (2000, 1024, 640, 0),
                                     (50, 96, 512, 8), (900, 256, 1024, 4)])
def test_a_wait_that_runs_out(M, N, K, E):
    """With a limit of zero the first wait for data runs out in every block, and a copy starts after it.  The call returns, leaves
    its status, stores nothing that is not a right result, and the next call is right.  (Split over a cluster or not, persistent,
    per expert.)"""
    import sm120_moe_bench_b200 as vm
    from sm120_moe_bench_b200._lib import lib
    plan = vm.plan_tokens((torch.arange(M, device="cuda", dtype=torch.int32) % E)[:, None].contiguous(), E) if E else None
    a, w = random_rows(vm, (M, K), 98), random_rows(vm, (E, 2 * N, K) if E else (2 * N, K), 99)
    assert vm.int8_status() == 0
    for swiglu in (False, True):
        want = vm.int8_matmul(a, w, plan, swiglu=swiglu, out_dtype=torch.float32)
        out = torch.full_like(want, 12345.0)
        try:
            assert lib.vmoe_int8_set_wait_limit(0) == 0
            vm.int8_matmul(a, w, plan, swiglu=swiglu, out=out)
        finally:
            lib.vmoe_int8_set_wait_limit(10 ** 6)
        assert vm.int8_status() == 6
        assert bool(((out == 12345) | (out == want)).all())
        assert torch.equal(vm.int8_matmul(a, w, plan, swiglu=swiglu, out_dtype=torch.float32), want)
        assert vm.int8_status() == 0


@pytest.mark.parametrize("E,per", [(8192, 130), (11495, 130), (11496, 130), (13000, 200), (15591, 40), (15592, 40), (16384, 130), (16384, 3), (16385, 3)])
def test_thousands_of_experts(E, per):
    """The experts' tables lie beside the operands in shared memory: item sizes that leave no room for them are not taken."""
    import sm120_moe_bench_b200 as vm
    M, N, K = E * per, 8, 16
    offsets = torch.arange(0, M + 1, per, device="cuda", dtype=torch.int32)
    pairs = torch.arange(M, device="cuda", dtype=torch.int32)
    plan = vm.TokenPlan(offsets, pairs[:, None], pairs, E)
    a, w = random_rows(vm, (M, K), 100), random_rows(vm, (E, N, K), 102)
    exact = torch.bmm(a.q.view(E, per, K).double(), w.q.double().transpose(1, 2))
    want = (exact * a.scale.view(E, per, 1).double() * w.scale.view(E, 1, N).double()).view(M, N)
    check_product(vm.int8_matmul(a, w, plan, out_dtype=torch.float32), want)
    check_swiglu(vm.int8_matmul(a, w, plan, swiglu=True, out_dtype=torch.float32), want, N // 2)
    odd = vm.Int8Rows(w.q[..., :K - 1].contiguous(), w.scale)         # packed first
    short = vm.Int8Rows(a.q[:, :K - 1], a.scale)
    exact = torch.bmm(short.q.reshape(E, per, K - 1).double(), odd.q.double().transpose(1, 2))
    want = (exact * a.scale.view(E, per, 1).double() * w.scale.view(E, 1, N).double()).view(M, N)
    check_product(vm.int8_matmul(short, odd, plan, out_dtype=torch.float32), want)
    assert vm.int8_status() == 0


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad
    import sm120_moe_bench_b200 as vm
    w = random_rows(vm, (8, 32), 104)
    w13, w2 = random_rows(vm, (2, 32, 32), 106), random_rows(vm, (2, 32, 16), 108)
    x, ids, wt = torch.randn(6, 32, generator=gen(110), device="cuda"), torch.zeros(6, 2, dtype=torch.int32, device="cuda"), torch.ones(6, 2, device="cuda")
    a, out = vm.quantize_int8(x), torch.zeros(6, 8, device="cuda")
    with forward_ad.dual_level():
        dx, dwt, dout = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, wt, out))
        for call in (lambda: vm.quantize_int8(dx), lambda: vm.quantize_int8(dx[None].contiguous()), lambda: vm.int8_linear(dx, w),
                     lambda: vm.int8_experts(dx, w13, w2, ids, wt), lambda: vm.int8_experts(x, w13, w2, ids, dwt),
                     lambda: vm.int8_linear(x, w, out=dout), lambda: vm.int8_matmul(a, w, out=dout)):
            for mode in (torch.enable_grad, torch.no_grad):
                with pytest.raises(ValueError, match="forward-mode"), mode():
                    call()
        vm.int8_linear(x, w)


def test_scales_that_require_a_gradient_are_refused():
    from torch.autograd import forward_ad
    import sm120_moe_bench_b200 as vm
    x, ids, wt = torch.randn(6, 32, generator=gen(111), device="cuda"), torch.zeros(6, 2, dtype=torch.int32, device="cuda"), torch.ones(6, 2, device="cuda")
    a, w = vm.quantize_int8(x), random_rows(vm, (8, 32), 112)
    w13, w2 = random_rows(vm, (2, 32, 32), 114), random_rows(vm, (2, 32, 16), 116)

    def calls(learn):
        return (lambda: vm.int8_matmul(learn(a), w), lambda: vm.int8_matmul(a, learn(w)), lambda: vm.int8_linear(x, learn(w)),
                lambda: vm.int8_experts(x, learn(w13), w2, ids, wt), lambda: vm.int8_experts(x, w13, learn(w2), ids, wt))

    learnt = lambda r: vm.Int8Rows(r.q, torch.nn.Parameter(r.scale))
    for call, plain in zip(calls(learnt), calls(lambda r: r)):
        with pytest.raises(ValueError, match="scale requires a gradient"):
            call()
        with torch.no_grad():
            assert torch.equal(call(), plain())
    with forward_ad.dual_level():
        for call in calls(lambda r: vm.Int8Rows(r.q, forward_ad.make_dual(r.scale, r.scale))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
    scale = torch.nn.Parameter(a.scale)
    g, = torch.autograd.grad(vm.Int8Rows(a.q, scale).dequantize().sum(), scale)       # this is torch's own and has one
    assert torch.equal(g, a.q.float().sum(1))


@pytest.mark.parametrize("K,N", [(256, 8192), (256, 8200), (1024, 16384), (1024, 16392), (4096, 2048), (4096, 2056), (4096, 6144), (4096, 6152), (8192, 24),
                                 (1001, 1047), (1001, 1048), (1001, 2095), (1001, 2096), (1000, 8388), (1000, 8390), (4095, 300), (9001, 64), (16392, 32)])
def test_both_sides_of_the_few_row_rule(K, N):
    """Where one launch does it all, where quantiser and product are two, where unaligned weights are packed: the same bits."""
    import sm120_moe_bench_b200 as vm
    from sm120_moe_bench_b200._lib import lib
    x, w = torch.randn(9, K, generator=gen(118), device="cuda").bfloat16(), random_rows(vm, (N, K), 119)
    a = vm.quantize_int8(x)
    pairs = vm.Int8Rows(w.q[:N // 2 * 2], w.scale[:N // 2 * 2])
    want, gated = vm.int8_linear(x, w), vm.int8_linear(x, pairs, swiglu=True)
    check_product(want, exact_product(a, w))
    for M in range(1, 9):
        part = vm.Int8Rows(a.q[:M], a.scale[:M])
        assert torch.equal(vm.int8_linear(x[:M], w), want[:M]) and torch.equal(vm.int8_matmul(part, w), want[:M])
        assert torch.equal(vm.int8_linear(x[:M], pairs, swiglu=True), gated[:M])
        if M * ((K + 15) // 16 * 16) <= 65536:            # from C without scratch
            out = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
            assert lib.vmoe_int8_linear(x.data_ptr(), K, 0, M, w.q.data_ptr(), K, w.scale.data_ptr(), N, K, 0, out.data_ptr(), N, 0, None, 0,
                                        torch.cuda.current_stream().cuda_stream) == 0
            assert torch.equal(out, want[:M])


def silu_points():
    inf = float("inf")
    at = [0.0, -0.0, 2.0 ** -149, -2.0 ** -149, 1e-40, 2.0 ** -126, 1e-30, -1e-30, 2.0 ** -24, -2.0 ** -12, 0.5, 1.0, -1.0, 8.0, -8.0, 16.0, -16.0, 16.635,
          20.0, -20.0, -87.0, -87.3, -87.33, -87.3365, -87.337, -87.5, -88.0, -88.72, -88.73, -89.0, -103.0, -104.0, -1000.0, 88.0, 1000.0, 3.4e38, -3.4e38]
    c = torch.tensor(at, device="cuda")
    near = [c]
    for way in (inf, -inf):
        n = c
        for _ in range(3):
            n = torch.nextafter(n, torch.full_like(n, way))
            near.append(n)
    g = gen(120)
    return torch.cat(near + [torch.linspace(-110, 110, 100001, device="cuda"), torch.linspace(-4, 4, 20001, device="cuda"),
                             20 * torch.randn(40000, generator=g, device="cuda"), torch.exp(20 * torch.randn(20000, generator=g, device="cuda")),
                             -torch.exp(6 * torch.randn(20000, generator=g, device="cuda"))])


@pytest.mark.parametrize("M", [1, 8, 9, 40])
def test_silu_over_its_range(M):
    """A code of 1 times a channel's scale is any gate, times an up of 1: the result is the silu itself, of each kernel.  It may be
    off by 6 * 2^-24 (expf 4, the sum and the quotient half a step each) and 2^-40 for products of those; half a step among
    the subnormals; and is flushed to 0 below -87.33, where silu is above -1.04e-36."""
    import sm120_moe_bench_b200 as vm
    x = silu_points()
    n = x.numel()
    a = vm.Int8Rows(torch.ones(M, 1, dtype=torch.int8, device="cuda"), torch.ones(M, device="cuda"))
    w = vm.Int8Rows(torch.ones(2 * n, 1, dtype=torch.int8, device="cuda"), torch.cat([x, torch.ones(n, device="cuda")]))
    y = vm.int8_matmul(a, w, swiglu=True, out_dtype=torch.float32)
    assert torch.equal(y, y[:1].expand(M, n))
    want = silu64(x.double())
    tol = (6 * 2.0 ** -24 + 2.0 ** -40) * want.abs() + 2.0 ** -150 + torch.where(x < -87.33, 1.04e-36, 0.0).double()
    assert bool(((y[0].double() - want).abs() <= tol).all())
    ends = vm.Int8Rows(torch.ones(8, 1, dtype=torch.int8, device="cuda"), torch.tensor([float("inf"), float("-inf"), float("nan"), 1.0, 1, 1, 1, 1], device="cuda"))
    y = vm.int8_matmul(a, ends, swiglu=True, out_dtype=torch.float32)
    assert bool((y[:, 0] == float("inf")).all()) and bool(y[:, 1:3].isnan().all()) and bool(y[:, 3].isfinite().all())


def test_status_while_capturing_is_refused():
    import sm120_moe_bench_b200 as vm
    x, w = torch.randn(40, 64, generator=gen(121), device="cuda"), random_rows(vm, (64, 64), 122)
    want = vm.int8_linear(x, w)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        with pytest.raises(RuntimeError, match="capture"):
            vm.int8_status()
        y = vm.int8_linear(x, w)                          # the capture goes on
    g.replay()
    assert torch.equal(y, want) and vm.int8_status() == 0
