"""Token rows sorted by expert and back against a plain implementation in 64 bits, with the gradients.

Tolerances: copies are bit-equal.  A sum of T products in f32 is off by at most (T + 1) * 2^-24 * sum |w| |r| before it is
rounded to the output type, which adds half a step (eps / 2 of the value; 2^-25 absolute among fp16's subnormals).  A dot
product over K elements in f32, in any order, is off by at most (K + 1) * 2^-24 * sum |r| |dy|."""
import copy
import os
import pickle

import pytest
import torch

os.environ.setdefault("VMOE_NO_VLLM", "1")
pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def rows_of(M, K, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(M, K, generator=g, device="cuda").to(dtype)


def ids_of(M, T, E, seed, repeat=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if repeat:                                            # the same expert several times in a token
        return torch.randint(0, E, (M, T), generator=g, device="cuda", dtype=torch.int32)
    return torch.topk(torch.randn(M, E, generator=g, device="cuda"), T, dim=1).indices.int()


def plain_plan(ids, E, expert_map=None):
    flat = ids.cpu().reshape(-1).tolist()
    emap = None if expert_map is None else expert_map.cpu().tolist()
    local = []
    for e in flat:
        if emap is not None:
            e = emap[e] if 0 <= e < len(emap) else -1
        local.append(e if 0 <= e < E else -1)
    order = sorted((e, p) for p, e in enumerate(local) if e >= 0)
    row_of_pair = [-1] * len(flat)
    for r, (_, p) in enumerate(order):
        row_of_pair[p] = r
    pair_of_row = [p for _, p in order] + [-1] * (len(flat) - len(order))
    offsets = [sum(1 for e in local if 0 <= e < x) for x in range(E + 1)] if E <= 64 else \
        torch.searchsorted(torch.tensor([e for e, _ in order], dtype=torch.int64), torch.arange(E + 1)).tolist()
    return (torch.tensor(offsets, dtype=torch.int32), torch.tensor(row_of_pair, dtype=torch.int32).reshape(ids.shape),
            torch.tensor(pair_of_row, dtype=torch.int32))


def check_plan(plan, ids, E, expert_map=None):
    offsets, row_of_pair, pair_of_row = plain_plan(ids, E, expert_map)
    assert torch.equal(plan.expert_offsets.cpu(), offsets)
    assert torch.equal(plan.row_of_pair.cpu(), row_of_pair)
    assert torch.equal(plan.pair_of_row.cpu(), pair_of_row)


def half_step(dtype, value):
    return torch.finfo(dtype).eps / 2 * value.abs() * (1 + 2.0 ** -20) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126)


def plain_unsort(rows, row_of_pair, w):
    """(sum, sum of magnitudes) in 64 bits"""
    kept = (row_of_pair >= 0).double()[:, :, None]
    r = rows.double()[row_of_pair.clamp(min=0).long()]
    r = torch.where(kept > 0, r, 0.0)
    w = torch.ones(row_of_pair.shape, dtype=torch.float64, device=rows.device) if w is None else w.double()
    w = torch.where(row_of_pair >= 0, w, 0.0)[:, :, None]
    return (r * w).sum(1), (r * w).abs().sum(1)


@pytest.mark.parametrize("M,T,E,repeat", [(0, 2, 4, False), (1, 1, 1, False), (1, 16, 16, False), (3, 2, 5, True), (64, 10, 512, False),
                                          (409, 10, 512, False), (410, 10, 512, False), (1000, 7, 33, True), (2049, 8, 8, False),
                                          (5000, 3, 8192, True), (700, 16, 1, True), (4097, 1, 2, False), (8192, 10, 512, False)])
def test_plan(M, T, E, repeat):
    import sm120_moe_bench_b200 as vm
    ids = ids_of(M, T, E, 1, repeat) if M else torch.zeros(0, T, dtype=torch.int32, device="cuda")
    check_plan(vm.plan_tokens(ids, E), ids, E)


def test_plan_drops_ids_outside_the_experts_and_the_map():
    import sm120_moe_bench_b200 as vm
    ids = ids_of(300, 6, 40, 2, True)
    ids[::7, 2] = -1
    ids[::5, 1] = 40
    ids[11] = 2 ** 31 - 1
    ids[12] = -2 ** 31
    check_plan(vm.plan_tokens(ids, 40), ids, 40)
    emap = torch.full((40,), -1, dtype=torch.int32, device="cuda")
    emap[8:20] = torch.arange(12, device="cuda", dtype=torch.int32)
    emap[3] = 12                                          # a map entry outside the local experts
    check_plan(vm.plan_tokens(ids, 12, emap), ids, 12, emap)
    nothing = torch.full((9, 3), -1, dtype=torch.int32, device="cuda")
    plan = vm.plan_tokens(nothing, 4)
    check_plan(plan, nothing, 4)
    x = rows_of(9, 24, torch.bfloat16, 3)
    assert torch.count_nonzero(vm.sort_tokens(x, plan)) == 0
    rows = torch.full((27, 24), float("nan"), dtype=torch.bfloat16, device="cuda")
    assert torch.count_nonzero(vm.unsort_tokens(rows, plan, torch.full((9, 3), float("inf"), device="cuda"))) == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,T,E,K", [(1, 1, 1, 1), (1, 10, 512, 4096), (5, 2, 3, 7), (33, 16, 64, 136), (64, 10, 512, 4096), (257, 3, 9, 1021),
                                     (100, 5, 20, 1026), (129, 4, 8, 2052), (31, 8, 16, 5000)])
def test_forward_and_gradients(M, T, E, K, dtype):
    import sm120_moe_bench_b200 as vm
    ids = ids_of(M, T, E, 5)
    if M > 4:
        ids[::4, T - 1] = -1
    plan = vm.plan_tokens(ids, E)
    check_plan(plan, ids, E)
    rp, pr = plan.row_of_pair, plan.pair_of_row
    x = rows_of(M, K, dtype, 6).requires_grad_()
    rows = vm.sort_tokens(x, plan)
    want = torch.where((pr >= 0)[:, None], x.detach()[(pr.clamp(min=0) // T).long()], 0.0)
    assert torch.equal(rows, want)
    g = rows_of(M * T, K, dtype, 7)
    dx, = torch.autograd.grad(rows, x, g)
    s, mag = plain_unsort(g, rp, None)
    assert dx.dtype == dtype and bool(((dx.double() - s).abs() <= (T + 1) * 2.0 ** -24 * mag + half_step(dtype, s)).all())

    w = torch.softmax(rows_of(M, T, torch.float32, 8), 1).requires_grad_()
    r = rows_of(M * T, K, dtype, 9).requires_grad_()
    y = vm.unsort_tokens(r, plan, w)
    s, mag = plain_unsort(r.detach(), rp, w.detach())
    assert y.dtype == dtype and bool(((y.double() - s).abs() <= (T + 1) * 2.0 ** -24 * mag + half_step(dtype, s)).all())
    dy = rows_of(M, K, dtype, 10)
    dr, dw = torch.autograd.grad(y, (r, w), dy)
    tok, flat = (pr.clamp(min=0) // T).long(), w.detach().reshape(-1)[pr.clamp(min=0).long()].double()
    want = torch.where((pr >= 0)[:, None], dy.double()[tok] * flat[:, None], 0.0)
    assert bool(((dr.double() - want).abs() <= 2.0 ** -24 * want.abs() + half_step(dtype, want)).all())
    assert torch.count_nonzero(dr[int(plan.expert_offsets[-1]):]) == 0
    rr = torch.where((rp >= 0)[:, :, None], r.detach().double()[rp.clamp(min=0).long()], 0.0)
    want, mag = (rr * dy.double()[:, None]).sum(2), (rr * dy.double()[:, None]).abs().sum(2)
    assert bool(((dw.double() - want).abs() <= (K + 1) * 2.0 ** -24 * mag).all())


def test_one_gradient_at_a_time():
    import sm120_moe_bench_b200 as vm
    plan = vm.plan_tokens(ids_of(20, 3, 6, 11), 6)
    r, w, dy = rows_of(60, 72, torch.float32, 12), torch.rand(20, 3, device="cuda"), rows_of(20, 72, torch.float32, 13)
    ra, wa = r.clone().requires_grad_(), w.clone().requires_grad_()
    both = torch.autograd.grad(vm.unsort_tokens(ra, plan, wa), (ra, wa), dy)
    rb = r.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(vm.unsort_tokens(rb, plan, w), rb, dy)[0], both[0])
    wb = w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(vm.unsort_tokens(r, plan, wb), wb, dy)[0], both[1])
    rc = r.clone().requires_grad_()
    ones = torch.autograd.grad(vm.unsort_tokens(rc, plan), rc, dy)[0]
    assert torch.equal(ones, vm.sort_tokens(dy, plan))
    with torch.no_grad():
        assert not vm.unsort_tokens(ra, plan, wa).requires_grad


def test_gradients_against_differences():
    """A scalar of the round trip is linear in x and in w: central differences are exact but for f32 rounding, which the step
    keeps at 2^-24 * |scalar parts| / step."""
    import sm120_moe_bench_b200 as vm
    plan = vm.plan_tokens(ids_of(6, 3, 4, 14, True), 4)
    x, w = rows_of(6, 10, torch.float32, 15).requires_grad_(), torch.rand(6, 3, device="cuda").requires_grad_()
    c, gain = rows_of(6, 10, torch.float32, 16), rows_of(18, 10, torch.float32, 17)

    def f(x, w):
        return (vm.unsort_tokens(vm.sort_tokens(x, plan) * gain, plan, w) * c).double().sum()

    dx, dw = torch.autograd.grad(f(x, w), (x, w))
    step = 2.0 ** -3
    scale = float((plain_unsort((vm.sort_tokens(x.detach(), plan) * gain), plan.row_of_pair, w.detach())[1] * c.double().abs()).sum())
    tol = 16 * 2.0 ** -24 * (scale + 10) / step
    with torch.no_grad():
        for t, d in ((x, dx), (w, dw)):
            for i in range(t.numel()):
                e = torch.zeros_like(t)
                e.view(-1)[i] = step
                a, b = ((f(x + e, w), f(x - e, w)) if t is x else (f(x, w + e), f(x, w - e)))
                assert abs(float((a - b) / (2 * step)) - float(d.view(-1)[i])) <= tol


def test_gradient_of_the_gradient():
    import sm120_moe_bench_b200 as vm
    plan = vm.plan_tokens(ids_of(9, 3, 5, 35), 5)
    x, g = rows_of(9, 12, torch.float32, 36).requires_grad_(), rows_of(27, 12, torch.float32, 37).requires_grad_()
    dx, = torch.autograd.grad(vm.sort_tokens(x, plan), x, g, create_graph=True)
    v = rows_of(9, 12, torch.float32, 38)
    dg, = torch.autograd.grad(dx, g, v)                    # dx is linear in g: its gradient sorts v
    assert torch.equal(dg, vm.sort_tokens(v, plan))
    w = torch.rand(9, 3, device="cuda").requires_grad_()
    dy = rows_of(9, 12, torch.float32, 39).requires_grad_()
    y = vm.unsort_tokens(g, plan, w)
    once = torch.autograd.grad(y, (g, w), dy, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(once, torch.autograd.grad(vm.unsort_tokens(g, plan, w), (g, w), dy)))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        once[0].sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_alignment(dtype):
    import sm120_moe_bench_b200 as vm
    M, T, E, K = 37, 3, 5, 64
    plan = vm.plan_tokens(ids_of(M, T, E, 18), E)
    base = rows_of(M + 1, 2 * K + 3, dtype, 19)
    for x in (base[:M, :K], base[:M, 1:K + 1], base[1:, 3:K + 3], base[::1][:M, K:2 * K], base[:1, :K].expand(M, K)):
        assert torch.equal(vm.sort_tokens(x, plan), vm.sort_tokens(x.contiguous(), plan))
    rows = rows_of(M * T, K + 5, dtype, 20)
    w = torch.rand(M, T, device="cuda")
    for r in (rows[:, :K], rows[:, 1:K + 1], rows[:, 5:]):
        assert torch.equal(vm.unsort_tokens(r, plan, w), vm.unsort_tokens(r.contiguous(), plan, w))
    # gradients that arrive expanded (of a sum) or strided
    x = base[:M, 1:K + 1].detach().requires_grad_()
    dx, = torch.autograd.grad(vm.sort_tokens(x, plan).sum(), x)
    assert torch.equal(dx, torch.full_like(dx, T))
    r = rows[:, 1:K + 1].detach().requires_grad_()
    dr, = torch.autograd.grad(vm.unsort_tokens(r, plan, w), r, base[:M, 2:K + 2])
    r2 = r.detach().contiguous().requires_grad_()
    assert torch.equal(dr, torch.autograd.grad(vm.unsort_tokens(r2, plan, w), r2, base[:M, 2:K + 2].contiguous())[0])


def test_out_keeps_what_is_behind_the_last_row():
    import sm120_moe_bench_b200 as vm
    ids = ids_of(10, 4, 6, 21)
    ids[:, 0] = -1
    plan = vm.plan_tokens(ids, 6)
    x = rows_of(10, 40, torch.float16, 22)
    buf = torch.full((41, 50), 7.0, dtype=torch.float16, device="cuda")
    got = vm.sort_tokens(x, plan, out=buf[:40, 3:43])
    assert got.data_ptr() == buf[:40, 3:43].data_ptr()
    assert torch.equal(buf[:30, 3:43], vm.sort_tokens(x, plan)[:30])
    assert bool((buf[30:] == 7).all()) and bool((buf[:, :3] == 7).all()) and bool((buf[:, 43:] == 7).all())
    y = torch.full((11, 44), 5.0, dtype=torch.float16, device="cuda")
    vm.unsort_tokens(buf[:40, 3:43], plan, out=y[:10, 2:42])
    assert torch.equal(y[:10, 2:42], vm.unsort_tokens(buf[:40, 3:43].contiguous(), plan))
    assert bool((y[10] == 5).all()) and bool((y[:, :2] == 5).all()) and bool((y[:, 42:] == 5).all())


def test_non_finite_values_stay_in_their_tokens():
    import sm120_moe_bench_b200 as vm
    ids = ids_of(12, 2, 4, 23)
    ids[5, 1] = -1
    plan = vm.plan_tokens(ids, 4)
    rows = rows_of(24, 16, torch.bfloat16, 24)
    clean = vm.unsort_tokens(rows, plan, torch.ones(12, 2, device="cuda"))
    w = torch.ones(12, 2, device="cuda")
    w[5, 1] = float("nan")                                # the weight of a dropped pair
    w[7, 0] = float("nan")
    rows[23] = float("inf")                               # behind the last kept row
    y = vm.unsort_tokens(rows, plan, w)
    assert bool(y[7].isnan().all())
    keep = torch.arange(12, device="cuda") != 7
    assert torch.equal(y[keep], clean[keep])


def test_a_copied_plan_outlives_the_original():
    import sm120_moe_bench_b200 as vm
    ids, x = ids_of(30, 3, 7, 46), rows_of(30, 40, torch.float32, 47)
    plan = vm.plan_tokens(ids, 7)
    want = vm.sort_tokens(x, plan)
    twin = copy.deepcopy(plan)
    check_plan(twin, ids, 7)
    assert twin._offsets_ptr == twin.expert_offsets.data_ptr() != plan._offsets_ptr
    del plan
    torch.full((4096,), -3, dtype=torch.int32, device="cuda")
    assert torch.equal(vm.sort_tokens(x, twin), want)


def test_more_than_four_gigabytes_of_rows():
    import sm120_moe_bench_b200 as vm
    M, T, E, K = 40000, 16, 32, 4096
    ids = ids_of(M, T, E, 25)
    plan = vm.plan_tokens(ids, E)
    x = rows_of(M, K, torch.bfloat16, 26)
    rows = vm.sort_tokens(x, plan)
    assert rows.numel() * 2 > 2 ** 32
    for r in (0, M * T // 2, M * T - 1):
        assert torch.equal(rows[r], x[int(plan.pair_of_row[r]) // T])
    w = torch.full((M, T), 1 / 16, device="cuda")
    assert torch.equal(vm.unsort_tokens(rows, plan, w), x)     # sixteen times a sixteenth, exact in f32
    rows.requires_grad_()
    dr, = torch.autograd.grad(vm.unsort_tokens(rows, plan, w), rows, x)
    assert torch.equal(dr[-1], x[int(plan.pair_of_row[-1]) // T] / 16)


def test_side_stream_and_graph():
    import sm120_moe_bench_b200 as vm
    M, T, E, K = 50, 4, 16, 256
    x, w = rows_of(M, K, torch.bfloat16, 27), torch.rand(M, T, device="cuda")
    ids = ids_of(M, T, E, 28)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        plan = vm.plan_tokens(ids, E)
        side = vm.unsort_tokens(vm.sort_tokens(x, plan), plan, w)
    torch.cuda.current_stream().wait_stream(s)
    plan.record_stream(torch.cuda.current_stream())
    assert torch.equal(side, vm.unsort_tokens(vm.sort_tokens(x, plan), plan, w))
    plan = vm.plan_tokens(ids, E)
    assert torch.equal(side, vm.unsort_tokens(vm.sort_tokens(x, plan), plan, w))
    # forward and backward captured together, replayed on other inputs
    xs, ws, ids_s, dy = x.clone().requires_grad_(), w.clone().requires_grad_(), ids.clone(), rows_of(M, K, torch.bfloat16, 29)

    def step():
        p = vm.plan_tokens(ids_s, E)
        y = vm.unsort_tokens(vm.sort_tokens(xs, p), p, ws)
        return (y.detach(), *torch.autograd.grad(y, (xs, ws), dy))

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for seed in (30, 31):
        with torch.no_grad():
            xs.copy_(rows_of(M, K, torch.bfloat16, seed))
            ids_s.copy_(ids_of(M, T, E, seed))
        g.replay()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))


def test_backward_in_a_graph_beside_an_eager_graph():
    import sm120_moe_bench_b200 as vm
    plan = vm.plan_tokens(ids_of(16, 2, 4, 40), 4)
    x, w = rows_of(16, 32, torch.float32, 41).requires_grad_(), torch.rand(16, 2, device="cuda").requires_grad_()
    eager = vm.unsort_tokens(vm.sort_tokens(x, plan), plan, w)
    for leaf in (lambda: vm.sort_tokens(x, plan), lambda: vm.unsort_tokens(vm.sort_tokens(x.detach(), plan), plan, w)):
        with pytest.raises(RuntimeError, match="eager graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                leaf()
    eager.sum().backward()
    want = x.grad.clone(), w.grad.clone()
    other = rows_of(16, 32, torch.float32, 45).requires_grad_()            # another leaf's graph is no hindrance
    held = vm.sort_tokens(other, plan)
    assert copy.deepcopy(x).equal(x)
    del eager
    x.grad = w.grad = None
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        vm.unsort_tokens(vm.sort_tokens(x, plan), plan, w).sum().backward()
    g.replay()
    assert torch.equal(x.grad, want[0]) and torch.equal(w.grad, want[1])
    held.sum().backward()
    p = torch.nn.Parameter(x.detach())
    graph = vm.sort_tokens(p, plan)                       # a parameter with a live graph is saved like any other
    assert torch.equal(pickle.loads(pickle.dumps(p)), p) and graph.requires_grad


def test_a_table_of_wild_rows_is_harmless():
    """Rows outside the tensor (a plan that plan_tokens did not make) drop their pair; nothing is read or written there."""
    import sm120_moe_bench_b200 as vm
    M, T, E, K = 8, 2, 4, 64
    good = vm.plan_tokens(ids_of(M, T, E, 42), E)
    rp = good.row_of_pair.clone()
    rp[2, 1], rp[5, 0], rp[6, 1] = M * T, 2 ** 31 - 1, -2 ** 31
    offsets = good.expert_offsets.clone()
    offsets[0], offsets[2], offsets[-1] = -7, 10 ** 6, 2 ** 31 - 1
    wild = vm.TokenPlan(offsets, rp, good.pair_of_row, E)
    x = rows_of(M, K, torch.float32, 43)
    fence = torch.full((M * T + 2, K), 3.0, device="cuda")
    vm.sort_tokens(x, wild, out=fence[1:-1])
    assert bool((fence[0] == 3).all()) and bool((fence[-1] == 3).all())
    rows = rows_of(M * T, K, torch.float32, 44)
    kept = (rp >= 0) & (rp < M * T)
    want = torch.where(kept[:, :, None], rows[rp.clamp(0, M * T - 1).long()], 0.0).sum(1)
    assert torch.equal(vm.unsort_tokens(rows, wild), want)
    r = rows.requires_grad_()
    torch.autograd.grad(vm.unsort_tokens(r, wild), r, x)
    q = vm.quantize_int8(x, wild)
    w = vm.quantize_int8(torch.randn(E, 32, K, device="cuda"))
    vm.int8_matmul(q, w, wild, out_dtype=torch.float32)
    odd = vm.Int8Rows(w.q[..., 1:62].contiguous(), w.scale)
    vm.int8_matmul(vm.Int8Rows(q.q[:, :61], q.scale), odd, wild, out_dtype=torch.float32)
    torch.cuda.synchronize()
    assert vm.int8_status() == 0


def test_refusals():
    import sm120_moe_bench_b200 as vm
    ids = ids_of(8, 2, 4, 32)
    for bad in (ids.long(), ids[0], ids[:, :1].expand(8, 2), ids.t()):
        with pytest.raises(ValueError):
            vm.plan_tokens(bad, 4)
    for E in (0, 8193):
        with pytest.raises(ValueError):
            vm.plan_tokens(ids, E)
    with pytest.raises(ValueError):
        vm.plan_tokens(torch.zeros(4, 17, dtype=torch.int32, device="cuda"), 4)
    for emap in (torch.zeros(4, dtype=torch.int32), torch.zeros(4, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")):
        with pytest.raises(ValueError):
            vm.plan_tokens(ids, 4, emap)
    plan = vm.plan_tokens(ids, 4)
    x = rows_of(8, 16, torch.float32, 33)
    for bad in (x.double(), x[:7], x[0], x.t().contiguous().t(), rows_of(8, 32, torch.float32, 33)[:, ::2], x.cpu()):
        with pytest.raises(ValueError):
            vm.sort_tokens(bad, plan)
    with pytest.raises(ValueError):
        vm.sort_tokens(x.clone().requires_grad_(), plan, out=torch.empty(16, 16, device="cuda"))
    for out in (torch.empty(15, 16, device="cuda"), torch.empty(16, 17, device="cuda"), torch.empty(16, 16, device="cuda").half(),
                torch.empty(1, 16, device="cuda").expand(16, 16)):
        with pytest.raises(ValueError):
            vm.sort_tokens(x, plan, out=out)
    rows, w = rows_of(16, 16, torch.float32, 34), torch.ones(8, 2, device="cuda")
    for bad in (w.half(), w[:7], w.t().contiguous().t(), w.cpu()):
        with pytest.raises(ValueError):
            vm.unsort_tokens(rows, plan, bad)
    with pytest.raises(ValueError):
        vm.unsort_tokens(rows[:15], plan, w)
    # the operator still answers afterwards
    assert torch.equal(vm.unsort_tokens(vm.sort_tokens(x, plan), plan), 2 * x)


def test_out_over_an_operand_is_refused():
    """Blocks read the operands and write out in no order: x under out would be sorted from rows that are overwritten already."""
    import sm120_moe_bench_b200 as vm
    M, T, E, K = 8, 2, 4, 16
    plan = vm.plan_tokens(ids_of(M, T, E, 50), E)
    copied = copy.deepcopy(plan)
    buf = rows_of(M * T, K, torch.float32, 51)
    for out in (buf, buf.as_strided((M * T, K), (K, 1), 0)):
        for p in (plan, copied):
            with pytest.raises(ValueError, match="shares memory with x"):
                vm.sort_tokens(buf[M:], p, out=out)
    for out in (buf[:M], buf[4:4 + M]):
        with pytest.raises(ValueError, match="shares memory with rows"):
            vm.unsort_tokens(buf, plan, out=out)
    one = vm.plan_tokens(ids_of(M, 1, E, 52), E)          # not even where every row stays a row
    x = rows_of(M, K, torch.float32, 53)
    with pytest.raises(ValueError, match="shares memory"):
        vm.sort_tokens(x, one, out=x)
    w = torch.ones(M, T, device="cuda")
    with pytest.raises(ValueError, match="shares memory with weights"):
        vm.unsort_tokens(rows_of(M * T, T, torch.float32, 54), plan, w, out=w)
    for p in (plan, copied):
        table = p.row_of_pair.view(torch.float32)
        with pytest.raises(ValueError, match="the plan"):
            vm.unsort_tokens(rows_of(M * T, T, torch.float32, 54), p, out=table)
    # columns of one buffer side by side are two tensors
    wide = rows_of(M * T, 2 * K, torch.float32, 55)
    want = vm.unsort_tokens(wide[:, :K].contiguous(), plan, w)
    vm.unsort_tokens(wide[:, :K], plan, w, out=wide[:M, K:])
    assert torch.equal(wide[:M, K:], want)


def test_forward_mode_is_refused():
    """A dual tensor does not require a gradient, and a result without its tangent would be a derivative of zero."""
    from torch.autograd import forward_ad
    import sm120_moe_bench_b200 as vm
    M, T, E, K = 6, 2, 4, 8
    plan = vm.plan_tokens(ids_of(M, T, E, 56), E)
    x, rows, w = rows_of(M, K, torch.float32, 57), rows_of(M * T, K, torch.float32, 58), torch.rand(M, T, device="cuda")
    want = vm.sort_tokens(x, plan), vm.unsort_tokens(rows, plan, w)
    with forward_ad.dual_level():
        dx, dr, dw = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, rows, w))
        for call in (lambda: vm.sort_tokens(dx, plan), lambda: vm.unsort_tokens(dr, plan, w), lambda: vm.unsort_tokens(rows, plan, dw),
                     lambda: vm.unsort_tokens(dr, plan), lambda: vm.sort_tokens(x, plan, out=dr), lambda: vm.unsort_tokens(rows, plan, w, out=dx),
                     lambda: vm.sort_tokens(forward_ad.make_dual(x.clone().requires_grad_(), x), plan)):
            for mode in (torch.enable_grad, torch.no_grad):
                with pytest.raises(NotImplementedError), mode():
                    call()
        assert torch.equal(vm.sort_tokens(x, plan), want[0]) and torch.equal(vm.unsort_tokens(rows, plan, w), want[1])
    xr, rr, wr = (t.clone().requires_grad_() for t in (x, rows, w))
    sorted_x, y = vm.sort_tokens(xr, plan), vm.unsort_tokens(rr, plan, wr)
    with forward_ad.dual_level():                         # the incoming gradient has a tangent
        dg, dy = forward_ad.make_dual(rows, rows), forward_ad.make_dual(x, x)
        for create in (False, True):
            for call in (lambda: torch.autograd.grad(sorted_x, xr, dg, retain_graph=True, create_graph=create),
                         lambda: torch.autograd.grad(y, rr, dy, retain_graph=True, create_graph=create),
                         lambda: torch.autograd.grad(y, wr, dy, retain_graph=True, create_graph=create)):
                with pytest.raises(NotImplementedError):
                    call()
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda t: vm.sort_tokens(t, plan), (x,), (x,))


def test_traces_are_refused():
    """torch.jit.trace and make_fx record torch's operators only: a trace would return the memory that was allocated for a result."""
    from torch.fx.experimental.proxy_tensor import make_fx
    import sm120_moe_bench_b200 as vm
    ids = ids_of(6, 2, 4, 59)
    plan = vm.plan_tokens(ids, 4)
    x, rows, w = rows_of(6, 32, torch.float32, 60), rows_of(12, 32, torch.float32, 61), torch.rand(6, 2, device="cuda")
    q = vm.quantize_int8(rows_of(8, 32, torch.float32, 62))
    w13, w2 = vm.quantize_int8(torch.randn(4, 32, 32, device="cuda")), vm.quantize_int8(torch.randn(4, 32, 16, device="cuda"))
    codes = vm.quantize_int8(x)
    calls = (lambda t: vm.sort_tokens(t, plan), lambda t: vm.unsort_tokens(torch.cat([t, t]), plan, w), lambda t: vm.int8_linear(t, q),
             lambda t: vm.quantize_int8(t).q, lambda t: t + vm.int8_matmul(codes, q).sum(), lambda t: vm.int8_experts(t, w13, w2, ids, w),
             lambda t: t + vm.plan_tokens(ids, 4).expert_offsets.sum(), lambda t: vm.sort_tokens(t * 1, plan, out=rows.clone()))
    for call in calls:
        for trace in (lambda: make_fx(call)(x), lambda: make_fx(call, pre_dispatch=True)(x), lambda: torch.jit.trace(call, x, check_trace=False),
                      lambda: make_fx(call)(x.clone().requires_grad_())):
            with pytest.raises((RuntimeError, ValueError)):
                trace()
    assert torch.equal(vm.unsort_tokens(vm.sort_tokens(x, plan), plan), 2 * x)
    # torch.compile runs the calls as they are
    def step(t, weights):
        return vm.unsort_tokens(vm.sort_tokens(t * 2, plan), plan, weights) + 1

    got = torch.compile(step, backend="eager")(x, w)
    assert torch.equal(got, step(x, w))
    a, b = (t.clone().requires_grad_() for t in (x, w)), (t.clone().requires_grad_() for t in (x, w))
    a, b = tuple(a), tuple(b)
    ga = torch.autograd.grad(torch.compile(step, backend="eager")(*a).sum(), a)
    gb = torch.autograd.grad(step(*b).sum(), b)
    assert all(torch.equal(p, r) for p, r in zip(ga, gb))


def test_a_graph_that_saved_out_notices():
    """Another graph holds the tensor that is overwritten: its backward pass must not use the new values."""
    import sm120_moe_bench_b200 as vm
    M, T, E, K = 6, 2, 4, 32
    plan = vm.plan_tokens(ids_of(M, T, E, 63), E)
    x, rows, weights = rows_of(M, K, torch.float32, 64), rows_of(M * T, K, torch.float32, 65), torch.rand(M, T, device="cuda")
    q, codes = vm.quantize_int8(rows_of(K, K, torch.float32, 66)), vm.quantize_int8(x)
    for n, call in ((M * T, lambda out: vm.sort_tokens(x, plan, out=out)), (M, lambda out: vm.unsort_tokens(rows, plan, weights, out=out)),
                    (M, lambda out: vm.int8_linear(x, q, out=out)), (M, lambda out: vm.int8_matmul(codes, q, out=out))):
        gain, wide = torch.ones(n, K, device="cuda", requires_grad=True), torch.zeros(n + 2, K + 4, device="cuda")
        for out in (torch.zeros(n, K, device="cuda"), wide[:n, 4:]):
            y = (gain * out).sum()
            assert call(out) is out
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                y.backward()
        with torch.inference_mode():                      # no versions there
            call(torch.zeros(n, K, device="cuda"))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_are_kept_for_the_weights_gradient_alone(dtype):
    import sm120_moe_bench_b200 as vm
    M, T, E, K = 40, 3, 6, 72
    plan = vm.plan_tokens(ids_of(M, T, E, 67), E)
    rows, dy = rows_of(M * T, K, dtype, 68), rows_of(M, K, dtype, 69)
    w = torch.rand(M, T, device="cuda")
    for weights, kept in ((None, 0), (w, 1), (w.clone().requires_grad_(), 2)):
        leaf = rows.clone().requires_grad_()
        saved = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: saved.append(t.shape) or t, lambda t: t):
            y = vm.unsort_tokens(leaf, plan, weights)
        assert saved == [rows.shape, w.shape][2 - kept:]
        want, = torch.autograd.grad(y, leaf, dy)
        # in between the rows may change
        inner = leaf * 1
        y = vm.unsort_tokens(inner, plan, weights)
        inner.mul_(2)
        if kept == 2:
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(y, leaf, dy)
        else:
            # d inner = the rows' gradient; the product with 2 is later than y
            assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], want)
