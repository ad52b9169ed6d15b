"""Workloads of the token sort (rows ordered by expert and back, with gradients) and of the 8-bit integer products.

A case is one pass through one operator:

  ``sort``    plan from the router's ids, then the token rows copied into expert order (``train``: and the gradient back);
  ``unsort``  plan, then a token's rows weighted and summed (``train``: and the gradients of the rows and of the weights);
  ``linear``  bf16 / fp16 / f32 rows quantised row by row, times 8-bit weights with a scale per output channel
              (``codes``: the rows arrive as codes already);
  ``experts`` the whole expert layer on 8-bit weights: sort, product, SwiGLU, product, weighted sum.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one decode step's dispatch: 64 tokens, ten of 512 experts each; latency counts
        dict(name="sort-decode", op="sort", M=64, T=10, E=512, K=4096, dtype="bf16", local=512, train=False),
        # a long prompt's dispatch: 81920 rows of 8 KB
        dict(name="sort-prompt", op="sort", M=8192, T=10, E=512, K=4096, dtype="bf16", local=512, train=False),
        # a training step's dispatch in f32 at sizes that divide nothing
        dict(name="sort-train-odd", op="sort", M=3001, T=3, E=37, K=1021, dtype="f32", local=37, train=True),
        # one decode step's weighted sum
        dict(name="unsort-decode", op="unsort", M=64, T=10, E=512, K=4096, dtype="bf16", local=512, train=False),
        # a training step's weighted sum with the gradients of rows and weights
        dict(name="unsort-train", op="unsort", M=4096, T=10, E=512, K=4096, dtype="bf16", local=512, train=True),
        # the same on one of eight ranks: seven of eight pairs have their expert elsewhere
        dict(name="unsort-train-shard", op="unsort", M=6000, T=8, E=256, K=2048, dtype="fp16", local=32, train=True),
        # one token through a projection: weights are read once, nothing else counts
        dict(name="linear-token", op="linear", M=1, K=4096, N=2048, dtype="bf16", codes=False),
        # a decode batch
        dict(name="linear-decode", op="linear", M=48, K=4096, N=4096, dtype="bf16", codes=False),
        # ragged sizes, f32 out: rows of 1000 bytes, which are no multiple of 16
        dict(name="linear-odd", op="linear", M=333, K=1000, N=1235, dtype="f32", codes=True),
        # a prompt through a projection: bound by the tensor cores
        dict(name="linear-prompt", op="linear", M=8192, K=4096, N=4096, dtype="bf16", codes=False),
        # a decode step of the whole expert layer: the weights of about 360 experts are read once
        dict(name="experts-decode", op="experts", M=64, T=10, E=512, K=4096, N=1024, dtype="bf16"),
        # a prompt on one rank's 64 experts
        dict(name="experts-prompt", op="experts", M=2048, T=10, E=64, K=4096, N=1024, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sort", "unsort", "linear", "experts"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "f32"])
    if op in ("sort", "unsort"):
        E = _log(rng, 4, 512)
        T = rng.randint(1, min(E, 12))
        K = rng.choice([_log(rng, 64, 4096), 8 * _log(rng, 8, 512), 64 * _log(rng, 1, 64)])
        b = DTYPES[dtype].itemsize
        M = min(_log(rng, 1, 8192), (1 << 29) // (T * K * b) + 1)
        return dict(op=op, M=M, T=T, E=E, K=K, dtype=dtype, local=rng.choice([E, E, max(1, E // 8)]), train=rng.random() < 0.5)
    if op == "linear":
        K = rng.choice([_log(rng, 64, 4096), 16 * _log(rng, 4, 256)])
        N = rng.choice([_log(rng, 64, 4096), 16 * _log(rng, 4, 256)])
        return dict(op=op, M=_log(rng, 1, 8192), K=K, N=N, dtype=dtype, codes=rng.random() < 0.25)
    E = _log(rng, 4, 128)
    T = rng.randint(1, min(E, 10))
    return dict(op=op, M=_log(rng, 1, 2048), T=T, E=E, K=16 * _log(rng, 8, 256), N=16 * _log(rng, 4, 64), dtype=rng.choice(["bf16", "bf16", "fp16"]))


def _ids(g, M, T, E):
    """Distinct experts of each token, some of them more popular than others, and the weights of the choice."""
    popular = 0.5 * torch.randn(E, generator=g, device="cuda")
    logits = torch.randn(M, E, generator=g, device="cuda") + popular
    top, ids = torch.topk(logits, T, dim=1)
    return ids.int(), torch.softmax(top, dim=1)


def _rows(g, shape, dtype):
    """Activations: unit variance with a few strong channels."""
    x = torch.randn(shape, generator=g, device="cuda")
    x *= 1 + 7 * (torch.rand(shape[-1], generator=g, device="cuda") < 0.01)
    return x.to(DTYPES[dtype])


def _codes(g, shape):
    return torch.randint(-127, 128, shape, generator=g, device="cuda", dtype=torch.int8)


def _scales(g, shape, K):
    return (0.5 + torch.rand(shape, generator=g, device="cuda")) / (73.0 * math.sqrt(K))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    op, M, K, dtype = case["op"], case["M"], case["K"], case["dtype"]
    if op == "linear":
        N = case["N"]
        if case["codes"]:
            s["q"], s["qs"] = _codes(g, (M, K)), _scales(g, (M,), 1)
        else:
            s["x"] = _rows(g, (M, K), dtype)
        s["w"], s["ws"] = _codes(g, (N, K)), _scales(g, (N,), K)
        return s
    T, E = case["T"], case["E"]
    s["ids"], s["weights"] = _ids(g, M, T, E)
    if op == "experts":
        N = case["N"]
        s["x"] = _rows(g, (M, K), dtype)
        s["w13"], s["w13s"] = _codes(g, (E, 2 * N, K)), _scales(g, (E, 2 * N), K)
        s["w2"], s["w2s"] = _codes(g, (E, K, N)), _scales(g, (E, K), N)
        return s
    s["map"] = None
    if case["local"] < E:
        first = int(torch.randint(0, E - case["local"] + 1, (1,), generator=g, device="cuda"))
        at = torch.arange(E, device="cuda", dtype=torch.int32) - first
        s["map"] = torch.where((at >= 0) & (at < case["local"]), at, -1).int()
    if op == "sort":
        s["x"] = _rows(g, (M, K), dtype)
        s["grad"] = _rows(g, (M * T, K), dtype)
    else:
        s["x"] = _rows(g, (M * T, K), dtype)
        s["grad"] = _rows(g, (M, K), dtype)
    if case["train"]:
        s["x"].requires_grad_()
        if op == "unsort":
            s["weights"].requires_grad_()
    return s


# ---------------------------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------------------------
def _plan(ids, experts, expert_map):
    """Experts of the pairs in expert order (``experts`` = dropped), the pairs in that order, the row of each pair, offsets."""
    e = ids.reshape(-1).long()
    if expert_map is not None:
        e = expert_map.long()[e]
    e = torch.where(e < 0, experts, e)
    e, order = torch.sort(e, stable=True)
    row = torch.empty_like(order)
    row[order] = torch.arange(order.numel(), device=order.device)
    offsets = torch.searchsorted(e, torch.arange(experts + 1, device=e.device))
    return e, order, row, offsets


def _gather(rows, row, kept, M, T):
    """[M, T, K] rows of each token's pairs in 32 bits, zero where the pair was dropped."""
    r = rows.float()[row].reshape(M, T, -1)
    return torch.where(kept.reshape(M, T, 1), r, 0.0)


def _quantize(x):
    """Codes as f32 values, scales.  The quotient in 64 bits: a code next to a border between two moves otherwise."""
    x = x.double()
    amax = x.abs().amax(dim=-1, keepdim=True)
    q = torch.where(amax > 0, torch.round(127.0 * x / amax), 0.0)
    return q.float(), (amax / 127.0).float()


def _grouped(q, qs, w, ws, e, offsets):
    """Rows in expert order times their expert's weights: every expert's rows padded to the longest, one batched product."""
    at = torch.arange(e.numel(), device=e.device) - offsets[e]
    longest = int((offsets[1:] - offsets[:-1]).max())
    padded = torch.zeros(w.shape[0], longest, q.shape[1], device=q.device)
    padded[e, at] = q
    y = torch.bmm(padded, w.float().transpose(1, 2))
    return y[e, at] * qs * ws[e]


def _plain(s):
    op, M, K = s["op"], s["M"], s["K"]
    dtype = DTYPES[s["dtype"]]
    if op == "linear":
        q, qs = (s["q"].float(), s["qs"][:, None]) if s["codes"] else _quantize(s["x"])
        return {"y": ((q @ s["w"].float().T) * qs * s["ws"]).to(dtype)}
    T = s["T"]
    if op == "experts":
        N = s["N"]
        e, order, row, offsets = _plan(s["ids"], s["E"], None)
        q, qs = _quantize(s["x"])
        gu = _grouped(q[order // T], qs[order // T], s["w13"], s["w13s"], e, offsets)
        gate, up = gu[:, :N], gu[:, N:]
        hq, hs = _quantize(gate / (1 + torch.exp(-gate)) * up)
        y = _grouped(hq, hs, s["w2"], s["w2s"], e, offsets)
        return {"y": (y[row].reshape(M, T, K) * s["weights"][:, :, None]).sum(1).to(dtype)}
    e, order, row, offsets = _plan(s["ids"], s["local"], s["map"])
    kept_row, kept_pair = e < s["local"], (e < s["local"])[row]
    x, grad = s["x"].detach(), s["grad"]
    out = {"offsets": offsets.int()}
    if op == "sort":
        out["rows"] = torch.where(kept_row[:, None], x[order // T], 0.0)
        if s["train"]:
            out["dx"] = _gather(grad, row, kept_pair, M, T).sum(1).to(dtype)
        return out
    w = s["weights"].detach()
    rows = _gather(x, row, kept_pair, M, T)
    out["y"] = (rows * w[:, :, None]).sum(1).to(dtype)
    if s["train"]:
        wr = torch.where(kept_row, w.reshape(-1)[order], 0.0)
        out["drows"] = (grad.float()[order // T] * wr[:, None]).to(dtype)
        out["dw"] = (rows * grad.float()[:, None, :]).sum(2)
    return out


# ---------------------------------------------------------------------------------------------
# The framework's operators, as a program calls them
# ---------------------------------------------------------------------------------------------
def _framework(s):
    import sm120_moe_bench_b200 as vm

    op, dtype = s["op"], DTYPES[s["dtype"]]
    if op == "linear":
        w = vm.Int8Rows(s["w"], s["ws"])
        if s["codes"]:
            return {"y": vm.int8_matmul(vm.Int8Rows(s["q"], s["qs"]), w, out_dtype=dtype)}
        return {"y": vm.int8_linear(s["x"], w)}
    if op == "experts":
        return {"y": vm.int8_experts(s["x"], vm.Int8Rows(s["w13"], s["w13s"]), vm.Int8Rows(s["w2"], s["w2s"]),
                                     s["ids"], s["weights"])}
    plan = vm.plan_tokens(s["ids"], s["local"], s["map"])
    out = {"offsets": plan.expert_offsets}
    if op == "sort":
        out["rows"] = vm.sort_tokens(s["x"], plan)
        if s["train"]:
            out["dx"], = torch.autograd.grad(out["rows"], s["x"], s["grad"])
            out["rows"] = out["rows"].detach()
        return out
    out["y"] = vm.unsort_tokens(s["x"], plan, s["weights"])
    if s["train"]:
        out["drows"], out["dw"] = torch.autograd.grad(out["y"], (s["x"], s["weights"]), s["grad"])
        out["y"] = out["y"].detach()
    return out


def run(state):
    return _framework(state) if own else _plain(state)


def work(case):
    op, M, K = case["op"], case["M"], case["K"]
    b = DTYPES[case["dtype"]].itemsize
    if op == "linear":
        N = case["N"]
        rows = M * K + 4 * M if case["codes"] else M * K * b
        return {"bytes": rows + N * K + 4 * N + M * N * b, "flops": 2 * M * N * K}
    T, E = case["T"], case["E"]
    P = M * T
    if op == "experts":
        N = case["N"]
        used = E * (1 - (1 - T / E) ** M)     # experts that some token chose, were they equally popular
        return {"bytes": used * (3 * N * K + 4 * (2 * N + K)) + 2 * M * K * b + 8 * P, "flops": 6 * P * N * K}
    kept = P * case["local"] // E
    tables = 4 * P + 4 * (case["local"] + 1)
    if op == "sort":
        # rows that nobody owns are defined to be zero: they are written too
        n = M * K * b + P * K * b
        more = (kept + M) * K * b if case["train"] else 0
        return {"bytes": tables + n + more, "flops": kept * K if case["train"] else 0}
    n = (kept + M) * K * b + 4 * P
    more = (P + M) * K * b + 4 * P if case["train"] else 0
    return {"bytes": tables + n + more, "flops": (5 if case["train"] else 2) * kept * K}


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _quantize64(x):
    x = x.double()
    top = x.abs().max(dim=1).values
    step = top / 127
    codes = torch.zeros_like(x)
    some = top > 0
    codes[some] = torch.round(x[some] * 127 / top[some, None])
    return codes, step


def _places(experts, count):
    """For each pair its row in a list ordered by expert, then by pair; dropped pairs (-1) behind all others."""
    key = [(int(e) if e >= 0 else count, p) for p, e in enumerate(experts)]
    place = [0] * len(key)
    for r, (_, p) in enumerate(sorted(key)):
        place[p] = r
    return place


def exact(case, seed):
    s = prepare(case, seed)
    op, M, K = case["op"], case["M"], case["K"]
    if op == "linear":
        a, sa = (s["q"].double(), s["qs"].double()) if case["codes"] else _quantize64(s["x"])
        return {"y": torch.einsum("mk,nk->mn", a, s["w"].double()) * sa[:, None] * s["ws"].double()[None]}
    T, E = case["T"], case["E"]
    if op == "experts":
        N = case["N"]
        if 6 * M * T * N * K > 6e14:
            return None
        a, sa = _quantize64(s["x"])
        ids, w = s["ids"].long(), s["weights"].double()
        y = torch.zeros(M, K, dtype=torch.float64, device="cuda")
        for expert in torch.unique(ids).tolist():
            token, slot = torch.nonzero(ids == expert, as_tuple=True)
            gu = (a[token] @ s["w13"][expert].double().T) * sa[token, None] * s["w13s"][expert].double()
            h, sh = _quantize64(gu[:, :N] * torch.sigmoid(gu[:, :N]) * gu[:, N:])
            d = (h @ s["w2"][expert].double().T) * sh[:, None] * s["w2s"][expert].double()
            y.index_add_(0, token, d * w[token, slot][:, None])
        return {"y": y}
    expert = s["ids"].long() if s["map"] is None else s["map"].long()[s["ids"].long()]
    place = torch.tensor(_places(expert.reshape(-1).tolist(), case["local"]), device="cuda").reshape(M, T)
    kept = (expert >= 0).double()[:, :, None]
    x, grad = s["x"].detach(), s["grad"]
    out = {"offsets": None}
    if op == "sort":
        rows = torch.zeros(M * T, K, dtype=torch.float64, device="cuda")
        dx = torch.zeros(M, K, dtype=torch.float64, device="cuda")
        for t in range(T):
            rows[place[:, t]] = x.double() * kept[:, t]
            if case["train"]:
                dx += grad[place[:, t]].double() * kept[:, t]
        out["rows"] = rows
        if case["train"]:
            out["dx"] = dx
        return out
    w = s["weights"].detach().double()
    y = torch.zeros(M, K, dtype=torch.float64, device="cuda")
    for t in range(T):
        y += x[place[:, t]].double() * kept[:, t] * w[:, t, None]
    out["y"] = y
    if case["train"]:
        drows = torch.zeros(M * T, K, dtype=torch.float64, device="cuda")
        dw = torch.zeros(M, T, dtype=torch.float64, device="cuda")
        for t in range(T):
            drows[place[:, t]] = grad.double() * kept[:, t] * w[:, t, None]
            dw[:, t] = (x[place[:, t]].double() * kept[:, t] * grad.double()).sum(1)
        out["drows"], out["dw"] = drows, dw
    return out
