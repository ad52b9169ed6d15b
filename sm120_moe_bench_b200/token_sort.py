"""Token rows sorted by expert and back, with the router's weights applied; both directions are differentiable.

    plan = plan_tokens(topk_ids, num_experts)            # once per batch
    rows = sort_tokens(hidden, plan)                     # [M * T, K], the rows of expert e at plan.expert_offsets[e]
    ...                                                  # the experts' own work on the rows
    out = unsort_tokens(rows, plan, topk_weights)        # [M, K] = sum over a token's rows of weight * row

Rows are bf16, fp16 or f32 with any row stride (elements of a row next to each other).  Sums run in f32 over a token's
choices in order and are rounded once; nothing depends on the order in which blocks run.  Dropped pairs (ids outside the
experts, or not local under an ``expert_map``) take part in nothing: they have no row, add nothing to a sum, and their
weights get a zero gradient.  They leave ``M * T - kept`` rows behind the last kept one; these are zero in every tensor
made here (rows and gradients) and left as they were in a tensor given as ``out``, which must not share memory with an operand.

A backward pass is captured into a CUDA graph together with its forward pass.  An eager graph of the same leaf tensor has
to be gone by then (a leaf's accumulator stays bound to the stream of the graph that made it, which the capture must not
wait for): with one of these operators' graphs still alive the captured call raises.  Derivatives are reverse-mode: a tensor
that carries a forward-mode tangent is refused.  So is recording a call with torch.jit.trace or make_fx; torch.compile runs it
as it is.
"""
from __future__ import annotations

import threading
import weakref

import torch
from torch.autograd import forward_ad

from ._lib import check, lib

DTYPE_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
MAX_TOPK = 16
MAX_ROWS = 2 ** 31 - 1025    # sizes travel as int32
MAX_EXPERTS = 8192
ONE_CTA_PAIRS = 4096      # up to here the plan needs no scratch (vmoe_plan_scratch_bytes is 0)


# The driver-level handle of a device's current stream and the current device's index, without the wrapper objects that
# torch.cuda.current_stream() makes (6 of a small call's 15 microseconds on the host).
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


_tracing, _dispatch_modes, _function_modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack, torch._C._len_torch_function_stack


def traced() -> bool:
    """Whether torch.jit.trace or make_fx records what runs now.  They see torch's own operators, not a kernel launched
    beside them: the recorded program would hold the allocations and return them as they are."""
    from torch.fx.experimental.proxy_tensor import get_proxy_mode
    return _tracing() or get_proxy_mode() is not None


# A tensor given as out is changed behind autograd's back: its version tells the graphs that saved it.
changed = torch.autograd.graph.increment_version


def launch(device: torch.device, name: str, fn, *args) -> None:
    """Call a C entry point on the device of its tensors, on that device's current stream."""
    # (make_fx pushes a mode of either kind; looking for them takes 0.15 us)
    if _tracing() or ((_dispatch_modes() or _function_modes()) and traced()):
        raise RuntimeError(f"{name}: a kernel of this library cannot be traced (its launch would be missing from the recorded program)")
    index = device.index
    if index == _current_device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        check(status, name)


def check_rows(t: torch.Tensor, name: str, rows: int | None = None, device: torch.device | None = None) -> torch.Tensor:
    """``t`` as a matrix of rows the kernels can read: 2-D, on the device, elements of a row next to each other."""
    if t.is_cuda and t.dtype in DTYPE_CODES and t.dim() == 2:
        n, k = t.shape
        if (rows is None or n == rows) and (device is None or t.device == device) and (k <= 1 or t.stride(1) == 1) \
                and n <= MAX_ROWS and k <= MAX_ROWS:
            return t
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype not in DTYPE_CODES:
        raise ValueError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name} must have two dimensions, got {t.dim()}")
    if rows is not None and t.shape[0] != rows:
        raise ValueError(f"{name} must have {rows} rows, got {t.shape[0]}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected on {device}")
    if t.shape[0] > MAX_ROWS or t.shape[1] > MAX_ROWS:
        raise ValueError(f"{name} has a dimension of more than {MAX_ROWS}")
    raise ValueError(f"the elements of a row of {name} must lie next to each other")


def has_tangent(*tensors: torch.Tensor | None) -> bool:
    """Whether one of them carries a forward-mode derivative: ``requires_grad`` does not tell, and the kernels would drop it."""
    return forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _refuse_tangent(*tensors: torch.Tensor | None) -> None:
    if has_tangent(*tensors):
        raise NotImplementedError("the token sort has no forward-mode derivatives, only reverse-mode ones")


def overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the two share memory; columns of one buffer that lie side by side do not.  Where row pitches differ and the
    byte ranges meet, yes."""
    def span(t):
        return t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))

    if a.numel() == 0 or b.numel() == 0:
        return False
    x, y = a.data_ptr(), b.data_ptr()
    if x + span(a) <= y or y + span(b) <= x:
        return False
    if a.dim() == b.dim() == 2:
        pitch = a.stride(0) * a.element_size()
        if pitch > 0 and pitch == b.stride(0) * b.element_size():
            wa, wb = (span(t[:1]) for t in (a, b))
            at = (y - x) % pitch
            return at < wa or at + wb > pitch
    return True


def refuse_overlap(out: torch.Tensor, plan: "TokenPlan | None" = None, **operands: torch.Tensor | None) -> None:
    """The kernels read their operands and write ``out`` in no order."""
    if plan is not None:
        operands["the plan"] = plan._buf if plan._buf is not None else plan.row_of_pair
        if plan._buf is None:
            operands["the plan's offsets"] = plan.expert_offsets
    for name, t in operands.items():
        if t is not None and overlap(out, t):
            raise ValueError(f"out shares memory with {name}")


def check_out(out: torch.Tensor, rows: int, like: torch.Tensor) -> torch.Tensor:
    check_rows(out, "out", rows, like.device)
    if out.dtype != like.dtype or out.shape[1] != like.shape[1]:
        raise ValueError(f"out must be {like.dtype} with {like.shape[1]} columns")
    if rows > 1 and out.stride(0) < out.shape[1]:
        raise ValueError("the rows of out must not overlap")
    return out


class TokenPlan:
    """Which row each (token, choice) pair has.  Made by ``plan_tokens``; the tensors stay on the device.

    ``expert_offsets`` int32 ``[E + 1]``: rows of expert e are ``expert_offsets[e] .. expert_offsets[e + 1] - 1``;
    ``row_of_pair`` int32 ``[M, T]``, -1 = dropped; ``pair_of_row`` int32 ``[M * T]``, -1 behind the last kept row."""

    __slots__ = ("tokens", "topk", "rows", "num_experts", "device", "_buf", "_offsets", "_rows", "_pairs", "_offsets_ptr", "_rows_ptr")

    def __init__(self, expert_offsets: torch.Tensor, row_of_pair: torch.Tensor, pair_of_row: torch.Tensor, num_experts: int):
        self.tokens, self.topk = row_of_pair.shape
        self.rows = self.tokens * self.topk
        self.num_experts = num_experts
        self.device = row_of_pair.device
        for t, n, name in ((expert_offsets, num_experts + 1, "expert_offsets"), (row_of_pair, self.rows, "row_of_pair"),
                           (pair_of_row, self.rows, "pair_of_row")):
            if t.dtype != torch.int32 or t.numel() != n or not t.is_contiguous() or t.device != self.device:
                raise ValueError(f"{name} must be a contiguous int32 tensor of {n} elements, on the device of the others")
        self._buf, self._offsets, self._rows, self._pairs = None, expert_offsets, row_of_pair, pair_of_row
        self._offsets_ptr, self._rows_ptr = expert_offsets.data_ptr(), row_of_pair.data_ptr()

    @classmethod
    def _over(cls, buf: torch.Tensor, tokens: int, topk: int, num_experts: int) -> "TokenPlan":
        """The three tables one behind another in ``buf``; views of them are made when they are asked for."""
        self = cls.__new__(cls)
        self.tokens, self.topk, self.rows, self.num_experts, self.device = tokens, topk, tokens * topk, num_experts, buf.device
        self._buf, self._offsets, self._rows, self._pairs = buf, None, None, None
        self._offsets_ptr = buf.data_ptr()
        self._rows_ptr = self._offsets_ptr + 4 * (num_experts + 1)
        return self

    def __reduce__(self):              # copies and pickles carry the tables, never the addresses
        return TokenPlan, (self.expert_offsets, self.row_of_pair, self.pair_of_row, self.num_experts)

    def record_stream(self, stream: torch.cuda.Stream) -> None:
        """As ``Tensor.record_stream``: for a plan that is used on another stream than the one it was made on."""
        for t in (self._buf,) if self._buf is not None else (self._offsets, self._rows, self._pairs):
            t.record_stream(stream)

    @property
    def expert_offsets(self) -> torch.Tensor:
        if self._offsets is None:
            self._offsets = self._buf[:self.num_experts + 1]
        return self._offsets

    @property
    def row_of_pair(self) -> torch.Tensor:
        if self._rows is None:
            at = self.num_experts + 1
            self._rows = self._buf[at:at + self.rows].view(self.tokens, self.topk)
        return self._rows

    @property
    def pair_of_row(self) -> torch.Tensor:
        if self._pairs is None:
            at = self.num_experts + 1 + self.rows
            self._pairs = self._buf[at:at + self.rows]
        return self._pairs


def plan_tokens(topk_ids: torch.Tensor, num_experts: int, expert_map: torch.Tensor | None = None) -> TokenPlan:
    """Tables of the stable sort of the ``[M, T]`` int32 expert ids by expert (one launch up to 4096 pairs, else two).

    With ``expert_map`` (int32, -1 = not local) the ids are global and ``num_experts`` counts the local ones.  Ids outside
    the map, or outside ``[0, num_experts)``, drop their pair.  ``T <= 16``, ``num_experts <= 8192``."""
    if not topk_ids.is_cuda:
        raise ValueError("topk_ids must be a CUDA tensor")
    if topk_ids.dtype != torch.int32 or topk_ids.dim() != 2:
        raise ValueError("topk_ids must be an int32 tensor [tokens, choices]")
    if not topk_ids.is_contiguous():
        raise ValueError("topk_ids must be contiguous")
    M, T = topk_ids.shape
    if not 1 <= T <= MAX_TOPK:
        raise ValueError(f"1 to {MAX_TOPK} choices per token, got {T}")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_EXPERTS} experts, got {num_experts}")
    if M * T > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} pairs, got {M * T}")
    dev = topk_ids.device
    if expert_map is not None:
        if expert_map.device != dev or expert_map.dtype != torch.int32 or expert_map.dim() != 1 or not expert_map.is_contiguous():
            raise ValueError("expert_map must be a contiguous int32 vector on the device of topk_ids")
        if expert_map.numel() == 0:
            raise ValueError("expert_map is empty")
    P = M * T
    need = 0 if P <= ONE_CTA_PAIRS else lib.vmoe_plan_scratch_bytes(M, T, num_experts)
    buf = topk_ids.new_empty(num_experts + 1 + 2 * P + need // 4)
    plan = TokenPlan._over(buf, M, T, num_experts)
    rows = plan._rows_ptr
    launch(dev, "vmoe_plan_tokens", lib.vmoe_plan_tokens, topk_ids.data_ptr(), None if expert_map is None else expert_map.data_ptr(),
           0 if expert_map is None else expert_map.numel(), M, T, num_experts, plan._offsets_ptr, rows, rows + 4 * P,
           rows + 8 * P if need else None, need)
    return plan


def _sort(x, plan: TokenPlan, out=None):
    K = x.shape[1]
    rows, stride = (x.new_empty((plan.rows, K)), K) if out is None else (out, max(out.stride(0), K))
    launch(plan.device, "vmoe_sort_tokens", lib.vmoe_sort_tokens, x.data_ptr(), x.stride(0), DTYPE_CODES[x.dtype], plan.tokens, plan.topk,
           plan.num_experts, K, plan._offsets_ptr, plan._rows_ptr, out is None, rows.data_ptr(),
           stride)
    return rows


def _unsort(rows, plan: TokenPlan, weights=None, out=None):
    K = rows.shape[1]
    y, stride = (rows.new_empty((plan.tokens, K)), K) if out is None else (out, max(out.stride(0), K))
    launch(plan.device, "vmoe_unsort_tokens", lib.vmoe_unsort_tokens, rows.data_ptr(), rows.stride(0), DTYPE_CODES[rows.dtype],
           plan.tokens, plan.topk, K, plan._rows_ptr, None if weights is None else weights.data_ptr(), y.data_ptr(),
           stride, DTYPE_CODES[rows.dtype])
    return y


def _dense_rows(g: torch.Tensor) -> torch.Tensor:
    """A gradient as torch hands it over may be expanded along its columns (the gradient of a sum)."""
    return g if g.shape[1] <= 1 or g.stride(1) == 1 else g.contiguous()


_capturing = torch._C._cuda_isCurrentStreamCapturing
_eager_graphs = weakref.WeakSet()      # nodes of live eager graphs; each knows its leaves (weakly)
_eager_lock = threading.Lock()


def _note_graph(ctx, *tensors: torch.Tensor | None) -> None:
    """Remembers an eager graph while it lives, and refuses to capture one of a leaf that has another alive."""
    leaves = [weakref.ref(t) for t in tensors if t is not None and t.requires_grad and t.is_leaf]
    if not leaves:
        return
    if not _capturing():
        ctx.leaves = leaves
        with _eager_lock:
            _eager_graphs.add(ctx)
        return
    with _eager_lock:
        others = [r() for g in _eager_graphs for r in g.leaves]
    if any(o is not None and o is r() for o in others for r in leaves):
        raise RuntimeError("an eager graph of this leaf tensor is still alive (an output of it is held): drop it before capturing a graph "
                           "that differentiates the leaf again")


class _SortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, plan):
        _note_graph(ctx, x)
        ctx.plan = plan
        return _sort(x, plan)

    @staticmethod
    def backward(ctx, grad):
        if forward_ad._current_level >= 0:
            _refuse_tangent(grad)
        grad = _dense_rows(grad)
        # with create_graph the gradient is differentiable itself
        return (unsort_tokens if torch.is_grad_enabled() else _unsort)(grad, ctx.plan), None


def _unsort_backward(ctx, grad):
    if forward_ad._current_level >= 0:
        _refuse_tangent(grad)
    rows, weights = ctx.saved_tensors
    want_rows, _, want_weights = ctx.needs_input_grad
    plan, grad = ctx.plan, _dense_rows(grad)
    M, T, K = plan.tokens, plan.topk, grad.shape[1]
    drows = grad.new_empty((plan.rows, K)) if want_rows else None
    dw = torch.empty((M, T), dtype=torch.float32, device=plan.device) if want_weights else None
    launch(plan.device, "vmoe_unsort_tokens_grad", lib.vmoe_unsort_tokens_grad, grad.data_ptr(), grad.stride(0),
           None if dw is None else rows.data_ptr(), 0 if dw is None else rows.stride(0), DTYPE_CODES[grad.dtype], M, T,
           plan.num_experts, K, plan._offsets_ptr, plan._rows_ptr,
           None if weights is None else weights.data_ptr(), None if drows is None else drows.data_ptr(), K,
           None if dw is None else dw.data_ptr())
    return drows, None, dw


_unsort_backward_once = torch.autograd.function.once_differentiable(_unsort_backward)


class _UnsortTokens(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, plan, weights):
        _note_graph(ctx, rows, weights)
        ctx.plan = plan
        ctx.save_for_backward(rows if ctx.needs_input_grad[2] else None, weights)      # rows: the weights' gradient alone
        return _unsort(rows, plan, weights)

    @staticmethod
    def backward(ctx, grad):
        # once_differentiable only matters, and only costs, where a graph of the gradient is asked for
        return (_unsort_backward_once if torch.is_grad_enabled() else _unsort_backward)(ctx, grad)


def sort_tokens(x: torch.Tensor, plan: TokenPlan, out: torch.Tensor | None = None) -> torch.Tensor:
    """``rows[r] = x[token of row r]``: the token rows ``[M, K]`` in expert order, ``[M * T, K]``.  Differentiable in ``x``
    (a token's gradient is the sum over its rows) unless ``out`` is given."""
    check_rows(x, "x", plan.tokens, plan.device)
    if forward_ad._current_level >= 0:
        _refuse_tangent(x, out)
    if out is not None:
        if torch.is_grad_enabled() and (x.requires_grad or out.requires_grad):
            raise ValueError("out cannot be given where a gradient is wanted")
        refuse_overlap(check_out(out, plan.rows, x), plan, x=x)
        _sort(x, plan, out)
        changed(out)
        return out
    if x.requires_grad and torch.is_grad_enabled():
        return _SortTokens.apply(x, plan)
    return _sort(x, plan)


def unsort_tokens(rows: torch.Tensor, plan: TokenPlan, weights: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``out[m] = sum_t weights[m, t] * rows[row of (m, t)]``: rows ``[M * T, K]`` in expert order back to tokens ``[M, K]``.
    ``weights`` f32 ``[M, T]`` (None = 1).  Differentiable in ``rows`` and ``weights`` unless ``out`` is given."""
    check_rows(rows, "rows", plan.rows, plan.device)
    if forward_ad._current_level >= 0:
        _refuse_tangent(rows, weights, out)
    if weights is not None:
        if weights.device != rows.device or weights.dtype != torch.float32 or weights.shape != (plan.tokens, plan.topk):
            raise ValueError(f"weights must be a float32 tensor [{plan.tokens}, {plan.topk}] on the device of rows")
        if not weights.is_contiguous():
            raise ValueError("weights must be contiguous")
    grad = torch.is_grad_enabled() and (rows.requires_grad or (weights is not None and weights.requires_grad))
    if out is not None:
        if grad or (torch.is_grad_enabled() and out.requires_grad):
            raise ValueError("out cannot be given where a gradient is wanted")
        refuse_overlap(check_out(out, plan.tokens, rows), plan, rows=rows, weights=weights)
        _unsort(rows, plan, weights, out)
        changed(out)
        return out
    if grad:
        return _UnsortTokens.apply(rows, plan, weights)
    return _unsort(rows, plan, weights)
