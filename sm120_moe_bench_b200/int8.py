"""8-bit integer products with a scale for each token and each output channel, dense and per expert.

    w = quantize_int8(weight)                            # once: codes [N, K] and a scale per output channel
    y = int8_linear(x, w)                                # quantises the rows of x, multiplies

    w13, w2 = quantize_int8(gate_up), quantize_int8(down)    # [E, 2N, K] (gate rows first) and [E, K, N]
    y = int8_experts(x, w13, w2, topk_ids, topk_weights)     # the whole expert layer

The integer sums are exact, the scales are applied in f32 and the result is rounded once; a result does not depend on the
batch around it.  These are inference operators: they have no gradient, and floating tensors that require one are refused
while gradients are enabled, as are those that carry a forward-mode tangent.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from ._lib import check, lib
from .token_sort import DTYPE_CODES, MAX_EXPERTS, MAX_ROWS, MAX_TOPK, TokenPlan, changed, check_out, check_rows, has_tangent, launch, refuse_overlap

MAX_K = 131071
TIMEOUT = 6               # VMOE_ERR_TIMEOUT


class Int8Rows:
    """Rows of 8-bit codes ``q`` int8 ``[..., rows, K]`` and a scale each, ``scale`` f32 ``[..., rows]``: row = q * scale.

    A row's codes lie next to each other; rows (and the matrices of several experts) may have any stride.  Where address
    and strides are multiples of 16 bytes the tensor cores read them as they are; ``quantize_int8`` makes them so."""

    __slots__ = ("q", "scale")

    def __init__(self, q: torch.Tensor, scale: torch.Tensor):
        shape = q.shape
        if not q.is_cuda or q.dtype != torch.int8 or len(shape) not in (2, 3):
            raise ValueError("q must be an int8 CUDA tensor [rows, K] or [experts, rows, K]")
        if scale.dtype != torch.float32 or scale.device != q.device or scale.shape != shape[:-1] or not scale.is_contiguous():
            raise ValueError("scale must be a contiguous float32 tensor, one value for each row of q, on its device")
        K = shape[-1]
        if K > 1 and q.stride(-1) != 1:
            raise ValueError("the codes of a row must lie next to each other")
        if K > MAX_K:
            raise ValueError(f"rows of at most {MAX_K} codes")
        if shape[-2] > MAX_ROWS:
            raise ValueError(f"at most {MAX_ROWS} rows")
        self.q = q
        self.scale = scale

    def dequantize(self) -> torch.Tensor:
        """f32 values."""
        return self.q.float() * self.scale[..., None]


def _no_grad(**tensors: torch.Tensor) -> None:
    for name, t in tensors.items():
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient: the 8-bit operators have none")
        if has_tangent(t):
            raise ValueError(f"{name} carries a forward-mode derivative: the 8-bit operators have none")


def _codes(rows: int, K: int, device) -> torch.Tensor:
    """Rows that start on 16-byte boundaries, whatever K is."""
    pitch = (K + 15) // 16 * 16
    q = torch.empty(rows, pitch, dtype=torch.int8, device=device)
    return q if pitch == K else q[:, :K]


def _quantize(x, plan: TokenPlan | None = None):
    M, K = x.shape
    rows = M if plan is None else plan.rows
    q = _codes(rows, K, x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    launch(x.device, "vmoe_int8_quantize", lib.vmoe_int8_quantize, x.data_ptr(), x.stride(0), DTYPE_CODES[x.dtype], M, K,
           0 if plan is None else plan.topk, None if plan is None else plan._rows_ptr, None, q.data_ptr(),
           max(q.stride(0), K), scale.data_ptr())
    return q, scale


def quantize_int8(x: torch.Tensor, plan: TokenPlan | None = None) -> Int8Rows:
    """bf16 / fp16 / f32 rows to 8-bit rows: ``scale = max|row| / 127``, codes = the exact ``127 * x / max|row|`` rounded to the
    nearest integer (ties to even).  A row of zeros has scale 0; a row with an infinity or NaN has scale NaN, so that what
    it is multiplied with becomes NaN.

    ``x`` is ``[rows, K]``, or ``[E, rows, K]`` contiguous for the weights of several experts.  With ``plan`` the rows of ``x``
    are tokens and the codes come sorted by expert, ``[M * T, K]`` (rows behind the last kept one are undefined)."""
    if x.requires_grad or forward_ad._current_level >= 0:
        _no_grad(x=x)
    if x.dim() == 3:
        if plan is not None:
            raise ValueError("a plan sorts token rows [M, K]")
        if not x.is_contiguous():
            raise ValueError("x must be contiguous")
        E, N, K = x.shape
        flat = quantize_int8(x.view(E * N, K))
        return Int8Rows(flat.q.as_strided((E, N, K), (N * flat.q.stride(0), flat.q.stride(0), 1)), flat.scale.view(E, N))
    check_rows(x, "x", None if plan is None else plan.tokens, None if plan is None else plan.device)
    if x.shape[1] > MAX_K:
        raise ValueError(f"rows of at most {MAX_K} elements")
    return Int8Rows(*_quantize(x, plan))


def _aligned(q: torch.Tensor) -> bool:
    """Whether the tensor cores can read these matrices as they are."""
    return (q.data_ptr() | q.stride(1) | q.stride(0)) % 16 == 0


def _one_launch(rows: int, n: int, k: int, address: int, stride: int) -> bool:
    """Whether a dense product of this many rows with weights ``[n, k]`` is done in one launch, without scratch."""
    if rows > 8:
        return False
    odd = (address | stride) & 15
    if rows <= 4 and n <= 8192 and 0 < k <= 8192 and stride >= k and n * k <= (1 << 21 if odd else 1 << 24):
        return True                                       # the C side says so too; asking costs half a microsecond
    return (n == 1 or stride >= k) and lib.vmoe_int8_one_launch(rows, n, k, 16 | odd) == 1


def _packs(q: torch.Tensor, rows: int) -> bool:
    """Whether unaligned matrices of several experts are worth a copy for a product with this many rows: not below one row per
    matrix, since the copy reads every matrix."""
    return rows >= q.shape[0]


def int8_status(device: torch.device | str | int = "cuda") -> int:
    """0, or the status of a bounded wait that ran out inside an 8-bit product on this device since the last call (6 = time-out,
    as ``Workspace.status``).  Waits for the current stream, so not while it is captured."""
    with torch.cuda.device(device):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("int8_status waits for the stream, which a capture does not allow")
        status = lib.vmoe_int8_read_status(torch.cuda.current_stream().cuda_stream)
    if status not in (0, TIMEOUT):
        check(status, "vmoe_int8_read_status")
    return status


def _out_columns(w: Int8Rows, K: int, device, swiglu: bool, experts: int | None) -> int:
    q = w.q
    shape = q.shape
    if q.device != device:
        raise ValueError(f"the weights are on {q.device}, the rows on {device}")
    if len(shape) != (2 if experts is None else 3):
        raise ValueError("weights of several experts go with a plan, a single matrix goes without")
    if experts is not None and shape[0] != experts:
        raise ValueError(f"the plan has {experts} experts, the weights {shape[0]}")
    if shape[-1] != K:
        raise ValueError(f"rows of {K} codes times weights of {shape[-1]}")
    n = shape[-2]
    if swiglu and n % 2:
        raise ValueError("swiglu needs gate and up rows")
    if n == 0:
        raise ValueError("the weights have no rows")
    return n // 2 if swiglu else n


def int8_matmul(a: Int8Rows, w: Int8Rows, plan: TokenPlan | None = None, *, swiglu: bool = False,
                out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """``out[m, n] = (a.q[m] . w.q[n]) * a.scale[m] * w.scale[n]``.

    With ``plan`` the rows are sorted by expert (``quantize_int8(x, plan)``) and each meets its expert's matrix of ``w``
    ``[E, N, K]``; rows behind the last kept one are zero (left as they were in a tensor given as ``out``, which must not share
    memory with an operand).  ``swiglu``: ``w`` holds gate rows and up rows (``[2N, K]``) and the result is ``silu(gate) * up``,
    ``[M, N]``."""
    if a.scale.requires_grad or w.scale.requires_grad or forward_ad._current_level >= 0:
        _no_grad(**{"a.scale": a.scale, "w.scale": w.scale})
    aq, wq = a.q, w.q
    if aq.dim() != 2:
        raise ValueError("a must be rows [M, K]")
    (M, K), device = aq.shape, aq.device
    if plan is not None and (M != plan.rows or plan.device != device):
        raise ValueError(f"the plan has {plan.rows} rows on {plan.device}, a {M} on {device}")
    N = _out_columns(w, K, device, swiglu, None if plan is None else plan.num_experts)
    if out is None:
        if out_dtype not in DTYPE_CODES:
            raise ValueError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
        y = torch.empty(M, N, dtype=out_dtype, device=device)
    else:
        y = check_out(out, M, out)
        if out.device != device or out.shape[1] != N:
            raise ValueError(f"out must have {N} columns on {device}")
        _no_grad(out=out)
        refuse_overlap(out, plan, **{"a": aq, "a's scales": a.scale, "w": wq, "w's scales": w.scale})
    E = 1 if plan is None else plan.num_experts
    need, channels, a_at, a_pitch, w_at, w_pitch = 0, 2 * N if swiglu else N, aq.data_ptr(), aq.stride(0), wq.data_ptr(), wq.stride(-2)
    each = 0 if plan is None else wq.stride(0)
    # unaligned operands are copied where that pays (figures at the C side's i8_product_any and i8_few_rows)
    if (a_at | a_pitch | w_at | w_pitch | each) & 15 and (_packs(wq, M) if plan is not None else not _one_launch(M, channels, K, w_at, w_pitch)):
        need = lib.vmoe_int8_pack_bytes(M, channels, K, E)
    scratch = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    launch(device, "vmoe_int8_matmul", lib.vmoe_int8_matmul, a_at, a_pitch, a.scale.data_ptr(), M, w_at,
           w_pitch, each, w.scale.data_ptr(), N, K, E, None if plan is None else plan._offsets_ptr,
           swiglu, out is None, y.data_ptr(), max(y.stride(0), N), DTYPE_CODES[y.dtype], scratch.data_ptr() if need else None, need)
    if out is not None:
        changed(out)
    return y


def int8_linear(x: torch.Tensor, w: Int8Rows, *, swiglu: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x [M, K]`` (bf16 / fp16 / f32) quantised row by row, times ``w [N, K]``: ``[M, N]`` in the type of ``x``.
    ``out`` must not share memory with ``x`` or ``w``."""
    if x.requires_grad or w.scale.requires_grad or forward_ad._current_level >= 0:
        _no_grad(**{"x": x, "w.scale": w.scale})
    check_rows(x, "x")
    (M, K), device, wq = x.shape, x.device, w.q
    N = _out_columns(w, K, device, swiglu, None)
    stride = N
    given = out is not None
    if not given:
        out = x.new_empty((M, N))
    else:
        stride = max(out.stride(0), N)
        check_rows(out, "out", M, device)
        if out.dtype != x.dtype or out.shape[1] != N or (M > 1 and out.stride(0) < N):
            raise ValueError(f"out must be {x.dtype} with {N} columns and rows that do not overlap")
        _no_grad(out=out)
        refuse_overlap(out, x=x, **{"w": wq, "w's scales": w.scale})
    need, address, pitch, channels = 0, wq.data_ptr(), wq.stride(0), 2 * N if swiglu else N
    if not _one_launch(M, channels, K, address, pitch):   # else the rows are quantised inside the product
        need = lib.vmoe_int8_linear_scratch_bytes(M, K)
        if (address | pitch) & 15:
            need += lib.vmoe_int8_pack_bytes(M, channels, K, 1)
    scratch = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    launch(device, "vmoe_int8_linear", lib.vmoe_int8_linear, x.data_ptr(), x.stride(0), DTYPE_CODES[x.dtype], M, address,
           pitch, w.scale.data_ptr(), N, K, swiglu, out.data_ptr(), stride, DTYPE_CODES[out.dtype],
           scratch.data_ptr() if need else None, need)
    if given:
        changed(out)
    return out


def int8_experts(x: torch.Tensor, w13: Int8Rows, w2: Int8Rows, topk_ids: torch.Tensor, topk_weights: torch.Tensor,
                 expert_map: torch.Tensor | None = None) -> torch.Tensor:
    """The expert layer on 8-bit weights: ``out[m] = sum_t weight[m, t] * w2[e] (silu(gate) * up)``, ``[gate; up] = w13[e] x[m]``.

    ``x [M, K]`` bf16 / fp16 / f32; ``w13 [E, 2N, K]`` (gate rows first); ``w2 [E, K, N]``; ids int32 and weights f32 ``[M, T]``.
    Tokens are quantised once and copied into expert order, the activations between the two products once more per row;
    everything between is f32, and the sum is rounded once to the type of ``x``.  ``expert_map`` as in ``plan_tokens``."""
    if x.requires_grad or topk_weights.requires_grad or w13.scale.requires_grad or w2.scale.requires_grad or forward_ad._current_level >= 0:
        _no_grad(**{"x": x, "topk_weights": topk_weights, "w13.scale": w13.scale, "w2.scale": w2.scale})
    if topk_ids.dim() != 2:
        raise ValueError("topk_ids must be an int32 tensor [tokens, choices]")
    check_rows(x, "x", topk_ids.shape[0], topk_ids.device)
    if w13.q.dim() != 3 or w2.q.dim() != 3:
        raise ValueError("w13 and w2 hold one matrix per expert")
    E, K = w13.q.shape[0], x.shape[1]
    N = _out_columns(w13, K, x.device, True, E)
    if _out_columns(w2, N, x.device, False, E) != K:
        raise ValueError(f"w2 must be [{E}, {K}, {N}]")
    if topk_weights.dtype != torch.float32 or topk_weights.shape != topk_ids.shape or topk_weights.device != x.device \
            or not topk_weights.is_contiguous():
        raise ValueError("topk_weights must be a contiguous float32 tensor of the shape of topk_ids")
    if topk_ids.dtype != torch.int32 or not topk_ids.is_contiguous():
        raise ValueError("topk_ids must be a contiguous int32 tensor [tokens, choices]")
    M, T = topk_ids.shape
    if not 1 <= T <= MAX_TOPK or E > MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_TOPK} choices per token and at most {MAX_EXPERTS} experts, got {T} and {E}")
    if expert_map is not None and (expert_map.device != x.device or expert_map.dtype != torch.int32 or expert_map.dim() != 1
                                   or not expert_map.is_contiguous() or expert_map.numel() == 0):
        raise ValueError("expert_map must be a contiguous int32 vector on the device of topk_ids, not empty")
    q13, q2 = w13.q, w2.q
    pack = not (_aligned(q13) and _aligned(q2)) and _packs(q13, M * T)
    out = x.new_empty((M, K))
    need = lib.vmoe_int8_experts_scratch_bytes(M, T, E, K, N, pack)
    scratch = torch.empty(need, dtype=torch.uint8, device=x.device)
    launch(x.device, "vmoe_int8_experts", lib.vmoe_int8_experts, x.data_ptr(), x.stride(0), DTYPE_CODES[x.dtype], M, T, E, K, N,
           topk_ids.data_ptr(), topk_weights.data_ptr(), None if expert_map is None else expert_map.data_ptr(),
           0 if expert_map is None else expert_map.numel(), q13.data_ptr(), q13.stride(1), q13.stride(0), w13.scale.data_ptr(),
           q2.data_ptr(), q2.stride(1), q2.stride(0), w2.scale.data_ptr(), out.data_ptr(), K, DTYPE_CODES[out.dtype], scratch.data_ptr(),
           need)
    return out
