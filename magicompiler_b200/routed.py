"""Row movements of a routed (mixture-of-experts) SwiGLU block: tokens sorted by expert, gathered into expert order and
added up again with the router's weights, each with its gradient, and the fp8 quantiser with one scale per 128 columns.

    row_slot, slot_row, offsets = expert_sort(expert_ids, E)      # expert_ids [T, k]; R = T * k slots
    xs = expert_gather(x, row_slot, slot_row)                     # [T, H] -> [R, H], rows offsets[e]:offsets[e+1] = expert e
    out = expert_combine(y, weights, row_slot, slot_row)          # [R, H], [T, k] -> [T, H]

``row_slot[r] = t * k + j`` says which choice sorted row ``r`` holds, ``slot_row[t, j] = r`` is its inverse; the sort is
stable (equal experts keep slot order).  An expert id outside ``[0, E)`` (``-1`` by custom) means the slot has no expert,
as in a padded batch or where another rank owns the expert: its ``slot_row`` is -1, and the rows from ``offsets[E]`` on
have ``row_slot`` -1 and come out as zeros.  Nothing is read on the host: the calls can be captured in a CUDA graph.

Registration, argument checks, streams and errors follow ``ops.py``.  Every op also has a ``*_out`` form, the op's body
without the dispatcher and with an optional ``out=``, for eager serving loops where a call's host time counts.  The
reference has no routed block: MagiCompiler compiles whatever its models contain, and these ops are split points for it
like the fused SwiGLU (``magi_compiler/_magi_register_custom_op.py:168-204``).
"""
from __future__ import annotations

from typing import Optional

import torch
from torch.utils._device import DeviceContext

from . import _loader
from .ops import _raw_stream, _rows_view
from .register import magi_register_custom_op

BLOCK = 128  # columns that share one fp8 scale
FP8_MAX = 448.0
SCALE_FLOOR = 2.0 ** -126
MAX_EXPERTS = 1024


def _raise(name: str, rc: int) -> None:
    msg = f"{name} failed ({rc}): {_loader.last_error()}"
    raise (ValueError(msg) if rc < 0 else RuntimeError(msg))


def _rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """``t`` itself when the kernels can read it as it is (no view is made: a call's host time counts), else ``_rows_view``."""
    return t if t.is_contiguous() and t.data_ptr() % 16 == 0 else _rows_view(t, cols)


def _end(t: torch.Tensor) -> int:
    """Address of the byte behind ``t``'s last element."""
    if t.is_contiguous():
        return t.data_ptr() + t.nbytes
    return t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def _result(name: str, out: torch.Tensor | None, shape: tuple[int, ...], dtype: torch.dtype, device: torch.device,
            *others: torch.Tensor | None) -> torch.Tensor:
    """``out`` if it is what the kernel can write (contiguous, 16-byte aligned, apart from ``others``, the operands and the
    call's other results), a new tensor if it is None.  (``torch.empty`` takes 1.5 us with the sizes as arguments, 2.3 with a
    tuple.)"""
    if out is None:
        return torch.empty(*shape, dtype=dtype, device=device)
    lo = out.data_ptr()
    if out.dtype is not dtype or out.device != device or out.shape != shape or not out.is_contiguous() or lo % 16:
        raise ValueError(f"{name}: out must be a contiguous, 16-byte-aligned {dtype} tensor of shape {tuple(shape)} on {device}")
    hi = lo + out.nbytes
    for t in others:
        if t is not None and t.data_ptr() < hi and _end(t) > lo:
            raise ValueError(f"{name}: out must not overlap an operand or another result")
    return out


# ------------------------------------------------------------------------------------------------ sort
SORT_OP_NAME = "magi_swiglu::expert_sort"


def _expert_sort_meta(expert_ids: torch.Tensor, num_experts: int):
    return (expert_ids.new_empty((expert_ids.shape[0] * expert_ids.shape[1],), dtype=torch.int32),
            expert_ids.new_empty(expert_ids.shape, dtype=torch.int32),
            expert_ids.new_empty((num_experts + 1,), dtype=torch.int32))


def expert_sort_out(expert_ids: torch.Tensor, num_experts: int,
                    out: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None
                    ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The body of ``expert_sort``; ``out`` = (row_slot, slot_row, offsets) to write into."""
    if not isinstance(expert_ids, torch.Tensor) or expert_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError("expert_sort takes int32 or int64 expert ids")
    if expert_ids.dim() != 2 or expert_ids.shape[1] < 1:
        raise ValueError(f"expert_ids must be [tokens, choices]; got shape {tuple(expert_ids.shape)}")
    if not 1 <= num_experts <= MAX_EXPERTS:
        raise ValueError(f"num_experts must be in [1, {MAX_EXPERTS}]; got {num_experts}")
    dev = _check_device("expert_sort", expert_ids)
    ids = expert_ids.contiguous()
    slots, device = ids.numel(), ids.device
    if out is None:
        row_slot = torch.empty(slots, dtype=torch.int32, device=device)
        slot_row = torch.empty(*ids.shape, dtype=torch.int32, device=device)
        offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=device)
    else:
        row_slot = _result("expert_sort", out[0], (slots,), torch.int32, device, ids)
        slot_row = _result("expert_sort", out[1], ids.shape, torch.int32, device, ids, row_slot)
        offsets = _result("expert_sort", out[2], (num_experts + 1,), torch.int32, device, ids, row_slot, slot_row)
    rc = _loader.load_library().magi_swiglu_expert_sort(
        ids.data_ptr(), 1 if ids.dtype == torch.int64 else 0, slots, num_experts, row_slot.data_ptr(),
        slot_row.data_ptr(), offsets.data_ptr(), dev, _raw_stream(dev))
    if rc != 0:
        _raise("expert_sort", rc)
    return row_slot, slot_row, offsets


@magi_register_custom_op(name=SORT_OP_NAME, mutates_args=(), infer_output_meta_fn=_expert_sort_meta,
                         is_subgraph_boundary=True)
def expert_sort(expert_ids: torch.Tensor, num_experts: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(row_slot [T*k], slot_row [T, k], offsets [num_experts+1])``, int32, from ``expert_ids [T, k]`` (int32 or
    int64): one launch of a stable counting sort (``magi_swiglu_expert_sort``).  At most 1024 experts."""
    return expert_sort_out(expert_ids, num_experts)


# ------------------------------------------------------------------------------------------------ checks shared below
def _check_maps(name: str, row_slot: torch.Tensor, slot_row: torch.Tensor) -> tuple[int, int]:
    for what, t, dim in (("row_slot", row_slot, 1), ("slot_row", slot_row, 2)):
        if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32:
            raise TypeError(f"{name}: {what} must be an int32 tensor (expert_sort returns it)")
        if t.dim() != dim or not t.is_contiguous():
            raise ValueError(f"{name}: {what} must be a contiguous {dim}-D tensor; got shape {tuple(t.shape)}")
    tokens, k = slot_row.shape
    if k < 1 or row_slot.numel() != tokens * k:
        raise ValueError(f"{name}: row_slot has {row_slot.shape[0]} rows for slot_row {tuple(slot_row.shape)}")
    return tokens, k


def _check_rows(name: str, what: str, t: torch.Tensor, rows: int, multiple: int) -> int:
    if not isinstance(t, torch.Tensor) or t.dtype is not torch.bfloat16:
        raise TypeError(f"{name} moves bf16 rows only; {what} is {getattr(t, 'dtype', type(t))}")
    shape = t.shape
    if len(shape) != 2 or shape[0] != rows:
        raise ValueError(f"{name}: {what} must be [{rows}, H]; got shape {tuple(shape)}")
    h = shape[1]
    if h == 0 or h % multiple:
        raise ValueError(f"{name}: the row length {h} must be a positive multiple of {multiple}")
    return h


def _check_device(name: str, first: torch.Tensor, *others: torch.Tensor) -> int:
    """The index of the one CUDA device that all operands are on."""
    dev = first.get_device()  # -1 for a CPU tensor
    for t in others:
        if t.get_device() != dev or dev < 0:
            if dev < 0 or t.get_device() < 0:
                break
            raise ValueError(f"{name}: operands are on {first.device} and {t.device}")
    else:
        if dev >= 0:
            return dev
    raise TypeError(f"{name} runs on CUDA tensors only (there is no CPU implementation)")


def _check_weights(name: str, weights: torch.Tensor, tokens: int, k: int) -> None:
    if not isinstance(weights, torch.Tensor) or weights.dtype != torch.float32:
        raise TypeError(f"{name}: weights must be an fp32 tensor")
    if tuple(weights.shape) != (tokens, k):
        raise ValueError(f"{name}: weights must be [{tokens}, {k}]; got shape {tuple(weights.shape)}")


def _plain(*operands: torch.Tensor | None) -> bool:
    """Whether nothing but autograd looks at a call on these operands: no compiler, tracer, tracing or torch-function mode,
    tensor subclass or functorch transform.  Such a call may go to the op's body without the dispatcher, which with a
    registered autograd formula costs more host time than a small step's kernels run (113 us against 93 us for a gather and
    its gradient)."""
    for t in operands:
        if type(t) is not torch.Tensor and type(t) is not torch.nn.Parameter and t is not None:
            return False
    return not torch.compiler.is_compiling() and not torch._C._is_tracing() and torch._C._len_torch_dispatch_stack() == 0 \
        and (torch._C._len_torch_function_stack() == 0 or _only_a_default_device()) \
        and torch._C._functorch.peek_interpreter_stack() is None


def _only_a_default_device() -> bool:
    """Whether every torch-function mode is one of ``torch.set_default_device`` / ``with torch.device(..)``, which touch
    nothing but factory functions."""
    return all(type(m) is DeviceContext for m in torch.overrides._get_current_function_mode_stack())


def _ld(t2: torch.Tensor) -> int:
    return t2.stride(0) if t2.shape[0] > 1 else t2.shape[1]


# ------------------------------------------------------------------------------------------------ gather
GATHER_OP_NAME = "magi_swiglu::expert_gather"


def expert_gather_out(x: torch.Tensor, row_slot: torch.Tensor, slot_row: torch.Tensor,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """The body of ``expert_gather`` (no autograd)."""
    tokens, k = _check_maps("expert_gather", row_slot, slot_row)
    h = _check_rows("expert_gather", "x", x, tokens, 8)
    dev = _check_device("expert_gather", x, row_slot, slot_row)
    x2 = _rows(x, h)
    xs = _result("expert_gather", out, (tokens * k, h), torch.bfloat16, x.device, x, row_slot, slot_row)
    rc = _loader.load_library().magi_swiglu_expert_gather_bf16(
        x2.data_ptr(), row_slot.data_ptr(), slot_row.data_ptr(), xs.data_ptr(), tokens, k, h, _ld(x2), dev, _raw_stream(dev))
    if rc != 0:
        _raise("expert_gather", rc)
    return xs


def _gather_setup_context(ctx, inputs, output):
    ctx.save_for_backward(inputs[1], inputs[2])


def _gather_backward(ctx, grad):
    row_slot, slot_row = ctx.saved_tensors
    return expert_combine(grad, None, row_slot, slot_row), None, None


@magi_register_custom_op(
    name=GATHER_OP_NAME, mutates_args=(),
    infer_output_meta_fn=lambda x, row_slot, slot_row: x.new_empty((row_slot.shape[0], x.shape[1])),
    setup_context_fn=_gather_setup_context, backward_fn=_gather_backward, is_subgraph_boundary=True)
def _expert_gather_op(x: torch.Tensor, row_slot: torch.Tensor, slot_row: torch.Tensor) -> torch.Tensor:
    return expert_gather_out(x, row_slot, slot_row)


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, row_slot, slot_row):
        ctx.save_for_backward(row_slot, slot_row)
        return expert_gather_out(x, row_slot, slot_row)

    @staticmethod
    def backward(ctx, grad):
        if torch.is_grad_enabled() or not _plain(grad):
            return _gather_backward(ctx, grad)
        # the forward has checked the maps and autograd the gradient: not again (5 us on the thread of the backward pass)
        return _combine_rows(grad, None, ctx.saved_tensors[1], grad.shape[1], grad.get_device()), None, None


def expert_gather(x: torch.Tensor, row_slot: torch.Tensor, slot_row: torch.Tensor) -> torch.Tensor:
    """``xs[r] = x[row_slot[r] // k]`` (``[T, H]`` -> ``[T*k, H]`` bf16, H a multiple of 8), zeros where ``row_slot`` is -1
    (``magi_swiglu_expert_gather_bf16``).  Gradient: ``dx[t]`` is the fp32 sum of its rows' gradients in slot order,
    rounded once.  In compiled or traced code this is ``torch.ops.magi_swiglu.expert_gather``."""
    if not _plain(x, row_slot, slot_row):
        return torch.ops.magi_swiglu.expert_gather(x, row_slot, slot_row)
    if x.requires_grad and torch.is_grad_enabled():
        return _Gather.apply(x, row_slot, slot_row)
    return expert_gather_out(x, row_slot, slot_row)


# ------------------------------------------------------------------------------------------------ combine
COMBINE_OP_NAME = "magi_swiglu::expert_combine"
COMBINE_BWD_OP_NAME = "magi_swiglu::expert_combine_backward"


def expert_combine_out(y: torch.Tensor, weights: torch.Tensor | None, row_slot: torch.Tensor, slot_row: torch.Tensor,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """The body of ``expert_combine`` (no autograd)."""
    tokens, k = _check_maps("expert_combine", row_slot, slot_row)
    h = _check_rows("expert_combine", "y", y, tokens * k, 8)
    if weights is not None:
        _check_weights("expert_combine", weights, tokens, k)
        dev = _check_device("expert_combine", y, weights, row_slot, slot_row)
        weights = weights.contiguous()
    else:
        dev = _check_device("expert_combine", y, row_slot, slot_row)
    if out is not None:
        _result("expert_combine", out, (tokens, h), torch.bfloat16, y.device, y, weights, slot_row)
    return _combine_rows(y, weights, slot_row, h, dev, out)


def _combine_rows(y: torch.Tensor, weights: torch.Tensor | None, slot_row: torch.Tensor, h: int, dev: int,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """The launch of ``expert_combine`` on operands that have been checked."""
    tokens, k = slot_row.shape
    y2 = _rows(y, h)
    if out is None:
        out = torch.empty(tokens, h, dtype=torch.bfloat16, device=y.device)
    rc = _loader.load_library().magi_swiglu_expert_combine_bf16(
        y2.data_ptr(), weights.data_ptr() if weights is not None else None, slot_row.data_ptr(), out.data_ptr(), tokens, k,
        h, _ld(y2), dev, _raw_stream(dev))
    if rc != 0:
        _raise("expert_combine", rc)
    return out


def _combine_backward_meta(dout, y, weights, row_slot, slot_row, need_dy, need_dw):
    return (y.new_empty(y.shape if need_dy else (0,)),
            y.new_empty(slot_row.shape if need_dw else (0,), dtype=torch.float32))


def _combine_backward_body(dout: torch.Tensor, y: torch.Tensor, weights: torch.Tensor, row_slot: torch.Tensor,
                           slot_row: torch.Tensor, need_dy: bool, need_dw: bool) -> tuple[torch.Tensor, torch.Tensor]:
    name = "expert_combine_backward"
    tokens, k = _check_maps(name, row_slot, slot_row)
    h = _check_rows(name, "dout", dout, tokens, 8)
    if _check_rows(name, "y", y, tokens * k, 8) != h:
        raise ValueError(f"{name}: y {tuple(y.shape)} and dout {tuple(dout.shape)} differ in row length")
    _check_weights(name, weights, tokens, k)
    dev = _check_device(name, dout, y, weights, row_slot, slot_row)
    return _combine_backward_rows(dout, y, weights, row_slot, slot_row, need_dy, need_dw, h, dev)


def _combine_backward_rows(dout: torch.Tensor, y: torch.Tensor, weights: torch.Tensor, row_slot: torch.Tensor,
                           slot_row: torch.Tensor, need_dy: bool, need_dw: bool, h: int, dev: int
                           ) -> tuple[torch.Tensor, torch.Tensor]:
    """The launch of ``expert_combine_backward`` on operands that have been checked."""
    tokens, k = slot_row.shape
    d2, y2, w = _rows(dout, h), _rows(y, h), weights.contiguous()
    dy = torch.empty(*((tokens * k, h) if need_dy else (0,)), dtype=torch.bfloat16, device=y.device)
    dw = torch.empty(*((tokens, k) if need_dw else (0,)), dtype=torch.float32, device=y.device)
    rc = _loader.load_library().magi_swiglu_expert_combine_backward_bf16(
        d2.data_ptr(), y2.data_ptr(), w.data_ptr(), row_slot.data_ptr(), slot_row.data_ptr(),
        dy.data_ptr() if need_dy else None, dw.data_ptr() if need_dw else None, tokens, k, h, _ld(d2), _ld(y2), dev, _raw_stream(dev))
    if rc != 0:
        _raise("expert_combine_backward", rc)
    return dy, dw


@magi_register_custom_op(name=COMBINE_BWD_OP_NAME, mutates_args=(), infer_output_meta_fn=_combine_backward_meta)
def expert_combine_backward(dout: torch.Tensor, y: torch.Tensor, weights: torch.Tensor, row_slot: torch.Tensor,
                            slot_row: torch.Tensor, need_dy: bool, need_dw: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """``dy[slot_row[t, j]] = weights[t, j] * dout[t]`` (zeros in rows without a slot) and
    ``dw[t, j] = <dout[t], y[slot_row[t, j]]>`` in one pass (``magi_swiglu_expert_combine_backward_bf16``); the one that is
    not needed comes back empty."""
    return _combine_backward_body(dout, y, weights, row_slot, slot_row, need_dy, need_dw)


def _combine_setup_context(ctx, inputs, output):
    y, weights, row_slot, slot_row = inputs
    ctx.weighted = weights is not None
    if ctx.weighted:
        ctx.save_for_backward(y, weights, row_slot, slot_row)
    else:
        ctx.save_for_backward(row_slot, slot_row)


def _combine_backward(ctx, grad):
    if not ctx.weighted:
        return expert_gather(grad, *ctx.saved_tensors), None, None, None
    need_dy, need_dw = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
    if torch.is_grad_enabled() or not _plain(grad):
        dy, dw = torch.ops.magi_swiglu.expert_combine_backward(grad, *ctx.saved_tensors, need_dy, need_dw)
    else:  # checked by the forward and by autograd
        dy, dw = _combine_backward_rows(grad, *ctx.saved_tensors, need_dy, need_dw, grad.shape[1], grad.get_device())
    return dy if need_dy else None, dw if need_dw else None, None, None


@magi_register_custom_op(
    name=COMBINE_OP_NAME, mutates_args=(),
    infer_output_meta_fn=lambda y, weights, row_slot, slot_row: y.new_empty((slot_row.shape[0], y.shape[1])),
    setup_context_fn=_combine_setup_context, backward_fn=_combine_backward, is_subgraph_boundary=True)
def _expert_combine_op(y: torch.Tensor, weights: Optional[torch.Tensor], row_slot: torch.Tensor,
                       slot_row: torch.Tensor) -> torch.Tensor:
    return expert_combine_out(y, weights, row_slot, slot_row)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, row_slot, slot_row):
        _combine_setup_context(ctx, (y, weights, row_slot, slot_row), None)
        return expert_combine_out(y, weights, row_slot, slot_row)

    backward = staticmethod(_combine_backward)


def expert_combine(y: torch.Tensor, weights: Optional[torch.Tensor], row_slot: torch.Tensor,
                   slot_row: torch.Tensor) -> torch.Tensor:
    """``out[t] = sum_j weights[t, j] * y[slot_row[t, j]]`` (``[T*k, H]`` bf16 and ``[T, k]`` fp32 -> ``[T, H]`` bf16;
    fp32 sums in slot order, one rounding; ``weights`` None: ones; ``magi_swiglu_expert_combine_bf16``).  Slots without an
    expert add nothing.  Gradients with respect to ``y`` and ``weights`` (once differentiable where weights are given).  In
    compiled or traced code this is ``torch.ops.magi_swiglu.expert_combine``."""
    if not _plain(y, weights, row_slot, slot_row):
        return torch.ops.magi_swiglu.expert_combine(y, weights, row_slot, slot_row)
    if torch.is_grad_enabled() and (y.requires_grad or (weights is not None and weights.requires_grad)):
        return _Combine.apply(y, weights, row_slot, slot_row)
    return expert_combine_out(y, weights, row_slot, slot_row)


# ------------------------------------------------------------------------------------------------ block quantiser
QUANTIZE_OP_NAME = "magi_swiglu::quantize_fp8_block"
GATHER_FP8_OP_NAME = "magi_swiglu::expert_gather_fp8"


def _fp8_block_outputs(name, out, rows, cols, device, *operands):
    codes, scales = out if out is not None else (None, None)
    codes = _result(name, codes, (rows, cols), torch.float8_e4m3fn, device, *operands)
    return codes, _result(name, scales, (rows, -(-cols // BLOCK)), torch.float32, device, codes, *operands)


def quantize_fp8_block_out(x: torch.Tensor, out: tuple[torch.Tensor, torch.Tensor] | None = None
                           ) -> tuple[torch.Tensor, torch.Tensor]:
    """The body of ``quantize_fp8_block``; ``out`` = (codes, scales) to write into."""
    cols = _check_rows("quantize_fp8_block", "x", x, x.shape[0] if isinstance(x, torch.Tensor) and x.dim() else 0, 16)
    dev = _check_device("quantize_fp8_block", x)
    x2 = _rows(x, cols)
    codes, scales = _fp8_block_outputs("quantize_fp8_block", out, x.shape[0], cols, x.device, x)
    rc = _loader.load_library().magi_swiglu_quantize_fp8_block(
        x2.data_ptr(), codes.data_ptr(), scales.data_ptr(), x.shape[0], cols, _ld(x2), dev, _raw_stream(dev))
    if rc != 0:
        _raise("quantize_fp8_block", rc)
    return codes, scales


@magi_register_custom_op(
    name=QUANTIZE_OP_NAME, mutates_args=(),
    infer_output_meta_fn=lambda x: (x.new_empty(x.shape, dtype=torch.float8_e4m3fn),
                                    x.new_empty((x.shape[0], (x.shape[1] + BLOCK - 1) // BLOCK), dtype=torch.float32)))
def quantize_fp8_block(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)`` of ``x [M, K]`` bf16 (K a multiple of 16): per row and 128 columns
    ``scale = max(max|x| / 448, 2^-126)`` and ``code = e4m3(x / scale)`` (``magi_swiglu_quantize_fp8_block``), bit for bit
    the formula in fp32.  ``codes`` float8_e4m3fn ``[M, K]``, ``scales`` fp32 ``[M, ceil(K/128)]``.  Inference only."""
    return quantize_fp8_block_out(x)


def expert_gather_fp8_out(x: torch.Tensor, row_slot: torch.Tensor, slot_row: torch.Tensor,
                          out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The body of ``expert_gather_fp8``; ``out`` = (codes, scales) to write into."""
    tokens, k = _check_maps("expert_gather_fp8", row_slot, slot_row)
    cols = _check_rows("expert_gather_fp8", "x", x, tokens, 16)
    dev = _check_device("expert_gather_fp8", x, row_slot, slot_row)
    x2 = _rows(x, cols)
    codes, scales = _fp8_block_outputs("expert_gather_fp8", out, tokens * k, cols, x.device, x, row_slot, slot_row)
    rc = _loader.load_library().magi_swiglu_expert_gather_fp8_block(
        x2.data_ptr(), row_slot.data_ptr(), slot_row.data_ptr(), codes.data_ptr(), scales.data_ptr(), tokens, k, cols,
        _ld(x2), dev, _raw_stream(dev))
    if rc != 0:
        _raise("expert_gather_fp8", rc)
    return codes, scales


def _gather_fp8_meta(x, row_slot, slot_row):
    rows, cols = row_slot.shape[0], x.shape[1]
    return (x.new_empty((rows, cols), dtype=torch.float8_e4m3fn),
            x.new_empty((rows, (cols + BLOCK - 1) // BLOCK), dtype=torch.float32))


@magi_register_custom_op(name=GATHER_FP8_OP_NAME, mutates_args=(), infer_output_meta_fn=_gather_fp8_meta,
                         is_subgraph_boundary=True)
def expert_gather_fp8(x: torch.Tensor, row_slot: torch.Tensor, slot_row: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``quantize_fp8_block(expert_gather(x, row_slot, slot_row))`` with every token read and quantised once
    (``magi_swiglu_expert_gather_fp8_block``): ``(codes [T*k, K], scales [T*k, ceil(K/128)])``; rows without a slot hold
    zero codes and the scale 2^-126.  Inference only."""
    return expert_gather_fp8_out(x, row_slot, slot_row)
