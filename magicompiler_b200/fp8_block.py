"""Products that READ block-scaled fp8: ``gemm_fp8_block`` (a projection) and ``gemm_swiglu_fp8_block`` (the fused gate/up
projection with SwiGLU, whose result leaves in the same format), dense or over routed experts.

    C[m, n] = sum_b a_scale[m, b] * b_scale[n // 128, b] * sum_{k in block b} a[m, k] * b[n, k]

``a`` is float8_e4m3fn ``[M, K]`` with fp32 ``a_scale [M, ceil(K/128)]`` (``quantize_fp8_block`` / ``expert_gather_fp8``),
``b`` float8_e4m3fn ``[N, K]`` with one fp32 scale per 128 x 128 block, ``[ceil(N/128), ceil(K/128)]``
(``quantize_fp8_weight``, once at load).  With ``offsets`` (``expert_sort``) ``b`` is ``[E, N, K]`` and rows
``offsets[e]:offsets[e+1]`` of ``a`` meet ``b[e]`` (they start at 0 and do not fall; one that does counts as the largest
before it); nothing is read on the host.  Inference only: no autograd.

A SwiGLU block in 8 bits, routed (dense: leave out the routing and ``offsets``):

    row_slot, slot_row, offsets = expert_sort(ids, E)
    a, s = expert_gather_fp8(x, row_slot, slot_row)
    h, hs = gemm_swiglu_fp8_block(a, s, w13, w13_scale, offsets)
    y = gemm_fp8_block(h, hs, w2, w2_scale, offsets)
    out = expert_combine(y, weights, row_slot, slot_row)

Checks, streams and errors follow ``ops.py``; the ``*_out`` forms are the ops' bodies with an optional ``out=``.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import _loader
from .ops import _raw_stream
from .register import magi_register_custom_op
from .routed import BLOCK, FP8_MAX, SCALE_FLOOR, _check_device, _fp8_block_outputs, _raise, _result

GEMM_OP_NAME = "magi_swiglu::gemm_fp8_block"
SWIGLU_OP_NAME = "magi_swiglu::gemm_swiglu_fp8_block"


def _quantize_blocks(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    full = torch.zeros(nb * BLOCK, kb * BLOCK, dtype=torch.float32, device=w.device)
    full[:n, :k] = w
    blocks = full.view(nb, BLOCK, kb, BLOCK)
    scale = (blocks.abs().amax(dim=(1, 3)) / FP8_MAX).clamp_min(SCALE_FLOOR)
    codes = (blocks / scale[:, None, :, None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return codes.view(nb * BLOCK, kb * BLOCK)[:n, :k].contiguous(), scale


def _per_expert(w: torch.Tensor, fn) -> tuple[torch.Tensor, torch.Tensor]:
    if w.dim() == 2:
        return fn(w)
    if w.dim() != 3:
        raise ValueError(f"a weight is [N, K] or [E, N, K]; got shape {tuple(w.shape)}")
    parts = [fn(e) for e in w]  # expert by expert: one fp32 copy at a time
    return (torch.stack([p[0].view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn), torch.stack([p[1] for p in parts]))


@torch.no_grad()
def quantize_fp8_weight(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)`` of a weight ``[N, K]`` or ``[E, N, K]`` for ``gemm_fp8_block``: one scale ``max|w| / 448`` per
    128 x 128 block, ``scales [.., ceil(N/128), ceil(K/128)]``.  Plain torch, once at load; no gradients (a parameter may be
    given as it is)."""
    return _per_expert(w, _quantize_blocks)


@torch.no_grad()
def quantize_fp8_gate_up(w_gate_up: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)`` of a packed gate/up weight ``[2N, K]`` or ``[E, 2N, K]`` (``pack_gate_up``) for
    ``gemm_swiglu_fp8_block``: each half is cut into blocks from its own first row, ``scales [.., 2 * ceil(N/128),
    ceil(K/128)]`` hold the gate half's blocks, then the up half's."""
    if w_gate_up.dim() in (2, 3) and w_gate_up.shape[-2] % 2:
        raise ValueError(f"w_gate_up has {w_gate_up.shape[-2]} rows; it must hold N gate rows followed by N up rows")

    def halves(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        n = w.shape[0] // 2
        (g, gs), (u, us) = _quantize_blocks(w[:n]), _quantize_blocks(w[n:])
        return torch.cat([g.view(torch.uint8), u.view(torch.uint8)]).view(torch.float8_e4m3fn), torch.cat([gs, us])

    return _per_expert(w_gate_up, halves)


def _check(name: str, a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
           offsets: torch.Tensor | None, halves: int) -> tuple[int, int, int, int, int]:
    for what, t, dtype in (("a", a, torch.float8_e4m3fn), ("a_scale", a_scale, torch.float32),
                           ("b", b, torch.float8_e4m3fn), ("b_scale", b_scale, torch.float32)):
        if not isinstance(t, torch.Tensor) or t.dtype is not dtype:
            raise TypeError(f"{name}: {what} must be a {dtype} tensor; got {getattr(t, 'dtype', type(t))}")
    if a.dim() != 2 or a_scale.dim() != 2:
        raise ValueError(f"{name}: a and a_scale must be 2-D; got {tuple(a.shape)} and {tuple(a_scale.shape)}")
    experts = 1
    if offsets is not None:
        if not isinstance(offsets, torch.Tensor) or offsets.dtype != torch.int32:
            raise TypeError(f"{name}: offsets must be an int32 tensor (expert_sort returns it)")
        if b.dim() != 3 or not 1 <= b.shape[0] <= 1024:
            raise ValueError(f"{name}: with offsets the weight must be [experts, rows, K], at most 1024 experts; got {tuple(b.shape)}")
        experts = b.shape[0]
        if offsets.dim() != 1 or offsets.shape[0] != experts + 1 or not offsets.is_contiguous():
            raise ValueError(f"{name}: offsets must be a contiguous [{experts + 1}] tensor; got {tuple(offsets.shape)}")
    elif b.dim() != 2:
        raise ValueError(f"{name}: without offsets the weight must be [rows, K]; got {tuple(b.shape)}")
    m, k = a.shape
    rows, kw = b.shape[-2:]
    if rows % halves:
        raise ValueError(f"{name}: the weight has {rows} rows; it must hold N gate rows followed by N up rows")
    n = rows // halves
    if kw != k:
        raise ValueError(f"{name}: inner dimensions differ: a {tuple(a.shape)}, weight {tuple(b.shape)}")
    if k == 0 or n == 0 or k % 16 or n % (8 * halves):
        raise ValueError(f"{name}: K ({k}) must be a positive multiple of 16 and N ({n}) of {8 * halves}")
    kb, nb = (k + BLOCK - 1) // BLOCK, (n + BLOCK - 1) // BLOCK
    if a_scale.shape != (m, kb):
        raise ValueError(f"{name}: a_scale must be [{m}, {kb}]; got {tuple(a_scale.shape)}")
    if b_scale.shape != ((halves * nb, kb) if offsets is None else (experts, halves * nb, kb)):
        raise ValueError(f"{name}: the weight's scales must be {[] if offsets is None else [experts]}{[halves * nb, kb]}; got {tuple(b_scale.shape)}")
    if not b.is_contiguous() or not b_scale.is_contiguous():
        raise ValueError(f"{name}: the weight and its scales must be contiguous (a copy on every call would double their traffic)")
    if offsets is None:
        dev = _check_device(name, a, a_scale, b, b_scale)
    else:
        dev = _check_device(name, a, a_scale, b, b_scale, offsets)
    if b.data_ptr() % 16:
        raise ValueError(f"{name}: the weight must be 16-byte aligned")
    return m, n, k, experts, dev


def _operand(a: torch.Tensor, a_scale: torch.Tensor) -> tuple[torch.Tensor, int, torch.Tensor, int]:
    """``a`` and its scales as the kernels read them (a copy if they cannot), with their row strides."""
    m, k = a.shape
    if a.is_contiguous():
        if a.data_ptr() % 16:
            a = a.clone()
    elif not (a.stride(1) == 1 and a.stride(0) >= k and a.stride(0) % 16 == 0 and a.data_ptr() % 16 == 0):
        a = a.contiguous()
    if not (a_scale.is_contiguous() or (a_scale.stride(1) == 1 and a_scale.stride(0) >= a_scale.shape[1])):
        a_scale = a_scale.contiguous()
    return a, a.stride(0) if m > 1 else k, a_scale, a_scale.stride(0) if m > 1 else a_scale.shape[1]


def gemm_fp8_block_out(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                       offsets: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """The body of ``gemm_fp8_block``.  With ``out`` the rows from ``offsets[E]`` on are left as they were."""
    m, n, k, experts, dev = _check("gemm_fp8_block", a, a_scale, b, b_scale, offsets, 1)
    c = _result("gemm_fp8_block", out, (m, n), torch.bfloat16, a.device, a, a_scale, b, b_scale, offsets)
    if m == 0:
        return c
    a2, lda, s2, lds = _operand(a, a_scale)
    rc = _loader.load_library().magi_swiglu_gemm_fp8_block(
        a2.data_ptr(), s2.data_ptr(), b.data_ptr(), b_scale.data_ptr(), offsets.data_ptr() if offsets is not None else None,
        experts, c.data_ptr(), m, n, k, lda, lds, 0 if out is not None else 1, dev, _raw_stream(dev))
    if rc != 0:
        _raise("gemm_fp8_block", rc)
    return c


@magi_register_custom_op(name=GEMM_OP_NAME, mutates_args=(),
                         infer_output_meta_fn=lambda a, a_scale, b, b_scale, offsets=None: a.new_empty(
                             (a.shape[0], b.shape[-2]), dtype=torch.bfloat16),
                         is_compute_sensitive=True)
def gemm_fp8_block(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                   offsets: Optional[torch.Tensor] = None) -> torch.Tensor:
    """bf16 ``[M, N]`` from fp8 codes and block scales (formula above; ``magi_swiglu_gemm_fp8_block``): fp32 sums, one
    rounding.  K a multiple of 16, N of 8.  With ``offsets`` rows without an expert come out as zeros."""
    return gemm_fp8_block_out(a, a_scale, b, b_scale, offsets)


def gemm_swiglu_fp8_block_out(a: torch.Tensor, a_scale: torch.Tensor, w_gate_up: torch.Tensor, w_scale: torch.Tensor,
                              offsets: torch.Tensor | None = None, out: tuple[torch.Tensor, torch.Tensor] | None = None
                              ) -> tuple[torch.Tensor, torch.Tensor]:
    """The body of ``gemm_swiglu_fp8_block``; ``out`` = (codes, scales), whose rows from ``offsets[E]`` on are left as they
    were."""
    name = "gemm_swiglu_fp8_block"
    m, n, k, experts, dev = _check(name, a, a_scale, w_gate_up, w_scale, offsets, 2)
    codes, scales = _fp8_block_outputs(name, out, m, n, a.device, a, a_scale, w_gate_up, w_scale, offsets)
    if m == 0:
        return codes, scales
    a2, lda, s2, lds = _operand(a, a_scale)
    rc = _loader.load_library().magi_swiglu_gemm_swiglu_fp8_block(
        a2.data_ptr(), s2.data_ptr(), w_gate_up.data_ptr(), w_scale.data_ptr(),
        offsets.data_ptr() if offsets is not None else None, experts, codes.data_ptr(), scales.data_ptr(), m, n, k, lda, lds,
        0 if out is not None else 1, dev, _raw_stream(dev))
    if rc != 0:
        _raise(name, rc)
    return codes, scales


def _swiglu_meta(a, a_scale, w_gate_up, w_scale, offsets=None):
    n = w_gate_up.shape[-2] // 2
    return (a.new_empty((a.shape[0], n)), a.new_empty((a.shape[0], (n + BLOCK - 1) // BLOCK), dtype=torch.float32))


@magi_register_custom_op(name=SWIGLU_OP_NAME, mutates_args=(), infer_output_meta_fn=_swiglu_meta,
                         is_compute_sensitive=True, is_subgraph_boundary=True)
def gemm_swiglu_fp8_block(a: torch.Tensor, a_scale: torch.Tensor, w_gate_up: torch.Tensor, w_scale: torch.Tensor,
                          offsets: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)`` of ``silu(a · Wg^T) * (a · Wu^T)``, quantised per row and 128 columns from the fp32 sums
    (``magi_swiglu_gemm_swiglu_fp8_block``): float8_e4m3fn ``[M, N]`` and fp32 ``[M, ceil(N/128)]``, what
    ``gemm_fp8_block`` reads.  ``w_gate_up`` ``[2N, K]`` / ``[E, 2N, K]`` and ``w_scale`` from ``quantize_fp8_gate_up``.
    K and N multiples of 16.  With ``offsets`` rows without an expert hold zero codes and the scale 2^-126."""
    return gemm_swiglu_fp8_block_out(a, a_scale, w_gate_up, w_scale, offsets)
