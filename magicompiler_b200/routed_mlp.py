"""A routed (mixture-of-experts) SwiGLU MLP from the package's operators: the block that ``TensorParallelSwiGLUMLP`` is for a
dense model.  The router itself (logits, top-k) stays with the model; the module takes its choices and weights."""
from __future__ import annotations

import torch
import torch.nn.functional as F

from . import fp8_block, routed
from .fp8_block import quantize_fp8_gate_up, quantize_fp8_weight
from .ops import gemm_swiglu_auto


class RoutedSwiGLUMLP(torch.nn.Module):
    """``out[t] = sum_j weights[t, j] * mlp_e(x[t])`` with ``e = expert_ids[t, j]`` and
    ``mlp_e(x) = (silu(x Wg_e^T) * (x Wu_e^T)) Wd_e^T``; ids outside ``[0, E)`` add nothing.

    ``w_gate_up`` is ``[E, 2N, K]`` (gate rows first, ``pack_gate_up`` per expert), ``w_down`` ``[E, K_out, N]``, both bf16.

    * ``precision="bf16"``: trainable.  Experts run one after the other through ``gemm_swiglu_auto`` on their rows, so a
      forward reads the E + 1 row offsets on the host (it cannot be captured in a CUDA graph).
    * ``precision="fp8"``: inference.  The weights are quantised once, here (one fp32 scale per 128 x 128 block), and all
      experts run in one launch per projection (``gemm_swiglu_fp8_block``, ``gemm_fp8_block``); nothing is read on the host,
      a forward of fixed shape can be captured.  Moving the module to another dtype (``.bfloat16()``, ``.to(dtype)`` of a whole
      model) moves the codes and the fp32 scales to the device it names and leaves their types alone.
    """

    def __init__(self, w_gate_up: torch.Tensor, w_down: torch.Tensor, precision: str = "bf16"):
        super().__init__()
        if precision not in ("bf16", "fp8"):
            raise ValueError(f"precision must be 'bf16' or 'fp8', got {precision!r}")
        if w_gate_up.dim() != 3 or w_down.dim() != 3 or w_gate_up.shape[0] != w_down.shape[0] \
                or w_gate_up.shape[1] != 2 * w_down.shape[2]:
            raise ValueError(f"w_gate_up {tuple(w_gate_up.shape)} and w_down {tuple(w_down.shape)} must be [E, 2N, K] and "
                             "[E, K_out, N]")
        if w_gate_up.dtype != torch.bfloat16 or w_down.dtype != torch.bfloat16:
            raise TypeError(f"the weights must be bf16; got {w_gate_up.dtype} and {w_down.dtype}")
        self.precision, self.num_experts, self.k_out = precision, w_gate_up.shape[0], w_down.shape[1]
        if precision == "bf16":
            self.w_gate_up = torch.nn.Parameter(w_gate_up.contiguous())
            self.w_down = torch.nn.Parameter(w_down.contiguous())
            return
        for name, pair in (("gate_up", quantize_fp8_gate_up(w_gate_up)), ("down", quantize_fp8_weight(w_down))):
            self.register_buffer(f"{name}_codes", pair[0])
            self.register_buffer(f"{name}_scales", pair[1])

    def _apply(self, fn, recurse=True):
        if self.precision != "fp8":
            return super()._apply(fn, recurse)

        def keep_type(t: torch.Tensor) -> torch.Tensor:
            moved = fn(t)
            return moved if moved.dtype is t.dtype else t.to(moved.device)

        return super()._apply(keep_type, recurse)

    def forward(self, x: torch.Tensor, expert_ids: torch.Tensor, weights: torch.Tensor) -> torch.Tensor:
        """``x [..., K]`` bf16, ``expert_ids [..., k]`` int32 or int64, ``weights [..., k]`` fp32 -> ``[..., K_out]``."""
        if expert_ids.shape != weights.shape or expert_ids.shape[:-1] != x.shape[:-1]:
            raise ValueError(f"x {tuple(x.shape)}, expert_ids {tuple(expert_ids.shape)} and weights {tuple(weights.shape)} "
                             "must agree in their leading dimensions, ids and weights in all")
        if self.precision == "fp8" and torch.is_grad_enabled() and (x.requires_grad or weights.requires_grad):
            raise RuntimeError("precision='fp8' is for inference: it has no gradients (run it under torch.no_grad())")
        x2, k = x.reshape(-1, x.shape[-1]), expert_ids.shape[-1]
        ids, w = expert_ids.reshape(-1, k), weights.reshape(-1, k)
        out_form = "_out" if routed._plain(x, expert_ids, weights) else ""  # compiled and traced code calls the registered ops
        row_slot, slot_row, offsets = getattr(routed, "expert_sort" + out_form)(ids, self.num_experts)
        if self.precision == "fp8":
            a, a_scale = getattr(routed, "expert_gather_fp8" + out_form)(x2, row_slot, slot_row)
            h, h_scale = getattr(fp8_block, "gemm_swiglu_fp8_block" + out_form)(a, a_scale, self.gate_up_codes,
                                                                                self.gate_up_scales, offsets)
            y = getattr(fp8_block, "gemm_fp8_block" + out_form)(h, h_scale, self.down_codes, self.down_scales, offsets)
            return routed.expert_combine(y, w, row_slot, slot_row).view(*x.shape[:-1], self.k_out)
        xs = routed.expert_gather(x2, row_slot, slot_row)
        bounds = offsets.tolist()
        parts = []
        for e, (wg, wd) in enumerate(zip(self.w_gate_up.unbind(0), self.w_down.unbind(0))):
            lo, hi = bounds[e], bounds[e + 1]
            if hi > lo or (bounds[-1] == 0 and e == 0):  # without any routed row one empty call keeps the gradients zeros
                parts.append(F.linear(gemm_swiglu_auto(xs[lo:hi], wg), wd))
        parts.append(xs.new_zeros((xs.shape[0] - bounds[-1], self.k_out)))  # rows without an expert
        return routed.expert_combine(torch.cat(parts), w, row_slot, slot_row).view(*x.shape[:-1], self.k_out)
