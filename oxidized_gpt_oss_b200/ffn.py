"""SwiGLU — mirror of src/ffn.rs of the reference.

The reference's ``swiglu(gate, up)`` (src/ffn.rs:5-13) is the plain
``silu(g) * u``. gpt-oss experts use the clamped form, which is what this
library computes (and fuses into the mlp1 epilogue of the MoE kernels):
``g <- min(g, limit); u <- clamp(u, -limit, limit); g * sigmoid(alpha g) * (u + 1)``.
"""
from __future__ import annotations

import torch

from . import abi
from .mxfp4 import _DTYPES, _context_on, check_status, device_context, quantized_like, rows_of, scale_rule_code

ALPHA = 1.702
LIMIT = 7.0


def swiglu(gate: torch.Tensor, up: torch.Tensor, alpha: float = ALPHA, limit: float = LIMIT, *,
           ctx: abi.Context | None = None) -> torch.Tensor:
    if gate.shape != up.shape:
        raise ValueError(f"gate and up shapes differ: {tuple(gate.shape)} vs {tuple(up.shape)}")
    index = gate.get_device()
    if gate.dtype != torch.float32 or up.dtype != torch.float32 or index < 0 or up.get_device() != index:
        if gate.dtype == up.dtype == torch.float32 and gate.is_cuda and up.is_cuda:
            raise ValueError("gate and up must be on one device")
        raise ValueError("gate and up must be float32 CUDA tensors")
    g = gate.contiguous()
    u = up.contiguous()
    out = torch.empty_like(g)
    c = _context_on(index, ctx)
    abi.check(c.lib.oxg_swiglu(c.handle, g.data_ptr(), u.data_ptr(), g.numel(), float(alpha), float(limit),
                               out.data_ptr()), c.handle)
    return out


def swiglu_quantize_mxfp4(gate_up: torch.Tensor, alpha: float = ALPHA, limit: float = LIMIT, *,
                          scale_rule: str = "floor", tiled: bool = False,
                          ctx: abi.Context | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The clamped SwiGLU of gate_up [..., 2 cols] (gate in the even columns, up
    in the odd ones, as the experts' first product gives them; float32, bfloat16
    or float16), as MXFP4 [..., cols]: (blocks, scales) as
    ``mxfp4.quantize_mxfp4`` returns them, with the codes of the exact values."""
    x2, rows, ld = rows_of(gate_up, "gate_up")
    if gate_up.shape[-1] % 2:
        raise ValueError(f"gate_up must hold pairs, got {gate_up.shape[-1]} columns")
    cols = gate_up.shape[-1] // 2
    blocks, scales = quantized_like(gate_up, cols, rows, tiled)
    c = device_context(gate_up, ctx)
    check_status(c.lib.oxg_swiglu_quantize_mxfp4(c.handle, x2.data_ptr(), _DTYPES[gate_up.dtype], rows, cols, ld,
                                                 float(alpha), float(limit), scale_rule_code(scale_rule), int(tiled),
                                                 blocks.data_ptr(), scales.data_ptr()), c)
    return blocks, scales
