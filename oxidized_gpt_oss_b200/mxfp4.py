"""MXFP4 dequantisation — mirror of src/mxfp4.rs of the reference.

``dequantize_mxfp4(blocks, scales, rows, cols)`` keeps the reference's
signature and meaning (src/mxfp4.rs:15): ``blocks`` are packed E2M1 codes
(low nibble = even element), ``scales`` one per 32-element block, the result
``rows * cols`` bf16 bit patterns. Inputs are CUDA tensors; the work runs in
liboxg_b200.so on torch's current stream. Shape violations raise
``ValueError`` with the reference's assert text where the reference panics.

The way back and what 4-bit operands are for (no counterpart in the reference):
``quantize_mxfp4`` makes blocks and scales of floating-point rows,
``mxfp4_matmul`` multiplies two MXFP4 operands on the 4-bit tensor cores, and
``mxfp4_grouped_matmul`` does so for runs of rows that each have a matrix of
their own (experts). The products read scales in the tiled layout
``[ceil(k / 128), rows, 4]``, which the quantisers write with ``tiled=True`` and
``tile_scales`` makes of a checkpoint's ``[rows, k / 32]``; given the latter,
they convert it first, on every call. Making a context allocates no device
memory, so a process's first call may be captured.
"""
from __future__ import annotations

import threading

import torch

from . import abi

_default_ctx = None  # one of the next
_device_ctx: dict[int, abi.Context] = {}  # the main thread's, by device
_making = threading.Lock()
# the raw stream handle where this torch has it: the Stream object costs 3 us a call
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _bind(ctx: abi.Context) -> abi.Context:
    """Puts the context on torch's current stream of its device."""
    stream = _raw_stream(ctx.device) if _raw_stream is not None else torch.cuda.current_stream(ctx.device).cuda_stream
    abi.check(ctx.lib.oxg_ctx_set_stream(ctx.handle, stream), ctx.handle)
    return ctx


def context(ctx: abi.Context | None = None) -> abi.Context:
    """The given context, or a per-process default one (the main thread's on the
    device that was current when it was first asked for), bound to torch's
    current stream. A context serves one thread at a time: a MoE layer that is
    called from other threads than the main one wants a context of its own."""
    global _default_ctx
    if ctx is None:
        if _default_ctx is None:
            _default_ctx = _main_context(torch.cuda.current_device())
        ctx = _default_ctx
    return _bind(ctx)


def _main_context(index: int) -> abi.Context:
    """The main thread's context on a device. Any thread may ask for the default one."""
    with _making:
        ctx = _device_ctx.get(index)
        if ctx is None:
            ctx = _device_ctx[index] = abi.Context(index)
        return ctx


def dequantize_mxfp4(blocks: torch.Tensor, scales: torch.Tensor, rows: int, cols: int, *,
                     ctx: abi.Context | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """blocks: uint8 CUDA tensor; scales: int16/uint16 (bf16 bits) or uint8 (E8M0),
    on the same device, which the work runs on.

    Returns an int16 tensor of rows*cols bf16 bit patterns."""
    index = blocks.get_device()
    if index < 0 or scales.get_device() != index:
        if not (blocks.is_cuda and scales.is_cuda):
            raise ValueError("blocks and scales must be CUDA tensors")
        raise ValueError("blocks and scales must be on one device")
    if out is not None and out.get_device() != index and (out.is_cuda or not out.is_pinned()):
        raise ValueError(f"out must be on cuda:{index} or in pinned host memory")
    blocks = blocks.contiguous()
    scales = scales.contiguous()
    if scales.dtype == torch.uint8:
        fmt = abi.OXG_SCALE_E8M0
    elif scales.dtype in (torch.int16, torch.uint16, torch.bfloat16):
        fmt = abi.OXG_SCALE_BF16
    else:
        raise ValueError(f"unsupported scale dtype {scales.dtype}")
    c = _context_on(index, ctx)
    if out is None:
        out = torch.empty_strided((max(rows * cols, 0),), (1,), dtype=torch.int16, device=blocks.device)
    st = c.lib.oxg_dequant_mxfp4(c.handle, blocks.data_ptr(), blocks.numel(), scales.data_ptr(),
                                 scales.numel(), fmt, rows, cols, out.data_ptr())
    if st == abi.OXG_ERR_SHAPE:
        raise ValueError(c.lib.oxg_last_error(c.handle).decode())
    abi.check(st, c.handle)
    return out


_DTYPES = {torch.float32: abi.OXG_DTYPE_F32, torch.bfloat16: abi.OXG_DTYPE_BF16, torch.float16: abi.OXG_DTYPE_F16}
_RULES = {"floor": abi.OXG_MX_FLOOR, "noclip": abi.OXG_MX_NOCLIP}
_main_thread = threading.main_thread().ident
# Other threads' contexts, by thread and device. They stay when a thread ends (ending one would synchronise, in the
# middle of whatever other threads do, a capture perhaps); a later thread that is given the same identity takes them over.
_thread_ctx: dict[tuple[int, int], abi.Context] = {}
_MOST = 0x7FFFFE00  # rows, columns and k of a product: 32-bit numbers with room for a tile


def device_context(x: torch.Tensor, ctx: abi.Context | None) -> abi.Context:
    """The given context, or the calling thread's own on x's device (the main
    thread's is the process's default one), bound to torch's current stream there.

    A thread's context outlives it. What a graph that was captured in the thread
    finds wrong in a later replay is reported by that context's ``sync``: keep
    what ``device_context(x, None)`` returns there."""
    return _context_on(x.get_device(), ctx)


def _context_on(index: int, ctx: abi.Context | None) -> abi.Context:
    if ctx is None:
        thread = threading.get_ident()
        if thread != _main_thread:
            ctx = _thread_ctx.get((thread, index))
            if ctx is None:
                ctx = _thread_ctx[thread, index] = abi.Context(index)
        else:
            ctx = _device_ctx.get(index)
            if ctx is None:
                ctx = _main_context(index)
    elif ctx.device != index:
        raise ValueError(f"the context is on cuda:{ctx.device}, the input on cuda:{index}")
    return _bind(ctx)


def check_status(status: int, ctx: abi.Context) -> None:
    """ValueError where the library refuses shapes or arguments, OxgError else."""
    if status in (abi.OXG_ERR_SHAPE, abi.OXG_ERR_INVALID_ARG):
        raise ValueError(ctx.lib.oxg_last_error(ctx.handle).decode())
    abi.check(status, ctx.handle)


def rows_of(x: torch.Tensor, name: str) -> tuple[torch.Tensor, int, int]:
    """x [..., width] as a 2-D view (a copy only where its rows have no common
    pitch or are not contiguous) with its row count and pitch in elements."""
    if not x.is_cuda or x.dtype not in _DTYPES:
        raise ValueError(f"{name} must be a float32, bfloat16 or float16 CUDA tensor")
    if x.dim() == 0:
        raise ValueError(f"{name} must have at least one dimension")
    if x.dim() == 2 and x.is_contiguous():
        return x, x.shape[0], x.shape[1]
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1]) if x.shape[-1] else x.reshape(0, 0)
    if x.shape[1] > 1 and x.stride(1) != 1 or x.shape[0] > 1 and x.stride(0) < x.shape[1]:
        x = x.contiguous()
    return x, x.shape[0], x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _empty(rows: int, cols: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    """A new matrix (empty_strided is torch's quickest way to one: 1.5 us, new_empty 2.0, empty 2.4)."""
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=device)


def scale_rule_code(rule: str) -> int:
    if rule not in _RULES:
        raise ValueError(f"unknown scale rule {rule!r}: one of {', '.join(_RULES)}")
    return _RULES[rule]


def quantized_like(x: torch.Tensor, cols: int, rows: int, tiled: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """Empty blocks and scales for the MXFP4 form of x's rows at `cols` columns."""
    if cols % 32:
        raise ValueError(f"cols must be divisible by 32, got {cols}")
    if tiled and x.dim() != 2:
        raise ValueError(f"tiled scales are those of one matrix: the input must have 2 dimensions, got {x.dim()}")
    blocks = _empty(rows, cols // 2, torch.uint8, x.device)
    if tiled:
        return blocks, x.new_empty(((cols + 127) // 128, rows, 4), dtype=torch.uint8)
    scales = _empty(rows, cols // 32, torch.uint8, x.device)
    if x.dim() == 2:
        return blocks, scales
    lead = x.shape[:-1]
    return blocks.view(*lead, cols // 2), scales.view(*lead, cols // 32)


def quantize_mxfp4(x: torch.Tensor, *, row_scale: torch.Tensor | None = None, scale_rule: str = "floor",
                   tiled: bool = False, ctx: abi.Context | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., cols] (float32, bfloat16 or float16 CUDA tensor, cols a multiple
    of 32) -> (blocks [..., cols / 2] uint8, scales [..., cols / 32] uint8), the
    nearest E2M1 codes under a power-of-two scale for each 32 elements.

    row_scale: float32 factor for each row, applied first. scale_rule: "floor"
    (the largest element of a block lands in [4, 8) and what is above 6 becomes
    6) or "noclip" (it lands in (3, 6]). tiled: scales as the products read
    them, [ceil(cols / 128), rows, 4] (x must be a matrix). A block that holds an
    infinity or a NaN reads as NaN."""
    x2, rows, ld = rows_of(x, "x")
    cols = x.shape[-1]
    blocks, scales = quantized_like(x, cols, rows, tiled)
    if row_scale is not None:
        if row_scale.dtype != torch.float32 or row_scale.numel() != rows or row_scale.device != x.device:
            raise ValueError(f"row_scale must be {rows} float32 values on {x.device}")
        row_scale = row_scale.contiguous()
    c = device_context(x, ctx)
    check_status(c.lib.oxg_quantize_mxfp4(c.handle, x2.data_ptr(), _DTYPES[x.dtype], rows, cols, ld,
                                          None if row_scale is None else row_scale.data_ptr(),
                                          scale_rule_code(scale_rule), int(tiled), blocks.data_ptr(),
                                          scales.data_ptr()), c)
    return blocks, scales


def tile_scales(scales: torch.Tensor, *, ctx: abi.Context | None = None) -> torch.Tensor:
    """Scales [..., rows, k / 32] uint8 as the products read them:
    [..., ceil(k / 128), rows, 4], zero where k ends inside a 128-element stretch."""
    if not scales.is_cuda or scales.dtype != torch.uint8 or scales.dim() < 2:
        raise ValueError("scales must be a uint8 CUDA tensor [..., rows, k / 32]")
    scales = scales.contiguous()
    *lead, rows, kb = scales.shape
    out = torch.empty(*lead, (kb + 3) // 4, rows, 4, dtype=torch.uint8, device=scales.device)
    c = device_context(scales, ctx)
    groups = 1
    for n in lead:
        groups *= n
    check_status(c.lib.oxg_mxfp4_tile_scales(c.handle, scales.data_ptr(), groups, rows, 32 * kb, out.data_ptr()), c)
    return out


def _operand(blocks: torch.Tensor, scales: torch.Tensor, name: str, dim: int, index: int,
             ctx: abi.Context | None) -> tuple[torch.Tensor, torch.Tensor]:
    """One operand's blocks and tiled scales, contiguous, checked against each other."""
    if blocks.dtype != torch.uint8 or scales.dtype != torch.uint8 or not blocks.is_cuda or \
            blocks.get_device() != index or scales.get_device() != index:
        raise ValueError(f"{name}'s blocks and scales must be uint8 tensors on one CUDA device with the other operand")
    shape = blocks.shape
    if len(shape) != dim:
        raise ValueError(f"{name}'s blocks must have {dim} dimensions, got {tuple(shape)}")
    lead, rows, k = shape[:-2], shape[-2], 2 * shape[-1]
    if k == 0 or k % 32:
        raise ValueError(f"k must be a positive multiple of 32, got {k}")
    if rows > _MOST or k > _MOST:
        raise ValueError(f"{name} is too large: {rows} rows of {k} elements")
    if scales.shape != (*lead, (k + 127) // 128, rows, 4):
        if scales.shape != (*lead, rows, k // 32):
            raise ValueError(f"{name}'s scales must be {(*lead, (k + 127) // 128, rows, 4)} (tiled) or "
                             f"{(*lead, rows, k // 32)}, got {tuple(scales.shape)}")
        scales = tile_scales(scales, ctx=ctx)
    return blocks.contiguous(), scales.contiguous()


def _output(out: torch.Tensor | None, out_dtype: torch.dtype, m: int, n: int, a: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """The output tensor (a new one on a's device), its type's code and its row pitch."""
    if out is None:
        if out_dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"out_dtype must be float32 or bfloat16, got {out_dtype}")
        return _empty(m, n, out_dtype, a.device), _DTYPES[out_dtype], n
    if out.shape != (m, n) or out.dtype not in (torch.float32, torch.bfloat16) or out.device != a.device or \
            (n > 1 and out.stride(1) != 1) or (m > 1 and out.stride(0) < n):
        raise ValueError(f"out must be a float32 or bfloat16 [{m}, {n}] on {a.device} with contiguous rows")
    return out, _DTYPES[out.dtype], out.stride(0) if m > 1 else n


def _bias(bias: torch.Tensor | None, shape: tuple, index: int) -> torch.Tensor | None:
    if bias is None:
        return None
    if bias.dtype != torch.bfloat16 or bias.shape != shape or bias.get_device() != index:
        raise ValueError(f"bias must be bfloat16 {shape} on cuda:{index}, got {bias.dtype} {tuple(bias.shape)}")
    return bias.contiguous()


def mxfp4_matmul(a_blocks: torch.Tensor, a_scales: torch.Tensor, b_blocks: torch.Tensor, b_scales: torch.Tensor, *,
                 bias: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16,
                 out: torch.Tensor | None = None, ctx: abi.Context | None = None) -> torch.Tensor:
    """a [m, k] times b [n, k] transposed, plus ``bias`` [n] (bfloat16), both
    operands MXFP4 (blocks [rows, k / 2], scales tiled [ceil(k / 128), rows, 4] or
    [rows, k / 32]); f32 sums, returned as ``out_dtype`` (float32 or bfloat16) or
    in ``out``, in its own type (contiguous rows of any pitch)."""
    index = a_blocks.get_device()
    a_blocks, a_scales = _operand(a_blocks, a_scales, "a", 2, index, ctx)
    b_blocks, b_scales = _operand(b_blocks, b_scales, "b", 2, index, ctx)
    m, half = a_blocks.shape
    n, k = b_blocks.shape[0], 2 * half
    if 2 * b_blocks.shape[1] != k:
        raise ValueError(f"a has rows of {k} elements, b of {2 * b_blocks.shape[1]}")
    out, code, ldo = _output(out, out_dtype, m, n, a_blocks)
    bias = _bias(bias, (n,), index)
    c = _context_on(index, ctx)
    check_status(c.lib.oxg_mxfp4_matmul(c.handle, a_blocks.data_ptr(), a_scales.data_ptr(), m, b_blocks.data_ptr(),
                                        b_scales.data_ptr(), n, k, None if bias is None else bias.data_ptr(),
                                        out.data_ptr(), code, ldo), c)
    return out


def mxfp4_grouped_matmul(a_blocks: torch.Tensor, a_scales: torch.Tensor, counts: torch.Tensor, b_blocks: torch.Tensor,
                         b_scales: torch.Tensor, *, bias: torch.Tensor | None = None,
                         out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None,
                         ctx: abi.Context | None = None) -> torch.Tensor:
    """Runs of a's rows, each times a matrix of its own: the first counts[0] rows
    of a [m, k] times b[0] [n, k] transposed, the next counts[1] times b[1] and so
    on (counts: int32 CUDA tensor, zeros allowed; ``MoELayer.dispatch`` returns
    them). bias [groups, n] bfloat16. Rows past the last group keep what ``out``
    held (nothing in particular in a new one). Counts that are negative or add
    up to more than m are reported by the context's next ``sync``
    (``device_context(a_blocks, None).sync()`` without one of your own)."""
    index = a_blocks.get_device()
    a_blocks, a_scales = _operand(a_blocks, a_scales, "a", 2, index, ctx)
    b_blocks, b_scales = _operand(b_blocks, b_scales, "b", 3, index, ctx)
    m, half = a_blocks.shape
    k = 2 * half
    groups, n = b_blocks.shape[:2]
    if 2 * b_blocks.shape[2] != k:
        raise ValueError(f"a has rows of {k} elements, b of {2 * b_blocks.shape[2]}")
    if counts.dtype != torch.int32 or counts.shape != (groups,) or counts.get_device() != index:
        raise ValueError(f"counts must be int32 [{groups}] on cuda:{index}, got {counts.dtype} {tuple(counts.shape)}")
    counts = counts.contiguous()
    out, code, ldo = _output(out, out_dtype, m, n, a_blocks)
    bias = _bias(bias, (groups, n), index)
    c = _context_on(index, ctx)
    check_status(c.lib.oxg_mxfp4_grouped_matmul(c.handle, a_blocks.data_ptr(), a_scales.data_ptr(), m, counts.data_ptr(),
                                                groups, b_blocks.data_ptr(), b_scales.data_ptr(), n, k,
                                                None if bias is None else bias.data_ptr(), out.data_ptr(), code, ldo), c)
    return out
