"""Low-bit decoder-layer work around the verify path.

* :func:`add_rms_norm` -- the residual's addition and ``LlamaRMSNorm``
  (``runtime/llama_target_model.py:124-138``) in one pass, with a 16-bit output
  or an e4m3 one with a scale per row.
* :func:`w4_linear` -- the projections of such a layer with 4-bit weights and
  group scales, laid out by :func:`quantize_w4`.

CUDA tensors only; errors raise :class:`specverify.SpecVerifyError`.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple, Union

import torch

from .. import _lib

__all__ = ["add_rms_norm", "dequantize_w4", "quantize_w4", "w4_linear"]

_HALF = {torch.bfloat16: _lib.TV_BF16, torch.float16: _lib.TV_F16}


def _rows_ok(t: torch.Tensor, shape, dtype, what: str) -> None:
    if t.shape != shape or (t.stride(1) != 1 and shape[1] > 1):
        raise _lib.SpecVerifyError(-1, f"{what} must be {tuple(shape)} with unit column stride, got "
                                       f"{tuple(t.shape)} strides {t.stride()}")
    if t.dtype != dtype:
        raise _lib.SpecVerifyError(-2, f"{what} must be {dtype}, got {t.dtype}")


def add_rms_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, eps: float, *, fp8: bool = False,
                 residual_out: Optional[torch.Tensor] = None
                 ) -> Union[Tuple[torch.Tensor, torch.Tensor], Tuple[torch.Tensor, torch.Tensor, torch.Tensor]]:
    """``h = x + residual`` and the RMSNorm of ``h``, one launch (``tv_add_rms_norm``).

    x, residual [rows, cols] and weight [cols], bf16 or fp16 (one type), unit
    column stride.  Returns ``(y, h)``: ``y`` as
    :func:`specverify.draft.spec_decode.rms_norm` of ``h``, or with ``fp8``
    ``(y, scale, h)``: ``y`` float8_e4m3fn and ``scale`` [rows] fp32 with
    ``y * scale[:, None]`` the normalised row (largest magnitude at 448;
    scale 0 for a row of zeros, NaN for a row with a NaN).  ``h`` is written to
    ``residual_out`` when given, which may be ``residual`` itself.
    """
    shape, dtype = x.shape, x.dtype
    # one look at what every call has right; the exact complaint is looked for when it is not
    if not (x.is_cuda and len(shape) == 2 and dtype in _HALF and x.stride()[1] == 1 and residual.shape == shape
            and residual.stride()[1] == 1 and residual.dtype is dtype and weight.dtype is dtype
            and weight.shape == shape[1:] and weight.stride()[0] == 1 and residual.device == x.device == weight.device
            and residual_out is None):
        _check_add_rms_norm(x, residual, weight, residual_out)
    rows, cols = shape
    _lib.fit_i32("tv_add_rms_norm", rows, cols)
    h = torch.empty_like(x, memory_format=torch.contiguous_format) if residual_out is None else residual_out
    if fp8:
        y = torch.empty_like(x, dtype=torch.float8_e4m3fn, memory_format=torch.contiguous_format)
        scale = x.new_empty(rows, dtype=torch.float32)
        scale_ptr = scale.data_ptr()
    else:
        y, scale_ptr = torch.empty_like(x, memory_format=torch.contiguous_format), None
    st = _lib.launch(x.device, _lib.load().tv_add_rms_norm, x.data_ptr(), x.stride(0), residual.data_ptr(),
                     residual.stride(0), weight.data_ptr(), h.data_ptr(), h.stride(0), y.data_ptr(), cols, scale_ptr,
                     rows, cols, eps, _HALF[dtype])
    if st != 0:
        _lib.check(st, "tv_add_rms_norm")
    return (y, scale, h) if fp8 else (y, h)


def _check_add_rms_norm(x, residual, weight, residual_out) -> None:
    _lib.require_cuda(x, residual, weight, residual_out)
    if x.dim() != 2:
        raise _lib.SpecVerifyError(-1, f"x must be [rows, cols], got {tuple(x.shape)}")
    if x.dtype not in _HALF:
        raise _lib.SpecVerifyError(-2, f"x must be bfloat16 or float16, got {x.dtype}")
    rows, cols = x.shape
    _rows_ok(x, x.shape, x.dtype, "x")
    _rows_ok(residual, x.shape, x.dtype, "residual")
    if weight.shape != (cols,) or weight.dtype != x.dtype or (cols > 1 and weight.stride(0) != 1):
        raise _lib.SpecVerifyError(-1, f"weight must be a dense [{cols}] {x.dtype}, got {tuple(weight.shape)} "
                                       f"{weight.dtype}")
    if residual_out is not None:
        _rows_ok(residual_out, x.shape, x.dtype, "residual_out")
        if rows > 1 and residual_out.stride(0) < cols:
            raise _lib.SpecVerifyError(-1, f"residual_out's rows overlap (stride {residual_out.stride(0)})")


# nibble i of a packed word holds weight 8 c + _ORDER[i]
_ORDER = (0, 2, 4, 6, 1, 3, 5, 7)


def quantize_w4(weight: torch.Tensor, group: int = 128) -> Tuple[torch.Tensor, torch.Tensor]:
    """Round a weight [N, K] (bf16 or fp16) to 4 bits with a scale per ``group``
    consecutive k of a row: ``scale = max|w| / 7`` rounded to the weight's type,
    ``q = round(w / scale)`` in -8 .. 7.  Returns ``(qweight, scales)``: int32
    [N, K / 8] (layout at ``tv_w4_linear``) and [N, K / group].  Plain torch
    operations on the weight's device, done once when a model is loaded.
    :func:`w4_linear` takes scales of 2^-80 to 2^30 in bf16 (weights of 2^-78 to
    2^32 as a group's largest) and up to 8188 in fp16, or 0.
    """
    if weight.dim() != 2 or weight.dtype not in _HALF:
        raise _lib.SpecVerifyError(-1, f"weight must be [N, K] in bfloat16 or float16, got {tuple(weight.shape)} "
                                       f"{weight.dtype}")
    n, k = weight.shape
    if group < 32 or group % 32 or k < group or k % group:
        raise _lib.SpecVerifyError(-1, f"group {group} must be a multiple of 32 that divides K {k}")
    w = weight.float().view(n, k // group, group)
    scales = (w.abs().amax(-1) / 7.0).to(weight.dtype)
    s = scales.float()[:, :, None]
    u = torch.where(s > 0, torch.round(w / s), 0.0).clamp(-8, 7).to(torch.int32).view(n, k // 8, 8) + 8
    q = torch.zeros((n, k // 8), dtype=torch.int32, device=weight.device)
    for i, o in enumerate(_ORDER):
        q |= u[:, :, o] << (4 * i)
    return q, scales


def dequantize_w4(qweight: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The weight [N, K] that ``(qweight, scales)`` stand for, in the scales' type."""
    n, k = qweight.shape[0], qweight.shape[1] * 8
    u = torch.empty((n, k // 8, 8), dtype=torch.float32, device=qweight.device)
    for i, o in enumerate(_ORDER):
        u[:, :, o] = ((qweight >> (4 * i)) & 15).float() - 8.0
    w = u.view(n, scales.shape[1], -1) * scales.float()[:, :, None]
    return w.view(n, k).to(scales.dtype)


def w4_linear(x: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, *, x_scale: Optional[torch.Tensor] = None,
              out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ W.T`` for a 4-bit weight W [N, K] (``tv_w4_linear``), W as
    :func:`dequantize_w4` has it, rounded to the scales' type.

    x [..., K]: the scales' type (bf16 or fp16), or float8_e4m3fn with
    ``x_scale`` (fp32, one per row, shape [...]) as :func:`add_rms_norm`
    returns them; unit stride on K.  qweight [N, K / 8] int32 and scales
    [N, K / group] as :func:`quantize_w4` lays them out (group a multiple of
    32).  Returns [..., N] in the scales' type, summed in fp32; ``out``, when
    given, is [rows, N] with unit stride on N and overlaps no input.  ``status`` (int32 [1], zeroed by
    the caller) receives a nonzero code if a bounded wait on the device ran out;
    the outputs it concerns are NaN.
    """
    n, words = qweight.shape if qweight.dim() == 2 else (0, 0)
    k, fp8 = words * 8, x.dtype is torch.float8_e4m3fn
    groups = scales.shape[-1]
    if not (x.is_cuda and x.dim() == 2 and x.shape[1] == k and x.stride()[1] == 1 and scales.dim() == 2
            and scales.shape[0] == n > 1 and qweight.dtype is torch.int32 and scales.dtype in _HALF
            and qweight.stride()[1] == 1 and scales.stride()[1] == 1 and (x.dtype is scales.dtype if not fp8 else False)
            and x_scale is None and out is None and groups and k % (32 * groups) == 0
            and (status is None or (status.dtype is torch.int32 and status.numel() == 1 and status.device == x.device))
            and x.device == qweight.device == scales.device):
        _check_w4_linear(x, qweight, scales, x_scale, out, status)
    x2 = x if x.dim() == 2 else x.reshape(-1, k)
    rows = x2.shape[0]
    _lib.fit_i32("tv_w4_linear", rows, n, k)
    if out is None:
        res = scales.new_empty((rows, n) if x.dim() == 2 else x.shape[:-1] + (n,))
        o_sm = n
    else:
        res, o_sm = out, out.stride(0)
    kind = _HALF[scales.dtype]
    a = _lib.W4Args(_lib.TV_E4M3 if fp8 else kind, kind, rows, n, k, k // groups, x2.data_ptr(), x2.stride(0),
                    x_scale.data_ptr() if fp8 else None, qweight.data_ptr(), qweight.stride(0) if n > 1 else words,
                    scales.data_ptr(), scales.stride(0), res.data_ptr(), o_sm)
    if status is not None:
        a.status = status.data_ptr()
    lib = _lib.load()
    st = _lib.launch(x.device, lib.tv_w4_linear, a)
    if st == _lib.TV_ERR_WORKSPACE:      # rows that have to be laid out anew first; nothing was launched
        need = ctypes.c_size_t(0)
        st = lib.tv_w4_workspace_size(a, need)
        if st == 0:
            ws = x.new_empty(need.value, dtype=torch.uint8)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need.value
            st = _lib.launch(x.device, lib.tv_w4_linear, a)
    if st != 0:
        _lib.check(st, "tv_w4_linear")
    return res


def _check_w4_linear(x, qweight, scales, x_scale, out, status) -> None:
    _lib.require_cuda(x, qweight, scales, x_scale, out, status)
    if status is not None and (status.dtype != torch.int32 or status.numel() != 1):
        raise _lib.SpecVerifyError(-2, f"status must be one int32, got {tuple(status.shape)} {status.dtype}")
    if x.dim() < 1 or qweight.dim() != 2 or scales.dim() != 2 or qweight.shape[0] != scales.shape[0]:
        raise _lib.SpecVerifyError(-1, f"x {tuple(x.shape)}, qweight {tuple(qweight.shape)}, scales "
                                       f"{tuple(scales.shape)}")
    n, k = qweight.shape[0], qweight.shape[1] * 8
    groups = scales.shape[1]
    if x.shape[-1] != k or groups < 1 or k % groups or (k // groups) % 32 or n < 1:
        raise _lib.SpecVerifyError(-1, f"x {tuple(x.shape)} and scales {tuple(scales.shape)} do not fit a "
                                       f"[{n}, {k}] weight with groups of a multiple of 32")
    if qweight.dtype != torch.int32 or scales.dtype not in _HALF:
        raise _lib.SpecVerifyError(-2, f"qweight {qweight.dtype} must be int32, scales {scales.dtype} 16-bit")
    fp8 = x.dtype == torch.float8_e4m3fn
    if not fp8 and x.dtype != scales.dtype:
        raise _lib.SpecVerifyError(-2, f"x {x.dtype} must be {scales.dtype} or float8_e4m3fn")
    if fp8 != (x_scale is not None):
        raise _lib.SpecVerifyError(-8, "x_scale goes with a float8_e4m3fn x, and only with it")
    if x.stride(-1) != 1 or qweight.stride(1) != 1 or (groups > 1 and scales.stride(1) != 1):
        raise _lib.SpecVerifyError(-3, "x, qweight and scales must have unit stride on their last dimension")
    if fp8 and (x_scale.dtype != torch.float32 or x_scale.shape != x.shape[:-1] or not x_scale.is_contiguous()):
        raise _lib.SpecVerifyError(-1, f"x_scale must be a contiguous float32 {list(x.shape[:-1])}")
    rows = x.numel() // k
    if out is not None and (out.shape != (rows, n) or out.dtype != scales.dtype or (n > 1 and out.stride(1) != 1)
                            or (rows > 1 and out.stride(0) < n)):
        raise _lib.SpecVerifyError(-1, f"out must be [{rows}, {n}] {scales.dtype} with unit column stride")
