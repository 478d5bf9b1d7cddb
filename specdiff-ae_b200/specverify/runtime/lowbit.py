"""Low-bit decoder-layer work around the verify path.

* :func:`add_rms_norm` -- the residual's addition and ``LlamaRMSNorm``
  (``runtime/llama_target_model.py:124-138``) in one pass, with a 16-bit output
  or an e4m3 one with a scale per row.

CUDA tensors only; errors raise :class:`specverify.SpecVerifyError`.
"""

from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _lib

__all__ = ["add_rms_norm"]

_HALF = (torch.bfloat16, torch.float16)


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
    dev = _lib.require_cuda(x, residual, weight, residual_out)
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
    if residual_out is None:
        residual_out = torch.empty((rows, cols), dtype=x.dtype, device=dev)
    else:
        _rows_ok(residual_out, x.shape, x.dtype, "residual_out")
        if rows > 1 and residual_out.stride(0) < cols:
            raise _lib.SpecVerifyError(-1, f"residual_out's rows overlap (stride {residual_out.stride(0)})")
    y = torch.empty((rows, cols), dtype=torch.float8_e4m3fn if fp8 else x.dtype, device=dev)
    scale = torch.empty(rows, dtype=torch.float32, device=dev) if fp8 else None
    st = _lib.launch(dev, _lib.load().tv_add_rms_norm, x.data_ptr(), x.stride(0), residual.data_ptr(),
                     residual.stride(0), weight.data_ptr(), residual_out.data_ptr(), residual_out.stride(0),
                     y.data_ptr(), cols, scale.data_ptr() if fp8 else None, rows, cols, float(eps),
                     _lib.TV_BF16 if x.dtype == torch.bfloat16 else _lib.TV_F16)
    _lib.check(st, "tv_add_rms_norm")
    return (y, scale, residual_out) if fp8 else (y, residual_out)
