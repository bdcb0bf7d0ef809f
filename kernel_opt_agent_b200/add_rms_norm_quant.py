"""add_rms_norm_quant plugin module: residual addition, RMS norm and FP8 quantisation of a layer's
input in one kernel -- what ``rms_norm`` and the block quantisation of ``swiglu_input_quant`` do
apart, with the module contract of the reference's plugins (``kernels/__init__.py:3-8``); the
reference registers no fused form.

    kernel_fn(x, residual, weight, eps=1e-6, *, group=128, inplace=False) -> (y_fp8, y_scale, residual_out)

x, residual [..., N] bf16 or fp16, weight [N] of the same type; ``residual=None`` leaves the addition
out (the first layer; residual_out is then x itself).

    h = T(x + residual)                       returned as residual_out
    y = h / sqrt(mean(h^2) + eps) * weight    (fp32), held as y_fp8 * y_scale

``group`` columns share a scale: 128 or 32 (N a multiple of it; y_scale is [N / group, M], M the number
of rows, as ``swiglu_input_quant`` lays its scales out) or None, one scale per row (y_scale [M]).
y_fp8 is e4m3, shaped like x; the largest magnitude of a group is held as 448.  Scales are fp32 and no powers of two in any
grouping: they go to products that scale partial sums in fp32, not to block-scaled ones that want e8m0 scales.  ``inplace=True`` writes
residual_out over ``residual``, so that a decode loop keeps one residual buffer (x may be the residual
itself; it must not overlap it otherwise).

``kernel_fn`` runs ``tokmix_add_rms_norm_quant`` (``csrc/add_rms_norm_quant.cu``), no fallback."""

from __future__ import annotations

import torch

from . import _lib

KERNEL_TYPE = "add_rms_norm_quant"
_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
MAX_N = 65536
MAX_ROWS = 2 ** 31 - 256


def kernel_fn(x: torch.Tensor, residual: torch.Tensor | None, weight: torch.Tensor, eps: float = 1e-6, *,
              group: int | None = 128, inplace: bool = False):
    dtype, shape, dev = x.dtype, x.shape, x.device
    if dtype not in _DTYPES or weight.dtype != dtype or not shape:
        raise ValueError("x and weight must both be bfloat16 or both float16")
    if residual is not None and (residual.dtype != dtype or residual.shape != shape):
        raise ValueError("residual must have the shape and type of x")
    if not x.is_cuda or weight.device != dev or (residual is not None and residual.device != dev):
        raise ValueError("x, residual and weight must be CUDA tensors on one device")
    if group not in (None, 32, 128):
        raise ValueError("group must be 32, 128 or None (one scale per row)")
    n = shape[-1]
    if n == 0 or n % (group or 8) != 0 or n > MAX_N:
        raise ValueError(f"the last dimension of x must be a multiple of {group or 8} and at most {MAX_N} (got {n})")
    if weight.shape != (n,):
        raise ValueError("weight must be [N], N the last dimension of x")
    if inplace and (residual is None or not residual.is_contiguous() or residual.data_ptr() % 16):
        raise ValueError("inplace=True needs a contiguous, 16-byte aligned residual")
    rows = x.numel() // n
    if rows > MAX_ROWS:
        raise ValueError(f"at most {MAX_ROWS} rows (got {rows})")
    given, x, w = x, _lib.aligned(x), _lib.aligned(weight)
    if inplace and 0 < abs(x.data_ptr() - residual.data_ptr()) < 2 * rows * n:
        raise ValueError("inplace=True: x must be the residual itself or share no memory with it")
    y = torch.empty_like(x, dtype=torch.float8_e4m3fn)
    y_scale = _lib.empty((n // group, rows) if group else (rows,), torch.float32, dev)
    if residual is None:
        res_out, res_ptr, out_ptr = given, None, None
    else:
        res = residual if inplace else _lib.aligned(residual)
        res_out = res if inplace else torch.empty_like(x)
        res_ptr, out_ptr = res.data_ptr(), res_out.data_ptr()
    rc = _lib.call_on(dev, _lib.load().tokmix_add_rms_norm_quant, x.data_ptr(), res_ptr, w.data_ptr(), out_ptr, y.data_ptr(),
                      y_scale.data_ptr(), rows, n, group or 0, _DTYPES[dtype], eps, _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc, "add_rms_norm_quant")
    return y, y_scale, res_out


def get_inputs(M: int = 2048, N: int = 4096, dtype: torch.dtype = torch.bfloat16, seed: int = 42,
               group: int | None = 128, device: str = "cuda") -> dict:
    gen = torch.Generator().manual_seed(seed)
    return {"x": torch.randn(M, N, generator=gen).to(dtype).to(device),
            "residual": (4 * torch.randn(M, N, generator=gen)).to(dtype).to(device),
            "weight": (1 + 0.2 * torch.randn(N, generator=gen)).to(dtype).to(device), "group": group}


def get_flops(M: int = 2048, N: int = 4096) -> int:
    return 7 * M * N


def get_bytes(M: int = 2048, N: int = 4096, element_size: int = 2, group: int | None = 128) -> int:
    """x and residual read, residual_out and y_fp8 written, one scale per group, the weight read once."""
    return M * N * (3 * element_size + 1) + N * element_size + M * (N // group if group else 1) * 4
