"""qk_norm_rope plugin module: the RMS norm of every query and key head and the position rotation in one
pass -- what ``rms_norm`` and ``qkv_part_rope`` do apart, between a layer's projection and its attention; with the
module contract of the reference's plugins (``kernels/__init__.py:3-8``).  The reference registers no fused form.

    kernel_fn(q, k, q_weight, k_weight, cos, sin, positions=None, *, eps=1e-6, nope_dim=None, sections=None,
              interleaved=False) -> (q_out, k_out)

q [B, S, Hq, D] and k [B, S, Hkv, D] bf16 or fp16, D 64, 128 or 256, any lengths (a decode step: S = 1); they may be
slices of a packed projection and are read where they lie.  q_weight, k_weight [D], of that type or fp32.

    n = x / sqrt(mean(x^2) + eps) * weight             for every head row x
    y_j = n_j cos_j - n_{j+half} sin_j,   y_{j+half} = n_j sin_j + n_{j+half} cos_j

cos, sin [rows, half] fp32 are tables by position; the 2 * half columns behind the first ``nope_dim`` are rotated
(default: the last ones, as in ``qkv_part_rope``; ``nope_dim=0`` with 2 * half < D: the first ones), half and nope_dim multiples of
8.  fp32 arithmetic, rounded once; the outputs are contiguous, ready for ``flash_attention_2`` (layout "bshd"),
``kv8_append`` and ``kv8_attention``.

positions: int32 [B, S], the table row of every token; None: its index in its sequence.  With ``sections`` =
(n_0, .., n_{A-1}), which add up to half (images: time, height, width), positions is [A, B, S] and every pair takes the row of one
axis: the first n_0 pairs axis 0, the next n_1 axis 1, and so on; or, ``interleaved``, pair j axis j % A while j < A * n_axis
and axis 0 behind that.  A position outside the tables makes the token's rotated columns NaN and is reported as
``TokmixDeviceError`` by a later call of this module or of its gradient, or by ``check_device_status``.

Squares are summed in fp32: a row whose squares add up to 2^128 overflows (magnitudes of 2^60, D 256).  ``eps`` may be 0: a row of
zeros is then 0 / 0 (NaN, in the weights' gradients too), and one of magnitudes below 2^-62 loses digits of its squares, below 2^-74
all of them.

``kernel_fn`` runs ``tokmix_qk_norm_rope_fwd`` (``csrc/qk_norm_rope.cu``), no fallback.  ``training.qk_norm_rope`` is this with
its gradient (``qk_norm_rope_bwd``) behind autograd."""

from __future__ import annotations

import ctypes
import functools

import torch

from . import _kv8, _lib

KERNEL_TYPE = "qk_norm_rope"
HEAD_DIMS = (64, 128, 256)
MAX_AXES = 4
_NO_STRIDES = (0,) * 6


@functools.lru_cache(maxsize=64)
def _pair_axis(half: int, sections: tuple, interleaved: bool):
    """The axis of every pair as a C array."""
    axes = len(sections)
    if not 1 <= axes <= MAX_AXES or any(n < 0 for n in sections) or sum(sections) != half:
        raise ValueError(f"sections must be 1 to {MAX_AXES} counts that add up to the {half} pairs (got {sections})")
    if interleaved:
        axis = [j % axes if j < axes * sections[j % axes] else 0 for j in range(half)]
    else:
        axis = [a for a, n in enumerate(sections) for _ in range(n)]
    if any(axis.count(a) != n for a, n in enumerate(sections)):
        raise ValueError(f"{half} interleaved pairs cannot hold sections {sections}")
    return (ctypes.c_uint8 * half)(*axis)


def describe(q, k, q_weight, k_weight, cos, sin, positions, eps, nope_dim, sections, interleaved, grads=None):
    """Checks a call (of the gradient, with grads = (dq_out, dk_out)) and allocates its outputs; returns its C
    description as bytes, the outputs and the tensors it points to."""
    qs, ks, dev, dtype = q.shape, k.shape, q.device, q.dtype
    if len(qs) != 4 or len(ks) != 4 or qs[0] != ks[0] or qs[1] != ks[1] or qs[3] != ks[3]:
        raise ValueError("q and k must be [B, S, heads, D] with equal B, S and D")
    batch, seq, hq, d = qs
    hk = ks[2]
    if dtype not in _kv8.IO_DTYPES or k.dtype != dtype:
        raise ValueError("q and k must both be bfloat16 or both float16")
    if d not in HEAD_DIMS or hq == 0 or hk == 0:
        raise ValueError(f"head_dim must be one of {HEAD_DIMS}, with at least one head of each kind")
    if batch >= 1 << 31 or seq >= 1 << 31:
        raise ValueError("fewer than 2^31 sequences and tokens per sequence")
    if not q.is_cuda or k.device != dev or q_weight.device != dev or k_weight.device != dev or cos.device != dev or (
            sin.device != dev):
        raise ValueError("all tensors must be CUDA tensors on one device")
    wtype = q_weight.dtype
    if q_weight.shape != (d,) or k_weight.shape != (d,):
        raise ValueError(f"q_weight and k_weight must be [{d}]")
    if k_weight.dtype != wtype or wtype not in (dtype, torch.float32):
        raise ValueError("q_weight and k_weight must have the type of q or be float32")
    if cos.ndim != 2 or cos.shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos and sin must be float32 [rows, pairs]")
    rows, half = cos.shape
    if half == 0 or half % 8 or 2 * half > d:
        raise ValueError("the number of pairs must be a positive multiple of 8, at most head_dim / 2")
    if nope_dim is None:
        nope_dim = d - 2 * half
    if nope_dim < 0 or nope_dim % 8 or nope_dim + 2 * half > d:
        raise ValueError("nope_dim must be a multiple of 8 with nope_dim + 2 * pairs <= head_dim")
    if rows == 0 or rows >= 1 << 31:
        raise ValueError("cos and sin need between 1 and 2^31 - 1 rows")
    axes, pair_axis = 1, None
    if sections is not None:
        pair_axis, axes = _pair_axis(half, tuple(sections), bool(interleaved)), len(sections)
    elif interleaved:
        raise ValueError("interleaved needs sections")
    if positions is None:
        if sections is not None:
            raise ValueError("sections need positions [axes, B, S]")
        if rows < seq:
            raise ValueError(f"cos and sin have {rows} rows for {seq} positions")
    else:
        shape = (batch, seq) if sections is None else (axes, batch, seq)
        if positions.dtype != torch.int32 or positions.shape != shape or positions.device != dev:
            raise ValueError(f"positions must be int32 {list(shape)} on the device of q")
        positions = positions.contiguous()
    dq = dk = None
    gs = _NO_STRIDES
    if grads is not None:
        dq, dk = grads
        if dq.shape != qs or dq.dtype != dtype or dq.device != dev:
            raise ValueError("dq_out must have the shape, type and device of q")
        if dk.shape != ks or dk.dtype != dtype or dk.device != dev:
            raise ValueError("dk_out must have the shape, type and device of k")
        dq, gq = _kv8.token_strides(dq)
        dk, gk = _kv8.token_strides(dk)
        gs = gq + gk
    q, sq = _kv8.token_strides(q)
    k, sk = _kv8.token_strides(k)
    cos, sin, q_weight, k_weight = _lib.aligned(cos), _lib.aligned(sin), _lib.aligned(q_weight), _lib.aligned(k_weight)
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
    args = _lib.QK_NORM_ROPE.pack(
        q.data_ptr(), k.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(), cos.data_ptr(), sin.data_ptr(),
        0 if positions is None else positions.data_ptr(), ctypes.addressof(pair_axis) if axes > 1 else 0,
        0 if dq is None else dq.data_ptr(), 0 if dk is None else dk.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), *sq, *sk, *gs,
        batch, seq, hq, hk, d, half, nope_dim, axes, rows, _kv8.IO_DTYPES[dtype],
        _lib.DTYPE_FP32 if wtype == torch.float32 else _kv8.IO_DTYPES[dtype], eps)
    return args, q_out, k_out, (q, k, q_weight, k_weight, cos, sin, positions, pair_axis, dq, dk)


def kernel_fn(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor, cos: torch.Tensor,
              sin: torch.Tensor, positions: torch.Tensor | None = None, *, eps: float = 1e-6,
              nope_dim: int | None = None, sections: tuple | None = None, interleaved: bool = False):
    args, q_out, k_out, keep = describe(q, k, q_weight, k_weight, cos, sin, positions, eps, nope_dim, sections, interleaved)
    dev = q.device
    status = _lib.host_status_ptr(dev, "qk_norm_rope")
    rc = _lib.call_on(dev, _lib.load().tokmix_qk_norm_rope_fwd, args, status, _lib.stream_ptr(dev))
    del keep
    if rc:
        _lib.check(rc, "qk_norm_rope")
    _lib.after_host_status_launch(dev, "qk_norm_rope")
    return q_out, k_out


def check_device_status(device: torch.device | None = None) -> None:
    """Synchronise and raise if a call on `device` met positions outside its tables."""
    dev = torch.device(device) if device is not None else torch.device("cuda")
    dev = torch.device("cuda", dev.index if dev.index is not None else torch.cuda.current_device())
    torch.cuda.synchronize(dev)
    _lib.take_host_status(dev, "qk_norm_rope")


def rotary_tables(rows: int, half: int, theta: float = 10000.0, device: str = "cuda"):
    """cos and sin [rows, half] of position * theta^(-j / half), the angles formed in 64 bits."""
    freq = theta ** (-torch.arange(half, dtype=torch.float64) / half)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * freq
    return angle.cos().float().to(device), angle.sin().float().to(device)


def get_inputs(batch: int = 4, seq_len: int = 2048, q_heads: int = 16, kv_heads: int = 2, head_dim: int = 256,
               pairs: int = 32, dtype: torch.dtype = torch.bfloat16, seed: int = 42, device: str = "cuda") -> dict:
    gen = torch.Generator().manual_seed(seed)
    heads = q_heads + 2 * kv_heads
    qkv = (2 * torch.randn(batch, seq_len, heads, head_dim, generator=gen)).to(dtype).to(device)
    cos, sin = rotary_tables(seq_len, pairs, device=device)
    w = [(1 + 0.2 * torch.randn(head_dim, generator=gen)).to(dtype).to(device) for _ in range(2)]
    return {"q": qkv[:, :, :q_heads], "k": qkv[:, :, q_heads:q_heads + kv_heads], "q_weight": w[0], "k_weight": w[1],
            "cos": cos, "sin": sin}


def get_flops(batch: int = 4, seq_len: int = 2048, q_heads: int = 16, kv_heads: int = 2, head_dim: int = 256) -> int:
    return 8 * batch * seq_len * (q_heads + kv_heads) * head_dim


def get_bytes(batch: int = 4, seq_len: int = 2048, q_heads: int = 16, kv_heads: int = 2, head_dim: int = 256,
              pairs: int = 32, element_size: int = 2) -> int:
    """q and k read and written once, the tables' rows and the weights read once."""
    return (batch * seq_len * (q_heads + kv_heads) * head_dim * element_size * 2 + seq_len * pairs * 8
            + 2 * head_dim * element_size)
