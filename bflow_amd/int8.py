"""8-bit integers with a scale for each row: quantisation, and the product of two such operands (csrc/int8_gemm.hip).

    q, s = quantize_rows(x)                   rows of any float type (tokens, the output channels of a weight matrix)
    q, s = quantize_pixels(maps)              feature maps, one row of channels for each pixel
    y    = matmul(qa, sa, qb, sb)             y[i, j] = sa[i] sb[j] sum_k qa[i, k] qb[j, k], sums exact

scale = max|x| / 127 of the row; q = the nearest whole number to 127 x / max|x|, halves to even.  A row of zeros has scale 0; a row with an
infinity or a NaN has q = 0 and an infinite or NaN scale: its products are NaN, as they would be without quantisation.
The correlation volume runs on it with `correlation.precision: i8` (corr.py).
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import hip


def _padded(k: int) -> int:
    return (k + 15) & ~15


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x (..., rows, K) float32 / float16 / bfloat16 -> int8 (..., rows, K), float32 scales (..., rows).  The rows of the result start 16 bytes
    apart or a multiple (zeros in between), as `matmul` wants them; x (K,) is one row."""
    hip._dev(x, None, "x", contiguous=False)
    if x.dtype not in hip.FLOAT_CODES or x.dim() < 1:
        raise hip.BflowHipError(f"quantize_rows: rows of {sorted(str(d) for d in hip.FLOAT_CODES)}, got {tuple(x.shape)} {x.dtype}")
    K, lead = x.shape[-1], x.shape[:-1]
    rows = x.numel() // K if K else 0
    q = torch.empty(lead + (_padded(K),), dtype=torch.int8, device=x.device)
    scale = torch.zeros(lead, device=x.device) if not K else torch.empty(lead, device=x.device)
    if rows:
        flat = x.reshape(rows, K)                          # a view where the rows are evenly spaced
        flat = flat if flat.stride(1) == 1 or K == 1 else flat.contiguous()
        with torch.cuda.device(x.device):
            hip._check(hip.lib().bflow_i8_quantize_rows(flat.data_ptr(), hip.FLOAT_CODES[x.dtype], flat.stride(0), rows, K, q.data_ptr(), _padded(K), scale.data_ptr(),
                                                        hip._stream()), "bflow_i8_quantize_rows")
    return q[..., :K], scale


def quantize_pixels(maps: torch.Tensor, tiled: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """maps (..., D, h, w) float32, D a multiple of 16 -> int8 (..., P, D), float32 scales (..., P): P = h * w pixels in order, or (tiled) the
    `hip.tiled_plane_size(h, w)` places of the tiled correlation volume, those outside the map zero with scale 0."""
    if maps.dim() < 3:
        raise hip.BflowHipError(f"quantize_pixels: maps (..., D, h, w), got {tuple(maps.shape)}")
    lead, (D, h, w) = maps.shape[:-3], maps.shape[-3:]
    hip._dev(maps, torch.float32, "maps", contiguous=False)
    maps = maps.contiguous()
    return _quantize_pixels(maps.data_ptr(), None, None, 0, maps.device, lead, D, h, w, tiled)


def quantize_packed(planes: torch.Tensor, h: int, w: int, tiled: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """quantize_pixels of maps in the conv engine's operand form (2, R, D/32, Np, 32) (hip.split_pack): int8 (R, P, D), scales (R, P)."""
    _, R, KB, Np, width = planes.shape
    if planes.dtype != torch.float16 or not planes.is_cuda or width != 32 or not (planes[0].is_contiguous() and planes[1].is_contiguous()):
        raise hip.BflowHipError("quantize_packed: the operand planes of hip.split_pack")
    return _quantize_pixels(None, planes[0].data_ptr(), planes[1].data_ptr(), Np, planes.device, (R,), KB * 32, h, w, tiled)


def _quantize_pixels(x, hi, lo, np_rows, device, lead, D, h, w, tiled):
    rows = hip.tiled_plane_size(h, w) if tiled else h * w
    q = torch.empty(tuple(lead) + (rows, D), dtype=torch.int8, device=device)
    scale = torch.empty(tuple(lead) + (rows,), device=device)
    B = scale.numel() // rows if rows else 0
    if D < 16 or D % 16:
        raise hip.BflowHipError(f"quantize_pixels: {D} channels, a multiple of 16 is needed")
    if B:
        with torch.cuda.device(device):
            hip._check(hip.lib().bflow_i8_quantize_pixels(x, hi, lo, np_rows, B, D, h, w, int(tiled), q.data_ptr(), scale.data_ptr(), hip._stream()),
                       "bflow_i8_quantize_pixels")
    return q, scale


def _operand(t: torch.Tensor, what: str) -> torch.Tensor:
    """(..., rows, K) as the kernel reads it: K contiguous, everything else at multiples of 16 bytes, every row readable up to K rounded up to 16."""
    hip._dev(t, torch.int8, what, contiguous=False)
    rows, K = t.shape[-2:]
    steps = [s for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n > 1]
    last = t.storage_offset() + sum((n - 1) * s for n, s in zip(t.shape[:-1], t.stride()[:-1])) + _padded(K)
    if (t.stride(-1) == 1 or K == 1) and t.data_ptr() % 16 == 0 and all(s % 16 == 0 for s in steps) and last <= t.untyped_storage().nbytes() \
            and (rows == 1 or _padded(K) <= t.stride(-2) <= 1 << 22):
        return t
    room = torch.empty(t.shape[:-1] + (_padded(K),), dtype=torch.int8, device=t.device)
    room[..., :K].copy_(t)
    return room[..., :K]


def _two(t: torch.Tensor, batch: Tuple[int, ...], tail: int) -> torch.Tensor:
    """t (..., tail dimensions) spread over `batch`, as (n0, n1, tail dimensions); repeated dimensions keep stride 0."""
    t = t.expand(tuple(batch) + tuple(t.shape[-tail:]))
    if len(batch) > 2:
        t = t.flatten(0, len(batch) - 2)
    while t.dim() < tail + 2:
        t = t.unsqueeze(0)
    return t


def matmul(a: torch.Tensor, scale_a: torch.Tensor, b: torch.Tensor, scale_b: torch.Tensor, out_dtype: torch.dtype = torch.float32, alpha: float = 1.0,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """a (..., M, K) int8 with scales (..., M), b (..., N, K) int8 with scales (..., N) -> (..., M, N) of out_dtype (float32, float16, bfloat16):
    alpha * scale_a * scale_b * (a @ b^T), rounded once.  Leading dimensions broadcast.  Operands whose rows are not spaced by multiples of 16 bytes
    are copied first (quantize_rows spaces them).  out: where the result goes, dense in its last dimension.  Not differentiable."""
    if a.dim() < 2 or b.dim() < 2 or a.shape[-1] != b.shape[-1]:
        raise hip.BflowHipError(f"matmul: rows of the same length, got {tuple(a.shape)} and {tuple(b.shape)}")
    if tuple(scale_a.shape) != tuple(a.shape[:-1]) or tuple(scale_b.shape) != tuple(b.shape[:-1]):
        raise hip.BflowHipError(f"matmul: a scale for each row, got {tuple(scale_a.shape)}, {tuple(scale_b.shape)} for {tuple(a.shape)}, {tuple(b.shape)}")
    for t, name in ((scale_a, "scale_a"), (scale_b, "scale_b")):
        hip._dev(t, torch.float32, name, contiguous=False)
    if out_dtype not in hip.FLOAT_CODES:
        raise hip.BflowHipError(f"matmul: out_dtype {out_dtype}, expected one of {sorted(str(d) for d in hip.FLOAT_CODES)}")
    M, N, K = a.shape[-2], b.shape[-2], a.shape[-1]
    try:
        batch = torch.broadcast_shapes(a.shape[:-2], b.shape[:-2])
    except RuntimeError:
        raise hip.BflowHipError(f"matmul: leading dimensions {tuple(a.shape[:-2])} and {tuple(b.shape[:-2])} do not broadcast") from None
    shape = tuple(batch) + (M, N)
    if out is None:
        hip._dev(a, torch.int8, "a", contiguous=False)
        out = torch.empty(shape, dtype=out_dtype, device=a.device)
    elif tuple(out.shape) != shape or out.dtype != out_dtype or not out.is_cuda or (N > 1 and out.stride(-1) != 1) or (M > 1 and out.stride(-2) < N):
        raise hip.BflowHipError(f"matmul: out {tuple(out.shape)} {out.dtype}, strides {out.stride()}: expected {shape} {out_dtype}, rows dense")
    if not (a.device == b.device == scale_a.device == scale_b.device == out.device):
        raise hip.BflowHipError("matmul: all tensors on one device")
    if not out.numel():
        return out
    if not K:
        return out.zero_()
    keep = (_operand(a, "a"), _operand(b, "b"), scale_a if scale_a.stride(-1) == 1 else scale_a.contiguous(), scale_b if scale_b.stride(-1) == 1 else scale_b.contiguous())
    # (_operand again: folding three or more leading dimensions may have made a dense copy)
    pa, pb, sa, sb = _operand(_two(keep[0], batch, 2), "a"), _operand(_two(keep[1], batch, 2), "b"), _two(keep[2], batch, 1), _two(keep[3], batch, 1)
    to = _two(out, batch, 2)
    if to.data_ptr() != out.data_ptr():
        raise hip.BflowHipError(f"matmul: out with strides {out.stride()}: its leading dimensions have to fold into two")
    d = hip.I8GemmDesc(a=pa.data_ptr(), b=pb.data_ptr(), scale_a=sa.data_ptr(), scale_b=sb.data_ptr(), out=to.data_ptr(), a_stride0=pa.stride(0), a_stride1=pa.stride(1),
                       b_stride0=pb.stride(0), b_stride1=pb.stride(1), sa_stride0=sa.stride(0), sa_stride1=sa.stride(1), sb_stride0=sb.stride(0), sb_stride1=sb.stride(1),
                       out_stride0=to.stride(0), out_stride1=to.stride(1), ldo=to.stride(2) if M > 1 else N, lda=pa.stride(2) if M > 1 else _padded(K),
                       ldb=pb.stride(2) if N > 1 else _padded(K), M=M, N=N, K=K, batch0=to.shape[0], batch1=to.shape[1], dtype=hip.FLOAT_CODES[out_dtype], alpha=alpha)
    for name in ("a", "b"):                                # a dimension of one element may carry any stride: it is never taken
        for k, n in ((0, d.batch0), (1, d.batch1)):
            if n == 1:
                setattr(d, f"{name}_stride{k}", 0)
    with torch.cuda.device(out.device):
        hip._check(hip.lib().bflow_i8_gemm(ctypes.byref(d), hip._stream()), "bflow_i8_gemm")
    return out
