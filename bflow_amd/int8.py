"""8-bit integers with a scale for each row: quantisation, and the product of two such operands (csrc/int8_gemm.hip).

    q, s = quantize_rows(x)                   rows of any float type (tokens, the output channels of a weight matrix)
    q, s = quantize_pixels(maps)              feature maps, one row of channels for each pixel
    y    = matmul(qa, sa, qb, sb)             y[i, j] = sa[i] sb[j] sum_k qa[i, k] qb[j, k], sums exact

scale = max|x| / 127 of the row; q = the nearest whole number to 127 x / max|x|, halves to even.  A row of zeros has scale 0; a row with an
infinity or a NaN has q = 0 and an infinite or NaN scale: its products are NaN, as they would be without quantisation.
The correlation volume runs on it with `correlation.precision: i8` (corr.py).
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

from . import hip


def _padded(k: int) -> int:
    return (k + 15) & ~15


def _sizes(what: str, *sizes: int):
    if any(n > hip.I8_MAX_SIZE for n in sizes):
        raise hip.BflowHipError(f"{what}: sizes {sizes}, at most {hip.I8_MAX_SIZE} are taken")


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x (..., rows, K) float32 / float16 / bfloat16 -> int8 (..., rows, K), float32 scales (..., rows).  The rows of the result start 16 bytes
    apart or a multiple (zeros in between), as `matmul` wants them; x (K,) is one row.  K is at most 2^31 - 512."""
    if isinstance(x, torch.Tensor) and x.dim():
        _sizes("quantize_rows", x.shape[-1])
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
        with hip._on(x.device):
            hip._check(hip.lib().bflow_i8_quantize_rows(flat.data_ptr(), hip.FLOAT_CODES[x.dtype], flat.stride(0), rows, K, q.data_ptr(), _padded(K), scale.data_ptr(),
                                                        hip._stream()), "bflow_i8_quantize_rows")
    return q[..., :K], scale


def quantize_pixels(maps: torch.Tensor, tiled: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """maps (..., D, h, w) float32, D a multiple of 16 -> int8 (..., P, D), float32 scales (..., P): P = h * w pixels in order, or (tiled) the
    `hip.tiled_plane_size(h, w)` places of the tiled correlation volume, those outside the map zero with scale 0.  Fewer than 2^28 places, 65535 maps
    at most."""
    lead, D, h, w = _maps_shape(maps)
    maps = maps.contiguous()
    return _quantize_maps([(maps.data_ptr(), 0, 0, 0, lead, tiled)], maps.device, D, h, w)[0]


def quantize_packed(planes: torch.Tensor, h: int, w: int, tiled: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """quantize_pixels of maps in the conv engine's operand form (2, R, D/32, Np, 32) (hip.split_pack): int8 (R, P, D), scales (R, P)."""
    return _quantize_maps([_packed(planes, tiled)], planes.device, planes.shape[2] * 32, h, w)[0]


def quantize_operands(f1: torch.Tensor, f2: torch.Tensor, packed_hw: Optional[Tuple[int, int]] = None):
    """Both sides of a correlation volume in one launch: quantize_pixels(f1), quantize_pixels(f2, tiled=True) of maps of one D, h, w; with `packed_hw`
    = (h, w) quantize_packed of operand planes."""
    if packed_hw is not None:
        items, (h, w), D = [_packed(f1, False), _packed(f2, True)], packed_hw, f1.shape[2] * 32
        if f2.shape[2] * 32 != D:
            raise hip.BflowHipError(f"quantize_operands: {D} and {f2.shape[2] * 32} channels")
    else:
        (lead1, D, h, w), (lead2, *size) = _maps_shape(f1), _maps_shape(f2)
        if size != [D, h, w]:
            raise hip.BflowHipError(f"quantize_operands: maps {tuple(f1.shape)} and {tuple(f2.shape)} of different channels or sizes")
        f1, f2 = f1.contiguous(), f2.contiguous()
        items = [(f1.data_ptr(), 0, 0, 0, lead1, False), (f2.data_ptr(), 0, 0, 0, lead2, True)]
    if f1.device != f2.device:
        raise hip.BflowHipError("quantize_operands: all tensors on one device")
    return _quantize_maps(items, f1.device, D, h, w)


def _maps_shape(maps):
    if maps.dim() < 3:
        raise hip.BflowHipError(f"quantize_pixels: maps (..., D, h, w), got {tuple(maps.shape)}")
    _sizes("quantize_pixels", maps.shape[-3], maps.shape[-2] * maps.shape[-1])
    hip._dev(maps, torch.float32, "maps", contiguous=False)
    shape = maps.shape
    return (tuple(shape[:-3]),) + tuple(shape[-3:])


def _packed(planes, tiled):
    if planes.dim() != 5 or planes.dtype != torch.float16 or not planes.is_cuda or planes.shape[4] != 32 or not (planes[0].is_contiguous() and planes[1].is_contiguous()):
        raise hip.BflowHipError("quantize_packed: the operand planes of hip.split_pack")
    return 0, planes[0].data_ptr(), planes[1].data_ptr(), planes.shape[3], (planes.shape[1],), tiled


def _quantize_maps(items, device, D, h, w):
    if D < 16 or D % 16:
        raise hip.BflowHipError(f"quantize_pixels: {D} channels, a multiple of 16 is needed")
    out, table = [], []
    for x, hi, lo, np_rows, lead, tiled in items:
        rows = hip.tiled_plane_size(h, w) if tiled else h * w
        q = torch.empty(lead + (rows, D), dtype=torch.int8, device=device)
        scale = torch.empty(lead + (rows,), device=device)
        out.append((q, scale))
        B = math.prod(lead)
        if B and rows:
            table.append(hip.I8_MAPS.pack(x, hi, lo, q.data_ptr(), scale.data_ptr(), np_rows, B, int(tiled), 0))
    if table:
        with hip._on(device):
            hip._check(hip.lib().bflow_i8_quantize_maps(b"".join(table), len(table), D, h, w, hip._stream()), "bflow_i8_quantize_maps")
    return out


def _ready(t: torch.Tensor, K: int) -> bool:
    """(..., rows, K) as the kernel reads it: K contiguous, everything else at multiples of 16 bytes, every row readable up to K rounded up to 16."""
    shape, strides = t.shape, t.stride()
    if (strides[-1] != 1 and K > 1) or t.data_ptr() % 16:
        return False
    need = (K + 15) & ~15
    if shape[-2] > 1 and not need <= strides[-2] <= 1 << 22:
        return False
    for n, s in zip(shape[:-1], strides[:-1]):
        if s % 16 and n > 1:
            return False
    if need == K:
        return True
    last = t.storage_offset() + sum((n - 1) * s for n, s in zip(shape[:-1], strides[:-1])) + need
    return last <= t.untyped_storage().nbytes()


def _operands(ts, K: int, device):
    """(address, strides) of the operands as the kernel reads them, and what holds them: those that are not ready are copied into one buffer, rows 16
    bytes apart or a multiple, in one launch where they are rows of bytes at even distances."""
    out, items, wanting, room, total = [], [], [], None, 0
    ldd = _padded(K)
    for i, t in enumerate(ts):
        if _ready(t, K):
            out.append((t.data_ptr(), t.stride()))
            continue
        rows, strides = 1, (1,)
        for n in reversed(t.shape[:-1]):
            strides = (rows * ldd,) + strides
            rows *= n
        out.append((total, strides))
        wanting.append((i, t, rows))
        total += rows * ldd
    if wanting:
        room = torch.empty(total, dtype=torch.int8, device=device)
        base = room.data_ptr()
        for i, t, rows in wanting:
            at, strides = out[i]
            out[i] = (base + at, strides)
            shape, from_ = t.shape, t.stride()
            if (from_[-1] == 1 or K == 1) and (len(shape) == 2 or (len(shape) == 3 and from_[0] == shape[1] * from_[1])):
                items.append(hip.I8_PAD.pack(t.data_ptr(), base + at, from_[-2], rows, K, ldd))
            else:
                room.as_strided(shape, strides, at).copy_(t)
        if items:
            hip._check(hip.lib().bflow_i8_pad_rows(b"".join(items), len(items), hip._stream()), "bflow_i8_pad_rows")
    return out, room


def _broadcast(a: Tuple[int, ...], b: Tuple[int, ...]) -> Tuple[int, ...]:
    n = max(len(a), len(b))
    a, b = (1,) * (n - len(a)) + tuple(a), (1,) * (n - len(b)) + tuple(b)
    for x, y in zip(a, b):
        if x != y and x != 1 and y != 1:
            raise hip.BflowHipError(f"matmul: leading dimensions {a} and {b} do not broadcast")
    return tuple(y if x == 1 else x for x, y in zip(a, b))


def _lead_strides(shape, strides, lead: int, batch: Tuple[int, ...]):
    """Strides of an operand's first `lead` dimensions over `batch`; 0 where an element is repeated or there is only one."""
    return [0] * (len(batch) - lead) + [s if n > 1 else 0 for n, s in zip(shape[:lead], strides[:lead])]


def _fold(batch, strides):
    """The batch dimensions as two, with each operand's strides: neighbours become one where every operand steps evenly over them.  None where more than
    two are left."""
    dims = [(n, [s[i] for s in strides]) for i, n in enumerate(batch) if n > 1]
    i = len(dims) - 2
    while i >= 0 and len(dims) > 2:
        (n0, s0), (n1, s1) = dims[i], dims[i + 1]
        if all(x == n1 * y for x, y in zip(s0, s1)):
            dims[i:i + 2] = [(n0 * n1, s1)]
        i -= 1
    if len(dims) > 2:
        return None
    return [(1, [0] * len(strides))] * (2 - len(dims)) + dims


def matmul(a: torch.Tensor, scale_a: torch.Tensor, b: torch.Tensor, scale_b: torch.Tensor, out_dtype: torch.dtype = torch.float32, alpha: float = 1.0,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """a (..., M, K) int8 with scales (..., M), b (..., N, K) int8 with scales (..., N) -> (..., M, N) of out_dtype (float32, float16, bfloat16):
    (alpha * scale_a) * scale_b * (a @ b^T): sums exact, rounded to 32 bits, as are the products with the scales, then to out_dtype.  Leading dimensions
    broadcast.  Operands whose rows are not spaced by multiples of 16 bytes are copied first (quantize_rows spaces them).  out: where the result goes,
    dense in its last dimension.  Refused: K above 131071, more than 65535 matrices, 2^28 rows or more on one side where the other has at most 32.
    Not differentiable."""
    ashape, bshape = a.shape, b.shape
    if len(ashape) < 2 or len(bshape) < 2 or ashape[-1] != bshape[-1]:
        raise hip.BflowHipError(f"matmul: rows of the same length, got {tuple(ashape)} and {tuple(bshape)}")
    if scale_a.shape != ashape[:-1] or scale_b.shape != bshape[:-1]:
        raise hip.BflowHipError(f"matmul: a scale for each row, got {tuple(scale_a.shape)}, {tuple(scale_b.shape)} for {tuple(ashape)}, {tuple(bshape)}")
    _sizes("matmul", ashape[-2], bshape[-2], ashape[-1])
    for t, kind, name in ((a, torch.int8, "a"), (b, torch.int8, "b"), (scale_a, torch.float32, "scale_a"), (scale_b, torch.float32, "scale_b")):
        hip._dev(t, kind, name, contiguous=False)
    code = hip.FLOAT_CODES.get(out_dtype)
    if code is None:
        raise hip.BflowHipError(f"matmul: out_dtype {out_dtype}, expected one of {sorted(str(d) for d in hip.FLOAT_CODES)}")
    M, N, K = ashape[-2], bshape[-2], ashape[-1]
    batch: Tuple[int, ...] = ()
    if len(ashape) > 2 or len(bshape) > 2:
        batch = _broadcast(ashape[:-2], bshape[:-2])
    shape, device = batch + (M, N), a.device
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=device)
    elif tuple(out.shape) != shape or out.dtype != out_dtype or not out.is_cuda or (N > 1 and out.stride(-1) != 1) or (M > 1 and out.stride(-2) < N) \
            or any(n > 1 and not s for n, s in zip(shape, out.stride())):
        raise hip.BflowHipError(f"matmul: out {tuple(out.shape)} {out.dtype}, strides {out.stride()}: expected {shape} {out_dtype}, rows dense")
    if not (device == b.device == scale_a.device == scale_b.device == out.device):
        raise hip.BflowHipError("matmul: all tensors on one device")
    if not (M and N and out.numel()):
        return out
    if not K:
        return out.zero_()
    with hip._on(device):
        ((pa, ra), (pb, rb)), held = _operands((a, b), K, device)         # (held: until the launches are enqueued)
        sa, sb = scale_a if scale_a.stride(-1) == 1 else scale_a.contiguous(), scale_b if scale_b.stride(-1) == 1 else scale_b.contiguous()
        strides, n0, n1 = (0,) * 10, 1, 1
        if batch:
            la, lb = len(ashape) - 2, len(bshape) - 2
            two = _fold(batch, [_lead_strides(ashape, ra, la, batch), _lead_strides(bshape, rb, lb, batch), _lead_strides(ashape, sa.stride(), la, batch),
                                _lead_strides(bshape, sb.stride(), lb, batch), _lead_strides(shape, out.stride(), len(batch), batch)])
            if two is None:                                # dense copies of what is spread over more than two dimensions
                whole = torch.empty(shape, dtype=out_dtype, device=device)
                spread = lambda t, tail: t.expand(batch + tuple(t.shape[-tail:])).contiguous()
                matmul(spread(a, 2).flatten(0, -3), spread(scale_a, 1).flatten(0, -2), spread(b, 2).flatten(0, -3), spread(scale_b, 1).flatten(0, -2), out_dtype, alpha,
                       out=whole.view((-1, M, N)))
                return out.copy_(whole)
            (n0, s0), (n1, s1) = two
            strides = tuple(v for pair in zip(s0, s1) for v in pair)
        ld = _padded(K)
        d = hip.I8_GEMM.pack(pa, pb, sa.data_ptr(), sb.data_ptr(), out.data_ptr(), *strides, out.stride(-2) if M > 1 else N,
                             ra[-2] if M > 1 else ld, rb[-2] if N > 1 else ld, M, N, K, n0, n1, code, alpha)
        hip._check(hip.lib().bflow_i8_gemm(d, hip._stream()), "bflow_i8_gemm")
    return out
