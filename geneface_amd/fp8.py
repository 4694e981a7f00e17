"""Linear products of block-scaled 8-bit values, with their gradients.

The arithmetic of `cond_encoder.MLP`'s bias-free layers (cond_encoder.py:92-111 of the reference) with both operands of every product brought to e4m3 in
blocks of 128 along the axis that is summed over, and added up in 32 bits (bfloat16 results: see `linear`):

    y  = Q_row(x)  Q_tile(W)^T        dx = Q_row(dy) Q_tile(W)        dW = Q_col(dy)^T Q_col(x)

Q_row has a scale for each 128 values of a row, Q_col for each 128 of a column, Q_tile for each 128 x 128 of the weight, which serves the forward
product and the one of dx.  A scale is 2^e with the smallest e >= -127 for which the block's largest magnitude is <= 448 * 2^e; codes are rounded
to nearest even.  Scales are powers of two because that is what the scaled matrix instructions take, and multiplying by them rounds nothing.  A
block that holds an infinity or a NaN is NaN as a whole, so an overflow reaches what looks for one (GradScaler).

`linear(x, weight)` quantises the weight at every call, as training needs; `quantize_weight` does it once for `linear(x, Fp8Weight)`.
`cond_encoder.MLP` takes this path with `mlp.precision = "fp8"`.  Nothing here keeps anything between calls.
"""
import ctypes as C

import torch

from .lib import check, current_stream, host, lib
from .optim import DTYPES

BLOCK = 128

_vp = C.c_void_p


class GfFp8Quantize(C.Structure):
    """ctypes mirror of gf_fp8_quantize_t (include/geneface_train_hip.h)."""
    _fields_ = [("src", _vp), ("rows", C.c_uint64), ("cols", C.c_uint64), ("ld", C.c_uint64), ("dtype", C.c_uint32), ("tiles", C.c_uint32)] + \
               [(n, _vp) for n in ("row_codes", "row_scales", "col_codes", "col_scales", "tile_scales")] + [("row_pitch", C.c_uint64), ("col_pitch", C.c_uint64)]


class GfFp8Linear(C.Structure):
    """ctypes mirror of gf_fp8_linear_t."""
    _fields_ = [("x", _vp), ("ldx", C.c_uint64), ("w", _vp), ("ldw", C.c_uint64), ("codes", _vp), ("scales", _vp), ("m", C.c_uint64), ("n", C.c_uint64),
                ("k", C.c_uint64), ("y", _vp), ("saved", _vp), ("workspace", _vp)] + [(n, C.c_uint32) for n in ("dtype", "w_dtype", "keep_w", "keep_x")] + \
               [(n, C.c_uint64) for n in ("saved_bytes", "workspace_bytes", "backward_bytes")]


class GfFp8LinearBackward(C.Structure):
    """ctypes mirror of gf_fp8_linear_backward_t."""
    _fields_ = [("dy", _vp), ("lddy", C.c_uint64), ("saved", _vp), ("m", C.c_uint64), ("n", C.c_uint64), ("k", C.c_uint64), ("dx", _vp), ("dw", _vp),
                ("workspace", _vp)] + [(n, C.c_uint32) for n in ("dtype", "w_dtype", "keep_w", "keep_x")]


def _blocks(n):
    return -(-n // BLOCK)


def _matrix(x):
    """x [..., K] as [M, K] whose rows are consecutive values, rows at any distance."""
    x = x.resolve_neg()
    m = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    return m if m.stride(1) == 1 and m.stride(0) >= m.shape[1] else m.contiguous()


def _quantize(m, rows, cols, tiles=False):
    """(row codes, row scales, column codes, column scales) of m [R, C]; with `tiles` one tensor of scales for both.  What is not wanted is None."""
    R, Cn = m.shape
    u8 = lambda *s: torch.empty(s, dtype=torch.uint8, device=m.device)      # noqa: E731
    rc, cc = u8(R, _blocks(Cn) * BLOCK) if rows else None, u8(Cn, _blocks(R) * BLOCK) if cols else None
    if tiles:
        rs = cs = ts = u8(_blocks(R), _blocks(Cn))
    else:
        rs, cs, ts = u8(_blocks(Cn), R) if rows else None, u8(_blocks(R), Cn) if cols else None, None
    p = lambda t: None if t is None else t.data_ptr()      # noqa: E731
    d = GfFp8Quantize(m.data_ptr(), R, Cn, m.stride(0) if R > 1 else Cn, DTYPES[m.dtype], int(tiles), p(rc), None if tiles else p(rs), p(cc),
                      None if tiles else p(cs), p(ts), R, Cn)
    check(lib().gf_fp8_quantize(C.byref(d), current_stream(m.device)))
    return rc, rs, cc, cs


class Fp8Weight:
    """A linear layer's weight [N, K] in 8 bits.

    values: float8_e4m3fn [N, up(K)], up(K) the multiple of 128 that holds K, zeros behind K; scales: float8_e8m0fnu [ceil(N / 128), ceil(K / 128)];
    in_features: K."""

    __slots__ = ("values", "scales", "in_features", "out_features")

    def __init__(self, values, scales, in_features):
        if values.dtype != torch.float8_e4m3fn or scales.dtype != torch.float8_e8m0fnu:
            raise RuntimeError(f"Fp8Weight: float8_e4m3fn values and float8_e8m0fnu scales are needed, got {values.dtype} and {scales.dtype}")
        n, kb = values.shape[0], _blocks(in_features)
        if values.dim() != 2 or in_features < 0 or values.shape[1] != kb * BLOCK or tuple(scales.shape) != (_blocks(n), kb):
            raise RuntimeError(f"Fp8Weight: values {tuple(values.shape)} and scales {tuple(scales.shape)} do not fit {in_features} input features")
        if not values.is_contiguous() or not scales.is_contiguous():
            raise RuntimeError("Fp8Weight: values and scales must be contiguous tensors")
        if values.device != scales.device:
            raise RuntimeError("Fp8Weight: values and scales must be on one device")
        self.values, self.scales, self.in_features, self.out_features = values, scales, in_features, n

    @property
    def device(self):
        return self.values.device

    def to(self, device):
        return Fp8Weight(self.values.to(device), self.scales.to(device), self.in_features)

    def dequantize(self):
        """The weight that is multiplied with, float32 [N, K]."""
        s = torch.ldexp(torch.ones((), dtype=torch.float64, device=self.device), self.scales.view(torch.uint8).double() - 127)
        s = s.masked_fill(self.scales.view(torch.uint8) == 255, float("nan"))
        s = s.repeat_interleave(BLOCK, 0)[:self.out_features].repeat_interleave(BLOCK, 1)
        return (self.values.float().double() * s).float()[:, :self.in_features]


@torch.no_grad()
def quantize_weight(weight):
    """Fp8Weight of weight [N, K] (float32, bfloat16 or float16)."""
    if weight.dtype not in DTYPES:
        raise RuntimeError(f"fp8: the weight must be float32, bfloat16 or float16, got {weight.dtype}")
    if weight.dim() != 2:
        raise RuntimeError(f"fp8: the weight must be a matrix, got {tuple(weight.shape)}")
    if not weight.is_cuda:
        raise RuntimeError("fp8: the weight must be a CUDA tensor")
    N, K = weight.shape
    with torch.cuda.device(weight.device):
        if N and K:
            codes, scales, _, _ = _quantize(_matrix(weight), True, False, tiles=True)
        else:
            codes, scales = (torch.empty(s, dtype=torch.uint8, device=weight.device) for s in ((N, _blocks(K) * BLOCK), (_blocks(N), _blocks(K))))
    return Fp8Weight(codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu), K)


def linear(x, weight):
    """x [..., K] times a weight's transpose, [..., N] in x's type (under autocast: in its type), both brought to 8 bits in blocks of 128.

    weight: a tensor [N, K], quantised in the call, with gradients to x and to the weight; or an Fp8Weight, without gradients.  x, weight: float32,
    bfloat16 or float16, each its own; the gradients have their input's type.  At most 8388480 values along each sum, unless both of the weight's
    sides are 128 or less.

    float32 and binary16 results (y and dx in x's type, dw in the weight's) are added up in 32 bits.  bfloat16 results come from the 8-bit matrix
    instructions, which line up the products of eight neighbours along the sum and drop what lies below 2^-13 of the largest: a sum loses at most
    7 * 2^-13 of each eight's largest product (8.5e-4, where bfloat16 rounds by 3.9e-3; normal operands: 2.5e-6), whatever its length.
    For less, give x (or the weight, for dw) in float32.  Values of blocks below 2^-115 (float32's least normal one is 2^-126) count as multiples of 2^-133
    in float32 and binary16 results.

    Both directions may be captured into a graph.  As with any torch node, a backward pass is captured only while no graph of the same leaves lives
    that was built outside the capture.  Gradients of the gradients are refused."""
    if isinstance(weight, Fp8Weight):
        return host().linear_packed(x, weight.values, weight.scales, weight.in_features)
    return host().linear(x, weight)
