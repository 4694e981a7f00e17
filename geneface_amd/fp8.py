"""Linear products of block-scaled 8-bit values, with their gradients.

The arithmetic of `cond_encoder.MLP`'s bias-free layers (cond_encoder.py:92-111 of the reference) with both operands of every product brought to e4m3 in
blocks of 128 along the axis that is summed over, and added up in 32 bits:

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

from .lib import check, current_stream, lib
from .optim import DTYPES

BLOCK = 128
FEW_ROWS = 16      # rows that gf_fp8_rows takes

_vp = C.c_void_p


class GfFp8Quantize(C.Structure):
    """ctypes mirror of gf_fp8_quantize_t (include/geneface_train_hip.h)."""
    _fields_ = [("src", _vp), ("rows", C.c_uint64), ("cols", C.c_uint64), ("ld", C.c_uint64), ("dtype", C.c_uint32), ("tiles", C.c_uint32)] + \
               [(n, _vp) for n in ("row_codes", "row_scales", "col_codes", "col_scales", "tile_scales")] + [("row_pitch", C.c_uint64), ("col_pitch", C.c_uint64)]


class GfFp8Operand(C.Structure):
    """ctypes mirror of gf_fp8_operand_t."""
    _fields_ = [("codes", _vp), ("scales", _vp), ("pitch", C.c_uint64), ("stride_row", C.c_uint64), ("stride_block", C.c_uint64)]


class GfFp8Matmul(C.Structure):
    """ctypes mirror of gf_fp8_matmul_t."""
    _fields_ = [("a", GfFp8Operand), ("b", GfFp8Operand), ("m", C.c_uint64), ("n", C.c_uint64), ("blocks", C.c_uint64), ("out", _vp),
                ("dtype", C.c_uint32), ("_pad", C.c_uint32), ("workspace", _vp)]


class GfFp8Rows(C.Structure):
    """ctypes mirror of gf_fp8_rows_t."""
    _fields_ = [("x", _vp), ("m", C.c_uint64), ("n", C.c_uint64), ("k", C.c_uint64), ("ldx", C.c_uint64), ("codes", _vp), ("scales", _vp), ("out", _vp),
                ("dtype", C.c_uint32), ("_pad", C.c_uint32)]


def _blocks(n):
    return -(-n // BLOCK)


def _matrix(x):
    """x [..., K] as [M, K] whose rows are consecutive values, rows at any distance."""
    m = x.reshape(-1, x.shape[-1])
    return m if m.stride(1) == 1 and m.stride(0) >= m.shape[1] else m.contiguous()


def _check_type(name, t):
    if t.dtype not in DTYPES:
        raise RuntimeError(f"fp8: {name} must be float32, bfloat16 or float16, got {t.dtype}")


def _check_device(name, t):
    if t.device.type != "cuda":
        raise RuntimeError(f"fp8: {name} must be a CUDA tensor")


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


def _by_row(codes, scales):
    return GfFp8Operand(codes.data_ptr(), scales.data_ptr(), scales.shape[1], 0, 0)


def _by_tile(codes, scales, transposed=False):
    """Scales [row block, block along the sum], or [block along the sum, row block] where the codes are the transposed ones."""
    a, b = scales.stride(0), scales.stride(1)
    return GfFp8Operand(codes.data_ptr(), scales.data_ptr(), 0, b if transposed else a, a if transposed else b)


def _matmul(a, b, m, n, blocks, dtype, device):
    out = torch.empty(m, n, dtype=dtype, device=device)
    L = lib()
    need = L.gf_fp8_matmul_workspace_bytes(m, n, blocks)
    work = torch.empty(need // 4, dtype=torch.float32, device=device) if need else None
    d = GfFp8Matmul(a, b, m, n, blocks, out.data_ptr(), DTYPES[dtype], 0, None if work is None else work.data_ptr())
    check(L.gf_fp8_matmul(C.byref(d), current_stream(device)))
    return out


class Fp8Weight:
    """A linear layer's weight [N, K] in 8 bits.

    values: float8_e4m3fn [N, up(K)], up(K) the multiple of 128 that holds K, zeros behind K; scales: float8_e8m0fnu [ceil(N / 128), ceil(K / 128)];
    in_features: K."""

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
    _check_type("the weight", weight)
    if weight.dim() != 2:
        raise RuntimeError(f"fp8: the weight must be a matrix, got {tuple(weight.shape)}")
    _check_device("the weight", weight)
    N, K = weight.shape
    with torch.cuda.device(weight.device):
        if N and K:
            codes, scales, _, _ = _quantize(_matrix(weight), True, False, tiles=True)
        else:
            codes, scales = (torch.empty(s, dtype=torch.uint8, device=weight.device) for s in ((N, _blocks(K) * BLOCK), (_blocks(N), _blocks(K))))
    return Fp8Weight(codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu), K)


def _linear_packed(x, w):
    K, N = w.in_features, w.out_features
    if not (x.numel() and N):
        return torch.zeros(*x.shape[:-1], N, dtype=x.dtype, device=x.device)
    m = _matrix(x)
    M = m.shape[0]
    with torch.cuda.device(x.device):
        if M <= FEW_ROWS:
            out = torch.empty(M, N, dtype=x.dtype, device=x.device)
            d = GfFp8Rows(m.data_ptr(), M, N, K, m.stride(0) if M > 1 else K, w.values.data_ptr(), w.scales.data_ptr(), out.data_ptr(), DTYPES[x.dtype], 0)
            check(lib().gf_fp8_rows(C.byref(d), current_stream(x.device)))
        else:
            codes, scales, _, _ = _quantize(m, True, False)
            out = _matmul(_by_row(codes, scales), _by_tile(w.values, w.scales), M, N, _blocks(K), x.dtype, x.device)
    return out.view(*x.shape[:-1], N)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight):
        (N, K), m = weight.shape, _matrix(x)
        M, need_x, need_w = m.shape[0], ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        with torch.cuda.device(x.device):
            wr, ws, wc, _ = _quantize(_matrix(weight), True, need_x, tiles=True)
            xr, xs, xc, xcs = _quantize(m, True, need_w)      # kept for the backward pass: x in 8 bits, not x
            y = _matmul(_by_row(xr, xs), _by_tile(wr, ws), M, N, _blocks(K), x.dtype, x.device)
        ctx.save_for_backward(wc, ws if need_x else None, xc, xcs)
        ctx.sizes, ctx.dtypes = (M, N, K), (x.dtype, weight.dtype)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        wc, ws, xc, xcs = ctx.saved_tensors
        (M, N, K), (tx, tw) = ctx.sizes, ctx.dtypes
        need_x, need_w = ctx.needs_input_grad
        dx = dw = None
        with torch.cuda.device(dy.device):
            gr, gs, gc, gcs = _quantize(_matrix(dy), need_x, need_w)
            if need_x:
                dx = _matmul(_by_row(gr, gs), _by_tile(wc, ws, transposed=True), M, K, _blocks(N), tx, dy.device)
            if need_w:
                dw = _matmul(_by_row(gc, gcs), _by_row(xc, xcs), N, K, _blocks(M), tw, dy.device)
        return dx, dw


def linear(x, weight):
    """x [..., K] times a weight's transpose, [..., N] in x's type (under autocast: in its type), both brought to 8 bits in blocks of 128.

    weight: a tensor [N, K], quantised in the call, with gradients to x and to the weight; or an Fp8Weight, without gradients.  x, weight: float32,
    bfloat16 or float16, each its own; the gradients have their input's type."""
    packed = isinstance(weight, Fp8Weight)
    if not packed:
        _check_type("the weight", weight)
        if weight.dim() != 2:
            raise RuntimeError(f"fp8: the weight must be a matrix, got {tuple(weight.shape)}")
    K = weight.in_features if packed else weight.shape[1]
    if x.dim() < 1 or x.shape[-1] != K:
        raise RuntimeError(f"fp8: x of shape {tuple(x.shape)} does not fit a weight of {K} input features")
    if x.is_cuda and torch.is_autocast_enabled("cuda"):
        x = x.to(torch.get_autocast_dtype("cuda"))
    _check_type("x", x)
    _check_device("x", x)
    if x.device != weight.device:
        raise RuntimeError(f"fp8: x is on {x.device}, the weight on {weight.device}")
    if packed:
        if torch.is_grad_enabled() and x.requires_grad:
            raise RuntimeError("fp8: an Fp8Weight has no backward pass: give the weight itself, or call under no_grad")
        return _linear_packed(x, weight)
    if not (x.numel() and weight.numel()):      # nothing to add up; differentiable
        return x @ weight.t().to(x.dtype)
    y = _Linear.apply(x.reshape(-1, K), weight)      # (a view made inside the node could not be written in place, as MLP's ReLU does)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], weight.shape[0])
