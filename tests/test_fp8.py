"""CPU: what the block-scaled 8-bit linear products refuse, the reference of their GPU tests against torch's own casts, and the library's checks."""
import ctypes as C

import pytest
import torch

import fp8_reference as R
from geneface_amd import fp8
from geneface_amd.cond_encoder import MLP


def _weight(n=130, k=200):
    return fp8.Fp8Weight(torch.zeros(n, 256, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(2, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu), k)


def test_reference_rounds_as_the_type_does():
    x = torch.cat([torch.linspace(-448, 448, 20001), torch.linspace(-0.02, 0.02, 4001), torch.tensor([0.0, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0])])
    assert torch.equal(R.to_grid(x.double()).float(), x.to(torch.float8_e4m3fn).float())


@pytest.mark.parametrize("a, e", [(448.0, 0), (448.0001, 1), (447.99, 0), (224.0, -1), (224.1, 0), (1.75, -8), (1.7500001, -7), (1.0, -8), (0.0, -127), (1e-45, -127),
                                  (3.4e38, 120)])
def test_reference_scale(a, e):
    assert float(R.scale_of(torch.tensor(a))) == 2.0 ** e
    s = 2.0 ** e
    assert float(torch.tensor(a)) <= 448 * s and (e == -127 or float(torch.tensor(a)) > 448 * s / 2)


@pytest.mark.parametrize("call, message", [
    (lambda: fp8.linear(torch.zeros(3, 5), torch.zeros(7, 5)), "CUDA"),
    (lambda: fp8.linear(torch.zeros(3, 5), torch.zeros(7, 6)), "does not fit"),
    (lambda: fp8.linear(torch.zeros(3, 5), torch.zeros(7, 5, 1)), "must be a matrix"),
    (lambda: fp8.linear(torch.zeros(()), torch.zeros(7, 5)), "does not fit"),
    (lambda: fp8.linear(torch.zeros(3, 5), torch.zeros(7, 5, dtype=torch.float64)), "must be float32"),
    (lambda: fp8.linear(torch.zeros(3, 200, dtype=torch.int32), _weight()), "must be float32"),
    (lambda: fp8.linear(torch.zeros(3, 201), _weight()), "does not fit"),
    (lambda: fp8.linear(torch.zeros(3, 200), _weight()), "CUDA"),
    (lambda: fp8.quantize_weight(torch.zeros(3)), "must be a matrix"),
    (lambda: fp8.quantize_weight(torch.zeros(3, 4)), "CUDA"),
    (lambda: fp8.Fp8Weight(torch.zeros(3, 128), torch.zeros(1, 1), 100), "float8_e4m3fn values"),
    (lambda: fp8.Fp8Weight(_weight().values[:, :128], _weight().scales, 200), "do not fit"),
    (lambda: fp8.Fp8Weight(_weight().values, _weight().scales[:1], 200), "do not fit"),
    (lambda: fp8.Fp8Weight(_weight().values, _weight().scales.t(), 200), "contiguous"),
])
def test_refusals(call, message):
    with pytest.raises(RuntimeError, match=message):
        call()


def test_mlp_precision():
    m = MLP(8, 3, 16, 2)
    x = torch.randn(5, 8)
    assert m.precision == "native" and torch.equal(m(x), m.net[1](torch.relu(m.net[0](x))))
    keys = set(m.state_dict())
    m.precision = "fp8"
    with pytest.raises(RuntimeError, match="CUDA"):
        m(x)
    m.precision = "fp7"
    with pytest.raises(ValueError, match="fp7"):
        m(x)
    assert set(m.state_dict()) == keys


def test_dequantized_weight():
    values = torch.tensor([[1.0, -448.0, 2.0 ** -9] + [0.0] * 125]).to(torch.float8_e4m3fn)
    for byte, s in ((127, 1.0), (130, 8.0), (1, 2.0 ** -126)):
        w = fp8.Fp8Weight(values, torch.tensor([[byte]], dtype=torch.uint8).view(torch.float8_e8m0fnu), 3)
        assert w.dequantize().tolist() == [[s, -448.0 * s, 2.0 ** -9 * s]]
    assert bool(fp8.Fp8Weight(values, torch.tensor([[255]], dtype=torch.uint8).view(torch.float8_e8m0fnu), 3).dequantize().isnan().all())


def test_the_library_refuses_bad_descriptors(hip_lib):
    def refused(rc, word):
        assert rc == 1 and word in hip_lib.gf_last_error(), hip_lib.gf_last_error()
    q = lambda **k: C.byref(fp8.GfFp8Quantize(**{"src": 16, "rows": 3, "cols": 5, "ld": 5, "row_codes": 16, "row_scales": 16, "row_pitch": 3, "col_pitch": 5, **k}))      # noqa: E731
    refused(hip_lib.gf_fp8_quantize(None, None), b"null")
    assert hip_lib.gf_fp8_quantize(q(rows=0), None) == 0 and hip_lib.gf_fp8_quantize(q(cols=0), None) == 0
    refused(hip_lib.gf_fp8_quantize(q(src=None), None), b"null")
    refused(hip_lib.gf_fp8_quantize(q(row_codes=None), None), b"null")
    refused(hip_lib.gf_fp8_quantize(q(row_scales=None), None), b"null scales")
    refused(hip_lib.gf_fp8_quantize(q(col_codes=16), None), b"null scales")
    refused(hip_lib.gf_fp8_quantize(q(tiles=1), None), b"null scales")
    refused(hip_lib.gf_fp8_quantize(q(dtype=9), None), b"dtype")
    refused(hip_lib.gf_fp8_quantize(q(ld=4), None), b"ld < cols")
    refused(hip_lib.gf_fp8_quantize(q(row_pitch=2), None), b"pitch")
    refused(hip_lib.gf_fp8_quantize(q(rows=1 << 40, cols=1 << 40, ld=1 << 40, row_pitch=1 << 40), None), b"too large")
    # gf_fp8_matmul_t as 64-bit words: a and b (codes, scales, pitch, stride of a tile's row and block), m, n, blocks, out, dtype, workspace
    base = {"a_codes": 16, "a_scales": 16, "a_pitch": 300, "b_codes": 16, "b_scales": 16, "b_pitch": 300, "m": 300, "n": 300, "blocks": 2, "out": 16}
    order = ["a_codes", "a_scales", "a_pitch", "a_row", "a_block", "b_codes", "b_scales", "b_pitch", "b_row", "b_block", "m", "n", "blocks", "out", "dtype", "workspace"]
    m = lambda **k: (C.c_uint64 * 16)(*[{**base, **k}.get(n, 0) for n in order])      # noqa: E731
    refused(hip_lib.gf_fp8_matmul(None, None), b"null")
    assert hip_lib.gf_fp8_matmul(m(m=0), None) == 0 and hip_lib.gf_fp8_matmul(m(n=0), None) == 0
    refused(hip_lib.gf_fp8_matmul(m(out=0), None), b"null output")
    refused(hip_lib.gf_fp8_matmul(m(dtype=3), None), b"dtype")
    refused(hip_lib.gf_fp8_matmul(m(blocks=0), None), b"no blocks")
    refused(hip_lib.gf_fp8_matmul(m(a_codes=0), None), b"a: null")
    refused(hip_lib.gf_fp8_matmul(m(b_scales=0), None), b"b: null")
    refused(hip_lib.gf_fp8_matmul(m(b_codes=24), None), b"multiple of 16")
    refused(hip_lib.gf_fp8_matmul(m(b_pitch=299), None), b"pitch")
    refused(hip_lib.gf_fp8_matmul(m(blocks=1 << 16), None), b"too large")
    refused(hip_lib.gf_fp8_matmul(m(blocks=1000), None), b"workspace")
    assert hip_lib.gf_fp8_matmul_workspace_bytes(300, 300, 1000) % (4 * 300 * 300) == 0 and hip_lib.gf_fp8_matmul_workspace_bytes(300, 300, 1) == 0
    f = lambda **k: fp8.GfFp8Linear(**{"x": 16, "ldx": 150, "w": 16, "ldw": 150, "m": 300, "n": 200, "k": 150, "y": 16, "workspace": 256, "saved": 256, "keep_x": 1, **k})      # noqa: E731
    refused(hip_lib.gf_fp8_linear_plan(None), b"null")
    refused(hip_lib.gf_fp8_linear_plan(C.byref(f(k=0))), b"empty")
    for change in (dict(m=1 << 24), dict(k=1 << 24), dict(n=1 << 24, keep_w=1)):
        refused(hip_lib.gf_fp8_linear_plan(C.byref(f(**change))), b"along a sum")
        refused(hip_lib.gf_fp8_linear(C.byref(f(**change)), None), b"along a sum")
    for change in (dict(m=1 << 24, keep_x=0), dict(n=1 << 24), dict(m=1 << 24, n=128, k=128)):
        assert hip_lib.gf_fp8_linear_plan(C.byref(f(**change))) == 0
    p = f(keep_w=1)
    assert hip_lib.gf_fp8_linear_plan(C.byref(p)) == 0 and p.saved_bytes >= 150 * 256 + 4 + 150 * 384 + 3 * 150 and p.workspace_bytes >= 300 * 256 and p.backward_bytes >= 300 * 256 + 200 * 384
    refused(hip_lib.gf_fp8_linear(None, None), b"null")
    for change in (dict(x=None), dict(y=None), dict(w=None)):
        refused(hip_lib.gf_fp8_linear(C.byref(f(**change)), None), b"null pointer")
    refused(hip_lib.gf_fp8_linear(C.byref(f(n=0)), None), b"empty")
    refused(hip_lib.gf_fp8_linear(C.byref(f(m=1 << 31)), None), b"too large")
    refused(hip_lib.gf_fp8_linear(C.byref(f(saved=None)), None), b"null buffer")
    refused(hip_lib.gf_fp8_linear(C.byref(f(workspace=16)), None), b"multiples of 256")
    refused(hip_lib.gf_fp8_linear(C.byref(f(w=None, codes=16, scales=16)), None), b"no backward")
    g = lambda **k: C.byref(fp8.GfFp8LinearBackward(**{"dy": 16, "lddy": 200, "saved": 256, "m": 300, "n": 200, "k": 150, "dx": 16, "dw": 16, "workspace": 256, "keep_w": 1, "keep_x": 1, **k}))      # noqa: E731
    refused(hip_lib.gf_fp8_linear_backward(None, None), b"null")
    assert hip_lib.gf_fp8_linear_backward(g(dx=None, dw=None), None) == 0
    refused(hip_lib.gf_fp8_linear_backward(g(dy=None), None), b"null")
    refused(hip_lib.gf_fp8_linear_backward(g(keep_x=0), None), b"not kept")
    refused(hip_lib.gf_fp8_linear_backward(g(keep_w=0), None), b"not kept")
    refused(hip_lib.gf_fp8_linear_backward(g(saved=16), None), b"multiples of 256")
    thin = ["x", "ldx", "m", "n", "k", "codes", "scale", "y", "col_codes", "col_scales", "dtype"]
    t = lambda **k: (C.c_uint64 * 11)(*[{**dict(x=16, ldx=5, m=300, n=7, k=5, codes=16, scale=16, y=16, col_codes=16, col_scales=16), **k}.get(n, 0) for n in thin])      # noqa: E731
    refused(hip_lib.gf_fp8_thin(None, None), b"null")
    for change, word in ((dict(n=129), b"1 to 128"), (dict(k=0), b"1 to 128"), (dict(m=0), b"rows"), (dict(dtype=3), b"dtype"), (dict(x=0), b"null"), (dict(scale=0), b"null"),
                         (dict(col_scales=0), b"null"), (dict(codes=24), b"multiple of 16"), (dict(ldx=4), b"ldx < k")):
        refused(hip_lib.gf_fp8_thin(t(**change), None), word)
    back = ["dy", "lddy", "m", "n", "k", "codes", "scale", "col_codes", "col_scales", "dx", "dw", "workspace", "dtype"]
    b = lambda **k: (C.c_uint64 * 13)(*[{**{n: 16 for n in back if n != "dtype"}, "lddy": 7, "m": 300, "n": 7, "k": 5, **k}.get(n, 0) for n in back])      # noqa: E731
    refused(hip_lib.gf_fp8_thin_backward(None, None), b"null")
    assert hip_lib.gf_fp8_thin_backward(b(dx=0, dw=0), None) == 0
    for change, word in ((dict(n=129), b"1 to 128"), (dict(m=1 << 31), b"rows"), (dict(dy=0), b"null"), (dict(codes=0), b"null"), (dict(col_codes=0), b"null"),
                         (dict(workspace=0), b"null"), (dict(lddy=6), b"lddy < n"), (dict(dtype=7 << 32), b"dtype"), (dict(dtype=7), b"dtype")):
        refused(hip_lib.gf_fp8_thin_backward(b(**change), None), word)
    assert hip_lib.gf_fp8_thin_workspace_bytes(300, 7, 5) == 3 * 7 * 5 * 4 and hip_lib.gf_fp8_thin_workspace_bytes(300, 129, 5) == 0
    rows = ["x", "m", "n", "k", "ldx", "codes", "scales", "out", "dtype"]
    r = lambda **k: (C.c_uint64 * 9)(*[{**{"x": 16, "m": 3, "n": 7, "k": 5, "ldx": 5, "codes": 16, "scales": 16, "out": 16}, **k}.get(n, 0) for n in rows])      # noqa: E731
    refused(hip_lib.gf_fp8_rows(None, None), b"null")
    assert hip_lib.gf_fp8_rows(r(m=0), None) == 0
    refused(hip_lib.gf_fp8_rows(r(x=0), None), b"null")
    refused(hip_lib.gf_fp8_rows(r(m=17), None), b"at most 16")
    refused(hip_lib.gf_fp8_rows(r(dtype=3), None), b"dtype")
    refused(hip_lib.gf_fp8_rows(r(k=0), None), b"k = 0")
    refused(hip_lib.gf_fp8_rows(r(ldx=4), None), b"ldx < k")
    refused(hip_lib.gf_fp8_rows(r(codes=24), None), b"multiple of 16")
