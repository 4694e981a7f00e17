"""The operators of an 8-bit training step, as cases that can be measured: block-scaled 8-bit linear products and AdamW over many tensors.

`run` with `own` false computes each operator from elementary torch operations, with `own` true through `geneface_amd.fp8` and
`geneface_amd.optim`.  The formats are those of these two modules:

* 8-bit values are e4m3 (largest 448) with a scale for each block of 128.
* the scales of the products are powers of two.  For the largest magnitude `a` of a block the exponent is the smallest e >= -127 with
  a <= 448 * 2^e; it is held as the byte e + 127.  Values are rounded to nearest even.  A block that holds an infinity or a NaN is NaN as a whole.
* a weight [N, K] has blocks of 128 x 128, an operand that is summed over an axis has blocks of 128 along that axis.  Rows are padded with
  zeros to a multiple of 128.
* the 8-bit moments of AdamW have blocks of 128 consecutive values of their tensor and 32-bit scales max(a, 2^-100) / 448.  The second moment
  is held as its square root.  They are rounded with a dither that is a function of the step and of the value's index, so that changes far
  below the spacing of the format add up.
"""
import math
import random

import torch

own = False

LR, BETA1, BETA2, EPS, DECAY = 5e-4, 0.9, 0.99, 1e-15, 0.01   # the framework's training step, with a weight decay
MAX_NORM, GRAD_SCALE = 1.0, 1024.0
DITHER_INDEX, DITHER_STEP = 3242174889, 2447445414            # 2^32 / rho and 2^32 / rho^2, rho the real root of x^3 = x + 1
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    adamw = lambda **k: {"op": "adamw", **k}          # noqa: E731
    serve = lambda **k: {"op": "serve", **k}          # noqa: E731
    train = lambda **k: {"op": "train", **k}          # noqa: E731
    return [
        # the 24 tensors of the condition encoder: all latency
        adamw(name="adamw-cond", tensors=24, total=53243, bits=32, dtype="float32", scaled=False, clip=False),
        # the RAD-NeRF head's 35 tensors under a gradient scaler: two tables hold most of it
        adamw(name="adamw-head", tensors=35, total=3112587, bits=32, dtype="float32", scaled=True, clip=False),
        # the head and torso together, 8-bit moments, clipped to a norm
        adamw(name="adamw8-torso-clip", tensors=43, total=4344011, bits=8, dtype="float32", scaled=True, clip=True),
        # a large model with 16-bit weights and 8-bit moments
        adamw(name="adamw8-200m-bf16", tensors=157, total=200_000_003, bits=8, dtype="bfloat16", scaled=False, clip=False),
        # the largest: 32-bit everything, clipped
        adamw(name="adamw-250m-clip", tensors=97, total=250_000_007, bits=32, dtype="float32", scaled=False, clip=True),
        # one row through a layer whose 8-bit weight is kept: what a frame-by-frame condition network does
        serve(name="linear8-one-row", M=1, N=4096, K=4096, dtype="bfloat16"),
        # a few rows, sizes that divide nothing
        serve(name="linear8-few-rows", M=7, N=1111, K=2050, dtype="float16"),
        # a window of rows through a wide layer
        serve(name="linear8-window", M=333, N=2048, K=8192, dtype="bfloat16"),
        # a large batch
        serve(name="linear8-large", M=8192, N=8192, K=4096, dtype="bfloat16"),
        # the field's first layer over the samples of a training batch (96 -> 128), 32-bit activations
        train(name="train8-tall", M=262221, N=128, K=96, dtype="float32"),
        # the density head's last layer (128 -> 129) beside the colour input's width, half precision
        train(name="train8-odd", M=1000, N=129, K=148, dtype="float16"),
        # a wide layer
        train(name="train8-wide", M=4096, N=4096, K=4096, dtype="bfloat16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    op = rng.choice(["adamw", "serve", "train"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    if op == "adamw":
        tensors = _log(rng, 1, 200)
        return {"op": op, "tensors": tensors, "total": max(tensors, _log(rng, 1000, 200_000_000)), "bits": rng.choice([8, 32]), "dtype": dtype,
                "scaled": rng.random() < 0.5, "clip": rng.random() < 0.5}
    if op == "serve":
        M, N, K = _log(rng, 1, 8192), _log(rng, 1, 8192), _log(rng, 1, 8192)
        if M * N * K > 8192 * 8192 * 4096:
            K = 4096 - rng.randrange(128)
    elif rng.random() < 0.5:
        M, N, K = _log(rng, 4096, 262144), _log(rng, 1, 128), _log(rng, 1, 96)
    else:
        M, N, K = _log(rng, 1, 4096), _log(rng, 1, 4096), _log(rng, 1, 4096)
    return {"op": op, "M": M, "N": N, "K": K, "dtype": dtype}


def _sizes(case):
    """The tensors' sizes: spread over a factor of some hundreds, as a model's are, most of them odd."""
    r = random.Random(case["tensors"] * 1000003 + case["total"])
    w = [math.exp(2.0 * r.gauss(0, 1)) for _ in range(case["tensors"])]
    return [max(1, int(case["total"] * v / sum(w))) for v in w]


def _up(n, m=128):
    return -(-n // m) * m


# ---------------------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")     # noqa: E731
    t = TYPES[case["dtype"]]
    if case["op"] == "adamw":
        return _prepare_adamw(case, g, normal, t)
    M, N, K = case["M"], case["N"], case["K"]
    # rows and columns of unlike size, as layers have them
    x = (normal(M, K) * (0.5 * normal(M, 1)).exp() * (0.5 * normal(K)).exp()).to(t)
    w = normal(N, K) * (0.5 * normal(N, 1)).exp() / math.sqrt(K)
    if case["op"] == "serve":
        values, scales = _encode_tiles(w)      # what such a program keeps: the weight in 8 bits and its scales
        return {"case": case, "x": x, "values": values, "scales": scales}
    dy = (normal(M, N) * (1.0 * normal(M, 1)).exp() / M).to(t)
    return {"case": case, "x": x.requires_grad_(True), "w": w.requires_grad_(True), "dy": dy}


def _prepare_adamw(case, g, normal, t):
    sizes = _sizes(case)
    room = [_up(n) for n in sizes]             # one buffer for all tensors, each at a multiple of 128 values
    at = [0]
    for n in room:
        at.append(at[-1] + n)
    total, dev = at[-1], "cuda"
    s = {"case": case, "sizes": sizes}
    keep = torch.zeros(total, dtype=torch.bool, device=dev)
    views = lambda flat: [flat[a:a + n] for a, n in zip(at, sizes)]     # noqa: E731
    for v in views(keep):
        v.fill_(True)
    spread = torch.repeat_interleave(normal(len(sizes)).exp(), torch.tensor(room, device=dev), output_size=total) * keep
    p = normal(total) * 0.1 * keep
    grad = normal(total) * spread
    grad = grad * (torch.rand(total, generator=g, device=dev) < 0.7)    # a table's rows that no sample touched have none
    m = 0.3 * spread * normal(total)
    r = spread * (0.2 * normal(total)).exp() * (torch.rand(total, generator=g, device=dev) < 0.9)
    m = m * (r > 0)
    if case["scaled"]:
        grad = grad * GRAD_SCALE
        s["grad_scale"], s["found_inf"] = torch.full((1,), GRAD_SCALE, device=dev), torch.zeros(1, device=dev)
    if t == torch.float16:
        grad = grad.clamp(-60000, 60000)
    s["p"], s["grad"] = p.to(t), grad.to(t)
    del p, grad, spread, keep
    if case["bits"] == 8:
        s["m"], s["m_scale"] = _nearest_blocks(m)
        s["r"], s["r_scale"] = _nearest_blocks(r)
        blocks = lambda flat: [flat[a // 128:a // 128 + _up(n) // 128] for a, n in zip(at, sizes)]     # noqa: E731
        s["m_scales"], s["r_scales"] = blocks(s["m_scale"]), blocks(s["r_scale"])
    else:
        s["m"], s["r"] = m, r * r
    s["steps"] = torch.randint(1, 2000, (len(sizes),), generator=g, device=dev).float()
    for k in ("p", "grad", "m", "r"):
        s[k + "s"] = views(s[k])
    s["step_list"] = [s["steps"][i] for i in range(len(sizes))]
    s["room"], s["start"] = torch.tensor(room, device=dev), torch.tensor(at[:-1], device=dev)
    return s


# ---------------------------------------------------------------------------------------------------------------- the formats

def _block_exponent(a):
    """The byte e + 127 of a block whose largest magnitude is `a` (any floating type), as int64: 255 where it is no finite number."""
    f, x = torch.frexp(a.double())
    e = torch.where(f <= 0.875, x - 9, x - 8).long()         # 448 = 0.875 * 2^9
    e = torch.where(a > 0, e.clamp(min=-127), -127) + 127
    return torch.where(torch.isfinite(a), e, 255)


def _power(byte):
    """2^(byte - 127) in 64 bits."""
    return ((byte.long() + (1023 - 127)) << 52).view(torch.float64)


def _encode_rows(x):
    """[R, K] -> (values e4m3 [R, up(K)], bytes int64 [R, up(K)/128])."""
    R, K = x.shape
    v = torch.zeros(R, _up(K), dtype=torch.float32, device=x.device)
    v[:, :K] = x
    v = v.view(R, -1, 128)
    byte = _block_exponent(v.abs().amax(-1))
    q = (v * (1.0 / _power(byte)).float()[..., None]).to(torch.float8_e4m3fn)
    return q.view(R, -1), byte


def _decode_rows(q, byte, K):
    return (q.float().view(q.shape[0], -1, 128) * _power(byte).float()[..., None]).view(q.shape[0], -1)[:, :K]


def _encode_tiles(w):
    """[N, K] -> (values e4m3 [N, up(K)], scales e8m0 [up(N)/128, up(K)/128])."""
    N, K = w.shape
    v = torch.zeros(_up(N), _up(K), dtype=torch.float32, device=w.device)
    v[:N, :K] = w
    v = v.view(_up(N) // 128, 128, _up(K) // 128, 128)
    byte = _block_exponent(v.abs().amax((1, 3)))
    q = (v * (1.0 / _power(byte)).float()[:, None, :, None]).view(_up(N), _up(K))[:N].to(torch.float8_e4m3fn)
    return q.contiguous(), byte.to(torch.uint8).view(torch.float8_e8m0fnu)


def _decode_tiles(q, scales, K):
    N = q.shape[0]
    s = _power(scales.view(torch.uint8)).float()
    s = s.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)
    return (q.float() * s)[:, :K]


def _moment_blocks(m):
    """A flat tensor of whole blocks -> (blocks divided by their scales, 32-bit scales)."""
    v = m.view(-1, 128)
    a = v.abs().amax(-1).clamp(min=2.0 ** -100)
    return v * (448 / a)[:, None], a / 448


def _nearest_blocks(m):
    """e4m3 values and scales, rounded to nearest: what a program's state may hold at some step."""
    y, scale = _moment_blocks(m)
    return y.clamp(-448, 448).to(torch.float8_e4m3fn).view(-1), scale


def _dithered_blocks(m, u, positive):
    """The same with each value rounded down or up by the dither u in [0, 1): floor(value / spacing + u).  `positive`: what is above zero stays so."""
    y, scale = _moment_blocks(m)
    spacing = _power((torch.frexp(y)[1].long() - 1).clamp(min=-6) - 3 + 127)
    k = torch.floor(y.abs().double() / spacing + u.view(-1, 128))
    if positive:
        k = torch.where(m.view(-1, 128) > 0, k.clamp(min=1), k)
    q = torch.copysign((k * spacing).clamp(max=448).float(), y).to(torch.float8_e4m3fn)
    return q.view(-1), scale


# ---------------------------------------------------------------------------------------------------------------- one pass

def run(s):
    return {"adamw": _run_adamw, "serve": _run_serve, "train": _run_train}[s["case"]["op"]](s)


def _run_serve(s):
    if own:
        from geneface_amd import fp8
        return fp8.linear(s["x"], fp8.Fp8Weight(s["values"], s["scales"], s["case"]["K"]))
    K = s["case"]["K"]
    x = _decode_rows(*_encode_rows(s["x"]), K)
    return (x @ _decode_tiles(s["values"], s["scales"], K).t()).to(s["x"].dtype)


def _run_train(s):
    x, w, dy = s["x"], s["w"], s["dy"]
    if own:
        from geneface_amd import fp8
        y = fp8.linear(x, w)
        dx, dw = torch.autograd.grad(y, (x, w), dy)
        return {"y": y.detach(), "dx": dx, "dw": dw}
    with torch.no_grad():
        (M, K), N = x.shape, w.shape[0]
        w8 = _decode_tiles(*_encode_tiles(w), K)
        y = _decode_rows(*_encode_rows(x), K) @ w8.t()
        dx = _decode_rows(*_encode_rows(dy), N) @ w8
        dw = _decode_rows(*_encode_rows(dy.t()), M) @ _decode_rows(*_encode_rows(x.t()), M).t()
        return {"y": y.to(x.dtype), "dx": dx.to(x.dtype), "dw": dw}


def _outputs(s, norm):
    got = {"p": s["p"], "m": s["m"], "v": s["r"], "steps": s["steps"]}
    if s["case"]["bits"] == 8:
        got |= {"m_scale": s["m_scale"], "v_scale": s["r_scale"]}
    if norm is not None:
        got["norm"] = norm
    return got


def _run_adamw(s):
    case, eight = s["case"], s["case"]["bits"] == 8
    if own:
        from geneface_amd import optim
        norm = optim.grad_norm(s["grads"], grad_scale=s.get("grad_scale")) if case["clip"] else None
        optim.adamw_step(s["ps"], s["grads"], s["ms"], s["rs"], s["step_list"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
                         exp_avg_scales=s["m_scales"] if eight else None, exp_avg_sq_scales=s["r_scales"] if eight else None,
                         grad_scale=s.get("grad_scale"), found_inf=s.get("found_inf"), grad_norm=norm, max_norm=MAX_NORM if case["clip"] else None)
        return _outputs(s, norm)
    total = s["p"].numel()
    each = lambda v: torch.repeat_interleave(v, s["room"], output_size=total)     # noqa: E731
    c, norm = 1.0, None
    if case["scaled"]:
        c = 1.0 / s["grad_scale"].double()
    if case["clip"]:
        norm = s["grad"].double().square().sum().sqrt() * c
        c = c * (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
        norm = norm.float().reshape(())
    grad = s["grad"].float() * (c.float() if isinstance(c, torch.Tensor) else c)
    new_steps = s["steps"] + 1
    t = new_steps.double()
    rate, root = each((LR / (1 - BETA1 ** t)).float()), each((1 - BETA2 ** t).sqrt().float())
    if eight:
        wide = lambda q, scale: (q.float().view(-1, 128) * scale[:, None]).view(-1)     # noqa: E731
        m, v = wide(s["m"], s["m_scale"]), wide(s["r"], s["r_scale"]).square()
    else:
        m, v = s["m"], s["r"]
    m = m + (1 - BETA1) * (grad - m)
    v = BETA2 * v + (1 - BETA2) * grad * grad
    r = v.sqrt()
    p = s["p"].float() * (1 - LR * DECAY)
    p = (p - rate * m / (r / root + EPS)).to(s["p"].dtype)
    new = {"p": p, "steps": new_steps}
    if eight:
        index = torch.arange(total, device=p.device) - each(s["start"])
        word = (index * DITHER_INDEX + each(new_steps.long()) * DITHER_STEP) & 0xffffffff
        u = (word >> 12).double() * 2.0 ** -20
        new["m"], new["m_scale"] = _dithered_blocks(m, u, False)
        new["r"], new["r_scale"] = _dithered_blocks(r, (u + 0.5) % 1.0, True)
    else:
        new["m"], new["r"] = m, v
    for k, value in new.items():
        if case["scaled"]:                     # a step whose gradients overflowed leaves everything as it was
            value = torch.where(s["found_inf"] == 0, value.float(), s[k].float()).to(s[k].dtype)
        s[k].copy_(value)
    return _outputs(s, norm)


# ---------------------------------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    b = torch.empty(0, dtype=TYPES[case["dtype"]]).element_size()
    if case["op"] == "adamw":
        n = sum(_sizes(case))
        state = 16 if case["bits"] == 32 else 4 * (1 + 4 / 128)          # two moments, read and written
        return {"bytes": n * (3 * b + state) + 8 * case["tensors"], "flops": n * (18 + 2 * case["clip"])}
    M, N, K = case["M"], case["N"], case["K"]
    if case["op"] == "serve":
        return {"bytes": M * K * b + N * K + N * K / 16384 + M * N * b, "flops": 2 * M * N * K}
    return {"bytes": 2 * M * K * b + 2 * M * N * b + 8 * N * K, "flops": 6 * M * N * K}


# ---------------------------------------------------------------------------------------------------------------- the definitions in 64 bits

def _grid(x, axis):
    """x in 64 bits on the 8-bit grid of its blocks of 128 along `axis`: nearest even on a grid of four significant bits, 2^-9 apart at least."""
    n = x.shape[axis]
    v = x.double().movedim(axis, -1)
    v = torch.nn.functional.pad(v, (0, -n % 128)).unflatten(-1, (-1, 128))
    return _on_grid(v, v.abs().amax(-1, keepdim=True)).flatten(-2)[..., :n].movedim(-1, axis)


def _tile_grid(x):
    N, K = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -K % 128, 0, -N % 128)).unflatten(1, (-1, 128)).unflatten(0, (-1, 128))
    return _on_grid(v, v.abs().amax((1, 3), keepdim=True)).flatten(2, 3).flatten(0, 1)[:N, :K]


def _scale_of(a):
    """The smallest power of two s with a <= 448 s."""
    s = torch.exp2(torch.ceil(torch.log2(a.clamp(min=2.0 ** -110) / 448)).round())
    s = torch.where(a > 448 * s, 2 * s, s)
    return torch.where(a <= 224 * s, s / 2, s)


def _on_grid(v, a):
    s = _scale_of(a)
    y = v / s
    gap = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))) / 8
    gap = torch.where(y.abs() >= 16 * gap, 2 * gap, gap)
    return torch.round(y / gap) * gap * s          # torch.round takes ties to even


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(case, s)
    with torch.no_grad():
        x = s["x"]
        if case["op"] == "serve":
            w = s["values"].double()[:, :case["K"]]
            byte = s["scales"].view(torch.uint8).double()
            rows, cols = torch.arange(case["N"], device="cuda") // 128, torch.arange(case["K"], device="cuda") // 128
            return _grid(x, 1) @ (w * torch.exp2(byte - 127)[rows][:, cols]).t()
        w8, dy = _tile_grid(s["w"]), s["dy"]
        return {"y": _grid(x, 1) @ w8.t(), "dx": _grid(dy, 1) @ w8, "dw": _grid(dy, 0).t().contiguous() @ _grid(x, 0)}


def _exact_adamw(case, s):
    eight = case["bits"] == 8
    whole = s["p"].double()
    out = {k: torch.zeros_like(whole) for k in ("p", "m", "v")}
    out["p"].copy_(whole)
    out |= {"steps": s["steps"].double() + 1}
    if eight:
        out |= {k + "_scale": torch.zeros_like(s["m_scale"], dtype=torch.float64) for k in ("m", "v")}
    c = 1.0 / GRAD_SCALE if case["scaled"] else 1.0
    if case["clip"]:
        norm = math.sqrt(sum(float((g.double() * c).pow(2).sum()) for g in s["grads"]))
        out["norm"] = torch.tensor(norm, dtype=torch.float64)
        c *= min(1.0, MAX_NORM / (norm + 1e-6))
    at = 0
    for i, n in enumerate(s["sizes"]):
        here, t = slice(at, at + n), float(out["steps"][i])
        blocks = slice(at // 128, (at + _up(n)) // 128)
        g, m, v = s["grads"][i].double() * c, s["ms"][i].double(), s["rs"][i].double()
        if eight:
            m = m * s["m_scales"][i].double().repeat_interleave(128)[:n]
            v = (v * s["r_scales"][i].double().repeat_interleave(128)[:n]) ** 2
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g * g
        step = (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
        out["p"][here] = s["ps"][i].double() * (1 - LR * DECAY) - LR * step
        if eight:
            k = torch.arange(n, device="cuda")
            u = torch.remainder(k * DITHER_INDEX + int(t) * DITHER_STEP, 2 ** 32) // 4096
            for name, value, shift in (("m", m, 0.0), ("v", v.sqrt(), 0.5)):
                b = torch.nn.functional.pad(value, (0, -n % 128)).view(-1, 128)
                scale = b.abs().amax(1).clamp(min=2.0 ** -100) / 448
                y = (b / scale[:, None]).view(-1)[:n]
                gap = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6)))) / 8
                steps = torch.floor(y.abs() / gap + torch.remainder(u / 2.0 ** 20 + shift, 1.0))
                if name == "v":
                    steps = torch.where(y > 0, steps.clamp(min=1), steps)
                out[name][here] = torch.sign(y) * (steps * gap).clamp(max=448)
                out[name + "_scale"][blocks] = scale
        else:
            out["m"][here], out["v"][here] = m, v
        at += _up(n)
    return out
