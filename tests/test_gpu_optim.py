"""GPU: AdamW over many tensors and the gradients' norm (geneface_amd.optim) against the formulas in 64 bits.

Tolerances are counts of roundings.  eps = 2^-24 is half a step of a 32-bit value.  One step makes at most 4 roundings on the first moment, each
relative to |m| + |g|, 4 on the second relative to itself, 6 more on the quotient, 2 on the parameter, then one to the parameter's type.  The tests
allow twice that.  An 8-bit code is floor(value / spacing + u): it can differ only where that sum is within the value's own error of a whole number.
"""
import copy
import math

import pytest
import torch

from geneface_amd import optim

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24
A, B = 3242174889, 2447445414


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _place(x, offset):
    """x on the GPU, `offset` values behind an aligned address."""
    flat = torch.zeros(x.numel() + 16, dtype=torch.uint8 if x.dtype == torch.float8_e4m3fn else x.dtype, device="cuda").view(x.dtype)
    out = flat[offset:offset + x.numel()].view(x.shape)
    out.copy_(x) if x.dtype != torch.float8_e4m3fn else out.view(torch.uint8).copy_(x.view(torch.uint8))
    return out


class Case:
    def __init__(self, sizes, dtype, bits, seed, offset=0, sparse=0.3):
        g = _gen(seed)
        r = lambda n: torch.randn(n, generator=g)      # noqa: E731
        self.sizes, self.dtype, self.bits = sizes, dtype, bits
        self.p = [_place((0.3 * r(n)).to(dtype), offset) for n in sizes]
        self.g = [_place((r(n) * (torch.rand(n, generator=g) > sparse)).to(dtype), offset) for n in sizes]
        self.steps = [torch.tensor(float(i % 5), device="cuda") for i in range(len(sizes))]
        self.ms = self.vs = None
        if bits == 32:
            self.m = [_place(0.3 * r(n), offset) for n in sizes]
            self.v = [_place(torch.rand(n, generator=g) ** 4, offset) for n in sizes]
        else:
            code = lambda n, lo: torch.randint(lo, 127, (n,), generator=g).to(torch.uint8)      # noqa: E731
            self.m = [_place((code(n, 0) + 128 * code(n, 0).remainder(2)).view(torch.float8_e4m3fn), offset) for n in sizes]
            self.v = [_place(code(n, 0).view(torch.float8_e4m3fn), offset) for n in sizes]
            self.ms = [torch.rand(-(-n // 128), generator=g).cuda() / 448 for n in sizes]
            self.vs = [torch.rand(-(-n // 128), generator=g).cuda() / 448 for n in sizes]

    def before(self):
        wide = lambda q, s, n: q.double().cpu() * (s.double().cpu().repeat_interleave(128)[:n] if s is not None else 1)      # noqa: E731
        none = [None] * len(self.sizes)
        m = [wide(q, s, n) for q, s, n in zip(self.m, self.ms or none, self.sizes)]
        v = [wide(q, s, n) for q, s, n in zip(self.v, self.vs or none, self.sizes)]
        return {"p": [p.double().cpu() for p in self.p], "g": [g.double().cpu() for g in self.g], "m": m, "v": v if self.bits == 32 else [x * x for x in v],
                "t": [int(s) + 1 for s in self.steps]}

    def step(self, **kw):
        optim.adamw_step(self.p, self.g, self.m, self.v, self.steps, exp_avg_scales=self.ms, exp_avg_sq_scales=self.vs, **kw)


def _check(case, old, lr, betas, eps, weight_decay, c=1.0):
    b1, b2 = betas
    half = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[case.dtype]
    for i, n in enumerate(case.sizes):
        p0, g, m0, v0, t = old["p"][i], old["g"][i] * c, old["m"][i], old["v"][i], old["t"][i]
        assert float(case.steps[i]) == t
        m, v = m0 + (1 - b1) * (g - m0), b2 * v0 + (1 - b2) * g * g
        root = v.sqrt() / math.sqrt(1 - b2 ** t) + eps
        rate = lr / (1 - b1 ** t)
        p = p0 * (1 - lr * weight_decay) - rate * m / root
        big = m0.abs() + g.abs()
        off_m, off_v = 8 * EPS * big + 1e-44, 8 * EPS * v + 1e-44
        off_p = 4 * EPS * p0.abs() + rate * (off_m + 12 * EPS * m.abs()) / root + (half + 2 * EPS) * p.abs() + (2.0 ** -25 if case.dtype == torch.float16 else 1e-44)
        got = case.p[i].double().cpu()
        # half a step above the largest value of the type (binary16: 65504 + 16) the nearest is infinity
        top = torch.finfo(case.dtype).max * (1 + half / 2)
        fine = (got - p).abs() <= off_p
        fine |= torch.isinf(got) & (torch.sign(got) * p + off_p.nan_to_num(0.0, 0.0) >= top)
        worst = float(((got - p).abs() - off_p)[~fine].max()) if not bool(fine.all()) else 0.0
        assert worst == 0.0, (i, n, worst)
        if case.bits == 32:
            assert bool(((case.m[i].double().cpu() - m).abs() <= off_m).all()) and bool(((case.v[i].double().cpu() - v).abs() <= off_v).all()), (i, n)
            continue
        k = torch.arange(n)
        u = ((k * A + t * B) % 2 ** 32 // 4096).double() / 2 ** 20
        for value, off, q, s, shift in ((m, off_m, case.m[i], case.ms[i], 0.0), (v.sqrt(), 8 * EPS * v.sqrt(), case.v[i], case.vs[i], 0.5)):
            a = torch.nn.functional.pad(value.abs(), (0, -n % 128)).view(-1, 128).amax(1).clamp(min=2.0 ** -100)
            loose = torch.nn.functional.pad(off, (0, -n % 128)).view(-1, 128).amax(1) / a
            assert bool(((s.double().cpu() * 448 / a - 1).abs() <= loose + 4 * EPS).all())
            y = value.abs() / (a / 448).repeat_interleave(128)[:n]
            gap = 2.0 ** (torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
            x = y / gap + (u + shift) % 1
            slack = (off / (a / 448).repeat_interleave(128)[:n] + y * (loose.repeat_interleave(128)[:n] + 6 * EPS)) / gap + 2.0 ** -20
            code = q.double().cpu()
            assert bool((torch.signbit(code) == torch.signbit(value))[code != 0].all())
            # a value within its error of a power of two may be taken from the other side, where the spacing is another: its code is the power then
            steps = code.abs() / gap
            want = torch.floor(x)
            if shift:
                want = torch.where(value > 0, want.clamp(min=1), want)
            near = (x - torch.round(x)).abs() <= slack
            same = steps == (want * gap).clamp(max=448) / gap
            assert bool((same | (near & ((steps - x).abs() <= 1 + slack))).all()), (i, n)
            assert float((~same).double().mean()) < 0.01 or n < 1000


SIZES = [1, 3, 4, 5, 127, 128, 129, 1000, 1023, 1024, 1025, 4099, 100003]
HYPER = dict(lr=3e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("offset", [0, 1, 4])
def test_one_step_matches_the_formula(dtype, bits, offset):
    case = Case(SIZES, dtype, bits, 1 + offset, offset)
    for _ in range(3):
        old = case.before()
        case.step(**HYPER)
        _check(case, old, **HYPER)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_among_them_empty_ones(bits):
    sizes = [(i * i) % 300 if i % 7 else 0 for i in range(1, 200)]
    case = Case(sizes, torch.float32, bits, 5)
    old = case.before()
    case.step(**HYPER)
    _check(case, old, **HYPER)


@pytest.mark.parametrize("bits", [32, 8])
def test_nothing_else_is_written(bits):
    """Guard values around every tensor stay as they were: sizes that end inside a vector, a block and a workgroup's chunk."""
    for n in (1, 5, 130, 1027, 9001):
        flat = {k: torch.full((n + 64,), 7.0, device="cuda") for k in "pmv"}
        codes = {k: torch.full((n + 64,), 77, dtype=torch.uint8, device="cuda") for k in "mv"}
        nb = -(-n // 128)
        scale = {k: torch.full((nb + 8,), 0.5, device="cuda") for k in "mv"}
        mid = lambda x: x[32:32 + n]      # noqa: E731
        if bits == 32:
            optim.adamw_step([mid(flat["p"])], [torch.ones(n, device="cuda")], [mid(flat["m"])], [mid(flat["v"])], [torch.zeros((), device="cuda")], lr=0.1)
            whole = list(flat.values())
        else:
            optim.adamw_step([mid(flat["p"])], [torch.ones(n, device="cuda")], *([mid(codes[k]).view(torch.float8_e4m3fn)] for k in "mv"),
                             [torch.zeros((), device="cuda")], lr=0.1, exp_avg_scales=[scale["m"][4:4 + nb]], exp_avg_sq_scales=[scale["v"][4:4 + nb]])
            whole = [flat["p"], *codes.values()]
            for s in scale.values():
                assert bool((s[:4] == 0.5).all()) and bool((s[4 + nb:] == 0.5).all())
        for x in whole:
            assert bool((x[:32] == x[0]).all()) and bool((x[32 + n:] == x[0]).all()) and float(x[0]) in (7.0, 77.0)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_scale_and_clip(dtype, bits):
    case = Case([5, 1000, 40001], dtype, bits, 9)
    scale = torch.full((1,), 64.0, device="cuda")
    for max_norm in (1e-3, 1e9):
        old = case.before()
        norm = optim.grad_norm(case.g, grad_scale=scale)
        want = math.sqrt(sum(float(x.pow(2).sum()) for x in old["g"])) / 64
        assert abs(float(norm) - want) <= 2 * EPS * want
        case.step(**HYPER, grad_scale=scale, found_inf=torch.zeros((), device="cuda"), grad_norm=norm, max_norm=max_norm)
        c = min(1.0, max_norm / (float(norm) + 1e-6)) / 64
        _check(case, old, **HYPER, c=c)


@pytest.mark.parametrize("bits", [32, 8])
def test_an_overflowed_step_changes_nothing(bits):
    case = Case([5, 1000, 40001], torch.float32, bits, 11)
    case.g[1][3] = math.inf
    tensors = [*case.p, *case.m, *case.v, *case.steps, *(case.ms or []), *(case.vs or [])]
    raw = lambda t: t.view(torch.uint8).clone() if t.dtype == torch.float8_e4m3fn else t.clone()      # noqa: E731
    old = [raw(t) for t in tensors]
    for found in (1.0, 2.0, math.nan):
        case.step(**HYPER, found_inf=torch.full((1,), found, device="cuda"))
        assert all(torch.equal(raw(t), o) for t, o in zip(tensors, old))


def test_infinities_and_nan_without_a_scaler():
    """As torch's: the value itself is lost, and with 8-bit moments its block of 128."""
    for bits in (32, 8):
        case = Case([1000], torch.float32, bits, 13, sparse=0.0)
        case.g[0][300], case.g[0][700] = math.inf, math.nan
        case.step(**HYPER)
        bad = ~torch.isfinite(case.p[0])
        assert bad.nonzero().flatten().tolist() == [300, 700]
        m = torch.isnan(case.m[0].float()) if bits == 32 else torch.isnan(case.m[0].float()).view(-1)
        hit = (~torch.isfinite(case.m[0].float())).nonzero().flatten().tolist()
        if bits == 32:
            assert hit == [300, 700]
        else:
            case.step(**HYPER)
            blocks = {i // 128 for i in (~torch.isfinite(case.p[0])).nonzero().flatten().tolist()}
            assert blocks == {300 // 128, 700 // 128}
        del m


def test_eps_zero_and_untouched_rows():
    """Rows of a table that no sample touched have no gradient and no moments: with eps > 0 only the decay moves them."""
    for bits in (32, 8):
        p = torch.nn.Parameter(torch.ones(1000, device="cuda"))
        o = optim.AdamW([p], lr=0.1, betas=(0.9, 0.99), eps=1e-15, weight_decay=0.5, state_bits=bits)
        p.grad = torch.zeros_like(p)
        for _ in range(3):
            o.step()
        want = torch.full((1000,), (1 - 0.1 * 0.5) ** 3)
        assert float((p.detach().cpu() - want).abs().max()) <= 8 * EPS
        p.grad[7] = 1e-6
        o.step()
        assert bool(torch.isfinite(p).all()) and float(p[7]) < float(p[6])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_against_torch(dtype):
    """Twenty steps beside torch.optim.AdamW on the same gradients, two groups, in 32 bits: each step's roundings (eps / 2 of the parameter's type and
    20 of 32 bits on the update) add up at most."""
    g = _gen(17)
    init = [torch.randn(n, generator=g).to(dtype) for n in (3, 700, 5001)]
    a, b = ([torch.nn.Parameter(x.clone().cuda()) for x in init] for _ in range(2))
    kw = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    ours = optim.AdamW([{"params": a[:1]}, {"params": a[1:], "lr": 3e-3}], **kw)
    theirs = torch.optim.AdamW([{"params": b[:1]}, {"params": b[1:], "lr": 3e-3}], **kw, fused=True)
    for i in range(20):
        for x, y in zip(a, b):
            grad = torch.randn(x.shape, generator=g).to(dtype).cuda()
            x.grad, y.grad = grad, grad.clone()
        ours.step()
        theirs.step()
    for x, y in zip(a, b):
        step = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
        bound = 20 * (step * 2 * y.double().abs() + 1e-2 * 60 * EPS) * 2
        if dtype == torch.bfloat16:      # torch keeps the moments in bfloat16 too: 20 x 2^-8 of an update of at most lr each
            bound = bound + 20 * 1e-2 * 20 * 2.0 ** -8
        assert bool(((x.double() - y.double()).abs() <= bound).all())


def test_8_bit_moments_follow_32_bit_ones():
    """Slow changes add up: under a constant gradient the second moment closes 63 % of its way to g^2 in 1 / (1 - beta2) steps, though one step moves it by
    less than a tenth of the format's spacing.  The dither's error after n steps is below two spacings (1/8 of the value) and its mean over 512
    values far below one."""
    n, b2 = 512, 0.999
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    o = optim.AdamW([p], lr=1e-4, betas=(0.9, b2), eps=1e-8, weight_decay=0.0, state_bits=8)
    first = torch.rand(n, generator=_gen(3)).cuda() + 0.5
    p.grad = first * 4
    for i in range(1001):
        o.step()
        if i == 0:
            p.grad = first.clone()
    _, v = o.moments(p)
    want = (first * 4) ** 2 * (1 - b2) * b2 ** 1000 + first ** 2 * (1 - b2 ** 1000)
    ratio = (v / want).double()
    assert abs(float(ratio.mean()) - 1) < 0.03 and float((ratio - 1).abs().max()) < 0.3


@pytest.mark.parametrize("bits", [32, 8])
def test_gradient_scaler(bits):
    """torch.amp.GradScaler: same result as unscaled gradients (the scale is a power of two), a skipped step on overflow, a halved scale after it."""
    g = _gen(23)
    init = torch.randn(3001, generator=g)
    grads = [torch.randn(3001, generator=g).cuda() for _ in range(4)]
    a, b = (torch.nn.Parameter(init.clone().cuda()) for _ in range(2))
    kw = dict(lr=1e-2, betas=(0.9, 0.99), state_bits=bits, max_grad_norm=0.5)
    oa, ob = optim.AdamW([a], **kw), optim.AdamW([b], **kw)
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0)
    for i, x in enumerate(grads):
        scaler.scale((a * x).sum()).backward()
        if i == 2:
            a.grad[17] = math.inf
        else:
            b.grad = x.clone()
            ob.step()
        scaler.step(oa)
        scaler.update()
        oa.zero_grad()
    assert torch.equal(a.detach(), b.detach()) and float(oa.state[a]["step"]) == 3 and scaler.get_scale() == 512.0


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_continues_bit_for_bit(bits, tmp_path):
    g = _gen(29)
    init = [torch.randn(n, generator=g).to(torch.bfloat16) for n in (3, 1000)]
    grads = [[torch.randn(n, generator=g).to(torch.bfloat16).cuda() for n in (3, 1000)] for _ in range(4)]
    a = [torch.nn.Parameter(x.clone().cuda()) for x in init]
    oa = optim.AdamW(a, lr=1e-2, state_bits=bits)

    def steps(params, opt, which):
        for i in which:
            for p, x in zip(params, grads[i]):
                p.grad = x
            opt.step()
    steps(a, oa, (0, 1))
    torch.save(oa.state_dict(), tmp_path / "o.pt")
    b = [torch.nn.Parameter(x.detach().clone()) for x in a]
    ob = optim.AdamW(b, lr=1.0, state_bits=bits)
    ob.load_state_dict(torch.load(tmp_path / "o.pt", weights_only=True))
    steps(a, oa, (2, 3))
    steps(b, ob, (2, 3))
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and ob.param_groups[0]["lr"] == 1e-2


@pytest.mark.parametrize("bits", [32, 8])
def test_a_copied_optimizer_continues(bits):
    p = torch.nn.Parameter(torch.randn(300, generator=_gen(3)).cuda())
    p.grad = torch.randn(300, generator=_gen(4)).cuda()
    o = optim.AdamW([p], lr=1e-2, state_bits=bits, max_grad_norm=1.0)
    o.step()
    c = copy.deepcopy(o)
    q = c.param_groups[0]["params"][0]
    q.grad = p.grad.clone()
    o.step()
    c.step()
    assert q is not p and c.state_bits == bits and torch.equal(p.detach(), q.detach())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_replays(bits):
    """Norm and step in a graph, replayed between eager work of the same kind: each replay is what an eager step gives, with the learning rate that its
    tensor holds at that time."""
    def make():
        g = _gen(31)
        ps = [torch.nn.Parameter(torch.randn(n, generator=g).cuda()) for n in (5, 3000, 20000)]
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g).cuda()
        lr = torch.tensor(1e-2, device="cuda")
        return ps, lr, optim.AdamW(ps, lr=lr, state_bits=bits, max_grad_norm=3.0)
    a, lra, oa = make()
    b, lrb, ob = make()
    for o in (oa, ob):
        o.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        oa.step()
    for i in range(4):
        for lr in (lra, lrb):
            lr.fill_(1e-2 / (i + 1))
        for x, y in zip(a, b):
            x.grad.mul_(0.9)
            y.grad.mul_(0.9)
        graph.replay()
        ob.step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(a, b)), i
    assert float(oa.state[a[0]]["step"]) == 5


def test_on_a_side_stream():
    case = Case([100003], torch.float32, 8, 37)
    old = case.before()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        norm = optim.grad_norm(case.g)
        case.step(**HYPER, grad_norm=norm, max_norm=1.0)
    torch.cuda.current_stream().wait_stream(s)
    _check(case, old, **HYPER, c=min(1.0, 1.0 / (float(norm) + 1e-6)))


def test_gradients_in_another_order_and_the_version_counter():
    p = torch.nn.Parameter(torch.randn(30, 50, generator=_gen(1)).cuda())
    q = torch.nn.Parameter(p.detach().clone())
    x = torch.randn(50, 30, generator=_gen(2)).cuda()
    oa, ob = optim.AdamW([p]), optim.AdamW([q])
    p.grad, q.grad = x.t(), x.t().contiguous()
    version = p._version
    oa.step()
    ob.step()
    assert torch.equal(p.detach(), q.detach()) and p._version > version


def test_the_same_tensor_twice_is_refused():
    a = [torch.zeros(5, device="cuda") for _ in range(8)]
    with pytest.raises(RuntimeError, match="twice"):
        optim.adamw_step([a[0], a[0]], a[1:3], a[3:5], a[5:7], [torch.zeros((), device="cuda") for _ in range(2)], lr=1e-3)
    with pytest.raises(RuntimeError, match="twice"):
        step = torch.zeros((), device="cuda")
        optim.adamw_step(a[:2], a[2:4], a[4:6], a[6:8], [step, step], lr=1e-3)
    with pytest.raises(RuntimeError, match="grad_scale must be"):
        optim.adamw_step(a[:1], a[1:2], a[2:3], a[3:4], [torch.zeros((), device="cuda")], lr=1e-3, grad_scale=torch.ones(2, device="cuda"))
    with pytest.raises(RuntimeError, match="must be contiguous"):
        optim.adamw_step([torch.zeros(10, device="cuda")[::2]], a[1:2], a[2:3], a[3:4], [torch.zeros((), device="cuda")], lr=1e-3)
    with pytest.raises(RuntimeError, match="must all be on"):
        optim.adamw_step(a[:1], a[1:2], [torch.zeros(5)], a[3:4], [torch.zeros((), device="cuda")], lr=1e-3)
    assert all(float(x.abs().max()) == 0 for x in a)


def test_tensors_that_share_memory_are_refused():
    flat = torch.zeros(40, device="cuda")
    z = lambda n: [torch.zeros(n, device="cuda") for _ in range(2)]      # noqa: E731
    steps = [torch.zeros((), device="cuda") for _ in range(2)]
    with pytest.raises(RuntimeError, match="share memory"):
        optim.adamw_step([flat[:10], flat[9:19]], z(10), z(10), z(10), steps, lr=1.0)
    with pytest.raises(RuntimeError, match="share memory"):
        optim.adamw_step([flat[:10], flat[20:30]], z(10), [flat[29:39], z(10)[0]], z(10), steps, lr=1.0)
    many, n = torch.zeros(200, 8, device="cuda"), 40
    rows = lambda: list(torch.zeros(n, 8, device="cuda"))      # noqa: E731
    for at in range(0, n, 13):      # one of many, at some place among the others
        p = [many[5 * i] for i in range(n)]
        p[at] = many[5 * ((at + 7) % n)].view(-1)[:3] if at else many.view(-1)[5 * 8 * 7 + 4:5 * 8 * 7 + 12]
        like = lambda: [torch.zeros_like(x) for x in p]      # noqa: E731
        with pytest.raises(RuntimeError, match="share memory"):
            optim.adamw_step(p, like(), like(), like(), list(torch.zeros(n, device="cuda")), lr=1.0)
    optim.adamw_step([many[5 * i] for i in range(n)], rows(), rows(), rows(), list(torch.zeros(n, device="cuda")), lr=1.0)
    optim.adamw_step([flat[:10], flat[10:20]], [torch.ones(10, device="cuda")] * 2, z(10), z(10), steps, lr=1.0, weight_decay=0.0)
    assert bool((flat[:20] < -0.9).all()) and not bool(flat[20:].any())


def test_a_gradient_whose_sign_is_still_to_be_applied():
    c = torch.randn(300, dtype=torch.complex64, generator=_gen(3)).cuda()
    g = c.conj().imag
    assert g.is_neg()
    got = []
    for grad in (g, g.clone().contiguous() + 0.0):
        p, m, v = (torch.zeros(300, device="cuda") for _ in range(3))
        optim.adamw_step([p], [grad], [m], [v], [torch.zeros((), device="cuda")], lr=0.1)
        got.append(p)
    assert torch.equal(*got) and bool((got[0] != 0).any())


def test_a_first_step_is_not_captured(monkeypatch):
    p = torch.nn.Parameter(torch.ones(5, device="cuda"))
    p.grad = torch.ones(5, device="cuda")
    o = optim.AdamW([p])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="first step"):
        o.step()
    monkeypatch.undo()
    o.step()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    o.step()
    assert float(o.state[p]["step"]) == 2


@pytest.mark.parametrize("g", [1e-15, 1e-21, 1e-25])
def test_gradients_far_below_the_range_of_their_squares(g):
    """g^2 is a subnormal number, or nothing: the second moment is the root of what a 32-bit square leaves of it, between nothing and its value."""
    p, grad = torch.zeros(256, device="cuda"), torch.full((256,), g, device="cuda")
    m, v = (torch.zeros(256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    ms, vs = (torch.zeros(2, device="cuda") for _ in range(2))
    optim.adamw_step([p], [grad], [m], [v], [torch.zeros((), device="cuda")], lr=0.1, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.0, exp_avg_scales=[ms], exp_avg_sq_scales=[vs])
    first, root = m.float() * ms[0], v.float() * vs[0]
    assert bool(((first / (0.1 * g) - 1).abs() <= 2.0 ** -3).all())                      # a code is at most a spacing below or above
    assert bool((root <= 0.1 * g * (1 + 2.0 ** -3) + 448 * 2.0 ** -100 / 448).all()) and bool((root >= 0).all())
    assert float(p.abs().max()) <= 0.1 * g / 1e-8 * 1.01


def _written_out(q, scale, n):
    return q.float().cpu() * scale.cpu().repeat_interleave(128)[:n]


def _held(x, u, positive):
    """Codes and scales of the moment x in single 32-bit operations (sums with the dither in 64 bits, where they are exact)."""
    n = x.numel()
    a = torch.nn.functional.pad(x.abs(), (0, -n % 128)).view(-1, 128).amax(1).clamp(min=2.0 ** -100)
    y = (x * (a.reciprocal() * 448.0).repeat_interleave(128)[:n]).clamp(-448, 448)
    gap = 2.0 ** ((torch.frexp(y)[1].double() - 1).clamp(min=-6) - 3)
    k = torch.floor(y.abs().double() / gap + u)
    if positive:
        k = torch.where(x > 0, k.clamp(min=1), k)
    return torch.copysign((k * gap).clamp(max=448).float(), y), a * torch.tensor(1.0 / 448.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_8_bit_state_is_the_formula_written_out_bit_for_bit(dtype):
    """No tolerance: every operation of the moments rounds as the formula's own does, so after any number of steps the codes are its codes."""
    b1, b2, scale = 0.9, 0.99, 1024.0
    one = lambda x: torch.tensor(x, dtype=torch.float32)      # noqa: E731
    n, g = 70001, _gen(77)
    p = (0.3 * torch.randn(n, generator=g)).to(dtype).cuda()
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    ms, vs = (torch.zeros(-(-n // 128), device="cuda") for _ in range(2))
    step, loss_scale = torch.zeros((), device="cuda"), torch.full((), scale, device="cuda")
    for t in range(1, 9):
        grad = (torch.randn(n, generator=g) * 2.0 ** torch.randint(-9, 5, (n,), generator=g) * (torch.rand(n, generator=g) > 0.3)).to(dtype)
        m0, r0 = _written_out(m, ms, n), _written_out(v, vs, n)
        norm = optim.grad_norm([grad.cuda()], grad_scale=loss_scale)
        wide = float(norm.wide)
        assert wide == pytest.approx(math.sqrt(float(grad.double().pow(2).sum())) / scale, rel=1e-13) and float(norm) == float(one(wide))
        optim.adamw_step([p], [grad.cuda()], [m], [v], [step], lr=1e-3, betas=(b1, b2), exp_avg_scales=[ms], exp_avg_sq_scales=[vs], grad_scale=loss_scale,
                         grad_norm=norm, max_norm=0.01)
        x = grad.float() * one(min(1.0, 0.01 / (wide + 1e-6)) / scale)
        u = ((torch.arange(n) * A + t * B) % 2 ** 32 // 4096).double() / 2 ** 20
        # (torch's float32 square root on the CPU is a unit off for one value in 170; by way of 64 bits it is the nearest)
        for value, q, s, shift in ((m0 + one(1 - b1) * (x - m0), m, ms, 0.0), ((one(b2) * (r0 * r0) + one(1 - b2) * x * x).double().sqrt().float(), v, vs, 0.5)):
            code, held = _held(value, (u + shift) % 1, shift > 0)
            assert torch.equal(s.cpu(), held), t
            assert torch.equal(q.float().cpu(), code), t


def test_a_norm_changed_by_the_caller_is_the_one_that_counts():
    grad = torch.full((1000,), 1.0, device="cuda")
    moved = []
    for change in (lambda x: x, lambda x: x.mul_(4.0), lambda x: x.clone() * 4.0, lambda x: torch.full_like(x, 4.0 * float(x))):
        p, m, v = (torch.zeros(1000, device="cuda") for _ in range(3))
        norm = change(optim.grad_norm([grad]))
        optim.adamw_step([p], [grad], [m], [v], [torch.zeros((), device="cuda")], lr=0.1, betas=(0.5, 0.5), eps=1.0, grad_norm=norm, max_norm=1.0)
        moved.append(float(m[0]))
    assert moved[0] == pytest.approx(0.5 / math.sqrt(1000), rel=1e-6) and all(x == pytest.approx(moved[0] / 4, rel=1e-6) for x in moved[1:])


@pytest.mark.parametrize("scale", [1e-30, 1.0, 1e30])
def test_norm_over_mixed_types(scale):
    g = _gen(41)
    grads = [torch.randn(n, generator=g).to(dt).cuda() * (scale if dt == torch.float32 else 1) for n, dt in
             [(1, torch.float32), (1003, torch.float32), (77, torch.bfloat16), (100001, torch.float16), (0, torch.float32)] + [(9, torch.float32)] * 200]
    grads[1] = _place(grads[1].cpu(), 3)
    want = math.sqrt(sum(float(x.double().pow(2).sum()) for x in grads))
    got = [float(optim.grad_norm(grads)) for _ in range(3)]
    assert got[0] == got[1] == got[2] and abs(got[0] - want) <= 2 * EPS * want
    assert abs(float(optim.grad_norm(grads, grad_scale=torch.tensor(3.0, device="cuda"))) - want / 3) <= 2 * EPS * want
    grads[3][5] = math.nan
    assert math.isnan(float(optim.grad_norm(grads)))
    grads[3][5] = math.inf
    assert math.isinf(float(optim.grad_norm(grads)))


def test_norm_of_nothing():
    assert float(optim.grad_norm([torch.zeros(0, device="cuda")])) == 0.0
    assert float(optim.grad_norm([None, torch.zeros(7, device="cuda")])) == 0.0


def test_more_values_than_32_bits_count():
    """2^32 + 5 values in one tensor: its first and last values, and those around 2^32, move as the formula says; one gradient among them."""
    n = 2 ** 32 + 5
    p, grad = (torch.zeros(n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    m, v = (torch.zeros(n, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2))
    ms, vs = (torch.zeros(-(-n // 128), device="cuda") for _ in range(2))
    step = torch.zeros((), device="cuda")
    at = [0, 5, 2 ** 32 - 1, 2 ** 32, n - 1]
    for i in at:
        grad[i] = 2.0
    norm = optim.grad_norm([grad])
    assert abs(float(norm) - 2 * math.sqrt(5)) <= 4 * EPS * 2 * math.sqrt(5)
    optim.adamw_step([p], [grad], [m], [v], [step], lr=0.5, betas=(0.9, 0.99), weight_decay=0.0, exp_avg_scales=[ms], exp_avg_sq_scales=[vs])
    for i in at:
        assert float(p[i]) == -0.5, i           # the first step is lr sign(g), exact in bfloat16 up to eps
    assert float(p[1]) == 0 and float(p[2 ** 32 - 2]) == 0 and float(p[n - 2]) == 0 and float(step) == 1
    assert int((p[:2 ** 20] != 0).sum()) == 2 and int((p[-2 ** 20:] != 0).sum()) == 3
