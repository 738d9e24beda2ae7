"""AdamW on the device against its formula in 64 bits, and its 8-bit codes against their fp32 definition."""
import math

import pytest
import torch

import gefen
import adamw_reference as ref

pytestmark = pytest.mark.gpu

LR, B1, B2, EPS, WD = 1e-2, 0.9, 0.99, 1e-8, 0.1
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def tensors(sizes, dtype, seed, dev, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(dtype).to(dev) for s in sizes]


def storage(t):
    """The elements in the order they are stored in, on the CPU."""
    dims = sorted(range(t.dim()), key=lambda d: -t.stride(d)) if not t.is_contiguous() else list(range(t.dim()))
    return t.detach().permute(dims).reshape(-1).cpu()


class Mirror:
    """The optimizer's parameters stepped on the CPU, each step from the device's own state before it."""

    def __init__(self, params, bits, seed=0, **hyper):
        self.params, self.bits, self.seed, self.hyper = params, bits, seed, hyper

    def before(self, opt):
        self.old = []
        for p, mv in zip(self.params, opt.moments(self.params)):
            m, v = (torch.zeros(p.numel()),) * 2 if mv is None else (storage(x) for x in mv)
            self.old.append((storage(p), storage(p.grad) if p.grad is not None else None, m.clone(), v.clone()))

    def check(self, opt, t, coef=1.0, index=None):
        h = dict(lr=LR, beta1=B1, beta2=B2, eps=EPS, wd=WD, **self.hyper)
        got = opt.moments(self.params)
        for i, (p, old) in enumerate(zip(self.params, self.old)):
            p0, g, m0, v0 = old
            if g is None:
                assert torch.equal(storage(p), p0)
                continue
            want, m64, v64 = ref.step64(p0, g, m0, v0, t, coef=coef, **h)
            upd = (p0.double() * (1 - h["lr"] * h["wd"]) - want).abs()
            off = (storage(p).double() - want).abs()
            tol = ref.tolerance(want, upd, p.dtype)
            assert torch.all(off <= tol), (i, p.shape, (off / tol).max())
            if self.bits == 32:
                # two roundings of each term and one of the sum
                gm, gv = g.double().abs() * coef, (g.double() * coef) ** 2
                for a, b, size in ((got[i][0], m64, B1 * m0.double().abs() + (1 - B1) * gm),
                                   (got[i][1], v64, B2 * v0.double() + (1 - B2) * gv)):
                    assert torch.all((storage(a).double() - b).abs() <= 6 * 2.0 ** -24 * size + 2.0 ** -148), i
            else:
                state = opt.state[p]
                m, v = ref.moments32(m0, v0, g.float() * torch.tensor(coef, dtype=torch.float32), B1, B2)
                mc, ms = ref.codes_m(m)
                key = ref.step_key(self.seed, index[i] if index else i, t)
                vc, vs = ref.codes_v(v, ref.random16(key, v.numel()))
                assert torch.equal(state["exp_avg_scale"].cpu(), ms) and torch.equal(state["exp_avg_sq_scale"].cpu(), vs), i
                assert torch.equal(state["exp_avg_sq"].cpu(), vc), i
                assert torch.equal(state["exp_avg"].cpu().view(torch.uint8), mc.view(torch.uint8)), i
                assert torch.equal(got[i][0].cpu(), ref.value_m(mc, ms)) and torch.equal(got[i][1].cpu(), ref.value_v(vc, vs))


def run(params, grads, bits, dev, seed=0, **kw):
    opt = gefen.AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=bits, seed=seed, **kw)
    mirror = Mirror(params, bits, seed)
    for t, step in enumerate(grads, 1):
        for p, g in zip(params, step):
            p.grad = g
        mirror.before(opt)
        opt.step()
        mirror.check(opt, t)
    return opt


SIZES = [(1,), (7,), (8,), (9,), (255,), (256,), (257,), (4095,), (3, 683), (33, 129), (4097,), (2, 3, 5), ()]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_step_matches_the_formula(dev, dtype, bits):
    params = [torch.nn.Parameter(t) for t in tensors(SIZES, dtype, 1, dev)]
    run(params, [tensors(SIZES, dtype, 2 + k, dev, 0.1) for k in range(3)], bits, dev)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_a_launch_holds(dev, bits):
    sizes = [(1 + 13 * k % 300,) for k in range(90)]
    params = [torch.nn.Parameter(t) for t in tensors(sizes, torch.bfloat16, 1, dev)]
    run(params, [tensors(sizes, torch.bfloat16, 2, dev)], bits, dev)


def test_large_launches_take_longer_workgroups(dev):
    """Past 8192 workgroup passes a workgroup takes four: the tail of a tensor ends inside one."""
    n = 8192 * 2048 + 2048 * 5 + 3
    for bits, n in ((32, n), (8, 2 * n)):
        p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device=dev))
        g = torch.randn(n, generator=torch.Generator(dev).manual_seed(1), device=dev).to(torch.bfloat16)
        opt = gefen.AdamW([p], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=bits)
        p.grad = g
        opt.step()
        # first step from zero: p = -lr g / (|g| + eps), m = (1-b1) g, v = (1-b2) g^2
        want = (-LR * g.double() / (g.double().abs() + EPS)).to(torch.bfloat16)
        assert (p.detach().double() - want.double()).abs().max() <= LR * 2.0 ** -8 * 1.01
        m, v = opt.moments()[0]
        if bits == 32:
            assert torch.equal(m, g.float() * torch.tensor(1 - B1)) and torch.equal(v, g.float() ** 2 * torch.tensor(1 - B2))
        else:
            # half a code of E4M3 (or of its smallest step), a whole code of v rounded either way
            scale = opt.state[p]["exp_avg_scale"].double().repeat_interleave(256)[:n]
            off = (m.double() - g.double() * (1 - B1)).abs()
            assert torch.all(off <= g.double().abs() * (1 - B1) / 16 * 1.001 + scale * 2.0 ** -10 * 1.001)
            nz = v > 0
            ratio = v[nz].double() / (g[nz].double() ** 2 * (1 - B2))
            big = g[nz].float().abs() > 1e-3
            assert ratio[big].max() <= 1.126 and ratio[big].min() >= 0.888


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_unaligned_and_turned_parameters(dev, dtype, bits):
    flat = tensors([(5000,), (5000,)], dtype, 1, dev)
    base = [flat[0][1:2002], flat[0][2003:3003].view(40, 25).t(), tensors([(31, 65)], dtype, 4, dev)[0].t(),
            tensors([(4, 6, 5, 7)], dtype, 5, dev)[0].to(memory_format=torch.channels_last)]
    params = [torch.nn.Parameter(t) for t in base]
    grads = [flat[1][3:2004], flat[1][2005:3005].view(40, 25).t(), tensors([(31, 65)], dtype, 6, dev)[0].t(),
             tensors([(4, 6, 5, 7)], dtype, 7, dev)[0].to(memory_format=torch.channels_last)]
    before = flat[0].clone()
    opt = run(params, [grads, grads], bits, dev)
    untouched = torch.ones(5000, dtype=torch.bool)
    untouched[1:2002] = untouched[2003:3003] = False
    assert torch.equal(flat[0].cpu()[untouched], before.cpu()[untouched])
    if bits == 32:
        assert opt.state[params[1]]["exp_avg"].stride() == params[1].stride()


@pytest.mark.parametrize("bits", [32, 8])
def test_gaps_and_gradients_of_another_layout(dev, bits):
    wide = tensors([(40, 100)], torch.float32, 1, dev)[0]
    keep = wide.clone()
    a = torch.nn.Parameter(wide[:, 10:43])            # rows with gaps
    b = torch.nn.Parameter(tensors([(20, 30)], torch.float32, 2, dev)[0])
    c = torch.nn.Parameter(tensors([(20, 30)], torch.float32, 3, dev)[0].t())
    g = tensors([(40, 33), (30, 20), (30, 20)], torch.float32, 4, dev)
    like = [torch.nn.Parameter(p.detach().clone(memory_format=torch.contiguous_format)) for p in (a, b, c)]
    kw = dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=bits)
    opt, plain = gefen.AdamW([a, b], **kw), gefen.AdamW(like[:2], **kw)
    for _ in range(2):
        a.grad, b.grad = g[0], g[1].t()
        like[0].grad, like[1].grad = g[0].clone(), g[1].t().contiguous()
        opt.step()
        plain.step()
    assert torch.equal(a, like[0]) and torch.equal(b, like[1])
    outside = torch.ones(100, dtype=torch.bool, device=dev)
    outside[10:43] = False
    assert torch.equal(wide[:, outside], keep[:, outside])
    # a turned parameter with a contiguous gradient, and one gradient value for all elements
    opt, plain = gefen.AdamW([c], **dict(kw, state_bits=32)), gefen.AdamW([like[2]], **dict(kw, state_bits=32))
    for grad in (g[2], torch.full((1, 1), 0.5, device=dev).expand(30, 20)):
        c.grad, like[2].grad = grad, grad.contiguous()
        opt.step()
        plain.step()
    assert torch.equal(c, like[2])


def test_moments_of_a_turned_parameter_with_gaps(dev):
    """Row by row, as a contiguous parameter's, whose checkpoint goes on from there bit for bit."""
    wide, g = tensors([(40, 100)], torch.float32, 1, dev)[0], tensors([(33, 40)] * 2, torch.float32, 2, dev)
    turned = torch.nn.Parameter(wide[:, 10:43].t())
    flat = torch.nn.Parameter(turned.detach().contiguous())
    opts = [gefen.AdamW([p], state_bits=8) for p in (turned, flat)]
    for p, o in zip((turned, flat), opts):
        p.grad = g[0]
        o.step()
    assert all(torch.equal(a, b) for a, b in zip(opts[0].moments()[0], opts[1].moments()[0]))
    opts[1].load_state_dict(opts[0].state_dict())
    for p, o in zip((turned, flat), opts):
        p.grad = g[1]
        o.step()
    assert torch.equal(turned, flat)
    assert all(torch.equal(a, b) for a, b in zip(opts[0].moments()[0], opts[1].moments()[0]))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_clipping_by_the_global_norm(dev, dtype, bits):
    sizes = [(300,), (5, 700), (1,)]
    params = [torch.nn.Parameter(t) for t in tensors(sizes, dtype, 1, dev)]
    opt = gefen.AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=bits, max_grad_norm=0.75)
    mirror = Mirror(params, bits)
    for t, scale in ((1, 0.5), (2, 1e-4)):  # one step clipped, one not
        grads = tensors(sizes, dtype, 1 + t, dev, scale)
        for p, g in zip(params, grads):
            p.grad = g.clone()
        mirror.before(opt)
        opt.step()
        norm = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
        got = opt.grad_norm.cpu()
        assert abs(float(got) - norm) <= 2.0 ** -23 * norm
        coef = torch.tensor(0.75) / (got + torch.tensor(1e-6))
        assert (coef < 1) == (t == 1)
        mirror.check(opt, t, coef=float(coef.clamp(max=1.0)))
        assert all(torch.equal(p.grad, g) for p, g in zip(params, grads))


def test_norm_of_many_elements_and_types(dev):
    """The sum's order depends on no other tensor of the call beyond their sizes; float64 sums of 20M terms."""
    g = torch.randn(20_000_003, generator=torch.Generator(dev).manual_seed(3), device=dev)
    parts = [g[:9_000_001].clone(), g[9_000_001:17_000_000].half(), g[17_000_000:].bfloat16()]
    params = [torch.nn.Parameter(torch.zeros_like(x)) for x in parts]
    for p, x in zip(params, parts):
        p.grad = x
    opt = gefen.AdamW(params, max_grad_norm=1.0)
    opt.step()
    first = opt.grad_norm.clone()
    opt.step()
    want = math.sqrt(sum(float(x.double().square().sum()) for x in parts))
    assert torch.equal(first, opt.grad_norm) and abs(float(first) - want) <= 2.0 ** -23 * want


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients_and_zero_state(dev, bits):
    p = torch.nn.Parameter(torch.linspace(-1, 1, 700, device=dev))
    p.grad = torch.zeros(700, device=dev)
    old = p.detach().clone()
    opt = gefen.AdamW([p], lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=bits)
    opt.step()
    assert torch.equal(p.detach(), old * torch.tensor(1 - LR * WD))
    m, v = opt.moments()[0]
    assert not m.any() and not v.any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_bad_gradient_stays_where_it_is(dev, dtype):
    """32 bits: its own element.  8 bits: its own block, whose scales turn NaN."""
    for value in (float("nan"), float("inf")):
        for bits in (32, 8):
            p = torch.nn.Parameter(torch.ones(1000, dtype=dtype, device=dev))
            g = torch.full((1000,), 0.5, dtype=dtype, device=dev)
            g[300] = value
            opt = gefen.AdamW([p], lr=LR, betas=(B1, B2), state_bits=bits)
            for _ in range(2):
                p.grad = g
                opt.step()
                g = torch.full((1000,), 0.5, dtype=dtype, device=dev)
            bad = ~torch.isfinite(p.detach())
            want = torch.zeros(1000, dtype=torch.bool, device=dev)
            want[300] = True
            if bits == 8:
                want[256:512] = True
            assert torch.equal(bad, want)


def test_extreme_scales_of_8_bit_blocks(dev):
    """Gradients from the smallest normal numbers to the largest whose square is finite, in blocks of their own."""
    scales = [1e-30, 1e-18, 1e-10, 1.0, 1e10, 1e18]
    g0 = torch.cat([torch.linspace(0.1, 1.0, 256) * s for s in scales]).to(dev)
    p = torch.nn.Parameter(torch.zeros_like(g0))
    opt = gefen.AdamW([p], lr=LR, betas=(B1, B2), eps=0.0, weight_decay=0.0, state_bits=8)
    p.grad = g0
    opt.step()
    m, v = (x.cpu() for x in opt.moments()[0])
    want_m, want_v = ref.moments32(torch.zeros(g0.numel()), torch.zeros(g0.numel()), g0.cpu(), B1, B2)
    mc, ms = ref.codes_m(want_m)
    vc, vs = ref.codes_v(want_v, ref.random16(ref.step_key(0, 0, 1), want_v.numel()))
    assert torch.equal(m, ref.value_m(mc, ms)) and torch.equal(v, ref.value_v(vc, vs))
    # the first step's size is lr wherever the square neither vanishes nor loses bits
    sound = want_v > 1e-30
    assert (p.detach().cpu()[sound] + LR).abs().max() <= LR * 1e-6


@pytest.mark.parametrize("eps", [1e-12, 1e-10, 1e-9, 1e-8])
@pytest.mark.parametrize("beta2", [0.9, 0.9999, 1 - 2.0 ** -23])
def test_second_moments_below_the_normal_numbers(dev, beta2, eps):
    """v below 2^-126 where 1 / sqrt(1 - beta2) lifts its root to a share of eps: 8 bits step as the formula says, to 16
    roundings (fewer than that many operations are in it)."""
    g = torch.cat([torch.linspace(0.05, 1.0, 256) * 2.0 ** -63 / math.sqrt(1 - beta2), torch.linspace(0.1, 1, 256) * 1e-3])
    p = torch.nn.Parameter(torch.zeros(512, device=dev))
    p.grad = g.to(dev)
    opt = gefen.AdamW([p], lr=LR, betas=(B1, beta2), eps=eps, weight_decay=0.0, state_bits=8)
    opt.step()
    m, v = ref.moments32(torch.zeros(512), torch.zeros(512), g, B1, beta2)
    assert v[:256].max() < 2.0 ** -125 and (v[:256] > 0).all()
    # from the rounded moments: those of denormal v are no matter of the step
    want = -LR / (1 - B1) * m.double() / (v.double().sqrt() / math.sqrt(1 - beta2) + eps)
    assert torch.all((p.detach().cpu().double() - want).abs() <= 16 * U * want.abs())


def test_every_float8_code_decodes_and_encodes_as_torch_does(dev):
    """m codes 0..255 through moments(), and values between them through a step with beta1 = 0."""
    n = 256
    p = torch.nn.Parameter(torch.zeros(n, device=dev))
    opt = gefen.AdamW([p], betas=(0.0, 0.5), state_bits=8)
    codes = torch.arange(256, dtype=torch.uint8)
    codes[127] = codes[255] = 0  # the NaN codes
    opt.load_state_dict({"state": {0: {"step": 1, "exp_avg": codes.view(torch.float8_e4m3fn), "exp_avg_sq": codes,
                                       "exp_avg_scale": torch.tensor([0.37]), "exp_avg_sq_scale": torch.tensor([2.5])}},
                         "param_groups": opt.state_dict()["param_groups"]})
    m, v = opt.moments()[0]
    assert torch.equal(m.cpu(), codes.view(torch.float8_e4m3fn).float() * torch.tensor(0.37))
    assert torch.equal(v.cpu(), ref.value_v(codes, torch.tensor([2.5])))
    # largest value 448: scale 448 * RN(1/448), values at, just beside and between all codes
    mag = codes[:127].view(torch.float8_e4m3fn).float()
    mid = (mag[1:] + mag[:-1]) / 2
    x = torch.cat([mag, -mag, mid, torch.nextafter(mid, torch.tensor(0.0)), torch.nextafter(mid, torch.tensor(1e9))])
    x = torch.cat([torch.cat([part, torch.tensor([448.0])]) for part in x.split(255)])
    x = torch.nn.functional.pad(x, (0, -x.numel() % 256))
    q = torch.nn.Parameter(torch.zeros(x.numel(), device=dev))
    q.grad = x.to(dev)
    opt = gefen.AdamW([q], betas=(0.0, 0.5), state_bits=8)
    opt.step()
    m, _ = ref.moments32(torch.zeros_like(x), torch.zeros_like(x), x, 0.0, 0.5)  # -0 becomes 0 + -0 = 0
    want, scale = ref.codes_m(m)
    assert torch.equal(opt.state[q]["exp_avg"].cpu().view(torch.uint8), want.view(torch.uint8))
    assert torch.equal(opt.state[q]["exp_avg_scale"].cpu(), scale)


def test_second_moment_in_8_bits_is_unbiased(dev):
    """400 steps of noise: the mean of v over 2^17 elements stays that of 32 bits.  An element's v strays by
    about a third (each step moves a share 1 - b2 of it by whole codes), so the mean by 0.33 / 362 = 0.1%;
    nearest rounding would stay off by tens of percent."""
    n = 1 << 17
    p8, p32 = (torch.nn.Parameter(torch.zeros(n, device=dev)) for _ in range(2))
    o8 = gefen.AdamW([p8], lr=0.0, betas=(0.9, 0.999), state_bits=8)
    o32 = gefen.AdamW([p32], lr=0.0, betas=(0.9, 0.999))
    gen = torch.Generator(dev).manual_seed(0)
    for _ in range(400):
        p8.grad = p32.grad = torch.randn(n, generator=gen, device=dev)
        o8.step()
        o32.step()
    v8, v32 = o8.moments()[0][1].double(), o32.moments()[0][1].double()
    assert abs((v8.mean() / v32.mean()).item() - 1) < 0.005
    assert ((v8 / v32 - 1) ** 2).mean().sqrt().item() < 0.5


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_graphs_that_saved_a_parameter_end_with_the_step(dev, bits, capturable):
    """A second backward pass through weights that were stepped in between raises; through others it does not."""
    x = torch.ones(5, 8, device=dev, requires_grad=True)
    w, idle = (torch.nn.Parameter(torch.ones(8, 8, device=dev)) for _ in range(2))
    turned = torch.nn.Parameter(torch.ones(8, 8, device=dev).t())
    opt = gefen.AdamW([w, idle, turned], state_bits=bits, capturable=capturable)
    for p in (w, turned, idle):
        out = (x @ p).sum()
        out.backward(retain_graph=True)
        if p is idle:
            idle.grad = None
        opt.step()
        opt.zero_grad()
        if p is idle:
            out.backward()
        else:
            with pytest.raises(RuntimeError, match="modified"):
                out.backward()


def test_same_seed_same_run(dev):
    def go(seed):
        p = torch.nn.Parameter(torch.ones(5000, device=dev))
        opt = gefen.AdamW([p], state_bits=8, seed=seed)
        for k in range(3):
            p.grad = tensors([(5000,)], torch.float32, k, dev)[0]
            opt.step()
        return opt.state[p]["exp_avg_sq"]
    assert torch.equal(go(3), go(3)) and not torch.equal(go(3), go(4))


@pytest.mark.parametrize("bits", [32, 8])
def test_groups_of_unlike_settings_and_missing_gradients(dev, bits):
    dtypes = [torch.float32, torch.bfloat16, torch.float16, torch.float32]
    params = [torch.nn.Parameter(tensors([(300 + k,)], d, k, dev)[0]) for k, d in enumerate(dtypes)]
    opt = gefen.AdamW([{"params": params[:2], "lr": 1e-3}, {"params": params[2:3], "betas": (0.8, 0.95)},
                       {"params": params[3:], "weight_decay": 0.3, "eps": 1e-3, "state_bits": 40 - bits}], state_bits=bits)
    old = [p.detach().clone() for p in params]
    for k, p in enumerate(params):
        if k != 1:
            p.grad = tensors([(300 + k,)], dtypes[k], 10 + k, dev)[0]
    opt.step()
    assert torch.equal(params[1], old[1]) and params[1] not in opt.state
    hyper = [(1e-3, 0.9, 0.999, 1e-8, 1e-2), None, (1e-3, 0.8, 0.95, 1e-8, 1e-2), (1e-3, 0.9, 0.999, 1e-3, 0.3)]
    for k in (0, 2, 3):
        z = torch.zeros(300 + k)
        lr, b1, b2, eps, wd = hyper[k]
        want, _, _ = ref.step64(old[k].cpu(), params[k].grad.cpu(), z, z, 1, lr, b1, b2, eps, wd)
        off = (params[k].detach().cpu().double() - want).abs()
        assert torch.all(off <= ref.tolerance(want, torch.full_like(want, lr), dtypes[k]))


@pytest.mark.parametrize("bits", [32, 8])
def test_resumed_run_goes_on_the_same(dev, bits):
    def grads(k):
        return tensors([(700,), (20, 33)], torch.bfloat16, 50 + k, dev)
    params = [torch.nn.Parameter(t) for t in tensors([(700,), (20, 33)], torch.bfloat16, 1, dev)]
    opt = gefen.AdamW(params, state_bits=bits, max_grad_norm=1.0, seed=9)
    for k in range(2):
        for p, g in zip(params, grads(k)):
            p.grad = g
        opt.step()
    others = [torch.nn.Parameter(p.detach().clone()) for p in params]
    other = gefen.AdamW(others, state_bits=bits, max_grad_norm=1.0, seed=9)
    other.load_state_dict(opt.state_dict())
    for ps, o in ((params, opt), (others, other)):
        for p, g in zip(ps, grads(2)):
            p.grad = g
        o.step()
    assert all(torch.equal(a, b) for a, b in zip(params, others))
    assert all(torch.equal(a, b) for x, y in zip(opt.moments(), other.moments()) for a, b in zip(x, y))


def test_steps_as_torch_does(dev):
    """The same run through torch.optim.AdamW in fp32, and from its checkpoint."""
    a, b = (torch.nn.Parameter(tensors([(513,)], torch.float32, 1, dev)[0]) for _ in range(2))
    kw = dict(lr=1e-2, betas=(B1, B2), weight_decay=WD)
    theirs, ours = torch.optim.AdamW([a], **kw), gefen.AdamW([b], **kw)
    for k in range(4):
        a.grad = b.grad = tensors([(513,)], torch.float32, 2 + k, dev)[0]
        theirs.step()
        if k == 2:
            ours.load_state_dict(dict(theirs.state_dict(), state={0: {**theirs.state_dict()["state"][0], "step": 2}}))
            b.data.copy_(b0)
            ours.state[b]["exp_avg"].copy_(m0)
            ours.state[b]["exp_avg_sq"].copy_(v0)
        ours.step()
        b0, (m0, v0) = b.detach().clone(), (x.clone() for x in ours.moments()[0])
        # about 16 roundings a step of terms no larger than 1 and lr
        assert (a - b).abs().max().item() <= (k + 1) * 16 * 2.0 ** -24 * (a.abs().max().item() + 1e-2)


def test_work_goes_to_the_current_stream(dev):
    p = torch.nn.Parameter(torch.zeros(1 << 20, device=dev))
    opt = gefen.AdamW([p], lr=LR, weight_decay=0.0, max_grad_norm=1e9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.zeros(1 << 20, device=dev)
        for _ in range(50):
            g += 0.02
        p.grad = g
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    assert (p.detach() + LR).abs().max().item() <= LR * 1e-5


def test_scaled_fp16_gradients(dev):
    p = torch.nn.Parameter(torch.ones(64, dtype=torch.float16, device=dev))
    opt = gefen.AdamW([p], lr=LR)
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0)
    scaler.scale((p.float() * 0.25).sum()).backward()
    scaler.step(opt)
    scaler.update()
    assert abs(opt.moments()[0][0][0].item() - 0.025) < 1e-6
    old = p.detach().clone()
    p.grad.fill_(float("inf"))
    scaler.scale(torch.zeros((), device=dev))
    scaler.step(opt)
    assert torch.equal(p, old) and opt.state[p]["step"] == 1


def test_refusals(dev):
    p = torch.nn.Parameter(torch.ones(8, device=dev))
    opt = gefen.AdamW([p])
    p.grad = torch.ones(8, device=dev).to_sparse()
    with pytest.raises(RuntimeError, match="sparse"):
        opt.step()
    q = torch.nn.Parameter(torch.ones(8, device=dev, dtype=torch.float64))
    opt = gefen.AdamW([q])
    q.grad = torch.ones_like(q)
    with pytest.raises(NotImplementedError):
        opt.step()
    r = torch.nn.Parameter(torch.ones(1, 4, device=dev).expand(8, 4))
    r.grad = torch.ones(8, 4, device=dev)
    opt = gefen.AdamW([r])
    with pytest.raises(ValueError, match="share memory"):
        opt.step()
    s = torch.nn.Parameter(torch.ones(600, device=dev))
    s.grad = torch.ones(600, device=dev)
    opt = gefen.AdamW([s], state_bits=8)
    opt.step()
    opt.state[s]["exp_avg_scale"] = opt.state[s]["exp_avg_scale"][:1]
    with pytest.raises(ValueError, match="exp_avg_scale"):
        opt.step()
    graph = torch.cuda.CUDAGraph()
    t = torch.nn.Parameter(torch.ones(8, device=dev))
    t.grad = torch.ones(8, device=dev)
    opt = gefen.AdamW([t])
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step()


def captured(opt, warm):
    """A graph of opt.step(), after one eager step."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm()
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    return graph


@pytest.mark.parametrize("bits", [32, 8])
def test_replays_equal_eager_steps(dev, bits):
    """A captured step, replayed with other gradients, a device lr that changes and eager work between: the eager
    run's moments bit for bit (8-bit codes follow the counters' random bits), its parameters but for roundings of the
    bias corrections (computed in float64 on either side, a unit of fp32 apart at most)."""
    sizes = [(300,), (40, 33), (1,), (0,), (5000,)] + [(17,)] * 60
    base = tensors(sizes, torch.float32, 1, dev)
    base[1] = base[1].t()
    ps = [[torch.nn.Parameter(t.detach().clone()) for t in base] for _ in range(2)]
    lr = torch.tensor(1e-2, device=dev, dtype=torch.float64)
    kw = dict(betas=(B1, B2), weight_decay=WD, state_bits=bits, max_grad_norm=3.0, seed=4)
    graphed = gefen.AdamW([{"params": ps[0][:2], "lr": lr}, {"params": ps[0][2:], "lr": 5e-3}], capturable=True, **kw)
    eager = gefen.AdamW([{"params": ps[1][:2], "lr": 1e-2}, {"params": ps[1][2:], "lr": 5e-3}], **kw)
    grads = [[torch.zeros_like(p) for p in side] for side in ps]
    for side, g in zip(ps, grads):
        for p, x in zip(side, g):
            p.grad = x

    def fill(step):
        for i, s in enumerate(sizes):
            x = tensors([s], torch.float32, 100 * step + i, dev)[0]
            for g in grads:
                g[i].copy_(x.t() if i == 1 else x)
    graph = captured(graphed, lambda: fill(0))
    fill(0)
    eager.step()
    for step in range(1, 5):
        fill(step)
        lr.fill_(1e-2 * step)
        eager.param_groups[0]["lr"] = 1e-2 * step
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        _ = (base[0] * 2).sum().item()
        assert torch.equal(graphed.grad_norm, eager.grad_norm)
        for a, b in zip(graphed.moments(), eager.moments()):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        for a, b in zip(*ps):
            assert (a - b).abs().max().item() <= 2.0 ** -22 * (1 + step) if a.numel() else True
        assert all(float(graphed.state[p]["step"]) == step + 1 for p in ps[0])
    again = gefen.AdamW([{"params": ps[1][:2]}, {"params": ps[1][2:]}], **kw)
    again.load_state_dict(graphed.state_dict())
    assert again.state[ps[1][0]]["step"] == 5


def test_captures_that_are_refused(dev):
    def grab(opt):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    p = torch.nn.Parameter(torch.ones(8, device=dev))
    p.grad = torch.ones(8, device=dev)
    with pytest.raises(RuntimeError, match="first step"):
        grab(gefen.AdamW([p], capturable=True))
    opt = gefen.AdamW([p], capturable=True)
    opt.step()
    opt.state[p]["step"] = 1
    with pytest.raises(ValueError, match="step counter"):
        opt.step()
    with pytest.raises(ValueError, match="device lr"):
        opt = gefen.AdamW([p], lr=torch.tensor(0.1, device=dev, dtype=torch.float16), capturable=True)
        opt.step()


def test_a_device_lr_of_another_device_is_refused(dev, monkeypatch):
    """Before anything moves: its pointer would go to the parameters' kernels."""
    import types
    p = torch.nn.Parameter(torch.ones(8, device=dev))
    p.grad = torch.ones(8, device=dev)
    opt = gefen.AdamW([p], capturable=True)
    elsewhere = types.SimpleNamespace(get_device=lambda: dev.index + 1, dtype=torch.float32)  # no pointer to follow
    monkeypatch.setattr(gefen.AdamW, "_lr_of", staticmethod(lambda lr: (0.0, elsewhere)))
    with pytest.raises(ValueError, match="device lr"):
        opt.step()
    assert not opt.state and torch.equal(p.detach(), torch.ones(8, device=dev))


def test_bad_descriptors_are_refused(dev):
    from gefen.kernels import _native
    lib = _native.load()
    x = torch.zeros(64, device=dev)
    d = _native.AdamWDesc(p=x.data_ptr(), grad=x.data_ptr(), exp_avg=x.data_ptr(), exp_avg_sq=x.data_ptr(), numel=64,
                          dtype=0, bits=32)
    import ctypes
    for change, status in (({"dtype": 3}, -2), ({"bits": 16}, -1), ({"numel": -1}, -1), ({"p": None}, -1), ({"bits": 8}, -1)):
        bad = _native.AdamWDesc.from_buffer_copy(d)
        for k, v in change.items():
            setattr(bad, k, v)
        assert lib.gefenx_adamw_step(ctypes.byref(bad), 1, None, None) == status, change
        assert _native.last_error()
    assert lib.gefenx_adamw_step(None, 1, None, None) == -1 and lib.gefenx_adamw_step(None, 0, None, None) == 0
    assert lib.gefenx_adamw_norm(ctypes.byref(d), 1, 0.0, x.data_ptr(), x.data_ptr(), 256, None) == -1
    assert lib.gefenx_adamw_norm(ctypes.byref(d), 1, 1.0, x.data_ptr(), x.data_ptr(), 0, None) == -1
    assert lib.gefenx_adamw_moments(ctypes.byref(d), 1, None) == -1
    torch.cuda.synchronize()


@pytest.mark.parametrize("bits", [32, 8])
def test_past_2_31_elements(dev, bits):
    n = (1 << 31) + 4096 + 5
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device=dev))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    p.grad[-1000:] = 1.0
    p.grad[:1000] = -1.0
    opt = gefen.AdamW([p], lr=LR, weight_decay=0.0, state_bits=bits, max_grad_norm=1e9)
    opt.step()
    assert abs(opt.grad_norm.item() - math.sqrt(2000)) < 1e-5
    want = torch.tensor(LR).bfloat16().item()
    assert torch.all(p.detach()[-1000:] == -want) and torch.all(p.detach()[:1000] == want)
    assert not p.detach()[1000:1 << 20].any() and not p.detach()[-(1 << 20):-1000].any()
    m, v = opt.moments()[0]
    assert torch.all(m[-1000:] == m[-1]) and abs(m[-1].item() - 0.1) < 1e-6 and abs(m[0].item() + 0.1) < 1e-6
