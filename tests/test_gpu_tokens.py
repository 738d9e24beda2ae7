"""Token statistics and distillation against their formulas in 64 bits (values, gradients, differences), masks and refusals."""
import math

import pytest
import torch
from torch.autograd import forward_ad

import gefen

pytestmark = pytest.mark.gpu

IGNORE = -100
INF = math.inf
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


def bits(t):
    return t.detach().contiguous().reshape(-1).view(torch.uint8)


# ------------------------------------------------ the formulas, in float64 on the CPU

def finite(t):
    return torch.where(t.isfinite(), t, torch.zeros_like(t))


def statistics64(z, k):
    """z: [T, V] float64, divided by the temperature: (log softmax, entropy, ids of the k largest)."""
    lq = torch.log_softmax(z, -1)
    return lq, -(lq.exp() * finite(lq)).sum(-1), torch.sort(z, dim=-1, descending=True, stable=True)[1][:, :k]


def distill64(x, labels, spans, ids, logps, temperature, rest, hard, reduction):
    """(loss, divergence, nll, per row), differentiable in x; spans: the sequences' rows."""
    T, V = x.shape
    live = torch.zeros(T, dtype=torch.bool)
    for a, b in spans:
        live[a:b] = True
    valid = (labels != IGNORE) & live
    lq = torch.log_softmax(x / temperature, -1)
    held = logps != -INF
    at = torch.where(held, ids, torch.zeros_like(ids))
    p = torch.where(held, logps.double().exp(), torch.zeros_like(logps, dtype=torch.float64))
    lp = torch.where(held, logps.double(), torch.zeros_like(p))
    mass = p.sum(1)
    if rest == "normalize":
        some = mass > 0
        lp = lp - torch.where(some, mass, torch.ones_like(mass)).log()[:, None]
        p = p / torch.where(some, mass, torch.ones_like(mass))[:, None]
    each = (torch.where(held, p * (lp - lq.gather(1, at)), torch.zeros_like(p))).sum(1)
    if rest == "bucket":
        named = torch.zeros(T, V + 1, dtype=torch.bool).scatter_(1, torch.where(held, ids, torch.full_like(ids, V)), True)[:, :V]
        left = (1 - mass).clamp(min=0)
        open_ = (left > 0) & (~named & (x > -INF)).any(1)
        # from the largest of the others: next to the type's lowest value a logsumexp loses the log of how many there are,
        # and its gradient gives each of them all of the weight
        apart = (x / temperature).masked_fill(named, -INF)
        most = torch.where(open_, apart.detach().amax(1), torch.zeros_like(left))
        total = torch.where(open_, (apart - most[:, None]).exp().sum(1), torch.ones_like(left))
        others = total.log() + most - torch.logsumexp(x / temperature, 1)
        left = torch.where(open_, left, torch.ones_like(left))
        each = each + torch.where(open_, left * (left.log() - torch.where(open_, others, torch.zeros_like(others))), torch.zeros_like(left))
    each = torch.where(valid, each, torch.zeros_like(each))
    nll = torch.zeros_like(each)
    if hard:
        nll = torch.where(valid, -torch.log_softmax(x, -1).gather(1, labels.clamp(min=0)[:, None])[:, 0], nll)
    w = row_weights(valid, spans, reduction)
    divergence, mean = (each * w).sum(), (nll * w).sum()
    return (1 - hard) * temperature ** 2 * divergence + hard * mean, divergence, mean, each


def row_weights(valid, spans, reduction):
    n = [int(valid[a:b].sum()) for a, b in spans]
    w = torch.zeros(valid.numel(), dtype=torch.float64)
    for (a, b), count in zip(spans, n):
        if count:
            w[a:b] = 1.0 / sum(n) if reduction == "token" else 1.0 / (count * sum(1 for c in n if c))
    return w * valid


# ------------------------------------------------ tolerances

def sum_error(z):
    """Relative, of a row's sum of exp(z - max): a lane adds up V / 256 terms, a few dozen are joined; the exponents'
    (2 units each of an argument up to the distance from the maximum, weighted by the softmax)."""
    far = finite(z.amax(1, keepdim=True) - z)
    return U * (z.shape[1] / 256 + 64 + 4 * (finite(torch.softmax(z, -1)) * far).sum(1))


def entropy_error(z, h):
    """log S by its relative error; T / S by S's, its own sum's and its terms' (an exponent's 4 units, times the distance)."""
    far = finite(z.amax(1, keepdim=True) - z)
    p = finite(torch.softmax(z, -1))
    ratio, square = (p * far).sum(1), (p * far * far).sum(1)
    return sum_error(z) * (1 + ratio) + U * (ratio * (z.shape[1] / 256 + 64) + 4 * square + 2 * h)


# ------------------------------------------------ data

SHAPES = [(1, 1), (3, 2), (5, 7), (6, 8), (4, 9), (70, 1000), (5, 2048), (4, 2049), (3, 50257), (2300, 257), (3, 70001)]


def rows_of(T, V, dtype, seed=0, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, V, generator=g) * scale).to(dtype)
    labels = torch.randint(0, V, (T,), generator=g)
    labels[torch.rand(T, generator=g) < 0.2] = IGNORE
    return x, labels, g


# ------------------------------------------------ token statistics

@pytest.mark.parametrize("T,V", SHAPES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_statistics(dev, T, V, dtype):
    for top, temperature in ((0, 1.0), (1, 0.7), (min(V, 20), 1.0), (min(V, 128), 2.0)):
        x, labels, g = rows_of(T, V, dtype)
        z = x.double() / temperature
        lq, h, ids = statistics64(z, top)
        valid = labels != IGNORE
        logits = x.to(dev).requires_grad_()
        got = gefen.token_statistics(logits, labels.to(dev), top=top, temperature=temperature)
        assert got.logps.dtype is torch.float32 and got.top_ids.dtype is torch.int64 and got.top_ids.shape == (T, top)
        lp, err = lq.gather(1, labels.clamp(min=0)[:, None])[:, 0], sum_error(z)
        row = lambda t: t.detach().cpu().double()  # noqa: E731
        assert torch.all((row(got.logps) - lp).abs()[valid] <= (err + U * (2 * lp.abs() + 4))[valid])
        assert torch.all((row(got.entropy) - h).abs()[valid] <= entropy_error(z, h)[valid])
        assert torch.equal(got.top_ids.cpu()[valid], ids[valid])
        tl = lq.gather(1, ids)
        assert torch.all((row(got.top_logps) - tl).abs()[valid] <= (err[:, None] + U * (2 * tl.abs() + 4))[valid])
        assert torch.all(got.logps[~valid] == 0) and torch.all(got.entropy[~valid] == 0)
        assert torch.all(got.top_ids[~valid] == 0) and torch.all(got.top_logps[~valid] == -INF)
        plain = gefen.token_statistics(x.to(dev), labels.to(dev), top=top, temperature=temperature)
        assert all(torch.equal(a, b) for a, b in zip(got, plain)) and not plain.logps.requires_grad
        # the gradient, from gradients of all three
        up = [torch.randn(s, generator=g) for s in ((T,), (T,), (T, top))]
        torch.autograd.backward([got.logps, got.entropy, got.top_logps], [u.to(dev) for u in up])
        gl, gh, gt = (torch.where(valid.view(-1, *[1] * (u.dim() - 1)), u.double(), torch.zeros_like(u, dtype=torch.float64)) for u in up)
        p = lq.exp()
        far = z.amax(1, keepdim=True) - z
        hot = torch.zeros_like(p).scatter_add_(1, labels.clamp(min=0)[:, None], gl[:, None]).scatter_add_(1, ids, gt)
        sizes = torch.zeros_like(p).scatter_add_(1, labels.clamp(min=0)[:, None], gl.abs()[:, None]).scatter_add_(1, ids, gt.abs())
        want = (hot - p * ((gl + gt.sum(1))[:, None] + gh[:, None] * (lq + h[:, None]))) / temperature
        size = (gl.abs() + gt.abs().sum(1))[:, None] + gh.abs()[:, None] * (lq.abs() + h[:, None])
        tol = (p * size * (err[:, None] + U * (4 * far + top + 32)) + p * gh.abs()[:, None] * (entropy_error(z, h) + err)[:, None]
               + 8 * U * sizes) / temperature + UNIT[dtype] * want.abs() * 1.01 + LEAST[dtype]
        assert logits.grad.dtype is dtype and torch.all((logits.grad.cpu().double() - want).abs() <= tol)


@pytest.mark.parametrize("which", ["logps", "entropy", "top_logps"])
def test_statistics_gradient_of_one_output(dev, which):
    x, labels, g = rows_of(9, 300, torch.float32)
    up = torch.randn((9, 5) if which == "top_logps" else (9,), generator=g)
    one, all_ = x.to(dev).requires_grad_(), x.to(dev).requires_grad_()
    getattr(gefen.token_statistics(one, labels.to(dev), top=5), which).backward(up.to(dev))
    got = gefen.token_statistics(all_, labels.to(dev), top=5)
    names = ["logps", "entropy", "top_logps"]
    torch.autograd.backward([getattr(got, n) for n in names],
                            [up.to(dev) if n == which else torch.zeros_like(getattr(got, n)) for n in names])
    assert torch.equal(one.grad, all_.grad) and one.grad.abs().sum() > 0


def test_statistics_gradients_against_differences(dev):
    """Central differences of the 64-bit outputs, step 1e-5: third derivatives (below 10 here) leave 1e-9."""
    x, labels, g = rows_of(4, 6, torch.float32, seed=3, scale=1.0)
    up = [torch.randn(s, generator=g).double() for s in ((4,), (4,), (4, 2))]
    valid = (labels != IGNORE).double()

    def value(x):
        lq, h, ids = statistics64(x / 0.8, 2)
        lp = lq.gather(1, labels.clamp(min=0)[:, None])[:, 0]
        return ((lp * up[0] + h * up[1] + (lq.gather(1, ids) * up[2]).sum(1)) * valid).sum().item()

    logits = x.to(dev).requires_grad_()
    got = gefen.token_statistics(logits, labels.to(dev), top=2, temperature=0.8)
    torch.autograd.backward([got.logps, got.entropy, got.top_logps], [u.float().to(dev) for u in up])
    for r in range(4):
        for v in range(6):
            a, b = x.double().clone(), x.double().clone()
            a[r, v] += 1e-5
            b[r, v] -= 1e-5
            assert abs((value(a) - value(b)) / 2e-5 - logits.grad[r, v].item()) <= 1e-9 + 1e-6 + 1e-5 * abs(logits.grad[r, v].item())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [50, 300, 5000, 40001])
def test_ties_and_orders(dev, V, dtype):
    """Equal logits by index, rising and falling rows, few distinct values, both zeros: ids as a stable sort gives them."""
    g = torch.Generator().manual_seed(V)
    rising = torch.linspace(-3, 3, V)
    zeros = torch.where(torch.rand(V, generator=g) < 0.5, 0.0, -0.0)
    rows = [torch.zeros(V), rising, rising.flip(0), torch.randint(0, 3, (V,), generator=g).float(), zeros,
            torch.where(torch.arange(V) % 7 == 3, 1.0, 0.0), torch.where(torch.arange(V) >= V - 40, 2.0, torch.randn(V, generator=g)),
            torch.where(torch.arange(V) % 256 < 8, 5.0, 0.0) + torch.rand(V, generator=g),
            torch.where(torch.arange(V) % 2048 < 8, 5.0, 0.0) + torch.rand(V, generator=g)]
    x = torch.stack(rows).to(dtype)
    for top in (1, 20, min(V, 128)):
        for copies in (1, 300):  # rows of few and of many workgroups each
            got = gefen.token_statistics(x.repeat(copies, 1).to(dev), top=top)
            want = torch.sort(x.double(), dim=-1, descending=True, stable=True)[1][:, :top].repeat(copies, 1)
            assert got.logps is None and torch.equal(got.top_ids.cpu(), want)


# 2 or 4 splits of 5 steps of 1024 runs, the last of 4
UNEVEN = [(torch.bfloat16, 131072, 128), (torch.float16, 65536, 256), (torch.float32, 32768, 256)]


@pytest.mark.parametrize("dtype,V,T", UNEVEN)
@pytest.mark.parametrize("equal", [300, 600, 1000])
def test_ties_in_a_shorter_last_split(dev, dtype, V, T, equal):
    """The row's highest values in its last split alone, many of them equal, neighbours or a few apart."""
    g = torch.Generator().manual_seed(equal)
    x = torch.randn(T, V, generator=g).clamp(max=4.0)
    x[::2, V - 50 - equal:V - 50] = 9.0
    x[1::2, V - 50 - 3 * equal:V - 50:3] = 9.0
    x[:, V - 60] = 10.0
    x[:, V - 20] = 11.0
    x = x.to(dtype).to(dev)
    want = torch.sort(x.float(), dim=-1, descending=True, stable=True)[1][:, :128]
    lq = torch.log_softmax(x.double(), -1).gather(1, want)
    tol = sum_error(x.double())[:, None] + U * (2 * lq.abs() + 4)
    for top in (1, 20, 128):
        got = gefen.token_statistics(x, top=top)
        assert torch.equal(got.top_ids, want[:, :top])
        assert torch.all((got.top_logps.double() - lq[:, :top]).abs() <= tol[:, :top])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [40, 3001, 70001])
def test_masked_logits(dev, V, dtype):
    """-inf and the type's lowest value in masked places, rows that they leave nothing, NaN and +inf."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(8, V, generator=g).to(dtype)
    low = torch.finfo(dtype).min
    x[0, 5:] = -INF
    x[1, ::2] = low
    x[2] = -INF
    x[3] = low
    x[4, :-1] = -INF
    x[5, 7], x[5, 3] = math.nan, math.nan
    x[6, 2], x[6, 9] = INF, INF
    x[7, 1:] = low
    labels = torch.zeros(8, dtype=torch.long)
    logits = x.to(dev).requires_grad_()
    got = gefen.token_statistics(logits, labels.to(dev), top=12)
    (got.logps.sum() + got.entropy.sum()).backward()
    ids = got.top_ids.cpu()
    key = x.double().clone()
    key[5, 7], key[5, 3] = INF, INF  # NaN before all; no other +inf in that row
    assert torch.equal(ids, torch.sort(key, dim=-1, descending=True, stable=True)[1][:, :12])
    z = x.double()
    for r in (0, 1, 3, 4, 7):
        lq, h, _ = statistics64(z[r:r + 1], 12)
        want = lq[0, 0].item()
        assert got.logps[r].item() == want == -INF or abs(got.logps[r].item() - want) <= (sum_error(z[r:r + 1]) + U * (2 * abs(want) + 4)).item()
        assert abs(got.entropy[r].item() - h.item()) <= entropy_error(z[r:r + 1], h).item()
        assert torch.all(logits.grad[r].isfinite())
    assert torch.all(got.top_logps[0, 5:] == -INF) and torch.all(got.top_logps[0, :5].isfinite())
    for r in (2, 5, 6):
        assert math.isnan(got.logps[r].item()) and math.isnan(got.entropy[r].item())


FILLS = {torch.float32: [-1e7, -3e7, -1e9, -1e10, -1e12, 1e10, 2e30, -1e38], torch.float16: [-1e4, -65504.0, 6e4],
         torch.bfloat16: [-1e9, -1e10, 1e12, -1e38]}


@pytest.mark.parametrize("temperature", [1.0, 0.01, 50.0])
@pytest.mark.parametrize("V", [24, 3001, 9000])
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_logits(dev, dtype, V, temperature):
    """Rows that a large mask value leaves nothing, or one step above it, or some ordinary logits."""
    rows = []
    for fill in FILLS[dtype]:
        row = torch.full((V,), fill).to(dtype)
        next_ = row.clone()
        # one representable step towards 0, for every third
        step = torch.nextafter(row.float() if dtype is torch.float32 else row, torch.zeros_like(row))
        next_[::3] = step[::3].to(dtype)
        some = row.clone()
        some[5:15] = torch.linspace(-2, 2, 10).to(dtype)
        rows += [row, next_, some]
    x = torch.stack(rows)
    T = x.shape[0]
    labels = torch.arange(T) % V
    z = x.double() / temperature
    ids = statistics64(z, 7)[2]
    logits = x.to(dev).requires_grad_()
    got = gefen.token_statistics(logits, labels.to(dev), top=7, temperature=temperature)
    (got.logps.sum() + got.entropy.sum()).backward()
    err = sum_error(z)
    assert torch.equal(got.top_ids.cpu(), ids)
    for r in range(T):
        # relative to the maximum: a logsumexp of numbers like these rounds at their scale
        exact = ((z[r, labels[r]] - z[r].amax()) - torch.log(torch.exp(z[r] - z[r].amax()).sum())).item()
        if exact < -3.5e38:  # beyond fp32
            assert got.logps[r].item() == -INF
        else:
            assert abs(got.logps[r].item() - exact) <= err[r] + U * (2 * abs(exact) + 4), r
        p = torch.softmax(z[r] - z[r].amax(), 0)
        ent = -(p * torch.where(p > 0, p.log(), torch.zeros_like(p))).sum()
        assert abs(got.entropy[r].item() - ent.item()) <= entropy_error(z[r:r + 1] - z[r].amax(), ent[None]).item(), r
        assert torch.all(logits.grad[r].isfinite())
    # a student like that, held to its own top tokens: nothing to learn, and nothing lost
    own = gefen.token_statistics(x.to(dev), top=7, temperature=temperature)
    for rest in ("bucket", "drop", "normalize"):
        out, grad = gefen.distillation_loss_and_grad(x.to(dev), labels.to(dev), own.top_ids, own.top_logps, rest=rest,
                                                     temperature=temperature, hard_weight=0.25)
        if rest != "normalize":
            # of the difference of p log p and p log q the roundings of log p (up to 10) and the sums' errors are left
            assert torch.all(out.token_divergence.abs().cpu().double() <= 1e-5 + 2 * err), rest
        assert out.token_divergence.isfinite().all() and grad.isfinite().all()


LIMIT = 2.0 ** 24 / 1.4426950408889634  # of logits over their temperature that a lane takes by one fused operation
EDGES = [(1.0, LIMIT), (0.001, 0.001 * LIMIT), (1e-4, 1e-4 * LIMIT), (100.0, 100.0 * LIMIT), (2.0, LIMIT), (0.5, LIMIT)]


@pytest.mark.parametrize("T,V", [(4, 9000), (2304, 2800), (300, 40960)])  # a workgroup, a wave, splits and rows of their own
@pytest.mark.parametrize("temperature,edge", EDGES)
def test_rows_across_the_limit_of_fused_exponents(dev, temperature, edge, T, V):
    """Rows that rise by steps of fp32 from below 2^24 temperature / log2(e) to above it, and from -above to -below; where
    labels count at a temperature, the same of the logits themselves.  Formulas of the differences from the maximum, which
    are exact in 64 bits."""
    g = torch.Generator().manual_seed(V)
    step = 2.0 ** (math.floor(math.log2(edge)) - 23)
    rise = torch.arange(V) * 9 // V - 4 + torch.randint(-1, 2, (4, V), generator=g)
    rows = torch.tensor([1.0, -1.0, 1.0, -1.0], dtype=torch.float64)[:, None] * (round(edge / step) * step) + rise * step
    x = rows.float()
    assert torch.equal(x.double(), rows)
    keep = torch.tensor([0, 1, T // 2, T - 1])
    labels, y = torch.full((T,), IGNORE), torch.randint(0, V, (4,), generator=g)
    labels[keep] = y
    held = torch.zeros(T, V, device=dev)
    held[keep] = x.to(dev)
    labels = labels.to(dev)
    x64 = rows - rows.amax(1, keepdim=True)
    z = x64 / temperature
    lq, h, ids = statistics64(z, 5)
    leaf = held.clone().requires_grad_()
    got = gefen.token_statistics(leaf, labels, top=5, temperature=temperature)
    (got.logps.sum() + got.entropy.sum()).backward()
    of = lambda t: t.detach()[keep].cpu().double()  # noqa: E731
    err, lp, tl = sum_error(z), lq.gather(1, y[:, None])[:, 0], lq.gather(1, ids)
    assert torch.equal(got.top_ids[keep].cpu(), ids)
    assert torch.all((of(got.logps) - lp).abs() <= err + U * (2 * lp.abs() + 4))
    assert torch.all((of(got.top_logps) - tl).abs() <= err[:, None] + U * (2 * tl.abs() + 4))
    assert torch.all((of(got.entropy) - h).abs() <= entropy_error(z, h))
    p, far = lq.exp(), -z
    hot = torch.zeros_like(p).scatter_(1, y[:, None], 1.0)
    want = (hot - p * (1 + lq + h[:, None])) / temperature
    size = 1 + lq.abs() + h[:, None]
    tol = (p * size * (err[:, None] + U * (4 * far + 32)) + p * (entropy_error(z, h) + err)[:, None] + 8 * U * hot) / temperature
    assert torch.all((of(leaf.grad) - want).abs() <= tol + U * want.abs() * 1.01 + LEAST[torch.float32])
    # the same rows as a student's
    teacher = torch.stack([torch.randperm(V, generator=g)[:6] for _ in range(4)])
    logps = torch.full((4, 6), math.log(0.1))
    all_ids, all_lp = torch.zeros(T, 6, dtype=torch.long), torch.zeros(T, 6)
    all_ids[keep], all_lp[keep] = teacher, logps
    all_ids, all_lp = all_ids.to(dev), all_lp.to(dev)
    for rest, hard in (("bucket", 0.0), ("drop", 0.3)):
        at = x64.clone().requires_grad_()
        loss, _, _, each = distill64(at, y, [(0, 4)], teacher, logps, temperature, rest, hard, "token")
        loss.backward()
        kw = dict(rest=rest, hard_weight=hard, temperature=temperature)
        leaf = held.clone().requires_grad_()
        two = gefen.distillation_loss(leaf, labels, all_ids, all_lp, **kw)
        two.loss.backward()
        out, grad = gefen.distillation_loss_and_grad(held, labels, all_ids, all_lp, **kw)
        for o, d in ((two, leaf.grad), (out, grad)):
            off = check_distill(x64, y, [(0, 4)], teacher, logps, temperature, rest, hard, "token", at.grad, each.detach(), of(d),
                                of(o.token_divergence), torch.float32)
            assert abs(o.loss.item() - loss.item()) <= off + 2 * U * abs(loss.item())


def test_statistics_without_labels(dev):
    x, _, g = rows_of(6, 700, torch.float32)
    a, b = x.to(dev).requires_grad_(), x.to(dev).requires_grad_()
    one = gefen.token_statistics(a, top=3)
    two = gefen.token_statistics(b, torch.zeros(6, dtype=torch.long, device=dev), top=3)
    assert one.logps is None and torch.equal(one.entropy, two.entropy) and torch.equal(one.top_logps, two.top_logps)
    for o in (one, two):
        (o.entropy.sum() * 2 + o.top_logps[:, 1].sum()).backward()
    assert torch.equal(a.grad, b.grad)


def test_forward_mode_is_refused(dev):
    """Logits with a tangent, which none of the results would carry."""
    x = torch.randn(3, 50, device=dev)
    y = torch.zeros(3, dtype=torch.long, device=dev)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.randn_like(x))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                for call in (lambda: gefen.token_statistics(dual, y, top=3), lambda: gefen.token_statistics(dual),
                             lambda: gefen.token_logps(dual, y)):
                    with pytest.raises(NotImplementedError, match="jvp"):
                        call()
        inside = gefen.token_statistics(x, y, top=3)
    assert all(torch.equal(a, b) for a, b in zip(inside, gefen.token_statistics(x, y, top=3)))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("top", [129, 1 << 20, -1])
def test_bad_counts_of_tokens_take_no_memory(dev, top, grad):
    x = torch.zeros(64, 200, device=dev, requires_grad=grad)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats(dev)
    before = torch.cuda.memory_allocated(dev)
    with pytest.raises(ValueError, match="top"):
        gefen.token_statistics(x, top=top)
    assert torch.cuda.max_memory_allocated(dev) == before


def test_labels_outside_of_the_vocabulary(dev):
    x, _, _ = rows_of(4, 30, torch.float32)
    labels = torch.tensor([3, 30, -1, IGNORE])
    logits = x.to(dev).requires_grad_()
    got = gefen.token_statistics(logits, labels.to(dev), top=3)
    assert got.logps.isnan().tolist() == [False, True, True, False]
    assert got.entropy.isfinite().all() and got.top_logps[:3].isfinite().all()
    got.logps.sum().backward()
    assert logits.grad.isnan().any(1).tolist() == [False, True, True, False]


def test_leading_shapes_strides_and_sizes(dev):
    g = torch.Generator().manual_seed(2)
    for dtype in DTYPES:
        big = torch.randn(6, 11, 1003, generator=g).to(dtype).to(dev)
        labels = torch.randint(0, 1000, (6, 11), generator=g).to(dev)
        views = [big[:, :, 3:1003], big[:, :-1, :1000], big[:, 1:, 1:1001], big.transpose(0, 1)[:6, :6, 2:1002], big[::2, ::3, :1000],
                 big[:, :, :1000].transpose(1, 2).contiguous().transpose(1, 2), big[:1, :1].expand(6, 11, 1003)]
        for v in views:
            n, s = v.shape[:2]
            y = labels[:n, :s]
            leaf = v.detach().clone(memory_format=torch.preserve_format).requires_grad_(True)
            same = v.detach().contiguous().clone().requires_grad_(True)
            a, b = gefen.token_statistics(leaf, y, top=9), gefen.token_statistics(same, y.contiguous(), top=9)
            c = gefen.token_statistics(v, y, top=9)
            assert all(torch.equal(bits(i), bits(j)) and torch.equal(bits(i), bits(k)) for i, j, k in zip(a, b, c))
            for o in (a, b):
                (o.logps.sum() + o.entropy.sum() + o.top_logps[..., 2].sum()).backward()
            assert torch.equal(bits(leaf.grad), bits(same.grad))
    x = torch.randn(2, 3, 4, 50, device=dev)
    want = gefen.token_statistics(x.view(24, 50), top=3)
    for lead in ((24,), (2, 12), (2, 3, 4)):
        got = gefen.token_statistics(x.view(*lead, 50), top=3)
        assert got.entropy.shape == lead and torch.equal(got.entropy.view(-1), want.entropy)
        assert got.top_ids.shape == (*lead, 3) and torch.equal(got.top_ids.view(24, 3), want.top_ids)
    one = gefen.token_statistics(x[0, 0, 0], top=3)
    assert one.entropy.shape == () and torch.equal(one.top_ids, want.top_ids[0])
    none = gefen.token_statistics(x[:, :0], top=3)
    assert none.entropy.shape == (2, 0, 4) and none.top_ids.shape == (2, 0, 4, 3)
    empty = x[:0].clone().requires_grad_()
    gefen.token_statistics(empty).entropy.sum().backward()
    assert empty.grad.shape == (0, 3, 4, 50)
    with pytest.raises(ValueError):
        gefen.token_statistics(x, top=51)
    with pytest.raises(ValueError):
        gefen.token_statistics(x, top=-1)
    with pytest.raises(TypeError):
        gefen.token_statistics(x, top=1.5)
    with pytest.raises(NotImplementedError):
        gefen.token_statistics(x.double())


def test_rows_alone_and_among_many(dev):
    """A row alone and among thousands: the splits differ; ids agree, values to the sums' rounding."""
    for V in (4000, 40001):
        x = torch.randn(2500, V, device=dev, generator=torch.Generator(dev).manual_seed(V))
        many = gefen.token_statistics(x, top=20)
        for r in (0, 1234, 2499):
            one = gefen.token_statistics(x[r:r + 1], top=20)
            z = x[r:r + 1].double().cpu()
            assert torch.equal(one.top_ids[0], many.top_ids[r])
            assert abs(one.entropy.item() - many.entropy[r].item()) <= 2 * entropy_error(z, one.entropy.double().cpu()).item()
            tl = one.top_logps[0].double().cpu()
            assert torch.all((tl - many.top_logps[r].double().cpu()).abs() <= 2 * (sum_error(z) + U * (2 * tl.abs() + 4)))


def test_long_rows(dev):
    """Rows of more runs than a workgroup marks, among thousands, most of them masked."""
    T, V = 2100, 140001
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.randn(T, V, device=dev, dtype=dtype, generator=torch.Generator(dev).manual_seed(1)).requires_grad_()
        labels = torch.full((T,), IGNORE, device=dev)
        keep = torch.tensor([0, 1, 1000, T - 1], device=dev)
        labels[keep] = torch.tensor([0, V - 1, 131072, 70000], device=dev)
        z = x.detach()[keep].double().cpu()
        teacher = gefen.token_statistics(x.detach().roll(1, 0), labels, top=64)
        lq, h, ids = statistics64(torch.roll(x.detach(), 1, 0)[keep].double().cpu(), 64)
        assert torch.equal(teacher.top_ids[keep].cpu(), ids)
        ids_in, lp_in = teacher.top_ids[keep].cpu(), teacher.top_logps[keep].cpu()
        x64 = z.clone().requires_grad_()
        spans = [(0, 4)]
        loss, _, _, each = distill64(x64, labels[keep].cpu(), spans, ids_in, lp_in, 1.0, "bucket", 0.25, "token")
        loss.backward()
        out, grad = gefen.distillation_loss_and_grad(x.detach(), labels, teacher.top_ids, teacher.top_logps, hard_weight=0.25)
        check_distill(z, labels[keep].cpu(), spans, ids_in, lp_in, 1.0, "bucket", 0.25, "token", x64.grad, each.detach(),
                      grad[keep].cpu().double(), out.token_divergence[keep].cpu().double(), dtype)
        assert not grad[2:1000].any() and not grad[1001:-1].any()
        got = gefen.token_statistics(x, labels)
        got.entropy.sum().backward()
        lq, h, _ = statistics64(z, 0)
        want = -(lq.exp() * (lq + h[:, None]))
        p, far = lq.exp(), z.amax(1, keepdim=True) - z
        tol = (p * (lq.abs() + h[:, None]) * (sum_error(z)[:, None] + U * (4 * far + 32)) + p * (entropy_error(z, h) + sum_error(z))[:, None]
               + UNIT[dtype] * want.abs() * 1.01 + LEAST[dtype])
        assert torch.all((x.grad[keep].cpu().double() - want).abs() <= tol)
        assert not x.grad[2:1000].any()
        x.grad = None


def test_offsets_past_32_bits(dev):
    """More than 2^31 logits, of which a few rows count; and a row of 20 million."""
    T, V = 17000, 131072
    x = torch.zeros(T, V, device=dev, dtype=torch.bfloat16)
    keep = torch.tensor([3, T - 2, T - 1], device=dev)
    x[keep] = (torch.randn(3, V, device=dev, generator=torch.Generator(dev).manual_seed(2)) * 2).bfloat16()
    labels = torch.full((T,), IGNORE, device=dev)
    labels[keep] = torch.tensor([0, 70000, V - 1], device=dev)
    z, y = x[keep].double().cpu(), labels[keep].cpu()
    got = gefen.token_statistics(x.requires_grad_(), labels, top=16)
    lq, h, ids = statistics64(z, 16)
    assert torch.equal(got.top_ids[keep].cpu(), ids)
    lp = lq.gather(1, y[:, None])[:, 0]
    assert torch.all((got.logps[keep].detach().cpu().double() - lp).abs() <= sum_error(z) + U * (2 * lp.abs() + 4))
    got.logps.sum().backward()
    p = lq.exp()
    hot = torch.zeros_like(p).scatter_(1, y[:, None], 1.0)
    far = z.amax(1, keepdim=True) - z
    tol = UNIT[x.dtype] * (hot - p).abs() * 1.01 + p * (sum_error(z)[:, None] + U * (4 * far + 32)) + LEAST[x.dtype]
    assert torch.all((x.grad[keep].cpu().double() - (hot - p)).abs() <= tol)
    assert not x.grad[4:T - 2].any()
    x.grad = None
    x.requires_grad_(False)
    lps = torch.zeros(T, 16, device=dev)
    lps[keep] = got.top_logps.detach()[keep] - 0.125
    x64 = z.clone().requires_grad_()
    loss, _, _, each = distill64(x64, y, [(0, 3)], ids, lps[keep].cpu(), 1.0, "bucket", 0.0, "token")
    loss.backward()
    for hard in (0.0, 0.3):  # rows of their own, and two passes
        t = 1.0 if hard == 0.0 else 2.0
        x64 = z.clone().requires_grad_()
        loss, _, _, each = distill64(x64, y, [(0, 3)], ids, lps[keep].cpu(), t, "bucket", hard, "token")
        loss.backward()
        out, grad = gefen.distillation_loss_and_grad(x, labels, got.top_ids, lps, hard_weight=hard, temperature=t)
        check_distill(z, y, [(0, 3)], ids, lps[keep].cpu(), t, "bucket", hard, "token", x64.grad, each.detach(),
                      grad[keep].cpu().double(), out.token_divergence[keep].cpu().double(), x.dtype)
        del grad
    del x
    V = 20000003
    x = torch.randn(2, V, device=dev, generator=torch.Generator(dev).manual_seed(3)).half()
    got = gefen.token_statistics(x, top=128)
    ids = torch.sort(x.double(), dim=-1, descending=True, stable=True)[1][:, :128]
    assert torch.equal(got.top_ids, ids)
    lq = torch.log_softmax(x.double(), -1)
    assert (got.top_logps.double() - lq.gather(1, ids)).abs().max().item() <= U * (V / 256 + 100)
    out, grad = gefen.distillation_loss_and_grad(x, torch.zeros(2, dtype=torch.long, device=dev), ids, got.top_logps - 1.0, rest="drop",
                                                 grad_scale=1e5)
    q, p = lq.exp(), (got.top_logps - 1.0).double().exp()
    want = (q * p.sum(1, keepdim=True)).scatter_add_(1, ids, -p) * 5e4
    # the bound of a sum's error, V / 256 units, is 5e-3 here
    assert torch.all((grad.double() - want).abs() <= UNIT[x.dtype] * want.abs() * 1.01 + 5e4 * q * 1e-2 * p.sum(1, keepdim=True) + 5e4 * p.max() * 1e-5
                     + LEAST[x.dtype])


# ------------------------------------------------ distillation

class Data:
    """Sequences of given lengths, padded [N, S, V] or packed [T, V]; labels ignored in the first fifth (and in padding);
    a teacher near the student, some of whose entries hold no token."""

    def __init__(self, lengths, V, k, dtype, dev, packed, temperature=1.0, ids=torch.int64, seed=0, empty=(), scale=2.0):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.dev, self.V, self.packed, self.n, self.k = dtype, dev, V, packed, len(lengths), k
        S = max(lengths)
        T = self.T = sum(lengths) if packed else len(lengths) * S
        self.labels = torch.full((T,), IGNORE, dtype=torch.long)
        self.spans, at = [], 0
        for i, L in enumerate(lengths):
            start = at if packed else i * S
            at += L
            self.spans.append((start, start + (L if packed else S)))
            first = L if i in empty else L // 5
            self.labels[start + first:start + L] = torch.randint(0, V, (L - first,), generator=g)
        self.x = (torch.randn(T, V, generator=g) * scale).to(dtype)
        self.x64 = self.x.double()
        z = (self.x64 + torch.randn(T, V, generator=g)) / temperature
        logp, self.ids = torch.log_softmax(z, -1).topk(k, -1)
        gone = (torch.rand(T, 1, generator=g) < 0.3) & (torch.arange(k) >= (k + 1) // 2)
        self.ids = torch.where(gone, torch.full_like(self.ids, -7), self.ids).to(ids)  # an id of no token is not used
        self.logps = logp.float().masked_fill(gone, -INF)
        self.lead = (T,) if packed else (len(lengths), S)
        self.cu = torch.tensor([a for a, _ in self.spans] + [T], dtype=torch.int32, device=dev) if packed else None

    def logits(self, grad=False):
        return self.x.to(self.dev).view(*self.lead, self.V).requires_grad_(grad)

    def args(self):
        return self.labels.to(self.dev).view(self.lead), self.ids.to(self.dev).view(*self.lead, -1), self.logps.to(self.dev).view(*self.lead, -1)

    def exact(self, temperature, rest, hard, reduction):
        x = self.x64.clone().requires_grad_()
        out = distill64(x, self.labels, self.spans, self.ids.long(), self.logps, temperature, rest, hard, reduction)
        out[0].backward()
        return [t.detach() for t in out], x.grad


def distill_errors(x64, ids, logps, temperature, rest):
    """Per row: (error of the divergence, of sums relative, mass, r, rho): by the relative error of the student's sum
    (P of it), of the teacher's tokens' sum and of the others' (r (1 - rho) of either), the rest is in float64."""
    z = x64 / temperature
    held = logps != -INF
    named = torch.zeros(z.shape[0], z.shape[1] + 1, dtype=torch.bool)
    named = named.scatter_(1, torch.where(held, ids, torch.full_like(ids, z.shape[1])), True)[:, :-1]
    p = torch.where(held, logps.double().exp(), torch.zeros_like(logps, dtype=torch.float64))
    mass = p.sum(1)
    left = (1 - mass).clamp(min=0) if rest == "bucket" else torch.zeros_like(mass)
    if rest == "normalize":
        p = p / torch.where(mass > 0, mass, torch.ones_like(mass))[:, None]
        mass = p.sum(1)
    far = sum_error(z) + sum_error(z.masked_fill(named, -INF)) + sum_error(z.masked_fill(~named, -INF))
    lq = torch.log_softmax(z, -1)
    rho = lq.exp().masked_fill(named, 0.0).sum(1)
    return mass * far + left * far * (1 - rho) + 1e-10, far, p, mass, left, rho, named


def check_distill(x64, labels, spans, ids, logps, temperature, rest, hard, reduction, want, each, grad, token, dtype, scale=1.0):
    err, rel, p, mass, left, rho, named = distill_errors(x64, ids, logps, temperature, rest)
    assert torch.all((token - each).abs() <= (err + U * each.abs()) * (labels != IGNORE))
    w = row_weights(labels != IGNORE, spans, reduction)
    z = x64 / temperature
    q = torch.softmax(z, -1)
    far = finite(z.amax(1, keepdim=True) - z)
    held = torch.where(logps != -INF, ids, torch.zeros_like(ids))
    spread = torch.zeros_like(q).scatter_add_(1, held, p * (8 + 2 * finite(logps.double()).abs()))
    share = torch.where(named | (rho <= 0)[:, None], torch.zeros_like(q), (left / torch.where(rho > 0, rho, torch.ones_like(rho)))[:, None] * q)
    size = q * (mass + left)[:, None] + share
    soft = (1 - hard) * temperature
    tol = soft * (size * (rel[:, None] + U * (4 * far + 32)) + U * spread)
    if hard:
        q1 = torch.softmax(x64, -1)
        far1 = finite(x64.amax(1, keepdim=True) - x64)
        hot = torch.zeros_like(q).scatter_(1, labels.clamp(min=0)[:, None], 1.0)
        tol = tol + hard * (q1 * (sum_error(x64)[:, None] + U * (4 * far1 + 32)) + 4 * U * hot)
    tol = tol * (w * scale)[:, None] + UNIT[dtype] * (want * scale).abs() * 1.01 + LEAST[dtype]
    assert torch.all((grad - want * scale).abs() <= tol)
    return (w * ((1 - hard) * temperature ** 2 * err + (hard * sum_error(x64) if hard else 0.0))).sum().item()


LENGTHS = [([1], 2, 1), ([5, 3], 7, 3), ([1, 1, 1], 8, 8), ([9, 4], 9, 2), ([33, 20, 15, 40], 1000, 20), ([3, 2], 2048, 64), ([4, 7], 2049, 100),
           ([2, 3], 50257, 64), ([500, 700, 400, 600], 257, 40), ([300, 290], 513, 300)]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("lengths,V,k", LENGTHS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_distillation(dev, lengths, V, k, dtype, packed):
    for rest, hard, temperature, reduction, ids, empty in (
            ("bucket", 0.0, 1.0, "token", torch.int64, ()), ("bucket", 0.4, 2.0, "sequence", torch.int32, (len(lengths) - 1,)),
            ("drop", 0.3, 1.0, "sequence", torch.int64, (0,)), ("normalize", 0.2, 0.7, "token", torch.int32, ()),
            ("bucket", 0.5, 1.0, "token", torch.int32, ())):
        d = Data(lengths, V, k, dtype, dev, packed, temperature, ids, empty=empty)
        (loss, divergence, nll, each), want = d.exact(temperature, rest, hard, reduction)
        kw = dict(cu_seqlens=d.cu, temperature=temperature, rest=rest, hard_weight=hard, reduction=reduction)
        logits = d.logits(True)
        out = gefen.distillation_loss(logits, *d.args(), **kw)
        scale = 1024.0 if dtype is torch.float16 else 1.0
        (out.loss * scale).backward()
        fused, grad = gefen.distillation_loss_and_grad(d.logits(), *d.args(), grad_scale=scale, **kw)
        for o, g in ((out, logits.grad), (fused, grad)):
            assert g.shape == logits.shape and g.dtype is dtype
            off = check_distill(d.x64, d.labels, d.spans, d.ids.long(), d.logps, temperature, rest, hard, reduction, want, each,
                                g.cpu().double().view(d.T, V), o.token_divergence.detach().cpu().double().view(-1), dtype, scale)
            assert abs(o.loss.item() - loss.item()) <= off + 2 * U * abs(loss.item())
            assert abs(o.divergence.item() - divergence.item()) <= off / ((1 - hard) * temperature ** 2) + U * abs(divergence.item())
            assert abs(o.nll.item() - nll.item()) <= (sum_error(d.x64).max().item() + U * abs(nll.item()) if hard else 0.0)


ALONE = [  # many long rows, whose loss and gradient one workgroup each finds: type, rows, vocabulary, teacher's tokens, column
    (torch.bfloat16, 1050, 200000, 64, 0), (torch.bfloat16, 1700, 131072, 127, 3), (torch.float16, 1700, 131080, 5, 0),
    (torch.float32, 1100, 100000, 100, 1), (torch.bfloat16, 1700, 131072, 128, 0), (torch.float16, 1700, 131079, 20, 0),
    (torch.bfloat16, 1030, 49160, 33, 5), (torch.float32, 1030, 24576, 4, 0)]


@pytest.mark.parametrize("dtype,T,V,k,column", ALONE)
def test_many_long_rows(dev, dtype, T, V, k, column):
    """Most rows masked; those that are not against the formulas, by both calls."""
    g = torch.Generator(dev).manual_seed(k)
    held = torch.randn(T, V + (8 if column else 0), device=dev, dtype=dtype, generator=g) * 2
    x = held[:, column:column + V]
    keep = torch.tensor([0, 1, 77, 1024, T - 2], device=dev)
    labels = torch.full((T,), IGNORE, device=dev)
    near = (x[keep].float() + torch.randn(5, V, device=dev, generator=g)).log_softmax(-1)
    lp, ids = near.topk(k, -1)
    ids[0, -1], lp[0, -2], ids[1, 0] = V - 1, -INF, ids[1, 1]  # the last column, no token, one twice
    ids[3, :3] = torch.tensor([8, 9, 15], device=dev)  # of one run
    labels[keep] = torch.tensor([0, V - 1, int(ids[2, 0]), 16, V // 2], device=dev)  # one of them the teacher's
    all_ids, all_lp = torch.zeros(T, k, dtype=torch.long, device=dev), torch.zeros(T, k, device=dev)
    all_ids[keep], all_lp[keep] = ids, lp
    for rest, hard, temperature in (("bucket", 0.0, 1.0), ("bucket", 0.3, 2.0), ("drop", 0.2, 1.0), ("normalize", 0.5, 0.7)):
        y, spans = labels[keep].cpu(), [(0, 5)]
        x64 = x[keep].double().cpu().requires_grad_()
        loss, _, _, each = distill64(x64, y, spans, ids.cpu(), lp.cpu(), temperature, rest, hard, "token")
        loss.backward()
        kw = dict(rest=rest, hard_weight=hard, temperature=temperature)
        scale = torch.tensor(512.0, device=dev)
        out, grad = gefen.distillation_loss_and_grad(x, labels, all_ids, all_lp, grad_scale=scale, **kw)
        leaf = x.detach().clone().requires_grad_()
        two = gefen.distillation_loss(leaf, labels, all_ids, all_lp, **kw)
        (two.loss * 512.0).backward()
        masked = torch.ones(T, dtype=torch.bool, device=dev)
        masked[keep] = False
        for o, d in ((out, grad), (two, leaf.grad)):
            off = check_distill(x64.detach(), y, spans, ids.cpu(), lp.cpu(), temperature, rest, hard, "token", x64.grad, each.detach(),
                                d[keep].cpu().double(), o.token_divergence.detach()[keep].cpu().double(), dtype, 512.0)
            assert abs(o.loss.item() - loss.item()) <= off + 2 * U * abs(loss.item())
            assert not d[masked].any() and not o.token_divergence[masked].any()
    # a spoilt row is spoilt alone; a scale of 0 asks for no gradient
    all_ids[1, 2] = V
    out, grad = gefen.distillation_loss_and_grad(x, labels, all_ids, all_lp)
    assert out.token_divergence.isnan().nonzero().view(-1).tolist() == [1] and grad.isnan().any(1).nonzero().view(-1).tolist() == [1]
    out, grad = gefen.distillation_loss_and_grad(x, labels, all_ids, all_lp, grad_scale=0.0)
    assert not grad.any()
    cu = torch.tensor([1, 78, 1025], dtype=torch.int32, device=dev)  # rows 0 and T - 2 belong to none
    all_ids[1, 2] = 0
    one = gefen.distillation_loss_and_grad(x, labels, all_ids, all_lp, cu_seqlens=cu, reduction="sequence")
    assert not one[1][0].any() and not one[1][-2].any() and one[1][1].any()
    assert abs(one[0].loss.item() - (one[0].token_divergence[[1, 77]].mean() + one[0].token_divergence[1024]).item() / 2) <= 1e-6


def test_distillation_gradients_against_differences(dev):
    """Central differences of the 64-bit loss, step 1e-5: third derivatives (below 10 here) leave 1e-9."""
    d = Data([3, 2], 6, 2, torch.float32, dev, False, scale=1.0)
    for rest, hard, temperature in (("bucket", 0.3, 1.5), ("drop", 0.0, 1.0), ("normalize", 0.5, 1.0)):
        value = lambda x: distill64(x, d.labels, d.spans, d.ids, d.logps, temperature, rest, hard, "sequence")[0].item()  # noqa: E731, B023
        _, grad = gefen.distillation_loss_and_grad(d.logits(), *d.args(), temperature=temperature, rest=rest, hard_weight=hard,
                                                   reduction="sequence")
        grad = grad.cpu().double().view(d.T, 6)
        for r in range(d.T):
            for v in range(6):
                a, b = d.x64.clone(), d.x64.clone()
                a[r, v] += 1e-5
                b[r, v] -= 1e-5
                assert abs((value(a) - value(b)) / 2e-5 - grad[r, v].item()) <= 1e-9 + 1e-6 + 1e-5 * abs(grad[r, v].item())


@pytest.mark.parametrize("dtype", DTYPES)
def test_teachers_at_their_limits(dev, dtype):
    """All tokens named, none, one twice, a mass over 1, all of the mass; students that rule tokens out or are sure."""
    V, k = 12, 12
    g = torch.Generator().manual_seed(4)
    T = 9
    x = torch.randn(T, V, generator=g).to(dtype)
    logp, ids = torch.log_softmax(torch.randn(T, V, generator=g), -1).sort(-1, descending=True)
    logps = logp.float()
    logps[1] = -INF                        # none
    ids[2, 1], ids[2, 5] = ids[2, 0], ids[2, 0]  # one of them three times
    logps[2, 6:] = -INF
    logps[3, 3:] = -INF
    logps[3, :3] = math.log(0.5)           # a mass of 1.5
    logps[4, 1:] = -INF
    logps[4, 0] = 0.0                      # all of the mass on one
    logps[5, 4:] = -INF
    x[5] = torch.finfo(dtype).min
    x[5, ids[5, :4]] = 1.0                 # the others ruled out by the lowest value
    logps[6, 4:] = -INF
    x[6] = -INF
    x[6, ids[6, :6]] = 0.5                 # ... by -inf, two apart
    logps[7, 4:] = -INF
    x[7, ids[7, 0]] = 100.0                # sure
    logps[8, 2:] = -INF
    x[8, ids[8, 3]] = 300.0                # sure of a token that the teacher does not name
    labels = torch.zeros(T, dtype=torch.long)
    spans = [(0, T)]
    for rest in ("bucket", "drop", "normalize"):
        x64 = x.double().requires_grad_()
        loss, _, _, each = distill64(x64, labels, spans, ids, logps, 1.0, rest, 0.0, "token")
        loss.backward()
        out, grad = gefen.distillation_loss_and_grad(x.to(dev), labels.to(dev), ids.to(dev), logps.to(dev), rest=rest, grad_scale=T)
        got, g64 = out.token_divergence.cpu().double(), grad.cpu().double()
        err, rel, p, mass, left, rho, named = distill_errors(x.double(), ids, logps, 1.0, rest)
        for r in range(T):
            if not math.isfinite(each[r].item()):
                assert got[r].item() == each[r].item()
                continue
            # sums of 12 terms; sums that have to be told apart by e^100 and e^300 stay in range
            assert abs(got[r] - each[r]) <= 1e-6 * (1 + abs(each[r])), (rest, r)
            assert torch.all((g64[r] - T * x64.grad[r]).abs() <= UNIT[dtype] * T * x64.grad[r].abs() * 1.01 + 2e-6), (rest, r)


def test_bad_ids_spoil_their_rows_alone(dev):
    d = Data([6], 40, 4, torch.float32, dev, False)
    labels, ids, logps = d.args()
    labels[0] = torch.arange(6, device=dev)
    logps[0] = torch.tensor([-1.0, -2.0, -2.0, -3.0], device=dev)
    ids[0, :, :] = torch.tensor([1, 2, 3, 4], device=dev)
    ids[0, 1, 2], ids[0, 3, 0] = 40, -1
    ids[0, 5, 1], logps[0, 5, 1] = 1 << 40, -INF  # names none
    for rest in ("bucket", "drop", "normalize"):
        out, grad = gefen.distillation_loss_and_grad(d.logits(), labels, ids, logps, rest=rest)
        spoilt = [False, True, False, True, False, False]
        assert out.token_divergence[0].isnan().tolist() == spoilt and math.isnan(out.loss.item())
        assert grad[0].isnan().any(-1).tolist() == spoilt
    labels[0, 2], ids[0] = 40, torch.tensor([1, 2, 3, 4], device=dev)
    out, grad = gefen.distillation_loss_and_grad(d.logits(), labels, ids, logps, hard_weight=0.5)
    assert math.isnan(out.nll.item()) and out.divergence.isfinite() and grad[0].isnan().any(-1).tolist() == [r == 2 for r in range(6)]
    out, grad = gefen.distillation_loss_and_grad(d.logits(), labels, ids, logps)
    assert out.loss.isfinite() and grad.isfinite().all()


@pytest.mark.parametrize("T,V", [(6, 40), (2304, 40), (256, 24576)])  # a workgroup, a wave, rows of their own
@pytest.mark.parametrize("rest", ["bucket", "drop", "normalize"])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_labels_alone_leave_the_teacher_out(dev, T, V, rest, temperature):
    """hard_weight 1: a teacher that cannot be told spoils its divergence, neither the loss nor the gradient."""
    g = torch.Generator().manual_seed(11)
    x = torch.randn(T, V, generator=g)
    labels = torch.randint(V, (T,), generator=g)
    ids = torch.arange(4).repeat(T, 1)
    logps = torch.full((T, 4), -2.0)
    ids[1, 2], ids[4, 0] = V, -1
    logps[3, 1], logps[5, 0] = math.nan, INF
    out, grad = gefen.distillation_loss_and_grad(x.to(dev), labels.to(dev), ids.to(dev), logps.to(dev), rest=rest, hard_weight=1.0,
                                                 temperature=temperature, grad_scale=T)
    assert out.token_divergence[[1, 3, 4]].isnan().all() and out.token_divergence.isfinite().sum() == T - 4
    x64 = x.double()
    q = torch.softmax(x64, -1)
    nll = -torch.log_softmax(x64, -1).gather(1, labels[:, None])[:, 0]
    err = sum_error(x64)
    # each row's in float64 from sums in fp32, the loss rounded once
    assert abs(out.loss.item() - nll.mean().item()) <= err.max().item() + 2 * U * nll.mean().item()
    want = q.scatter_add(1, labels[:, None], -torch.ones(T, 1, dtype=torch.float64))
    # an exponent's units over distances up to 10 (32), six products and sums of values up to 1
    limit = (err[:, None] + 32 * U) * q + 8 * U
    assert torch.all((grad.cpu().double() - want).abs() <= limit)


def test_rows_outside_of_the_sequences(dev):
    d = Data([10], 50, 5, torch.float32, dev, True)
    labels, ids, logps = d.args()
    labels[:] = 1
    cu = torch.tensor([2, 5, 5, 8], dtype=torch.int32, device=dev)
    for reduction in ("token", "sequence"):
        out, grad = gefen.distillation_loss_and_grad(d.logits(), labels, ids, logps, cu_seqlens=cu, reduction=reduction)
        inside, g2 = gefen.distillation_loss_and_grad(d.logits()[2:8], labels[2:8], ids[2:8], logps[2:8], cu_seqlens=cu - 2,
                                                      reduction=reduction)
        assert torch.equal(out.loss, inside.loss) and torch.equal(grad[2:8], g2)
        assert not grad[:2].any() and not grad[8:].any()
        assert not out.token_divergence[:2].any() and not out.token_divergence[8:].any()


def test_many_short_rows(dev):
    """More rows than one workgroup adds up, without sequences and with them."""
    T, V, k = 70000, 24, 3
    g = torch.Generator(dev).manual_seed(9)
    x = torch.randn(T, V, device=dev, generator=g)
    lp, ids = (x + torch.randn(T, V, device=dev, generator=g)).log_softmax(-1).topk(k, -1)
    labels = torch.randint(0, V, (T,), device=dev, generator=g)
    labels[torch.rand(T, device=dev, generator=g) < 0.5] = IGNORE
    valid = labels != IGNORE
    out, grad = gefen.distillation_loss_and_grad(x, labels, ids, lp, hard_weight=0.5)
    n = int(valid.sum())
    each = out.token_divergence.double()
    assert abs(out.divergence.item() - each[valid].mean().item()) <= 2 * U * abs(out.divergence.item()) + 1e-9
    nll = -x.double().log_softmax(-1).gather(1, labels.clamp(min=0)[:, None])[:, 0][valid].mean().item()
    assert abs(out.nll.item() - nll) <= 70 * U + U * nll
    cu = torch.tensor([0, 30000, T], dtype=torch.int32, device=dev)
    two, g2 = gefen.distillation_loss_and_grad(x, labels, ids, lp, hard_weight=0.5, cu_seqlens=cu)
    assert torch.equal(out.token_divergence, two.token_divergence) and abs(out.loss.item() - two.loss.item()) <= 2 * U * out.loss.item()
    assert (grad - g2).abs().max().item() <= 4 * U / n


def test_nothing_to_learn_from(dev):
    d = Data([4, 3], 20, 3, torch.bfloat16, dev, False)
    _, ids, logps = d.args()
    none = torch.full(d.lead, IGNORE, device=dev)
    for reduction in ("token", "sequence"):
        out, grad = gefen.distillation_loss_and_grad(d.logits(), none, ids, logps, reduction=reduction, hard_weight=0.5)
        assert out.loss.item() == 0 and out.nll.item() == 0 and not grad.any()
        assert not out.token_divergence.any()
    x = torch.zeros(2, 0, 20, device=dev, requires_grad=True)
    out = gefen.distillation_loss(x, none[:, :0], ids[:, :0], logps[:, :0])
    out.loss.backward()
    assert out.loss.item() == 0 and x.grad.shape == x.shape


def test_distillation_strides_and_types(dev):
    """Views, other types of the teacher's numbers and ids give what their plain copies give, bit for bit."""
    g = torch.Generator().manual_seed(0)
    for dtype in DTYPES:
        big = torch.randn(4, 11, 1003, generator=g).to(dtype).to(dev)
        labels = torch.randint(0, 900, (4, 11), generator=g).to(dev)
        ids = torch.randint(0, 900, (4, 11, 24), generator=g).to(dev)
        logps = (torch.log_softmax(torch.randn(4, 11, 24, generator=g), -1) - 0.5).bfloat16().to(dev)
        for v in (big[:, :, 3:1003], big[:, :-1, :1000], big[:, 1:, 1:1001], big[::2, ::3, :1000],
                  big[:, :, :1000].transpose(1, 2).contiguous().transpose(1, 2)):
            n, s = v.shape[:2]
            y, i, p = labels[:n, :s], ids[:n, :s, ::2], logps[:n, :s, ::2]
            a, ga = gefen.distillation_loss_and_grad(v, y, i, p, hard_weight=0.2)
            b, gb = gefen.distillation_loss_and_grad(v.contiguous(), y.contiguous(), i.int().contiguous(), p.float().contiguous(),
                                                     hard_weight=0.2)
            assert all(torch.equal(bits(m), bits(o)) for m, o in zip(a, b)) and torch.equal(bits(ga), bits(gb))
            leaf = v.detach().clone(memory_format=torch.preserve_format).requires_grad_(True)
            gefen.distillation_loss(leaf, y, i, p, hard_weight=0.2).loss.backward()
            assert torch.equal(bits(leaf.grad), bits(gb))


def test_distillation_refusals(dev):
    d = Data([4, 4], 20, 3, torch.float32, dev, False)
    x, (labels, ids, logps) = d.logits(), d.args()
    ok = dict(rest="bucket", reduction="token")
    for args, kw, error in (
            ((x, labels, ids[:, :2], logps[:, :2]), {}, ValueError), ((x, labels, ids, logps[..., :2]), {}, ValueError),
            ((x, labels, ids.float(), logps), {}, ValueError), ((x, labels, ids, ids), {}, ValueError),
            ((x, labels, ids.cpu(), logps), {}, ValueError), ((x, labels, ids[..., :0], logps[..., :0]), {}, ValueError),
            ((x, labels, None, logps), {}, TypeError), ((x, None, ids, logps), {}, TypeError),
            ((x, labels, ids, logps), {"rest": "all"}, ValueError), ((x, labels, ids, logps), {"reduction": "sum"}, ValueError),
            ((x, labels, ids, logps), {"hard_weight": 1.1}, ValueError), ((x, labels, ids, logps), {"temperature": 0}, ValueError),
            ((x, labels, ids, logps), {"temperature": math.nan}, ValueError),
            ((x.double(), labels, ids, logps), {}, NotImplementedError),
            ((x[0], labels[0], ids[0], logps[0]), {"reduction": "sequence"}, ValueError),
            ((x, labels, torch.zeros(2, 4, 513, dtype=torch.long, device=dev), torch.zeros(2, 4, 513, device=dev)), {}, ValueError)):
        for call in (gefen.distillation_loss, gefen.distillation_loss_and_grad):
            with pytest.raises(error):
                call(*args, **{**ok, **kw})
    with pytest.raises(ValueError):
        gefen.distillation_loss_and_grad(x, labels, ids, logps, grad_scale=None)
    with pytest.raises(ValueError):
        gefen.distillation_loss_and_grad(x, labels, ids, logps, grad_scale=torch.ones(1))


def test_a_teacher_that_changed_is_noticed(dev):
    d = Data([4, 4], 20, 3, torch.float32, dev, False)
    labels, ids, logps = d.args()
    out = gefen.distillation_loss(d.logits(True), labels, ids, logps)
    logps.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.loss.backward()


# ------------------------------------------------ as they are used

def test_teacher_to_student(dev):
    """The teacher's statistics, the student's loss against them, a step: with the teacher's own logits the loss is nothing,
    and steps lead there.  Against plain autograd in float64."""
    V, k, temperature = 500, 16, 1.5
    g = torch.Generator().manual_seed(6)
    hidden = torch.randn(3, 7, 24, generator=g)
    head = torch.nn.Parameter((torch.randn(24, V, generator=g) * 0.3).to(dev))
    labels = torch.randint(0, V, (3, 7), generator=g)
    labels[0, :3] = IGNORE
    teacher = gefen.token_statistics((torch.randn(3, 7, V, generator=g) * 2).to(dev), labels.to(dev), top=k, temperature=temperature)
    opt = gefen.AdamW([head], lr=1e-2)
    for _ in range(2):
        opt.zero_grad()
        logits = hidden.to(dev) @ head
        out = gefen.distillation_loss(logits, labels.to(dev), teacher.top_ids, teacher.top_logps, temperature=temperature, hard_weight=0.1)
        stats = gefen.token_statistics(logits, labels.to(dev))
        valid = (labels != IGNORE).to(dev)
        (out.loss - 0.01 * stats.entropy[valid].mean()).backward()
        h64, w64 = hidden.double(), head.detach().cpu().double().requires_grad_()
        x = (h64 @ w64).view(21, V)
        loss = distill64(x, labels.view(-1), [(0, 21)], teacher.top_ids.cpu().view(21, k), teacher.top_logps.cpu().view(21, k),
                         temperature, "bucket", 0.1, "token")[0]
        lq = torch.log_softmax(x, -1)
        h = -(lq.exp() * lq).sum(-1)[labels.view(-1) != IGNORE].mean()
        (loss - 0.01 * h).backward()
        # products of 24 and 21 terms in fp32 on either side, values and gradients of order 1
        assert torch.allclose(head.grad.cpu().double(), w64.grad, rtol=1e-4, atol=1e-6)
        opt.step()
    same = torch.randn(3, 7, V, generator=g).to(dev)
    own = gefen.token_statistics(same, top=k, temperature=temperature)
    out, grad = gefen.distillation_loss_and_grad(same, labels.to(dev), own.top_ids, own.top_logps, temperature=temperature)
    # of a divergence of 0 the terms' errors are left: the log-probabilities' roundings (2^-24 of up to 10) on both sides
    assert abs(out.loss.item()) <= 1e-5 and grad.abs().max().item() <= 1e-6


def test_example_distills(dev):
    """The example's distillation runs, and its student's gradients are those of plain torch in float64."""
    import importlib.util
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    spec = importlib.util.spec_from_file_location("finetune", os.path.join(root, "examples", "finetune.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    torch.manual_seed(0)
    teacher, student = m.Model().to(dev), m.Model().to(dev)
    twin = m.Model().to(dev)
    twin.load_state_dict(student.state_dict())
    seen = {}
    real = gefen.distillation_loss_and_grad

    def watched(logits, labels, ids, logps, **kw):
        if not seen:
            seen.update(labels=labels, ids=ids, logps=logps, kw=kw)
        return real(logits, labels, ids, logps, **kw)

    class Watch:
        token_statistics, distillation_loss_and_grad = staticmethod(gefen.token_statistics), staticmethod(watched)

        class AdamW(gefen.AdamW):
            def step(self, closure=None):
                seen.setdefault("grads", [p.grad.clone() for g in self.param_groups for p in g["params"]])
                return super().step(closure)

    tokens = []
    sample, m.sample, m.gefen = m.sample, lambda *a: tokens.append(sample(*a)) or tokens[-1], Watch
    divergences = m.distill(teacher, student, 3)
    assert len(divergences) == 3 and all(math.isfinite(d) and d > 0 for d in divergences)
    twin = twin.double().cpu()
    logits = twin(tokens[0].cpu()).view(-1, m.VOCAB)
    labels, k = seen["labels"].cpu().view(-1), seen["ids"].shape[-1]
    loss = distill64(logits, labels, [(0, labels.numel())], seen["ids"].cpu().view(-1, k), seen["logps"].cpu().view(-1, k),
                     seen["kw"]["temperature"], "bucket", seen["kw"]["hard_weight"], "token")[0]
    loss.backward()
    for got, want in zip(seen["grads"], twin.parameters()):
        # an fp32 model against a float64 one: sums of hundreds of terms either way
        assert (got.cpu().double() - want.grad).abs().max().item() <= 1e-4 * want.grad.abs().max().item() + 1e-9


def test_repeats_are_equal(dev):
    d = Data([300, 200, 250], 5001, 40, torch.bfloat16, dev, True)
    first = None
    for _ in range(3):
        out, grad = gefen.distillation_loss_and_grad(d.logits(), *d.args(), cu_seqlens=d.cu, hard_weight=0.1)
        stats = gefen.token_statistics(d.logits(), d.args()[0], top=40)
        now = [bits(t) for t in (*out, grad, *stats)]
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(first, now))


def test_the_same_token_twice_adds_up_in_order(dev):
    d = Data([40], 600, 60, torch.float32, dev, False)
    labels, ids, logps = d.args()
    ids[:] = torch.randint(0, 20, ids.shape, device=dev)
    results = [gefen.distillation_loss_and_grad(d.logits(), labels, ids, logps - 2, rest=rest, hard_weight=0.3)[1]
               for rest in ("bucket", "drop") for _ in range(3)]
    for a in (0, 3):
        assert torch.equal(results[a], results[a + 1]) and torch.equal(results[a], results[a + 2])


def test_device_scales(dev):
    d = Data([6, 5], 300, 9, torch.float16, dev, False)
    scale = torch.tensor(256.0, device=dev)
    a, ga = gefen.distillation_loss_and_grad(d.logits(), *d.args(), grad_scale=scale)
    b, gb = gefen.distillation_loss_and_grad(d.logits(), *d.args(), grad_scale=256.0)
    assert torch.equal(ga, gb) and torch.equal(a.loss, b.loss)


def test_other_streams(dev):
    d = Data([50, 60], 3000, 20, torch.bfloat16, dev, False)
    want, grad = gefen.distillation_loss_and_grad(d.logits(), *d.args())
    stats = gefen.token_statistics(d.logits(), d.args()[0], top=10)
    torch.cuda.synchronize()
    args = d.args()
    x = d.logits()
    torch.cuda.synchronize()
    outs = []
    for _ in range(2):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            outs.append((gefen.distillation_loss_and_grad(x, *args), gefen.token_statistics(x, args[0], top=10)))
    torch.cuda.synchronize()
    for (out, g), st in outs:
        assert torch.equal(bits(g), bits(grad)) and all(torch.equal(bits(a), bits(b)) for a, b in zip(out, want))
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(st, stats))


def test_captured_calls(dev):
    """Two graphs, replayed in turn with new data and eager calls between them."""
    d = [Data([12, 9], 3001, 20, torch.bfloat16, dev, False, seed=s) for s in range(3)]
    held = []
    side = torch.cuda.Stream()
    for first in range(2):
        x, args = d[first].logits(), d[first].args()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            gefen.distillation_loss_and_grad(x, *args, hard_weight=0.2)
            gefen.token_statistics(x, args[0], top=20)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = gefen.distillation_loss_and_grad(x, *args, hard_weight=0.2)
            stats = gefen.token_statistics(x, args[0], top=20)
        held.append((graph, x, args, out, stats))
    for round_ in range(3):
        for i, (graph, x, args, (out, grad), stats) in enumerate(held):
            new = d[(round_ + i) % 3]
            x.copy_(new.logits())
            for a, b in zip(args, new.args()):
                a.copy_(b)
            graph.replay()
            want, g = gefen.distillation_loss_and_grad(new.logits(), *new.args(), hard_weight=0.2)
            st = gefen.token_statistics(new.logits(), new.args()[0], top=20)
            torch.cuda.synchronize()
            assert torch.equal(bits(grad), bits(g)) and all(torch.equal(bits(a), bits(b)) for a, b in zip(out, want))
            assert all(torch.equal(bits(a), bits(b)) for a, b in zip(stats, st))


def test_captured_backward(dev):
    """Forward and backward of fresh leaves in a graph, replayed with new data and eager calls between."""
    d = [Data([12, 9], 3001, 20, torch.bfloat16, dev, False, seed=s) for s in range(3)]

    def step(x, args):
        x.grad = None
        stats = gefen.token_statistics(x, args[0], top=5)
        out = gefen.distillation_loss(x, *args, hard_weight=0.2)
        (out.loss + stats.entropy.mean() + stats.top_logps[..., 0].mean()).backward()
        return out.loss.detach(), stats.entropy.detach(), x.grad

    x, args = d[0].logits(True), d[0].args()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, args)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, args)
    for new in (d[1], d[2], d[0]):
        with torch.no_grad():
            x.copy_(new.logits())
        for a, b in zip(args, new.args()):
            a.copy_(b)
        graph.replay()
        want = step(new.logits(True), new.args())
        torch.cuda.synchronize()
        assert all(torch.equal(bits(a), bits(b)) for a, b in zip(got, want))


def test_compiled_callers(dev):
    d = Data([5, 6], 200, 8, torch.float32, dev, False)

    def step(x, labels, ids, logps):
        return gefen.distillation_loss(x * 1.0, labels, ids, logps).loss + gefen.token_statistics(x, labels).entropy.sum()

    a, b = d.logits(True), d.logits(True)
    step(a, *d.args()).backward()
    torch.compile(step, backend="eager")(b, *d.args()).backward()
    assert torch.equal(a.grad, b.grad)
