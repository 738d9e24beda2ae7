"""Losses over the logits against their formulas in 64 bits (values, gradients, differences), masks and refusals."""
import math

import pytest
import torch

import gefen

pytestmark = pytest.mark.gpu

IGNORE = -100
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
U = 2.0 ** -24


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


# ------------------------------------------------ the formulas, in float64 on the CPU

def logps64(x, labels):
    """x: [T, V] float64; labels [T]: log-probabilities, 0 where ignored."""
    valid = labels != IGNORE
    lp = torch.log_softmax(x, -1).gather(1, labels.clamp(min=0)[:, None])[:, 0]
    return torch.where(valid, lp, torch.zeros_like(lp))


def per_sequence(values, spans):
    return torch.stack([values[a:b].sum() for a, b in spans]) if spans else values.new_zeros(0)


def preference64(x, labels, spans, ref, beta, smoothing, average):
    lp = logps64(x, labels)
    valid = (labels != IGNORE).double()
    n = per_sequence(valid, spans)
    reward = beta * per_sequence((lp - ref) * valid, spans) / (n.clamp(min=1) if average else 1.0)
    half = len(spans) // 2
    h = reward[:half] - reward[half:]
    sig = torch.nn.functional.logsigmoid
    return (-(1 - smoothing) * sig(h) - smoothing * sig(-h)).mean(), reward


def policy64(x, labels, spans, old, adv, ref, lo, hi, kl_coef, reduction):
    lp = logps64(x, labels)
    valid = (labels != IGNORE).double()
    n = per_sequence(valid, spans)
    q = torch.exp(lp - old)
    plain, clip = q * adv, q.clamp(1 - lo, 1 + hi) * adv
    d = ref - lp
    kl = torch.expm1(d) - d
    each = (kl_coef * kl - torch.minimum(plain, clip)) * valid
    tokens = n.sum().clamp(min=1)
    if reduction == "token":
        loss = each.sum() / tokens
    else:
        loss = (per_sequence(each, spans) / n.clamp(min=1)).sum() / (n > 0).double().sum().clamp(min=1)
    return loss, (kl * valid).sum() / tokens, ((clip < plain).double() * valid).sum() / tokens


# ------------------------------------------------ tolerances

def logp_tolerance(x, labels):
    """Per row: the sum's rounding (a lane adds up V / 256 terms, then a few dozen are joined), the exponents'
    (2 units each of an argument up to the distance from the maximum, weighted by the softmax), the result's own."""
    far = x.amax(1, keepdim=True) - x
    weighted = (torch.softmax(x, -1) * torch.where(far.isfinite(), far, torch.zeros_like(far))).sum(1)
    lp = logps64(x, labels).abs()
    return U * (x.shape[1] / 256 + 64 + 4 * weighted + 2 * lp + 4)


def grad_tolerance(g64, x, labels, k_rel, k, dtype):
    """Per element: the rounding to its type, and relative to |k| (softmax + one-hot) the coefficient's error, the
    sum's (as above) and the exponential's (its argument's distance from the maximum, 2 units each)."""
    p = torch.softmax(x, -1)
    far = (x.amax(1, keepdim=True) - x)
    far = torch.where(far.isfinite(), far, torch.zeros_like(far))
    hot = torch.zeros_like(p)
    hot.scatter_(1, labels.clamp(min=0)[:, None], 1.0)
    rel = logp_tolerance(x, labels)[:, None] + U * (4 * far + 16) + k_rel
    return UNIT[dtype] * g64.abs() * 1.01 + k.abs()[:, None] * (p + hot) * rel + LEAST[dtype]


# ------------------------------------------------ data

class Data:
    """Sequences of given lengths, padded [N, S, V] or packed [T, V]; labels ignored in the first fifth (and in padding)."""

    def __init__(self, lengths, V, dtype, dev, packed, seed=0, empty=(), scale=2.0):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.dev, self.V, self.packed, self.n = dtype, dev, V, packed, len(lengths)
        S = max(lengths) if lengths else 0
        T = sum(lengths) if packed else len(lengths) * S
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
        self.lead = (T,) if packed else (len(lengths), S)
        self.T = T
        lp = logps64(self.x64, self.labels).detach() if T else torch.zeros(0, dtype=torch.float64)
        d = torch.randn(T, generator=g, dtype=torch.float64) * 0.2
        for edge in (math.log(0.8), math.log(1.3)):  # ratios away from the clip's edges
            d = torch.where((d - edge).abs() < 1e-2, d + 0.03 * math.copysign(1, edge), d)
        self.old = (lp - d).float()
        self.ref = (lp + 0.1 * torch.randn(T, generator=g, dtype=torch.float64)).float()
        self.adv = torch.randn(T, generator=g)
        self.seq_adv = torch.randn(len(lengths), generator=g)
        self.cu = torch.tensor([a for a, _ in self.spans] + [T], dtype=torch.int32, device=dev) if packed else None

    def row(self, t):
        return t.to(self.dev).view(self.lead)

    def logits(self, grad=False):
        return self.x.to(self.dev).view(*self.lead, self.V).requires_grad_(grad)

    def seq_of_rows(self):
        s = torch.zeros(self.T, dtype=torch.long)
        for i, (a, b) in enumerate(self.spans):
            s[a:b] = i
        return s


LENGTHS = [
    ([5, 3], 1), ([1, 1], 2), ([9, 4], 7), ([6, 8], 8), ([2, 17], 9), ([33, 20, 15, 40], 1000), ([3, 2], 2048), ([4, 7], 2049),
    ([2, 3], 50257), ([260, 300, 400, 200, 310, 290, 150, 300], 257),
]


@pytest.mark.parametrize("lengths,V", LENGTHS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_token_logps(dev, lengths, V, dtype):
    d = Data(lengths, V, dtype, dev, packed=True)
    logits = d.logits(True)
    got = gefen.token_logps(logits, d.row(d.labels))
    x = d.x64.clone().requires_grad_(True)
    want = logps64(x, d.labels)
    assert got.dtype is torch.float32 and got.shape == d.lead
    assert torch.all((got.detach().cpu().double() - want.detach()).abs() <= logp_tolerance(d.x64, d.labels))
    up = torch.randn(d.T, generator=torch.Generator().manual_seed(5))
    (want * up.double()).sum().backward()
    got.backward(up.to(dev))
    k = torch.where(d.labels == IGNORE, 0.0, up.double())
    assert logits.grad.dtype is dtype
    assert torch.all((logits.grad.cpu().double() - x.grad).abs() <= grad_tolerance(x.grad, d.x64, d.labels, U, k, dtype))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("lengths,V", LENGTHS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_preference(dev, lengths, V, dtype, packed):
    for average, smoothing, with_ref, empty in ((False, 0.0, True, ()), (True, 0.1, True, (len(lengths) - 1,)),
                                                (False, 0.2, False, (0,))):
        d = Data(lengths, V, dtype, dev, packed, empty=empty)
        beta = 0.1
        ref = d.ref.double() if with_ref else torch.zeros(d.T, dtype=torch.float64)
        x = d.x64.clone().requires_grad_(True)
        loss, reward = preference64(x, d.labels, d.spans, ref, beta, smoothing, average)
        loss.backward()
        kw = dict(cu_seqlens=d.cu, beta=beta, label_smoothing=smoothing, average=average)
        args = (d.row(d.labels), d.row(d.ref) if with_ref else None)
        logits = d.logits(True)
        out = gefen.preference_loss(logits, *args, **kw)
        fused, grad = gefen.preference_loss_and_grad(d.logits(), *args, **kw)
        # a reward's error: its tokens' (sums are in float64), and one rounding
        tol = logp_tolerance(d.x64, d.labels) * (d.labels != IGNORE)
        n = per_sequence((d.labels != IGNORE).double(), d.spans).clamp(min=1) if average else 1.0
        off = beta * per_sequence(tol, d.spans) / n
        half = len(lengths) // 2
        for o in (out, fused):
            r = torch.cat([o.chosen_rewards, o.rejected_rewards]).detach().cpu().double()
            assert torch.all((r - reward.detach()).abs() <= off + U * reward.detach().abs())
            # the loss changes by at most as much as h
            assert abs(o.loss.item() - loss.item()) <= (off[:half] + off[half:]).max() + 2 * U * abs(loss.item())
            assert torch.all((o.logps.detach().cpu().double().view(-1) - logps64(d.x64, d.labels)).abs() <= tol)
        out.loss.backward()
        # |dk / k| <= the error of h: s(h) - 1 + e changes by s' <= 1/4, and |s(h) - (1 - e)| stays over 1/20 here
        s = torch.sigmoid(reward[:half] - reward[half:]).detach()
        assert (s - (1 - smoothing)).abs().min() > 0.01 or max(lengths) > 100 or V < 3
        k = beta * (s - (1 - smoothing)).abs() / half
        kk = (torch.cat([k, k]) / n)[d.seq_of_rows()] * (d.labels != IGNORE)
        dk = (beta * 0.25 * (off[:half] + off[half:]) / half)
        dkk = (torch.cat([dk, dk]) / n)[d.seq_of_rows()] * (d.labels != IGNORE)
        for g in (logits.grad, grad):
            g = g.cpu().double().view(d.T, V)
            tol_g = grad_tolerance(x.grad, d.x64, d.labels, 8 * U, kk, dtype)
            p = torch.softmax(d.x64, -1)
            hot = torch.zeros_like(p).scatter_(1, d.labels.clamp(min=0)[:, None], 1.0)
            assert torch.all((g - x.grad).abs() <= tol_g + dkk[:, None] * (p + hot))


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("lengths,V", LENGTHS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_policy(dev, lengths, V, dtype, packed):
    for reduction, per_token, kl_coef, empty in (("token", True, 0.05, ()), ("sequence", False, 0.2, (0,)),
                                                 ("token", False, 0.0, (len(lengths) - 1,))):
        d = Data(lengths, V, dtype, dev, packed, empty=empty)
        adv = d.adv if per_token else d.seq_adv[d.seq_of_rows()]
        x = d.x64.clone().requires_grad_(True)
        loss, kl, clipped = policy64(x, d.labels, d.spans, d.old.double(), adv.double(), d.ref.double(), 0.2, 0.3, kl_coef,
                                     reduction)
        loss.backward()
        kw = dict(cu_seqlens=d.cu, clip_low=0.2, clip_high=0.3, kl_coef=kl_coef, reduction=reduction)
        args = (d.row(d.labels), d.row(d.old), d.row(d.adv) if per_token else d.seq_adv.to(dev), d.row(d.ref))
        logits = d.logits(True)
        out = gefen.policy_loss(logits, *args, **kw)
        fused, grad = gefen.policy_loss_and_grad(d.logits(), *args, **kw)
        valid = (d.labels != IGNORE).double()
        lp = logps64(d.x64, d.labels)
        tol = logp_tolerance(d.x64, d.labels)
        q = torch.exp(lp - d.old.double())
        e = torch.expm1(d.ref.double() - lp)
        n = per_sequence(valid, d.spans)
        w = (torch.full_like(n, 1 / max(1.0, n.sum().item())) if reduction == "token"
             else 1 / (n.clamp(min=1) * (n > 0).double().sum().clamp(min=1)))[d.seq_of_rows()] * valid
        # a token's loss: its derivative in logp times the error of logp, and 8 roundings of its terms
        dl = (q * adv.abs() + kl_coef * e.abs()) * tol + 8 * U * (q * adv.abs() + kl_coef * (1 + d.ref.abs() + lp.abs()))
        for o in (out, fused):
            assert abs(o.loss.item() - loss.item()) <= (w * dl).sum() + 2 * U * abs(loss.item())
            assert abs(o.kl.item() - kl.item()) <= ((e.abs() * tol + 4 * U * (d.ref.abs() + lp.abs() + 1) * (e.abs() + U))
                                                    * valid).sum() / n.sum().clamp(min=1) + 2 * U * kl.item()
            assert abs(o.clip_fraction.item() - clipped.item()) <= U
            assert torch.all((o.logps.detach().cpu().double().view(-1) - lp).abs() <= tol * valid)
        out.loss.backward()
        part = w * (q * adv.abs() + kl_coef * e.abs())
        dk = w * (q * adv.abs() + kl_coef * (1 + e.abs())) * (tol + 8 * U * (1 + lp.abs() + d.ref.abs()))
        p = torch.softmax(d.x64, -1)
        hot = torch.zeros_like(p).scatter_(1, d.labels.clamp(min=0)[:, None], 1.0)
        for g in (logits.grad, grad):
            tol_g = grad_tolerance(x.grad, d.x64, d.labels, 8 * U, part, dtype) + dk[:, None] * (p + hot)
            assert torch.all((g.cpu().double().view(d.T, V) - x.grad).abs() <= tol_g)


@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_preference_of_decided_pairs(dev, smoothing):
    """Pairs won and lost by far: the gradient of a won one falls off as exp(-h), to the last digit."""
    hs = [25.0, 33.0, 36.5, 40.0, 60.0, 80.0, -30.0, -60.0]
    n, S, V = len(hs), 3, 50
    d = Data([S] * (2 * n), V, torch.float32, dev, packed=False)  # no row is masked: 3 // 5 = 0
    ref = logps64(d.x64, d.labels).view(2 * n, S)
    ref[:n] -= torch.tensor(hs, dtype=torch.float64)[:, None] / S
    ref = ref.float()
    x = d.x64.clone().requires_grad_(True)
    loss, reward = preference64(x, d.labels, d.spans, ref.double().view(-1), 1.0, smoothing, False)
    loss.backward()
    out, grad = gefen.preference_loss_and_grad(d.logits(), d.row(d.labels), ref.to(dev), beta=1.0, label_smoothing=smoothing)
    h = (reward[:n] - reward[n:]).detach()
    assert (h - torch.tensor(hs).double()).abs().max() < 1e-3
    # s(-h) changes by a share of at most the error of h, the tokens' of both answers
    tol = logp_tolerance(d.x64, d.labels)
    dh = (per_sequence(tol, d.spans)[:n] + per_sequence(tol, d.spans)[n:]).repeat(2)[d.seq_of_rows()]
    k = (torch.sigmoid(-h) - smoothing).abs() / n
    slip = torch.sigmoid(-h) / n
    k, slip = (t.repeat(2)[d.seq_of_rows()] for t in (k, slip))
    p = torch.softmax(d.x64, -1)
    hot = torch.zeros_like(p).scatter_(1, d.labels[:, None], 1.0)
    tol_g = grad_tolerance(x.grad, d.x64, d.labels, 8 * U, k, torch.float32) + (slip * dh)[:, None] * (p + hot)
    assert torch.all((grad.cpu().double().view(d.T, V) - x.grad).abs() <= tol_g)
    assert abs(out.loss.item() - loss.item()) <= dh.max() + 2 * U * abs(loss.item())


def test_gradients_against_differences(dev):
    """Central differences of the 64-bit losses, step 1e-5: third derivatives (below 10 here) leave 1e-9."""
    d = Data([4, 5], 6, torch.float32, dev, packed=False)
    pref = lambda x: preference64(x, d.labels, d.spans, d.ref.double(), 0.5, 0.1, False)[0]  # noqa: E731
    pol = lambda x: policy64(x, d.labels, d.spans, d.old.double(), d.adv.double(), d.ref.double(), 0.2, 0.3, 0.1, "token")[0]  # noqa: E731
    _, g1 = gefen.preference_loss_and_grad(d.logits(), d.row(d.labels), d.row(d.ref), beta=0.5, label_smoothing=0.1)
    _, g2 = gefen.policy_loss_and_grad(d.logits(), d.row(d.labels), d.row(d.old), d.row(d.adv), d.row(d.ref), clip_high=0.3,
                                       kl_coef=0.1)
    for f, g in ((pref, g1), (pol, g2)):
        g = g.cpu().double().view(d.T, 6)
        for r in range(d.T):
            for v in range(6):
                up, down = d.x64.clone(), d.x64.clone()
                up[r, v] += 1e-5
                down[r, v] -= 1e-5
                assert abs((f(up) - f(down)).item() / 2e-5 - g[r, v].item()) <= 1e-9 + 1e-5 * abs(g[r, v].item()) + 1e-7


def bits(t):
    return t.detach().contiguous().reshape(-1).view(torch.uint8)


def test_strides_and_alignment(dev):
    """Views read in place give what their contiguous copies give, bit for bit."""
    g = torch.Generator().manual_seed(0)
    for dtype in DTYPES:
        big = torch.randn(6, 11, 1003, generator=g).to(dtype).to(dev)
        labels = torch.randint(0, 1000, (6, 11), generator=g).to(dev)
        ref = torch.randn(6, 11, generator=g).to(dev) - 7
        views = [big[:, :, 3:1003], big[:, :-1, :1000], big[:, 1:, 1:1001], big.transpose(0, 1)[:6, :6, 2:1002],
                 big[::2, ::3, :1000], big[:, :, :1000].transpose(1, 2).contiguous().transpose(1, 2), big[:1, :1].expand(6, 11, 1003)]
        for v in views:
            n, s = v.shape[:2]
            y = labels[:n, :s].clamp(max=v.shape[2] - 1)
            if n % 2:
                v, y, n = v[:n - 1], y[:n - 1], n - 1
            r = ref[:n, :s]
            a, ga = gefen.preference_loss_and_grad(v, y, r)
            b, gb = gefen.preference_loss_and_grad(v.contiguous(), y.contiguous(), r.contiguous())
            assert torch.equal(bits(a.loss), bits(b.loss)) and torch.equal(bits(a.logps), bits(b.logps))
            assert torch.equal(bits(ga), bits(gb)) and ga.is_contiguous() and ga.shape == v.shape
            leaf = v.detach().clone(memory_format=torch.preserve_format).requires_grad_(True)
            gefen.preference_loss(leaf, y, r).loss.backward()
            assert torch.equal(bits(leaf.grad), bits(gb))


def test_leading_shapes_of_token_logps(dev):
    x = torch.randn(2, 3, 4, 50, device=dev)
    y = torch.randint(0, 50, (2, 3, 4), device=dev)
    want = gefen.token_logps(x.view(24, 50), y.view(24))
    for lead in ((24,), (2, 12), (6, 4), (2, 3, 4)):
        assert torch.equal(gefen.token_logps(x.view(*lead, 50), y.view(lead)).view(-1), want)
    assert torch.equal(gefen.token_logps(x[0, 0, 0], y[0, 0, 0]), want[0])
    assert gefen.token_logps(x[:, :0], y[:, :0]).shape == (2, 0, 4)


def test_results_do_not_depend_on_the_split(dev):
    """A row's statistics alone and among thousands: the splits differ, the values agree to the sum's rounding."""
    x = torch.randn(3000, 4000, device=dev)
    y = torch.randint(0, 4000, (3000,), device=dev)
    many, few = gefen.token_logps(x, y), gefen.token_logps(x[:2], y[:2])
    tol = logp_tolerance(x[:2].cpu().double(), y[:2].cpu())
    assert torch.all((many[:2] - few).abs().cpu().double() <= 2 * tol)


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_rows_are_not_looked_at(dev, dtype):
    """NaN and inf in rows without a label leave no trace, and their gradient is 0."""
    d = Data([40, 30, 20, 35], 600, dtype, dev, packed=False)
    clean = d.logits()
    dirty = clean.clone()
    off = d.row(d.labels) == IGNORE
    dirty[off] = float("nan")
    dirty[0, 0, 5] = float("inf")
    for f, args in ((gefen.preference_loss_and_grad, (d.row(d.ref),)),
                    (gefen.policy_loss_and_grad, (d.row(d.old), d.row(d.adv), d.row(d.ref)))):
        bad = [torch.where(off, torch.full_like(a, float("nan")), a) for a in args]
        a, ga = f(clean, d.row(d.labels), *args)
        b, gb = f(dirty, d.row(d.labels), *bad)
        assert torch.equal(a.loss, b.loss) and torch.equal(a.logps, b.logps) and torch.equal(ga, gb)
        assert not gb[off].any() and torch.all(b.logps[off] == 0)
    leaf = dirty.clone().requires_grad_(True)
    lp = gefen.token_logps(leaf, d.row(d.labels))
    lp.sum().backward()
    assert torch.equal(lp, b.logps) and not leaf.grad[off].any() and torch.isfinite(leaf.grad).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("low", ["inf", "lowest"])
def test_masked_vocabulary(dev, dtype, low):
    """Entries at -inf or at the type's lowest value have probability 0, also whole chunks and splits of them."""
    V = 9000
    value = -float("inf") if low == "inf" else torch.finfo(dtype).min
    x = torch.randn(4, V, generator=torch.Generator().manual_seed(0)).to(dtype)
    x[0, :4096] = value
    x[1, 1:] = value
    x[2, 8:V - 1] = value
    y = torch.tensor([5000, 0, V - 1, 17])
    leaf = x.to(dev).requires_grad_(True)
    lp = gefen.token_logps(leaf, y.to(dev))
    want = logps64(x.double(), y)
    kept = x.double().masked_fill(x == value, -1e9)
    assert torch.all((lp.detach().cpu().double() - want).abs() <= logp_tolerance(kept, y))
    assert lp[1].item() == 0.0
    lp.sum().backward()
    g = leaf.grad.cpu()
    assert torch.isfinite(g).all() and not g[0, :4096].any() and not g[1].any() and not g[2, 8:V - 1].any()


def test_labels_of_no_weight_and_rows_of_no_value(dev):
    """As torch: a label at -inf has log-probability -inf; a row of -inf alone, NaN and +inf give NaN."""
    x = torch.zeros(5, 300)
    x[0, 7] = -float("inf")
    x[1] = -float("inf")
    x[2, 100] = float("nan")
    x[3, 100] = float("inf")
    y = torch.tensor([7, 0, 3, 3, 3])
    leaf = x.to(dev).requires_grad_(True)
    lp = gefen.token_logps(leaf, y.to(dev))
    lp.sum().backward()
    assert lp[0].item() == -float("inf") and torch.isnan(lp[1:4]).all() and abs(lp[4].item() + math.log(300)) < 1e-5
    assert torch.isnan(leaf.grad[1:4]).all() and torch.isfinite(leaf.grad[4]).all()
    assert torch.isfinite(leaf.grad[0]).all() and leaf.grad[0, 7].item() == 1.0


def test_preference_of_impossible_answers(dev):
    """An answer with a label at -inf: rejected, its pair is won (loss 0, no gradient); chosen, it is lost (loss inf,
    the gradient that of a lost pair); both sides: NaN."""
    x = torch.zeros(6, 2, 40, device=dev)
    y = torch.full((6, 2), 3, dtype=torch.long, device=dev)
    x[3, 1, 3] = x[1, 0, 3] = -float("inf")
    out, g = gefen.preference_loss_and_grad(x[[0, 3]].contiguous(), y[:2])
    assert out.loss.item() == 0.0 and not g.any() and out.rejected_rewards[0].item() == -float("inf")
    out, g = gefen.preference_loss_and_grad(x[[1, 0]].contiguous(), y[:2], beta=0.5)
    assert out.loss.item() == float("inf") and torch.isfinite(g).all()
    assert g[0, 0, 3].item() == -0.5 and abs(g[1, 0, 3].item() - 0.5 * (1 - 1 / 40)) < 1e-6
    out, g = gefen.preference_loss_and_grad(x[[1, 3]].contiguous(), y[:2])
    assert torch.isnan(out.loss)


def test_labels_out_of_range_make_their_results_nan(dev):
    x = torch.randn(4, 100, device=dev, requires_grad=True)
    y = torch.tensor([100, -1, 1 << 40, 5], device=dev)
    lp = gefen.token_logps(x, y)
    lp.sum().backward()
    assert torch.isnan(lp[:3]).all() and torch.isfinite(lp[3])
    assert torch.isnan(x.grad[:3]).all() and torch.isfinite(x.grad[3]).all()
    out, g = gefen.preference_loss_and_grad(x.detach().view(2, 2, 100), y.view(2, 2))
    assert torch.isnan(out.loss) and torch.isnan(g).all()


def test_nothing_to_learn_from(dev):
    x = torch.randn(4, 7, 100, device=dev)
    y = torch.full((4, 7), IGNORE, device=dev)
    z = torch.zeros(4, 7, device=dev)
    out, g = gefen.preference_loss_and_grad(x, y, z, average=True)
    assert abs(out.loss.item() - math.log(2)) < 1e-6 and not g.any() and not out.chosen_rewards.any()
    for reduction in ("token", "sequence"):
        out, g = gefen.policy_loss_and_grad(x, y, z, torch.ones(4, device=dev), z, kl_coef=0.1, reduction=reduction)
        assert out.loss.item() == 0 and out.kl.item() == 0 and out.clip_fraction.item() == 0 and not g.any()
    out, g = gefen.preference_loss_and_grad(x[:, :0], y[:, :0])
    assert abs(out.loss.item() - math.log(2)) < 1e-6 and g.shape == (4, 0, 100)
    out, g = gefen.policy_loss_and_grad(x[:, :0], y[:, :0], z[:, :0], z[:, :0])
    assert out.loss.item() == 0 and g.shape == (4, 0, 100)
    cu = torch.tensor([0, 0, 0], dtype=torch.int32, device=dev)
    out, g = gefen.preference_loss_and_grad(x[0, :0], y[0, :0], cu_seqlens=cu)
    assert abs(out.loss.item() - math.log(2)) < 1e-6


def test_packed_sequences_with_empty_ones_and_rows_outside(dev):
    """Sequences without rows, and rows that belong to none: no loss, no gradient, logps 0."""
    x = torch.randn(20, 64, device=dev)
    y = torch.randint(0, 64, (20,), device=dev)
    ref = torch.randn(20, device=dev)
    cu = torch.tensor([2, 2, 9, 9, 15], device=dev)  # int64; rows 0-1 and 15-19 outside
    out, g = gefen.preference_loss_and_grad(x, y, ref, cu_seqlens=cu)
    want, gw = gefen.preference_loss_and_grad(x[2:15].contiguous(), y[2:15], ref[2:15], cu_seqlens=cu - 2)
    assert torch.equal(out.loss, want.loss) and torch.equal(out.chosen_rewards, want.chosen_rewards)
    assert torch.equal(g[2:15], gw) and not g[:2].any() and not g[15:].any()
    assert not out.logps[:2].any() and not out.logps[15:].any() and torch.equal(out.logps[2:15], want.logps)
    y[0], y[17] = 64, -5  # no logits of these numbers, but nobody asks for them
    again, g2 = gefen.preference_loss_and_grad(x, y, ref, cu_seqlens=cu)
    assert torch.equal(again.loss, out.loss) and torch.equal(g2, g)


def test_advantages_of_as_many_tokens_as_sequences(dev):
    """Packed logits with a row per sequence on average: what [N] advantages belong to has to be said, unless every
    sequence has one row."""
    x, y = torch.randn(3, 50, device=dev), torch.tensor([4, 5, 6], device=dev)
    old, adv = gefen.token_logps(x, y).detach(), torch.tensor([1.0, -2.0, 4.0], device=dev)
    for f in (gefen.policy_loss, gefen.policy_loss_and_grad):
        run = lambda cu, **kw: f(x, y, old, adv, cu_seqlens=torch.tensor(cu, device=dev), **kw)  # noqa: E731, B023
        loss = lambda out: (out if f is gefen.policy_loss else out[0]).loss.item()  # noqa: E731, B023
        for cu in ([0, 0, 2, 3], [0, 1, 2, 2]):
            with pytest.raises(ValueError, match="advantages_per"):
                run(cu)
        # ratios are 1: the loss is minus the mean advantage of the tokens
        assert abs(loss(run([0, 0, 2, 3], advantages_per="token")) + 1.0) < 1e-6
        assert abs(loss(run([0, 0, 2, 3], advantages_per="sequence")) - 0.0) < 1e-6   # -2, -2, 4
        for per in (None, "token", "sequence"):
            assert abs(loss(run([0, 1, 2, 3], advantages_per=per)) + 1.0) < 1e-6
        with pytest.raises(ValueError, match="advantages_per"):
            run([0, 1, 2, 3], advantages_per="row")
        with pytest.raises(ValueError, match="advantages"):  # two sequences, three tokens
            run([0, 1, 3], advantages_per="sequence")
        with pytest.raises(ValueError, match="advantages"):
            f(x, y, old, adv[:2], cu_seqlens=torch.tensor([0, 1, 3], device=dev), advantages_per="token")
    out, grad = gefen.policy_loss_and_grad(x, y, old, adv, cu_seqlens=torch.tensor([0, 0, 2, 3], device=dev),
                                           advantages_per="sequence")
    want, g = gefen.policy_loss_and_grad(x, y, old, adv[[1, 1, 2]], cu_seqlens=torch.tensor([0, 1, 2, 3], device=dev))
    assert torch.equal(out.loss, want.loss) and torch.equal(grad, g)


def test_padded_and_packed_agree(dev):
    d = Data([40, 31, 25, 33], 500, torch.bfloat16, dev, packed=False)
    keep = torch.cat([torch.arange(i * 40, i * 40 + n) for i, n in enumerate([40, 31, 25, 33])])
    cu = torch.tensor([0, 40, 71, 96, 129], dtype=torch.int32, device=dev)
    pick = lambda t: t.reshape(160, *t.shape[2:])[keep.to(dev)]  # noqa: E731
    a, ga = gefen.policy_loss_and_grad(d.logits(), d.row(d.labels), d.row(d.old), d.seq_adv.to(dev), d.row(d.ref), kl_coef=0.1,
                                       reduction="sequence")
    b, gb = gefen.policy_loss_and_grad(pick(d.logits()), pick(d.row(d.labels)), pick(d.row(d.old)), d.seq_adv.to(dev),
                                       pick(d.row(d.ref)), cu_seqlens=cu, kl_coef=0.1, reduction="sequence")
    assert abs(a.loss.item() - b.loss.item()) <= 1e-6 * abs(a.loss.item()) + 1e-8
    # splits differ with the number of rows, so sums may differ in their last bits: one rounding of the gradient
    assert torch.all((pick(ga).float() - gb.float()).abs() <= 2.0 ** -7 * gb.float().abs() + 1e-12)


def test_scales(dev):
    """grad_scale as a number, as a device scalar, and as the gradient of the loss: the same gradient."""
    d = Data([20, 30], 777, torch.float16, dev, packed=False)
    args = (d.row(d.labels), d.row(d.old), d.row(d.adv), d.row(d.ref))
    _, a = gefen.policy_loss_and_grad(d.logits(), *args, grad_scale=512.0)
    _, b = gefen.policy_loss_and_grad(d.logits(), *args, grad_scale=torch.tensor([512.0], device=dev))
    leaf = d.logits(True)
    out = gefen.policy_loss(leaf, *args)
    (out.loss * 512.0).backward()
    assert torch.equal(a, b) and torch.equal(leaf.grad, a)
    assert not out.kl.requires_grad and not out.logps.requires_grad and not out.clip_fraction.requires_grad
    with torch.no_grad():
        assert not gefen.policy_loss(leaf, *args).loss.requires_grad
    again = gefen.policy_loss(leaf, *args)
    again.loss.div_(2)  # in place, as accumulation loops do
    leaf.grad = None
    again.loss.backward()
    _, half = gefen.policy_loss_and_grad(d.logits(), *args, grad_scale=0.5)
    assert torch.equal(leaf.grad, half)


def test_backward_of_copies_and_of_moved_tensors(dev):
    """Logits, labels and cu_seqlens that the forward pass had to copy, and saved tensors that hooks moved away."""
    d = Data([30, 20], 500, torch.float32, dev, packed=True)
    y, ref = d.row(d.labels), d.row(d.ref)
    plain = d.logits(True)
    gefen.preference_loss(plain, y, ref, cu_seqlens=d.cu).loss.backward()
    odd = d.x.t().contiguous().to(dev).requires_grad_(True)  # [V, T]
    every = torch.stack([y, y], 1)[:, 0]                     # stride 2
    gefen.preference_loss(odd.t(), every, ref, cu_seqlens=d.cu.long()).loss.backward()
    assert torch.equal(odd.grad.t(), plain.grad)
    leaf = d.logits(True)
    with torch.autograd.graph.save_on_cpu():
        out = gefen.preference_loss(leaf * 1.0, y, ref, cu_seqlens=d.cu)
    torch.empty(1 << 20, device=dev).fill_(float("nan"))
    out.loss.backward()
    assert torch.equal(leaf.grad, plain.grad)
    twice = d.logits(True)
    out = gefen.preference_loss(twice, y, ref, cu_seqlens=d.cu)
    with torch.no_grad():
        twice.add_(1.0)
    with pytest.raises(RuntimeError, match="modified"):
        out.loss.backward()


@pytest.mark.parametrize("offsets", [None, torch.int32, torch.int64])
@pytest.mark.parametrize("which", ["logps", "preference", "policy"])
def test_backward_of_moved_views(dev, which, offsets):
    """Slices of padded logits and of every sequence's rows but the last, and either type of offsets, moved to the host
    and back between the passes while the memory they came from is free to be taken: the gradient of the plain call."""
    n, S, V = 4, 33, 1000
    g = torch.Generator().manual_seed(2)
    h = torch.randn(n, S + 1, V + 24, generator=g).to(dev)
    y = torch.randint(0, V, (n, S), generator=g).to(dev)
    ref, adv = torch.randn(n, S, generator=g).to(dev) - 7, torch.randn(n, generator=g).to(dev)
    cu = None if offsets is None else torch.arange(0, n * S + 1, S, dtype=offsets, device=dev)

    def loss(leaf):
        x, args = (leaf * 1.0)[:, :-1, :V], [y, ref]
        if cu is not None:  # rows of a padded vocabulary, one sequence after another
            x, args = (leaf[:, :-1] * 1.0).reshape(n * S, V + 24)[:, :V], [y.view(-1), ref.view(-1)]
        if which == "logps":
            return (gefen.token_logps(x, args[0]) * args[1]).sum()
        if which == "preference":
            return gefen.preference_loss(x, *args, cu_seqlens=cu).loss
        return gefen.policy_loss(x, *args, adv, args[1], cu_seqlens=cu, kl_coef=0.1).loss
    got = []
    for moved in (False, True):
        leaf = h.clone().requires_grad_(True)
        if moved:
            with torch.autograd.graph.save_on_cpu():
                out = loss(leaf)
        else:
            out = loss(leaf)
        out.backward()
        got.append(leaf.grad)
    assert got[0].any() and torch.equal(*got)


def test_runs_repeat_bit_for_bit_and_on_other_streams(dev):
    d = Data([200, 300, 250, 280], 3001, torch.bfloat16, dev, packed=True)
    args = (d.logits(), d.row(d.labels), d.row(d.old), d.row(d.adv), d.row(d.ref))
    kw = dict(cu_seqlens=d.cu, kl_coef=0.1)
    first, g = gefen.policy_loss_and_grad(*args, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = torch.zeros_like(args[0])
        for _ in range(20):
            x = x + args[0] / 20 * 0
        x = x + args[0]
        other, h = gefen.policy_loss_and_grad(x, *args[1:], **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other)) and torch.equal(g, h)


@pytest.mark.parametrize("V,S", [(3001, 20), (131080, 420)])
def test_captured_losses_replay(dev, V, S):
    """The fused calls in a graph, replayed on other logits with eager work between, against eager calls; both the
    split rows and the rows of their own."""
    n = 4
    x = torch.zeros(n, S, V, device=dev, dtype=torch.bfloat16)
    y = torch.randint(0, V, (n, S), device=dev)
    y[:, :3] = IGNORE
    old, adv = torch.full((n, S), -8.0, device=dev), torch.randn(n, device=dev)

    def both():
        return (gefen.preference_loss_and_grad(x, y, old, average=True),
                gefen.policy_loss_and_grad(x, y, old, adv, old, kl_coef=0.1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    for k in range(3):
        x.copy_(torch.randn(n, S, V, generator=torch.Generator(dev).manual_seed(k), device=dev))
        graph.replay()
        want = both()
        torch.cuda.synchronize()
        for (a, ga), (b, gb) in zip(got, want):
            assert all(torch.equal(i, j) for i, j in zip(a, b)) and torch.equal(ga, gb)


def test_positions_past_2_31_elements(dev):
    rows, V = 16500, 131072 + 8
    x = torch.zeros(rows, V, dtype=torch.bfloat16, device=dev)
    tail = torch.randn(3, V, generator=torch.Generator(dev).manual_seed(0), device=dev).bfloat16()
    x[-3:] = tail
    y = torch.full((rows,), IGNORE, device=dev)
    y[-3:] = torch.tensor([0, V - 1, 77], device=dev)
    y[0] = 1
    old = torch.full((rows,), -11.0, device=dev)
    cu = torch.tensor([0, 10, rows], dtype=torch.int32, device=dev)
    adv = torch.ones(2, device=dev)
    out, g = gefen.policy_loss_and_grad(x, y, old, adv, cu_seqlens=cu)
    want = logps64(tail.double().cpu(), y[-3:].cpu())
    assert torch.all((out.logps[-3:].cpu().double() - want).abs() <= logp_tolerance(tail.double().cpu(), y[-3:].cpu()))
    k = torch.exp(want + 11.0)
    k = torch.where(k > 1.2, torch.zeros_like(k), k) / 4
    soft = torch.softmax(tail.double().cpu(), -1)
    soft[torch.arange(3), y[-3:].cpu()] -= 1
    g64 = k[:, None] * soft
    tol = grad_tolerance(g64, tail.double().cpu(), y[-3:].cpu(), 32 * U, k, torch.bfloat16)
    assert torch.all((g[-3:].cpu().double() - g64).abs() <= tol)
    assert not g[1:-3].any()


@pytest.mark.parametrize("dtype,V", [(torch.bfloat16, 65541), (torch.bfloat16, 65600), (torch.bfloat16, 114696),
                                     (torch.float16, 70000), (torch.float32, 33333), (torch.float32, 33336)])
@pytest.mark.parametrize("packed", [False, True])
def test_long_rows_beyond_the_cache(dev, dtype, V, packed):
    """More than 400 MB of logits in rows of 128 KB and more take statistics and gradient of a row together: against
    the two passes of the autograd form, and a few rows against 64 bits; masked rows, rows outside, odd starts."""
    n, S = 8, 410
    T = n * S
    gen = torch.Generator(dev).manual_seed(3)
    wide = (torch.randn(T, V + 3, generator=gen, device=dev) * 2).to(dtype)
    x = wide[:, 2:V + 2]  # rows start anywhere
    y = torch.randint(0, V, (T,), generator=gen, device=dev)
    y[torch.rand(T, generator=gen, device=dev) < 0.3] = IGNORE
    y[5] = V - 1
    y[6] = 0
    old = torch.randn(T, generator=gen, device=dev) * 0.3 - 13
    ref = torch.randn(T, generator=gen, device=dev) * 0.3 - 13
    cu, lead = None, (n, S)
    if packed:
        cu, lead = torch.tensor([3, 500, 500, 1200, 1201, T - 7], dtype=torch.int32, device=dev), (T,)
    adv = torch.randn(n if not packed else 5, generator=gen, device=dev)
    kw = dict(cu_seqlens=cu, kl_coef=0.05, reduction="sequence")
    args = (y.view(lead), old.view(lead), adv, ref.view(lead))
    out, g = gefen.policy_loss_and_grad(x.view(*lead, V) if packed else x.unflatten(0, lead), *args, grad_scale=4096.0, **kw)
    leaf = x.contiguous().view(*lead, V).requires_grad_(True)
    two = gefen.policy_loss(leaf, *args, **kw)
    (two.loss * 4096.0).backward()
    x64 = x[:64].double().cpu()
    tol = logp_tolerance(x64, y[:64].cpu()).max().item()  # per row; about the same in all
    assert (out.logps - two.logps).abs().max().item() <= 2 * tol
    for a, b in ((out.loss, two.loss), (out.kl, two.kl)):
        assert abs(a.item() - b.item()) <= 1e-5 * (1 + abs(b.item()))
    assert abs(out.clip_fraction.item() - two.clip_fraction.item()) <= 2.0 / T
    off = (y.view(lead) == IGNORE).view(T)
    if packed:
        off[:3] = off[-7:] = True
    g, h = g.view(T, V), leaf.grad.view(T, V)
    assert not g[off].any() and not h[off].any()
    # ratios grow with the errors of logp: relative 4 tol, and one rounding of either; a token at the clip's edge may part
    near = (g.float() - h.float()).abs() <= (4 * tol + 2.02 * UNIT[dtype]) * h.float().abs() + 2 * LEAST[dtype]
    assert (~near.all(1)).sum().item() <= 1
    again, g2 = gefen.policy_loss_and_grad(x.view(*lead, V) if packed else x.unflatten(0, lead), *args, grad_scale=4096.0, **kw)
    assert torch.equal(out.loss, again.loss) and torch.equal(g, g2.view(T, V))
    keep = (~off[:64]).nonzero().view(-1)[:8].cpu()
    lp = logps64(x64, y[:64].cpu())[keep]
    assert torch.all((out.logps.view(T)[keep].cpu().double() - lp).abs() <= tol)


def test_long_rows_of_bad_values(dev):
    V, T = 66000, 3300
    x = torch.randn(T, V, device=dev).bfloat16()
    y = torch.randint(0, V, (T,), device=dev)
    y[7], y[8], y[9] = V, -1, IGNORE
    x[9] = float("nan")
    x[10, 5] = float("nan")
    x[11, :60000] = -float("inf")
    y[11] = 65000
    old = torch.full((T,), -11.0, device=dev)
    cu = torch.tensor([0, T], dtype=torch.int32, device=dev)
    out, g = gefen.policy_loss_and_grad(x, y, old, torch.ones(T, device=dev), cu_seqlens=cu, clip_high=1e9)
    bad = torch.isnan(g).all(1)
    assert bad.nonzero().view(-1).tolist() == [7, 8, 10] and torch.isnan(out.loss)
    assert not torch.isnan(g[~bad]).any() and not g[9].any() and not g[11, :60000].any() and g[11, 65000] != 0


def test_refusals(dev):
    x, y = torch.zeros(4, 6, 50, device=dev), torch.zeros(4, 6, dtype=torch.long, device=dev)
    z = torch.zeros(4, 6, device=dev)
    cu = torch.tensor([0, 3, 6], dtype=torch.int32, device=dev)
    with pytest.raises(NotImplementedError):
        gefen.token_logps(x.double(), y)
    for bad in (y.int(), y[:, :5], y.cpu()):
        with pytest.raises(ValueError, match="labels"):
            gefen.token_logps(x, bad)
    with pytest.raises(ValueError, match="vocabulary"):
        gefen.token_logps(x[..., :0], y)
    with pytest.raises(ValueError, match="pairs"):
        gefen.preference_loss(x[:3], y[:3])
    with pytest.raises(ValueError, match="sequences, tokens, vocab"):
        gefen.preference_loss(x[0], y[0])
    with pytest.raises(ValueError, match="cu_seqlens"):
        gefen.preference_loss(x, y, cu_seqlens=cu)
    for bad in (cu.float(), cu[:1], cu.cpu(), cu[None]):
        with pytest.raises(ValueError, match="cu_seqlens"):
            gefen.preference_loss(x[0], y[0], cu_seqlens=bad)
    for ref in (z[:, :5], z.cpu(), y, 3.0):
        with pytest.raises(ValueError, match="ref_logps"):
            gefen.preference_loss(x, y, ref)
    for kw in ({"beta": float("inf")}, {"beta": float("nan")}, {"label_smoothing": 0.5}, {"label_smoothing": -0.1}):
        with pytest.raises(ValueError):
            gefen.preference_loss(x, y, z, **kw)
    for kw in ({"clip_low": 1.0}, {"clip_low": -0.1}, {"clip_high": -0.1}, {"clip_high": float("nan")}, {"reduction": "mean"},
               {"kl_coef": float("nan")}, {"kl_coef": 0.1}):
        with pytest.raises(ValueError):
            gefen.policy_loss(x, y, z, z, **kw)
    for adv in (z[0], z[:3, 0], None, 1.0, y):
        with pytest.raises(ValueError, match="advantages"):
            gefen.policy_loss(x, y, z, adv)
    with pytest.raises(ValueError, match="old_logps"):
        gefen.policy_loss(x, y, None, z)
    for scale in (torch.ones(2, device=dev), torch.ones(())):
        with pytest.raises(ValueError, match="grad_scale"):
            gefen.policy_loss_and_grad(x, y, z, z, grad_scale=scale)
