"""The operators of a fine-tuning step that are timed: the loss over the logits with its gradient, and AdamW.

A case names an operator ("op") and its sizes:

  adamw        one AdamW step over a set of tensors ("shapes"), moments in 32 or 8 bits ("bits"), parameters and
               gradients of "dtype"; "clip": by the global gradient norm; "views": every n-th matrix is a
               transposed view, parameter and gradient alike (0: none); resumed in the middle of a run
  preference   the loss of "pairs" chosen / rejected answers of up to "tokens" tokens over "vocab" logits, and the
               gradient of the logits; "average": log ratios per token instead of summed
  policy       the clipped policy loss with a KL term of "seqs" sampled answers, and the gradient of the logits;
               "reduction": mean over tokens or over sequences; "advantages": one per "token" or per "sequence"

Both losses: "packed": the sequences lie one after another in [T, vocab], else padded in [N, tokens, vocab];
"call": "autograd" (loss, then backward()) or "fused" (loss and gradient in one call); "empty": one sequence
has no token to learn from.  Prompts and padding are masked.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LR, BETA1, BETA2, EPS, WD, STEP, CLIP = 6e-5, 0.9, 0.999, 1e-8, 0.01, 100, 1.0
BETA, SMOOTHING = 0.1, 0.05
CLIP_LOW, CLIP_HIGH, KL_COEF = 0.2, 0.28, 0.04
IGNORE = -100
SCALES = {"f32": 1.0, "f16": 4096.0, "bf16": 1.0}  # of the loss, as mixed-precision training sets it
BLOCK = 256             # elements per scale of the 8-bit moments
TINY = 2.0 ** -126      # smallest scale
GOLDEN, MIX1, MIX2 = 0x9E3779B97F4A7C15, 0xBF58476D1CE4E5B9, 0x94D049BB133111EB
SEED = 1234             # of the optimizer's stochastic rounding

ADAMW = {"op": "adamw", "bits": 32, "dtype": "bf16", "clip": False, "views": 0}
PREFERENCE = {"op": "preference", "dtype": "bf16", "packed": False, "call": "autograd", "average": False, "empty": False}
POLICY = {"op": "policy", "dtype": "bf16", "packed": False, "call": "fused", "reduction": "token",
          "advantages": "sequence", "empty": False}

# one decoder layer of the Llama-3-8B set: q, k, v, o, gate, up, down and two norms
LLAMA_LAYER = "4096x4096,1024x4096,1024x4096,4096x4096,14336x4096,14336x4096,4096x14336,4096,4096"
ADAPTERS = "16x768,768x16,16x768,768x16,768,10x768,10"
RAGGED = "50257x768,1023x768,769x2305,3001x1000,1000,2305,777"


def listed():
    return [
        # a few low-rank adapter pairs, clipped: the smallest step there is
        dict(ADAMW, name="adamw_adapters_f32", shapes=ADAPTERS, dtype="f32", clip=True),
        # a decoder layer's full fine-tuning step, clipped
        dict(ADAMW, name="adamw_llama_layer_bf16", shapes=LLAMA_LAYER, clip=True),
        # sizes that are multiples of nothing, half of the matrices held transposed
        dict(ADAMW, name="adamw_ragged_f16", shapes=RAGGED, dtype="f16", views=2),
        # 8-bit moments: the adapters, the layer, and embedding and head of the Llama-3-8B set (the largest step)
        dict(ADAMW, name="adamw8_adapters_f32", bits=8, shapes=ADAPTERS, dtype="f32"),
        dict(ADAMW, name="adamw8_llama_layer_bf16", bits=8, shapes=LLAMA_LAYER),
        dict(ADAMW, name="adamw8_embeddings_bf16", bits=8, shapes="128256x4096,128256x4096,4096"),
        # two short pairs of a small model in fp32: launches count
        dict(PREFERENCE, name="preference_small_f32", pairs=2, tokens=48, vocab=8000, dtype="f32"),
        # packed pairs of odd lengths, an odd vocabulary, one answer masked as a whole
        dict(PREFERENCE, name="preference_packed_f16", pairs=6, tokens=333, vocab=50257, dtype="f16", packed=True,
             average=True, empty=True),
        # a micro batch of long answers over the Llama-3-8B vocabulary
        dict(PREFERENCE, name="preference_llama_bf16", pairs=4, tokens=1024, vocab=128256, call="fused"),
        # few tokens of a large vocabulary: the work has to be split along the rows
        dict(POLICY, name="policy_few_tokens_bf16", seqs=2, tokens=24, vocab=128256),
        # packed answers, odd sizes, advantages per token, sequences weighted alike, through autograd
        dict(POLICY, name="policy_packed_f32", seqs=7, tokens=401, vocab=50257, dtype="f32", packed=True,
             call="autograd", reduction="sequence", advantages="token", empty=True),
        # a group of long samples over the Qwen3-4B vocabulary: the largest loss
        dict(POLICY, name="policy_qwen_bf16", seqs=8, tokens=2048, vocab=151936),
    ]


def _log_uniform(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(64, n // 64 * 64) if n >= 96 and rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["adamw", "adamw8", "preference", "policy"])
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    if op.startswith("adamw"):
        mats = []
        for _ in range(rng.randint(1, 4)):
            total = math.exp(rng.uniform(math.log(4096), math.log(1 << 27)))
            c = _log_uniform(rng, max(16, total / 131072), min(16384, total / 16))
            mats.append((max(16, int(total / c)), c))
        shapes = ",".join(["%dx%d" % m for m in mats] + ["%d" % c for _, c in mats[:rng.randint(0, 2)]])
        bits = 8 if op == "adamw8" else 32
        return dict(ADAMW, bits=bits, shapes=shapes, dtype=dtype, clip=bits == 32 and rng.random() < 0.5,
                    views=rng.choice([0, 0, 2]))
    vocab = _log_uniform(rng, 1000, 151936)
    seqs = rng.randint(1, 8)
    most = min(2048, (1 << 30) // (2 * seqs * vocab))  # logits of a drawn case: up to 2^30
    tokens = _log_uniform(rng, 8, max(9, most))
    shared = {"tokens": tokens, "vocab": vocab, "dtype": dtype, "packed": rng.random() < 0.5, "empty": rng.random() < 0.3,
              "call": rng.choice(["autograd", "fused"])}
    if op == "preference":
        return dict(PREFERENCE, pairs=seqs, average=rng.random() < 0.4, **shared)
    return dict(POLICY, seqs=2 * seqs, reduction=rng.choice(["token", "sequence"]),
                advantages=rng.choice(["token", "sequence"]), **shared)


# ------------------------------------------------------------------ inputs
def _shapes(case):
    return [tuple(int(n) for n in s.split("x")) for s in case["shapes"].split(",")]


def _lengths(case):
    """(prompt, whole) tokens of each sequence, by the case alone.  Padded: of `tokens`; packed: one after another."""
    n, S = (2 * case["pairs"] if case["op"] == "preference" else case["seqs"]), case["tokens"]
    r = random.Random("%d %d %d" % (n, S, case["vocab"]))
    got = []
    for i in range(n):
        whole = S if i == 0 else r.randint(S // 2, S)
        prompt = max(1, whole // 4)
        got.append((whole if case["empty"] and i == n - 1 else prompt, whole))
    return got


def _moments(shape, g, dtype, dev):
    """Gradient and moments of the middle of a run: rows of unlike scale, some rows that no batch has touched."""
    gen = torch.randn(shape, generator=g, device=dev)
    row = torch.exp(1.5 * torch.randn(shape[:1] + (1,) * (len(shape) - 1), generator=g, device=dev)) * 1e-3
    grad = (gen * row).to(dtype)
    m = torch.randn(shape, generator=g, device=dev) * row * 0.3
    v = (row * row) * torch.rand(shape, generator=g, device=dev).mul_(1.5).add_(0.1)
    if len(shape) > 1:
        idle = torch.rand(shape[:1] + (1,), generator=g, device=dev) < 0.02
        m, v, grad = (torch.where(idle, torch.zeros_like(t), t) for t in (m, v, grad))
    return grad, m, v


def _prepare_adamw(case, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"p": [], "g": [], "m": [], "v": [], "ms": [], "vs": []}
    mats = 0
    for shape in _shapes(case):
        mats += len(shape) == 2
        turned = case["views"] and len(shape) == 2 and mats % case["views"] == 0
        held = shape[::-1] if turned else shape
        p = (torch.randn(held, generator=g, device=dev) * 0.02).to(dtype)
        grad, m, v = _moments(held, g, dtype, dev)
        if case["bits"] == 8:
            m, ms = _encode_m(m.reshape(-1))
            v, vs = _encode_v(v.reshape(-1), torch.full((1,), 1 << 15, device=dev).expand(v.numel()))
            s["ms"].append(ms)
            s["vs"].append(vs)
        s["p"].append(p.t() if turned else p)
        s["g"].append(grad.t() if turned else grad)
        s["m"].append(m.t() if turned and case["bits"] == 32 else m)
        s["v"].append(v.t() if turned and case["bits"] == 32 else v)
    s["step"] = STEP
    if own:
        gefen = _gefen()
        params = [torch.nn.Parameter(p) for p in s["p"]]
        opt = gefen.AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=WD, state_bits=case["bits"],
                          max_grad_norm=CLIP if case["clip"] else None, seed=SEED)
        state = {}
        for i in range(len(params)):
            state[i] = {"step": STEP, "exp_avg": s["m"][i], "exp_avg_sq": s["v"][i]}
            if case["bits"] == 8:
                state[i].update(exp_avg_scale=s["ms"][i], exp_avg_sq_scale=s["vs"][i])
        opt.load_state_dict({"state": state, "param_groups": opt.state_dict()["param_groups"]})
        for p, grad in zip(params, s["g"]):
            p.grad = grad
        return {"case": case, "opt": opt, "params": params}
    return dict(s, case=case)


def _prepare_loss(case, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    lengths = _lengths(case)
    n, V = len(lengths), case["vocab"]
    dtype = DTYPES[case["dtype"]]
    starts = [0]
    for _, whole in lengths:
        starts.append(starts[-1] + whole)
    rows = starts[-1] if case["packed"] else n * case["tokens"]
    labels = torch.full((rows,), IGNORE, dtype=torch.long, device=dev)
    seq = torch.zeros(rows, dtype=torch.long, device=dev)
    for i, (prompt, whole) in enumerate(lengths):
        at = starts[i] if case["packed"] else i * case["tokens"]
        end = at + (whole if case["packed"] else case["tokens"])
        seq[at:end] = i
        labels[at + prompt:at + whole] = torch.randint(0, V, (whole - prompt,), generator=g, device=dev)
    logits = torch.empty(rows, V, dtype=dtype, device=dev)
    step = max(1, (1 << 28) // V)
    logps = torch.zeros(rows, device=dev)
    for a in range(0, rows, step):  # a trained model: the label stands out
        x = torch.randn(min(step, rows - a), V, generator=g, device=dev).mul_(2.0)
        y = labels[a:a + step].clamp(min=0)
        k = torch.arange(y.numel(), device=dev)
        x[k, y] += math.log(V) + 1.0 + torch.randn(y.numel(), generator=g, device=dev)
        logits[a:a + step] = x.to(dtype)
        x = logits[a:a + step].float()
        logps[a:a + step] = x[k, y] - x.logsumexp(-1)
    valid = labels != IGNORE
    noise = lambda scale: torch.randn(rows, generator=g, device=dev) * scale  # noqa: E731
    s = {"case": case, "seq": seq, "n": n}
    if case["op"] == "preference":
        # the trained policy has moved from the reference: up on chosen answers, down on rejected ones
        side = torch.where(torch.arange(n, device=dev) < n // 2, 1.0, -1.0)
        count = torch.tensor([float(max(1, w - q)) for q, w in lengths], device=dev)
        drift = side * (torch.rand(n, generator=g, device=dev) * 10 + 5) / (1.0 if case["average"] else count)
        s["ref"] = (logps - drift[seq] + noise(0.05)) * valid
    else:
        # ratios on both sides of the clip's edges, none within 1% of one, where two right programs may part
        d = noise(0.15)
        for edge in (math.log(1 - CLIP_LOW), math.log(1 + CLIP_HIGH)):
            d = torch.where((d - edge).abs() < 0.01, d + 0.03 * (1 if edge > 0 else -1), d)
        s["old"] = (logps - d) * valid
        s["ref"] = (logps + noise(0.1)) * valid
        if case["advantages"] == "token":
            s["adv"] = noise(1.0) + 0.2
        else:
            s["adv"] = torch.randn(n, generator=g, device=dev) + 0.2
    lead = (rows,) if case["packed"] else (n, case["tokens"])
    for k in ("ref", "old"):
        if k in s:
            s[k] = s[k].view(lead)
    if case["op"] == "policy" and case["advantages"] == "token":
        s["adv"] = s["adv"].view(lead)
    s["labels"] = labels.view(lead)
    s["logits"] = logits.view(*lead, V)
    s["cu"] = torch.tensor(starts, dtype=torch.int32, device=dev) if case["packed"] else None
    if own and case["call"] == "autograd":
        s["logits"].requires_grad_(True)
    return s


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    return (_prepare_adamw if case["op"] == "adamw" else _prepare_loss)(case, seed, dev)


# ------------------------------------------------------------------ the operators in their plain form
def _blocks(flat):
    pad = -flat.numel() % BLOCK
    return torch.nn.functional.pad(flat, (0, pad)).view(-1, BLOCK)


def _encode_m(m):
    """(E4M3 codes, scale of each block): the block's largest magnitude is 448 scales, nearest even."""
    b = _blocks(m)
    amax = b.abs().amax(1)
    scale = torch.where(torch.isfinite(amax), (amax / 448.0).clamp(min=TINY), amax * math.nan)
    code = (b * (1.0 / scale)[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return code.view(-1)[:m.numel()], scale


def _encode_v(v, bits16):
    """(codes, scale of each block): 5 exponent and 3 mantissa bits below the block's largest value, code 0 for zero
    alone; rounded up where the cut bits and the 16 random ones carry."""
    b = _blocks(v)
    amax = b.amax(1)
    scale = torch.where(torch.isfinite(amax), amax.clamp(min=TINY), amax * math.nan)
    x = (b * (1.0 / scale)[:, None]).view(-1)[:v.numel()].contiguous()
    code = ((x.view(torch.int32).long() + (bits16[:v.numel()].long() << 4)) >> 20) - 761
    return torch.where(v == 0, torch.zeros_like(code), code.clamp(1, 255)).to(torch.uint8), scale


def _decode_m(code, scale):
    return (_blocks(code.float()) * scale[:, None]).view(-1)[:code.numel()]


def _decode_v(code, scale):
    c = code.int()
    x = torch.where(c == 0, torch.zeros_like(c), (c + 761) << 20).view(torch.float32)
    return (_blocks(x) * scale[:, None]).view(-1)[:code.numel()]


def _signed(x):
    x &= (1 << 64) - 1
    return x - (1 << 64) if x >> 63 else x


def _mix(z):
    """SplitMix64's finalizer of a Python integer."""
    z &= (1 << 64) - 1
    z = (z ^ (z >> 30)) * MIX1 & ((1 << 64) - 1)
    z = (z ^ (z >> 27)) * MIX2 & ((1 << 64) - 1)
    return z ^ (z >> 31)


def _random16(index, step, n, dev):
    """16 random bits for each element of tensor `index` at `step`: four to a draw of the counter generator."""
    key = _mix(_mix(SEED + GOLDEN * (index + 1)) + GOLDEN * step)
    shr = lambda t, k: (t >> k) & ((1 << (64 - k)) - 1)  # noqa: E731
    z = (torch.arange(-(-n // 4), device=dev) + 1) * _signed(GOLDEN) + _signed(key)
    z = (z ^ shr(z, 30)) * _signed(MIX1)
    z = (z ^ shr(z, 27)) * _signed(MIX2)
    z = z ^ shr(z, 31)
    return ((z[:, None] >> torch.tensor([0, 16, 32, 48], device=dev)) & 0xFFFF).view(-1)


def _held(t):
    """A tensor's elements in the order it is stored in (itself, or transposed)."""
    return t.reshape(-1) if t.is_contiguous() else t.t().reshape(-1)


def _run_adamw(s):
    case = s["case"]
    s["step"] += 1
    bc1, bc2 = 1 - BETA1 ** s["step"], 1 - BETA2 ** s["step"]
    coef = None
    if case["clip"]:
        norm = torch.stack([g.float().square().sum() for g in s["g"]]).sum().sqrt()
        coef = (CLIP / (norm + 1e-6)).clamp(max=1.0)
    out = {"p": s["p"], "m": [], "v": []}
    if case["clip"]:
        out["norm"] = norm
    for i, (p, grad) in enumerate(zip(s["p"], s["g"])):
        g = grad.float() if coef is None else grad.float() * coef
        if case["bits"] == 8:
            g = _held(g)
            m, v = _decode_m(s["m"][i], s["ms"][i]), _decode_v(s["v"][i], s["vs"][i])
        else:
            m, v = s["m"][i], s["v"][i]
        m = m * BETA1 + g * (1 - BETA1)
        v = v * BETA2 + g * g * (1 - BETA2)
        update = m / (v.sqrt() / math.sqrt(bc2) + EPS)
        if case["bits"] == 8:
            update = update.view(p.shape) if p.is_contiguous() else update.view(p.t().shape).t()
            s["m"][i], s["ms"][i] = _encode_m(m)
            s["v"][i], s["vs"][i] = _encode_v(v, _random16(i, s["step"], v.numel(), v.device))
            m, v = _decode_m(s["m"][i], s["ms"][i]), _decode_v(s["v"][i], s["vs"][i])
        else:
            s["m"][i], s["v"][i] = m, v
        p.copy_((p.float() * (1 - LR * WD) - update * (LR / bc1)).to(p.dtype))
        out["m"].append(m)
        out["v"].append(v)
    return out


def _per_sequence(x, seq, n):
    """Sums of the rows of each sequence."""
    return torch.where(seq[None, :] == torch.arange(n, device=x.device)[:, None], x[None, :], torch.zeros_like(x)).sum(1)


def _run_loss(s):
    case, seq, n = s["case"], s["seq"], s["n"]
    labels = s["labels"].reshape(-1)
    x = s["logits"].detach().reshape(labels.numel(), -1).float()
    valid = labels != IGNORE
    row, at = torch.arange(labels.numel(), device=x.device), labels.clamp(min=0)
    x = x - x.amax(1, keepdim=True)
    picked = x[row, at]
    x = x.exp()
    total = x.sum(1)
    zero = torch.zeros_like(total)
    logps = torch.where(valid, picked - total.log(), zero)
    count = _per_sequence(valid.float(), seq, n)
    out = {"logps": logps.view(s["labels"].shape)}
    if case["op"] == "preference":
        ratio = _per_sequence(torch.where(valid, logps - s["ref"].reshape(-1), zero), seq, n)
        weight = 1.0 / count.clamp(min=1.0) if case["average"] else torch.ones_like(count)
        reward = BETA * ratio * weight
        h = reward[:n // 2] - reward[n // 2:]
        log_sigmoid = lambda t: t.clamp(max=0) - (-t.abs()).exp().log1p()  # noqa: E731
        out["loss"] = (-(1 - SMOOTHING) * log_sigmoid(h) - SMOOTHING * log_sigmoid(-h)).mean()
        out["chosen_rewards"], out["rejected_rewards"] = reward[:n // 2], reward[n // 2:]
        k = BETA * (1.0 / (1.0 + (-h).exp()) - (1 - SMOOTHING)) / (n // 2)
        k = (torch.cat([k, -k]) * weight)[seq]
    else:
        tokens = count.sum().clamp(min=1.0)
        if case["reduction"] == "token":
            weight = (1.0 / tokens).expand(n)
        else:
            weight = 1.0 / (count.clamp(min=1.0) * (count > 0).float().sum().clamp(min=1.0))
        weight = weight[seq]
        adv = s["adv"].reshape(-1) if case["advantages"] == "token" else s["adv"][seq]
        r = (logps - s["old"].reshape(-1)).exp()
        d = s["ref"].reshape(-1) - logps
        plain, clipped = r * adv, r.clamp(1 - CLIP_LOW, 1 + CLIP_HIGH) * adv
        kl = d.expm1() - d
        each = KL_COEF * kl - torch.minimum(plain, clipped)
        out["loss"] = torch.where(valid, each * weight, zero).sum()
        out["kl"] = torch.where(valid, kl, zero).sum() / tokens
        out["clip_fraction"] = torch.where(valid & (clipped < plain), torch.ones_like(zero), zero).sum() / tokens
        k = weight * (torch.where(plain <= clipped, -plain, zero) - KL_COEF * d.expm1())
    k = torch.where(valid, k * SCALES[case["dtype"]], zero)
    grad = x * (-k / total)[:, None]
    grad[row, at] += k
    grad = torch.where(valid[:, None], grad, torch.zeros_like(zero)[:, None])
    out["grad"] = grad.to(s["logits"].dtype).view(s["logits"].shape)
    return out


# ------------------------------------------------------------------ the framework's operators
def _gefen():
    path = os.path.join(os.getcwd(), "gefen-x_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import gefen
    return gefen


def _own_adamw(s):
    opt = s["opt"]
    opt.step()
    moments = opt.moments(s["params"])
    out = {"p": [p.detach() for p in s["params"]], "m": [m for m, _ in moments], "v": [v for _, v in moments]}
    if s["case"]["clip"]:
        out["norm"] = opt.grad_norm
    return out


def _own_loss(s):
    gefen, case = _gefen(), s["case"]
    scale = SCALES[case["dtype"]]
    if case["op"] == "preference":
        args = (s["logits"], s["labels"], s["ref"])
        kw = dict(cu_seqlens=s["cu"], beta=BETA, label_smoothing=SMOOTHING, average=case["average"], ignore_index=IGNORE)
        call, fused = gefen.preference_loss, gefen.preference_loss_and_grad
    else:
        args = (s["logits"], s["labels"], s["old"], s["adv"], s["ref"])
        kw = dict(cu_seqlens=s["cu"], clip_low=CLIP_LOW, clip_high=CLIP_HIGH, kl_coef=KL_COEF, reduction=case["reduction"],
                  ignore_index=IGNORE)
        call, fused = gefen.policy_loss, gefen.policy_loss_and_grad
    if case["call"] == "fused":
        got, grad = fused(*args, grad_scale=scale, **kw)
    else:
        s["logits"].grad = None
        got = call(*args, **kw)
        (got.loss if scale == 1.0 else got.loss * scale).backward()
        grad = s["logits"].grad
    return dict({k: v.detach() for k, v in got._asdict().items()}, grad=grad)


def run(s):
    if own:
        return (_own_adamw if s["case"]["op"] == "adamw" else _own_loss)(s)
    return (_run_adamw if s["case"]["op"] == "adamw" else _run_loss)(s)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case))
        blocks = sum(-(-math.prod(s) // BLOCK) for s in _shapes(case))
        # parameter in and out, gradient in; moments in and out; 8 bits: their scales, and their values handed out
        state = 16 * n if case["bits"] == 32 else 4 * n + 16 * blocks + 8 * n
        return {"bytes": 3 * size * n + state, "flops": 15 * n}
    lengths = _lengths(case)
    rows = sum(w for _, w in lengths) if case["packed"] else len(lengths) * case["tokens"]
    learned = sum(w - q for q, w in lengths)
    # logits of the rows with a token in, gradient of all rows out; label and a few numbers for each row
    return {"bytes": (learned + rows) * case["vocab"] * size + rows * 24, "flops": 8 * learned * case["vocab"]}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_m(m):
    b = _blocks(m)
    scale = (b.abs().amax(1, keepdim=True) / 448.0).clamp(min=TINY)
    x = b / scale
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -20))).clamp(min=-6.0)  # below 2^-6: steps of 2^-9
    unit = torch.exp2(e - 3.0)
    return (torch.round(x / unit) * unit * scale).view(-1)[:m.numel()]


def _exact_v(v, bits16):
    b = _blocks(v)
    scale = b.amax(1, keepdim=True).clamp(min=TINY)
    frac, e = torch.frexp(b / scale)  # frac in [0.5, 1)
    place = (e.double() - 1.0) * 8.0 + (frac * 2.0 - 1.0) * 8.0 + 255.0  # in codes
    place = place.view(-1)[:v.numel()] + bits16[:v.numel()].double() / 65536.0
    code = torch.where(v == 0, torch.zeros_like(v), torch.floor(place).clamp(1, 255))
    up = code - 255.0
    e = torch.floor(up / 8.0)
    x = torch.where(v == 0, torch.zeros_like(v), torch.exp2(e) * (1.0 + (up - 8.0 * e) / 8.0))
    return (_blocks(x) * scale).view(-1)[:v.numel()]


def _exact_adamw(case, seed, dev):
    s = _prepare_adamw(case, seed, dev)
    t = STEP + 1
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in s["g"]))
    coef = min(1.0, CLIP / (norm + 1e-6)) if case["clip"] else 1.0
    out = {"p": [], "m": [], "v": []}
    if case["clip"]:
        out["norm"] = norm
    for i, (p, g) in enumerate(zip(s["p"], s["g"])):
        g = g.double() * coef
        if case["bits"] == 8:
            g = _held(g)
            m, v = _decode_m(s["m"][i], s["ms"][i]).double(), _decode_v(s["v"][i], s["vs"][i]).double()
        else:
            m, v = s["m"][i].double(), s["v"][i].double()
        m = BETA1 * m + (1 - BETA1) * g
        v = BETA2 * v + (1 - BETA2) * g ** 2
        step = LR / (1 - BETA1 ** t) * m / ((v / (1 - BETA2 ** t)) ** 0.5 + EPS)
        if case["bits"] == 8:
            step = step.view(p.shape) if p.is_contiguous() else step.view(p.t().shape).t()
            m, v = _exact_m(m), _exact_v(v, _random16(i, t, v.numel(), dev))
        out["p"].append(p.double() - LR * WD * p.double() - step)
        out["m"].append(m)
        out["v"].append(v)
    return out


def _exact_loss(case, seed, dev):
    s = _prepare_loss(case, seed, dev)
    lead = s["labels"].shape
    labels, seq, n = s["labels"].reshape(-1), s["seq"].cpu(), s["n"]
    logits = s["logits"].detach().reshape(labels.numel(), -1)
    keep = (labels != IGNORE).nonzero().view(-1)
    where = seq[keep.cpu()]
    lse = torch.zeros(labels.numel(), dtype=torch.float64, device=dev)
    step = max(1, (1 << 28) // case["vocab"])
    for a in range(0, keep.numel(), step):
        lse[keep[a:a + step]] = torch.logsumexp(logits[keep[a:a + step]].double(), 1)
    lp = (logits[keep, labels[keep]].double() - lse[keep]).cpu()
    pick = lambda t: t.reshape(-1)[keep].double().cpu()  # noqa: E731
    count = torch.bincount(where, minlength=n).double()
    out = {}
    if case["op"] == "preference":
        d = torch.zeros(n, dtype=torch.float64).index_add_(0, where, lp - pick(s["ref"]))
        scale = BETA / (count.clamp(min=1) if case["average"] else torch.ones(n, dtype=torch.float64))
        d = (d * scale).requires_grad_(True)
        h = d[:n // 2] - d[n // 2:]
        sig = torch.nn.functional.logsigmoid
        loss = -((1 - SMOOTHING) * sig(h) + SMOOTHING * sig(-h)).mean()
        loss.backward()
        k = (d.grad * scale)[where]
        out["chosen_rewards"], out["rejected_rewards"] = d.detach()[:n // 2], d.detach()[n // 2:]
    else:
        l = lp.clone().requires_grad_(True)
        adv = pick(s["adv"]) if case["advantages"] == "token" else s["adv"].double().cpu()[where]
        r = torch.exp(l - pick(s["old"]))
        edge = torch.where(adv >= 0, torch.full_like(adv, 1 + CLIP_HIGH), torch.full_like(adv, 1 - CLIP_LOW))
        clipped = ((r - edge) * adv > 0).detach()
        gain = torch.where(clipped, edge, r) * adv
        back = pick(s["ref"]) - l
        kl = torch.expm1(back) - back
        per = KL_COEF * kl - gain
        if case["reduction"] == "token":
            loss = per.sum() / max(1, keep.numel())
        else:
            loss = (per / count[where]).sum() / max(1.0, float((count > 0).sum()))
        loss.backward()
        k = l.grad
        out["kl"] = kl.detach().sum() / max(1, keep.numel())
        out["clip_fraction"] = clipped.double().sum() / max(1, keep.numel())
    out["loss"] = loss.detach()
    grad = torch.zeros(logits.shape, dtype=torch.float64, device=dev)
    k = k.to(dev) * SCALES[case["dtype"]]
    for a in range(0, keep.numel(), step):
        at = keep[a:a + step]
        soft = torch.exp(logits[at].double() - lse[at][:, None])
        soft[torch.arange(at.numel(), device=dev), labels[at]] -= 1.0
        grad[at] = soft.mul_(-k[a:a + step, None])
    logps = torch.zeros(labels.numel(), dtype=torch.float64, device=dev)
    logps[keep] = lp.to(dev)
    return dict(out, grad=grad.view(s["logits"].shape), logps=logps.view(lead))


def exact(case, seed):
    global own
    dev, was = torch.device("cuda", 0), own
    own = False  # the inputs alone
    try:
        return (_exact_adamw if case["op"] == "adamw" else _exact_loss)(case, seed, dev)
    finally:
        own = was
