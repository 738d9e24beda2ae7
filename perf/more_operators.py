"""Operators between the logits of two models that are timed: the statistics of tokens and distillation.

A case names an operator ("op") and its sizes:

  statistics   log-probability of the label, entropy and the "top" likeliest tokens with their log-probabilities,
               per row of logits; "call": "forward" (serving, a teacher's pass) or "train" (the gradient of the
               logits from gradients of log-probabilities, entropy and top log-probabilities too)
  distill      loss against a teacher's "top" tokens and their log-probabilities, and the gradient of the logits;
               "rest": how the teacher's other tokens count; "hard": weight of the labels' own loss;
               "reduction": mean over tokens or over sequences; "ids": type of the teacher's ids;
               "call": "autograd" (loss, then backward()) or "fused" (loss and gradient in one call)

Both: "seqs" sequences of up to "tokens" tokens over "vocab" logits at a "temperature"; "packed": one after another
in [T, vocab], else padded in [N, tokens, vocab]; "head": the logits are the first "vocab" columns of a head padded
to a multiple of 64; "prompt": the first quarter of a sequence, and padding, is masked.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
IDS = {"i32": torch.int32, "i64": torch.int64}
IGNORE = -100
SCALES = {"f32": 1.0, "f16": 4096.0, "bf16": 1.0}  # of the loss, as mixed-precision training sets it
ENTROPY_COEF = 0.01
CHUNK = 1 << 27  # logits that are prepared at a time

STATISTICS = {"op": "statistics", "dtype": "bf16", "top": 0, "temperature": 1.0, "packed": False, "head": False,
              "prompt": False, "call": "forward"}
DISTILL = {"op": "distill", "dtype": "bf16", "temperature": 1.0, "packed": False, "head": False, "prompt": True,
           "rest": "bucket", "hard": 0.0, "reduction": "token", "ids": "i64", "call": "fused"}


def listed():
    return [
        # one decoded token with its alternatives: latency counts
        dict(STATISTICS, name="statistics_token_bf16", seqs=1, tokens=1, vocab=128256, top=20),
        # a decoded token of each sequence of a serving batch
        dict(STATISTICS, name="statistics_batch_bf16", seqs=64, tokens=1, vocab=151936, top=8),
        # odd sizes, a padded head, a temperature
        dict(STATISTICS, name="statistics_ragged_f16", seqs=5, tokens=333, vocab=50257, top=5, temperature=0.7, packed=True,
             head=True, dtype="f16"),
        # a teacher's pass over whole sequences
        dict(STATISTICS, name="statistics_teacher_bf16", seqs=4, tokens=1024, vocab=128256, top=64, prompt=True),
        # policy training with an entropy term over short answers of a small vocabulary
        dict(STATISTICS, name="statistics_short_rows_f32", seqs=16, tokens=256, vocab=4096, top=0, dtype="f32", prompt=True,
             call="train"),
        # ... and over long ones of the Qwen3-4B vocabulary, the top alternatives held to a reference too
        dict(STATISTICS, name="statistics_train_bf16", seqs=4, tokens=1024, vocab=151936, top=4, prompt=True, call="train"),
        # two short sequences of a small model: launches count
        dict(DISTILL, name="distill_small_f32", seqs=4, tokens=48, vocab=8000, top=8, dtype="f32"),
        # few tokens of a large vocabulary, a temperature, labels too
        dict(DISTILL, name="distill_few_tokens_bf16", seqs=2, tokens=24, vocab=128256, top=20, temperature=2.0, hard=0.3),
        # packed, odd sizes, sequences weighted alike, through autograd
        dict(DISTILL, name="distill_packed_f16", seqs=7, tokens=333, vocab=50257, top=100, dtype="f16", packed=True, ids="i32",
             rest="normalize", reduction="sequence", call="autograd"),
        # an fp32 head with labels, without the other tokens
        dict(DISTILL, name="distill_labels_f32", seqs=6, tokens=401, vocab=32000, top=32, dtype="f32", hard=0.5, rest="drop"),
        # long sequences of the Llama-3-8B vocabulary: the largest call
        dict(DISTILL, name="distill_llama_bf16", seqs=8, tokens=1024, vocab=128256, top=64),
    ]


def _log_uniform(rng, lo, hi):
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(64, n // 64 * 64) if n >= 96 and rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["serve", "teacher", "train", "distill", "distill", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f32", "f16"])
    vocab = _log_uniform(rng, 1000, 151936)
    seqs = rng.randint(1, 8)
    size = 4 if dtype == "f32" else 2
    most = min(2048, (1 << 31) // (size * seqs * vocab))  # logits of a drawn case: up to 2 GiB
    shared = {"seqs": seqs, "vocab": vocab, "dtype": dtype, "temperature": rng.choice([1.0, 1.0, 0.7, 2.0]),
              "head": rng.random() < 0.25}
    if op == "serve":
        return dict(STATISTICS, **dict(shared, seqs=_log_uniform(rng, 1, 256)), tokens=1, top=rng.randint(0, 20))
    shared.update(tokens=_log_uniform(rng, 8, max(9, most)), packed=rng.random() < 0.5, top=_log_uniform(rng, 1, 128))
    if op == "teacher":
        return dict(STATISTICS, prompt=rng.random() < 0.5, **shared)
    if op == "train":
        return dict(STATISTICS, **dict(shared, top=rng.choice([0, 0, rng.randint(1, 20)])), prompt=True, call="train")
    return dict(DISTILL, rest=rng.choice(["bucket", "drop", "normalize"]), hard=rng.choice([0.0, 0.0, 0.3]),
                reduction=rng.choice(["token", "sequence"]), ids=rng.choice(["i32", "i64"]),
                call=rng.choice(["autograd", "fused"]), **shared)


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """(prompt, whole) tokens of each sequence, by the case alone.  Padded: of `tokens`; packed: one after another."""
    n, S = case["seqs"], case["tokens"]
    r = random.Random("%d %d %d" % (n, S, case["vocab"]))
    got = []
    for i in range(n):
        whole = S if i == 0 or not case["prompt"] else r.randint((S + 1) // 2, S)
        got.append((whole // 4 if case["prompt"] else 0, whole))
    return got


def _top(case):
    return min(case["top"], case["vocab"])


def _teacher(x, k, temperature, g):
    """The k likeliest tokens of another model near x and their log-probabilities; some rows hold fewer."""
    z = x + torch.randn(x.shape, generator=g, device=x.device)
    logp = torch.log_softmax(z.div_(temperature), -1)
    top, ids = logp.topk(k, -1)
    few = torch.rand((x.shape[0], 1), generator=g, device=x.device) < 0.05
    gone = few & (torch.arange(k, device=x.device) >= (k + 1) // 2)
    return ids.masked_fill(gone, 0), top.masked_fill(gone, -math.inf)


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    g = torch.Generator(device=dev).manual_seed(seed)
    lengths = _lengths(case)
    n, V, k, temperature = len(lengths), case["vocab"], _top(case), case["temperature"]
    dtype = DTYPES[case["dtype"]]
    starts = [0]
    for _, whole in lengths:
        starts.append(starts[-1] + whole)
    rows = starts[-1] if case["packed"] else n * case["tokens"]
    labels = torch.full((rows,), IGNORE, dtype=torch.long, device=dev)
    seq = torch.zeros(rows, dtype=torch.long, device=dev)
    for i, (prompt, whole) in enumerate(lengths):
        at = starts[i] if case["packed"] else i * case["tokens"]
        seq[at:at + (whole if case["packed"] else case["tokens"])] = i
        labels[at + prompt:at + whole] = torch.randint(0, V, (whole - prompt,), generator=g, device=dev)
    held = torch.empty(rows, -(-V // 64) * 64 if case["head"] else V, dtype=dtype, device=dev)
    logits = held[:, :V]
    if case["head"]:
        held[:, V:] = 0
    ids = torch.zeros(rows, k, dtype=torch.long, device=dev)
    teacher = torch.zeros(rows, k, device=dev)
    step = max(1, CHUNK // V)
    for a in range(0, rows, step):  # a trained model: the label stands out
        x = torch.randn(min(step, rows - a), V, generator=g, device=dev).mul_(2.0)
        y = labels[a:a + step].clamp(min=0)
        row = torch.arange(y.numel(), device=dev)
        x[row, y] += math.log(V) + 1.0 + torch.randn(y.numel(), generator=g, device=dev)
        logits[a:a + step] = x.to(dtype)
        if case["op"] == "distill":
            ids[a:a + step], teacher[a:a + step] = _teacher(x, k, temperature, g)
    lead = (rows,) if case["packed"] else (n, case["tokens"])
    s = {"case": case, "seq": seq, "n": n, "labels": labels.view(lead), "logits": logits.view(*lead, V)}
    s["cu"] = torch.tensor(starts, dtype=torch.int32, device=dev) if case["packed"] else None
    if case["op"] == "distill":
        s["ids"], s["teacher"] = ids.view(*lead, k).to(IDS[case["ids"]]), teacher.view(*lead, k)
        training = case["call"] == "autograd"
    else:
        training = case["call"] == "train"
        if training:  # of a loss over advantages with an entropy term; the top tokens' held to a reference
            scale = SCALES[case["dtype"]] / rows
            s["up"] = [torch.randn(lead, generator=g, device=dev) * scale,
                       torch.full(lead, -ENTROPY_COEF * scale, device=dev)]
            if k:
                s["up"].append(torch.randn((*lead, k), generator=g, device=dev) * (0.1 * scale))
    if own and training:
        s["logits"].requires_grad_(True)
    return s


# ------------------------------------------------------------------ the operators in their plain form
def _ordered(x):
    """Whole numbers in the order of the fp32 values x, equal values by falling column: largest first, no two alike."""
    bits = (x + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    V = x.shape[1]
    return bits * V + (V - 1 - torch.arange(V, device=x.device))


def _run_statistics(s):
    case = s["case"]
    labels, k, temperature = s["labels"].reshape(-1), _top(case), case["temperature"]
    lead, rows = s["labels"].shape, labels.numel()
    x = s["logits"].detach().reshape(rows, -1).float()
    valid = labels != IGNORE
    row, at = torch.arange(rows, device=x.device), labels.clamp(min=0)
    zero = torch.zeros(rows, device=x.device)
    out = {}
    if k:
        ids = x.shape[1] - 1 - _ordered(x).topk(k, -1)[0] % x.shape[1]
        out["top_ids"] = torch.where(valid[:, None], ids, torch.zeros_like(ids))
    x = x - x.amax(1, keepdim=True)
    if temperature != 1.0:
        x = x / temperature
    e = x.exp()
    total = e.sum(1)
    lse = total.log()
    logp = x - lse[:, None]
    p = e / total[:, None]
    entropy = -(p * logp).sum(1)
    out["logps"] = torch.where(valid, logp[row, at], zero).view(lead)
    out["entropy"] = torch.where(valid, entropy, zero).view(lead)
    if k:
        out["top_logps"] = torch.where(valid[:, None], logp.gather(1, ids), torch.full_like(zero, -math.inf)[:, None]).view(*lead, k)
        out["top_ids"] = out["top_ids"].view(*lead, k)
    if case["call"] == "train":
        up = [torch.where(valid.view(lead + (1,) * (u.dim() - len(lead))), u, torch.zeros_like(u)).reshape(rows, -1) for u in s["up"]]
        all_of = up[0][:, 0] + up[2].sum(1) if k else up[0][:, 0]
        grad = -p * (all_of[:, None] + up[1] * (logp + entropy[:, None]))
        grad[row, at] += up[0][:, 0]
        if k:
            grad.scatter_add_(1, ids, up[2])
        grad = grad / temperature if temperature != 1.0 else grad
        out["grad"] = torch.where(valid[:, None], grad, zero[:, None]).to(s["logits"].dtype).view(s["logits"].shape)
    return out


def _per_sequence(x, seq, n):
    """Sums of the rows of each sequence."""
    return torch.where(seq[None, :] == torch.arange(n, device=x.device)[:, None], x[None, :], torch.zeros_like(x)).sum(1)


def _run_distill(s):
    case, seq, n = s["case"], s["seq"], s["n"]
    labels, k, temperature, hard = s["labels"].reshape(-1), _top(case), case["temperature"], case["hard"]
    rows = labels.numel()
    x = s["logits"].detach().reshape(rows, -1).float()
    ids, teacher = s["ids"].reshape(rows, k).long(), s["teacher"].reshape(rows, k)
    valid = labels != IGNORE
    row, at = torch.arange(rows, device=x.device), labels.clamp(min=0)
    zero = torch.zeros(rows, device=x.device)
    x = x - x.amax(1, keepdim=True)
    nll = zero
    if hard:
        e = x.exp()
        hard_total = e.sum(1)
        nll = torch.where(valid, hard_total.log() - x[row, at], zero)
    z = x / temperature if temperature != 1.0 else x
    q = z.exp()
    total = q.sum(1)
    # a row's few numbers in 64 bits: the divergence is what is left of terms that cancel
    wide = teacher.double()
    p = wide.exp()
    held = p > 0
    z_top = z.gather(1, ids)
    log_p = torch.where(held, wide, torch.zeros_like(wide))
    mass = p.sum(1)
    if case["rest"] == "normalize":
        safe = torch.where(mass > 0, mass, torch.ones_like(mass))
        p, log_p = p / safe[:, None], log_p - safe.log()[:, None]
        mass = torch.where(mass > 0, torch.ones_like(mass), torch.zeros_like(mass))
    each = torch.where(held, p * (log_p - z_top.double() + total.double().log()[:, None]), torch.zeros_like(p)).sum(1)
    if case["rest"] == "bucket":
        # the teacher's tokens leave the sum; places that hold none point behind it
        spot = torch.where(held, ids, torch.full_like(ids, q.shape[1]))
        others = torch.cat([q, zero[:, None]], 1).scatter_(1, spot, 0.0)[:, :-1].sum(1)
        left = (1.0 - mass).clamp(min=0.0)
        known = torch.where(held, z_top.exp(), torch.zeros_like(z_top)).double().sum(1)
        log_left = torch.where(left > 0, torch.log1p(-mass.clamp(max=1.0 - 1e-16)), torch.zeros_like(left))
        each = each + left * (log_left + torch.log1p(known / others.double()))
        share, whole = left.float(), (mass + left).float()
    p, mass, each = p.float(), mass.float(), each.float()
    each = torch.where(valid, each, zero)
    count = _per_sequence(valid.float(), seq, n)
    if case["reduction"] == "token":
        weight = (1.0 / count.sum().clamp(min=1.0)).expand(n)
    else:
        weight = 1.0 / (count.clamp(min=1.0) * (count > 0).float().sum().clamp(min=1.0))
    weight = torch.where(valid, weight[seq], zero)
    out = {"token_divergence": each.view(s["labels"].shape), "divergence": (each * weight).sum(), "nll": (nll * weight).sum()}
    soft = (1.0 - hard) * temperature * temperature
    out["loss"] = soft * out["divergence"] + hard * out["nll"]
    # d divergence / d logits
    up = weight * (soft / temperature * SCALES[case["dtype"]])
    if case["rest"] == "bucket":
        grad = q * (whole / total - share / others)[:, None]
        at_top = q.gather(1, ids) * (whole / total)[:, None] - p
        grad = torch.cat([grad, zero[:, None]], 1).scatter_(1, spot, at_top)[:, :-1]
    else:
        grad = q * (mass / total)[:, None]
        grad.scatter_add_(1, ids, torch.where(held, -p, torch.zeros_like(p)))
    grad = grad * up[:, None]
    if hard:
        down = weight * (hard * SCALES[case["dtype"]])
        e *= (down / hard_total)[:, None]
        e[row, at] -= down
        grad = grad + e
    grad = torch.where(valid[:, None], grad, zero[:, None])
    out["grad"] = grad.to(s["logits"].dtype).view(s["logits"].shape)
    return out


# ------------------------------------------------------------------ the framework's operators
def _gefen():
    path = os.path.join(os.getcwd(), "gefen-x_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import gefen
    return gefen


def _own_statistics(s):
    gefen, case = _gefen(), s["case"]
    s["logits"].grad = None
    got = gefen.token_statistics(s["logits"], s["labels"], top=_top(case), temperature=case["temperature"], ignore_index=IGNORE)
    out = {"logps": got.logps, "entropy": got.entropy}
    if case["top"]:
        out.update(top_ids=got.top_ids, top_logps=got.top_logps)
    if case["call"] == "train":
        torch.autograd.backward([got.logps, got.entropy] + ([got.top_logps] if case["top"] else []), s["up"])
        out = {name: t.detach() for name, t in out.items()}
        out["grad"] = s["logits"].grad
    return out


def _own_distill(s):
    gefen, case = _gefen(), s["case"]
    scale = SCALES[case["dtype"]]
    args = (s["logits"], s["labels"], s["ids"], s["teacher"])
    kw = dict(cu_seqlens=s["cu"], temperature=case["temperature"], rest=case["rest"], hard_weight=case["hard"],
              reduction=case["reduction"], ignore_index=IGNORE)
    if case["call"] == "fused":
        got, grad = gefen.distillation_loss_and_grad(*args, grad_scale=scale, **kw)
    else:
        s["logits"].grad = None
        got = gefen.distillation_loss(*args, **kw)
        (got.loss if scale == 1.0 else got.loss * scale).backward()
        grad = s["logits"].grad
    return {"token_divergence": got.token_divergence.detach(), "divergence": got.divergence.detach(), "nll": got.nll.detach(),
            "loss": got.loss.detach(), "grad": grad}


def run(s):
    if own:
        return (_own_statistics if s["case"]["op"] == "statistics" else _own_distill)(s)
    return (_run_statistics if s["case"]["op"] == "statistics" else _run_distill)(s)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    lengths, k = _lengths(case), _top(case)
    rows = sum(w for _, w in lengths) if case["packed"] else len(lengths) * case["tokens"]
    learned = sum(w - q for q, w in lengths)
    read, whole = learned * case["vocab"], rows * case["vocab"]
    if case["op"] == "statistics":
        # logits of the rows that count; label in, log-probability, entropy and the top tokens out
        count = read * size + rows * (8 + 4 + 4 + 12 * k)
        if case["call"] == "train":  # the gradient of all rows out, what flows into it in
            return {"bytes": count + whole * size + rows * (8 + 4 * k), "flops": 14 * read}
        return {"bytes": count, "flops": 6 * read}
    entry = (4 if case["ids"] == "i32" else 8) + 4
    return {"bytes": (read + whole) * size + learned * k * entry + rows * 12, "flops": (12 if case["hard"] else 8) * read}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_statistics(case, s):
    labels, k, temperature = s["labels"].reshape(-1), _top(case), case["temperature"]
    rows, V = labels.numel(), case["vocab"]
    logits = s["logits"].detach().reshape(rows, V)
    dev = logits.device
    keep = (labels != IGNORE).nonzero().view(-1)
    logps = torch.zeros(rows, dtype=torch.float64, device=dev)
    entropy = torch.zeros_like(logps)
    top_ids = torch.zeros(rows, k, dtype=torch.long, device=dev)
    top_logps = torch.full((rows, k), -math.inf, dtype=torch.float64, device=dev)
    grad = torch.zeros(rows, V, dtype=torch.float64, device=dev) if case["call"] == "train" else None
    step = max(1, CHUNK // V)
    for a in range(0, keep.numel(), step):
        at = keep[a:a + step]
        lq = torch.log_softmax(logits[at].double() / temperature, 1)
        q = torch.softmax(logits[at].double() / temperature, 1)
        logps[at] = lq.gather(1, labels[at][:, None])[:, 0]
        entropy[at] = h = torch.special.entr(q).sum(1)
        if k:
            order = torch.sort(logits[at].double(), dim=1, descending=True, stable=True)[1][:, :k]
            top_ids[at] = order
            top_logps[at] = lq.gather(1, order)
        if grad is not None:
            gl, gh = (u.reshape(-1)[at].double()[:, None] for u in s["up"][:2])
            d = -q * gh * (lq + h[:, None])
            d.sub_(q * gl).scatter_add_(1, labels[at][:, None], gl)
            if k:
                gt = s["up"][2].reshape(rows, k)[at].double()
                d.sub_(q * gt.sum(1, keepdim=True)).scatter_add_(1, order, gt)
            grad[at] = d / temperature
    lead = s["labels"].shape
    out = {"logps": logps.view(lead), "entropy": entropy.view(lead)}
    if k:
        out.update(top_ids=top_ids.view(*lead, k), top_logps=top_logps.view(*lead, k))
    if grad is not None:
        out["grad"] = grad.view(s["logits"].shape)
    return out


def _exact_distill(case, s):
    labels, k, temperature, hard = s["labels"].reshape(-1), _top(case), case["temperature"], case["hard"]
    rows, V = labels.numel(), case["vocab"]
    logits, ids, teacher = s["logits"].detach().reshape(rows, V), s["ids"].reshape(rows, k).long(), s["teacher"].reshape(rows, k)
    dev = logits.device
    keep = (labels != IGNORE).nonzero().view(-1)
    where = s["seq"][keep]
    count = torch.bincount(where, minlength=s["n"]).double()
    if case["reduction"] == "token":
        weight = torch.full_like(where, 1, dtype=torch.float64) / max(1, keep.numel())
    else:
        weight = 1.0 / (count[where] * (count > 0).sum().double())
    each = torch.zeros(rows, dtype=torch.float64, device=dev)
    nll = torch.zeros(rows, dtype=torch.float64, device=dev)
    grad = torch.zeros(rows, V, dtype=torch.float64, device=dev)
    soft = (1.0 - hard) * temperature ** 2
    scale = SCALES[case["dtype"]]
    step = max(1, CHUNK // V)
    for a in range(0, keep.numel(), step):
        at = keep[a:a + step]
        x = logits[at].double()
        lq = torch.log_softmax(x / temperature, 1)
        # the teacher as a distribution over the vocabulary, zero where it says nothing
        p = torch.zeros_like(x).scatter_add_(1, ids[at], teacher[at].double().exp())
        mass = p.sum(1, keepdim=True)
        if case["rest"] == "normalize":
            p = p / torch.where(mass > 0, mass, 1.0)
            mass = p.sum(1, keepdim=True)
        each[at] = (torch.special.xlogy(p, p) - p * lq).sum(1)
        d = lq.exp() * mass - p
        if case["rest"] == "bucket":
            # a student's token outside of the teacher's shares the rest by its own share
            other = lq.masked_fill(p > 0, -math.inf)
            log_other = torch.logsumexp(other, 1, keepdim=True)
            left = (1.0 - mass).clamp(min=0.0)
            each[at] += (torch.special.xlogy(left, left) - left * log_other)[:, 0]
            d = lq.exp() * (mass + left) - p - left * (other - log_other).exp()
        d *= (weight[a:a + step] * (soft * scale / temperature))[:, None]
        if hard:
            l1 = torch.log_softmax(x, 1)
            nll[at] = -l1.gather(1, labels[at][:, None])[:, 0]
            down = (weight[a:a + step] * (hard * scale))[:, None]
            d += l1.exp() * down
            d.scatter_add_(1, labels[at][:, None], -down)
        grad[at] = d
    divergence, hard_loss = (each[keep] * weight).sum(), (nll[keep] * weight).sum()
    return {"token_divergence": each.view(s["labels"].shape), "divergence": divergence, "nll": hard_loss,
            "loss": soft * divergence + hard * hard_loss, "grad": grad.view(s["logits"].shape)}


def exact(case, seed):
    global own
    was, own = own, False  # the inputs alone
    try:
        s = prepare(case, seed)
        return (_exact_statistics if case["op"] == "statistics" else _exact_distill)(case, s)
    finally:
        own = was
