"""Losses over the logits of a language model, and their gradient, on the MI355X.

What a fine-tuning loop computes before the optimizer steps: the
log-probability of each label, the preference loss over pairs of answers
(paired log ratios against a reference) and the clipped policy loss with a KL
term.  The reference has no losses.  Each reads the logits in their own type,
without a copy in fp32 and without their softmax in memory, and writes their
gradient once; rows whose label is ``ignore_index`` are not read and get a zero
gradient.

Logits are [..., vocab] (last dimension of stride 1; up to two leading
dimensions of any strides are read in place) in fp32, fp16 or bf16; labels are
int64 of the leading shape, and ``logits[..., t, :]`` predicts ``labels[..., t]``
(shift the labels, not the logits).  Per-token inputs have the labels' shape,
are constants (no gradient flows into them) and are taken in fp32.  Sequences are
the rows of logits [N, S, vocab], or, with ``cu_seqlens`` (int32 [N + 1] on the
device), lie one after another in [T, vocab].  Sums over tokens are in float64.

The plain calls are differentiable in the logits.  The ``*_and_grad`` calls return
the gradient with the loss, for a training loop that feeds it to
``logits.backward(grad)``; ``grad_scale`` (a number or a device scalar, such as a
GradScaler's) multiplies it before it is rounded to the logits' type.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from gefen.gefen import _on_device, _outside_graphs
from gefen.kernels import _native

_DTYPES = {torch.float32: _native.DT_F32, torch.float16: _native.DT_F16, torch.bfloat16: _native.DT_BF16}


class PreferenceLoss(NamedTuple):
    """loss (0-dim), beta times the log ratio of each chosen and rejected
    sequence [N / 2], the labels' log-probabilities (0 where ignored)."""
    loss: torch.Tensor
    chosen_rewards: torch.Tensor
    rejected_rewards: torch.Tensor
    logps: torch.Tensor


class PolicyLoss(NamedTuple):
    """loss, mean KL estimate (0 without ref_logps) and share of clipped tokens
    (0-dim), the labels' log-probabilities (0 where ignored)."""
    loss: torch.Tensor
    kl: torch.Tensor
    clip_fraction: torch.Tensor
    logps: torch.Tensor


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(device):
    """The current stream of a device; torch.cuda.current_stream makes an object of it first, which takes 3 us."""
    if _raw_stream is None or device.type != "cuda":
        return torch.cuda.current_stream(device).cuda_stream
    return _raw_stream(device.index)


class _Call:
    """The logits of one call, checked, and the descriptor that the kernels read them by.  labelled: whether there have to
    be labels; without them every row counts."""

    def __init__(self, logits, labels, ignore_index, cu_seqlens=None, sequences=True, labelled=True):
        if not isinstance(logits, torch.Tensor) or not (isinstance(labels, torch.Tensor) or (labels is None and not labelled)):
            raise TypeError("logits and labels must be tensors")
        if logits.device.type != "cuda":
            raise ValueError("Expected logits on a HIP device, got {}".format(logits.device))
        if logits.dtype not in _DTYPES:
            raise NotImplementedError("logits of {} are not implemented (fp32, fp16, bf16)".format(logits.dtype))
        if logits.dim() < 1 or logits.shape[-1] < 1:
            raise ValueError("logits need a vocabulary dimension, got shape {}".format(tuple(logits.shape)))
        if labels is not None and (labels.dtype != torch.int64 or labels.shape != logits.shape[:-1]
                                   or labels.device != logits.device):
            raise ValueError("labels must be int64 of shape {} on {}, got {} of shape {} on {}".format(
                tuple(logits.shape[:-1]), logits.device, labels.dtype, tuple(labels.shape), labels.device))
        self.device, self.shape, self.lead, self.vocab = logits.device, logits.shape, logits.shape[:-1], logits.shape[-1]
        self.n_seq, self.cu = 0, None
        if cu_seqlens is not None:
            if logits.dim() != 2:
                raise ValueError("with cu_seqlens logits are [tokens, vocab], got shape {}".format(tuple(logits.shape)))
            if (not isinstance(cu_seqlens, torch.Tensor) or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 2
                    or cu_seqlens.dtype not in (torch.int32, torch.int64) or cu_seqlens.device != logits.device):
                raise ValueError("cu_seqlens must be int32 or int64 [sequences + 1] on {}".format(logits.device))
            self.cu = cu_seqlens.to(torch.int32).contiguous()
            self.n_seq = cu_seqlens.numel() - 1
        elif sequences:
            if logits.dim() != 3 or logits.shape[0] < 1:
                raise ValueError("logits are [sequences, tokens, vocab], or [tokens, vocab] with cu_seqlens, got shape "
                                 "{}".format(tuple(logits.shape)))
            self.n_seq = logits.shape[0]
        x, placed = logits, self._placed(logits)
        if placed is None:
            x = x.detach().contiguous()
            placed = self._placed(x)
        self.logits, self.labels = x, labels if labels is None or labels.is_contiguous() else labels.contiguous()
        self.rows = self.lead.numel()
        self.desc = _native.Logits(
            x.data_ptr(), _ptr(self.labels), None if self.cu is None else self.cu.data_ptr(), self.rows, *placed,
            self.vocab, int(ignore_index), _DTYPES[x.dtype], self.n_seq)
        self.ref = ctypes.byref(self.desc)
        self.stream = _stream(self.device)

    @staticmethod
    def _placed(x):
        """How the rows of logits lie in memory: rows of a batch, batch stride, row stride; None: not so that the
        kernels read them in place."""
        if x.stride(-1) != 1 and x.shape[-1] > 1 and x.numel() > 0:
            return None
        if x.dim() == 3:
            return max(1, x.shape[1]), x.stride(0), x.stride(1)
        if x.dim() == 2:
            return max(1, x.shape[0]), 0, x.stride(0)
        if x.dim() > 3 and not x.is_contiguous():
            return None
        return max(1, x.numel() // x.shape[-1]), 0, x.shape[-1]

    @classmethod
    def again(cls, desc, logits, labels, ignore_index, cu_seqlens=None, sequences=True, labelled=True):
        """The call of a forward pass for its backward: by its descriptor, where that says how the saved tensors lie.
        An address alone does not: copies that the forward pass made are gone, hooks may have moved the tensors and
        laid them out anew, and either may have left its address to the other."""
        fits = (desc.logits == logits.data_ptr() and desc.dtype == _DTYPES.get(logits.dtype) and desc.vocab == logits.shape[-1]
                and cls._placed(logits) == (desc.rows_per_batch, desc.batch_stride, desc.row_stride)
                and desc.rows == logits.shape[:-1].numel() and desc.labels == _ptr(labels))
        if fits and labels is not None:
            fits = labels.shape == logits.shape[:-1] and labels.dtype is torch.int64 and labels.is_contiguous()
        if fits and cu_seqlens is not None:
            fits = (desc.cu_seqlens == cu_seqlens.data_ptr() and cu_seqlens.dtype is torch.int32
                    and cu_seqlens.is_contiguous() and desc.n_seq == cu_seqlens.numel() - 1)
        if not fits:
            return cls(logits, labels, ignore_index, cu_seqlens, sequences, labelled)
        call = cls.__new__(cls)
        call.desc, call.ref = desc, ctypes.byref(desc)
        call.device, call.shape, call.lead, call.logits, call.labels = (logits.device, logits.shape, logits.shape[:-1],
                                                                        logits, labels)
        call.stream = _stream(call.device)
        return call

    def per_token(self, t, name):
        """A per-token input as the kernels read it, or None."""
        if t is None:
            return None
        if not isinstance(t, torch.Tensor) or t.shape != self.lead or t.device != self.device \
                or not t.is_floating_point():
            raise ValueError("{} must be a floating tensor of the labels' shape {} on {}, got {}".format(
                name, tuple(self.lead), self.device,
                "{} of shape {} on {}".format(t.dtype, tuple(t.shape), t.device) if isinstance(t, torch.Tensor)
                else type(t).__name__))
        return t if t.dtype is torch.float32 and t.is_contiguous() else t.detach().to(torch.float32).contiguous()

    def empty(self, *shape):
        return torch.empty(shape, dtype=torch.float32, device=self.device)

    def saved(self):
        """One buffer for what the gradient needs (row statistics [rows, 2], row coefficients [rows], sequence weights
        [n_seq]), and the pointers of the three."""
        t = torch.empty(3 * self.desc.rows + self.desc.n_seq + 1, dtype=torch.float32, device=self.device)
        return t, self.saved_ptrs(t)

    def saved_ptrs(self, t):
        at, rows = t.data_ptr(), self.desc.rows
        return at, at + 8 * rows, at + 12 * rows

    def workspace(self):
        n = int(_native.load().gefenx_loss_workspace_bytes(self.ref))
        return torch.empty(max(n, 16), dtype=torch.uint8, device=self.device), n

    def scale(self, scale):
        """A gradient's scale as (device tensor or None, number)."""
        if not isinstance(scale, torch.Tensor):
            return None, float(scale)
        if scale.numel() != 1 or scale.device != self.device:
            raise ValueError("grad_scale must be a number or one value on {}".format(self.device))
        return scale if scale.dtype is torch.float32 else scale.detach().to(torch.float32), 1.0

    def empty_grad(self):
        return torch.empty(self.shape, dtype=self.logits.dtype, device=self.device)

    def grad(self, saved, k, weighted, scale):
        """The gradient of the logits, contiguous in their shape; k: pointer of the row coefficients, or None."""
        (scale_dev, factor), out = self.scale(scale), self.empty_grad()
        stats, _, weights = self.saved_ptrs(saved)
        with _on_device(self.device):
            _native.check(_native.load().gefenx_logits_grad(
                self.ref, stats, k, weights if weighted else None, _ptr(scale_dev), factor, out.data_ptr(), self.stream),
                "logits gradient")
        return out


def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _probability(value, name, most):
    value = float(value)
    if not 0.0 <= value < most:
        raise ValueError("{} must be in [0, {}) but is: {!r}".format(name, most, value))
    return value


def _finite(value, name):
    value = float(value)
    if not abs(value) < float("inf"):
        raise ValueError("{} must be finite but is: {!r}".format(name, value))
    return value


# ------------------------------------------------------------ forward passes

def _logps_forward(call):
    logps, (saved, ptrs) = call.empty(*call.labels.shape), call.saved()
    ws, n = call.workspace()
    with _on_device(call.device):
        _native.check(_native.load().gefenx_token_logps(call.ref, logps.data_ptr(), ptrs[0], ws.data_ptr(), n, call.stream),
                      "token_logps")
    return logps, saved


def _preference_forward(call, ref_logps, beta, smoothing, average):
    if call.n_seq % 2:
        raise ValueError("preference_loss needs pairs: the chosen sequences, then as many rejected ones, got {}".format(
            call.n_seq))
    ref = call.per_token(ref_logps, "ref_logps")
    beta, smoothing = _finite(beta, "beta"), _probability(smoothing, "label_smoothing", 0.5)
    pairs = call.n_seq // 2
    loss, chosen, rejected = call.empty(), call.empty(pairs), call.empty(pairs)
    logps, (saved, (stats, _, weights)) = call.empty(*call.labels.shape), call.saved()
    ws, n = call.workspace()
    with _on_device(call.device):
        _native.check(_native.load().gefenx_preference_loss(
            call.ref, _ptr(ref), beta, smoothing, 1 if average else 0, loss.data_ptr(), chosen.data_ptr(), rejected.data_ptr(),
            logps.data_ptr(), stats, weights, ws.data_ptr(), n, call.stream), "preference_loss")
    return PreferenceLoss(loss, chosen, rejected, logps), saved


def _advantages(call, advantages, per):
    """The advantages as the kernels read them, and whether they are one per token."""
    if per not in (None, "token", "sequence"):
        raise ValueError("advantages_per must be 'token' or 'sequence' but is: {!r}".format(per))
    each = isinstance(advantages, torch.Tensor) and advantages.shape == (call.n_seq,)
    if each and per is None and advantages.shape == call.labels.shape:
        # packed, with as many rows as sequences: the same either way where each has one row, which only the offsets know
        if torch.cuda.is_current_stream_capturing() or not torch.equal(
                call.cu, torch.arange(call.n_seq + 1, dtype=torch.int32, device=call.device)):
            raise ValueError("advantages of shape {} may be one per token or one per sequence: say which by "
                             "advantages_per".format(tuple(advantages.shape)))
        per = "token"
    if per == "token" or (per is None and not each):
        adv = call.per_token(advantages, "advantages (one per token or one per sequence)")
        if adv is None:
            raise ValueError("policy_loss needs advantages")
        return adv, 1
    if not each or advantages.device != call.device or not advantages.is_floating_point():
        raise ValueError("advantages per sequence must be a floating tensor of shape {} on {}".format(
            (call.n_seq,), call.device))
    return advantages.detach().to(torch.float32).contiguous(), 0


def _policy_forward(call, old_logps, advantages, ref_logps, clip_low, clip_high, kl_coef, reduction, advantages_per,
                    grad_scale=None):
    """The loss and what its gradient needs; with a grad_scale the gradient too."""
    old, ref = call.per_token(old_logps, "old_logps"), call.per_token(ref_logps, "ref_logps")
    if old is None:
        raise ValueError("policy_loss needs old_logps")
    if reduction not in ("token", "sequence"):
        raise ValueError("reduction must be 'token' or 'sequence' but is: {!r}".format(reduction))
    clip_low, clip_high = _probability(clip_low, "clip_low", 1.0), float(clip_high)
    if not clip_high >= 0.0:
        raise ValueError("clip_high must not be negative but is: {!r}".format(clip_high))
    kl_coef = _finite(kl_coef, "kl_coef")
    if kl_coef and ref is None:
        raise ValueError("kl_coef={} needs ref_logps".format(kl_coef))
    adv, per_row = _advantages(call, advantages, advantages_per)
    loss, kl, clipped, logps = call.empty(), call.empty(), call.empty(), call.empty(*call.labels.shape)
    saved, (stats, k, weights) = call.saved()
    args = [call.ref, old.data_ptr(), adv.data_ptr(), per_row, _ptr(ref), clip_low, clip_high, kl_coef,
            1 if reduction == "sequence" else 0, loss.data_ptr(), kl.data_ptr(), clipped.data_ptr(), logps.data_ptr(), stats, k,
            weights]
    entry, grad = _native.load().gefenx_policy_loss, None
    if grad_scale is not None:
        (scale_dev, factor), grad = call.scale(grad_scale), call.empty_grad()
        entry = _native.load().gefenx_policy_loss_grad
        args += [_ptr(scale_dev), factor, grad.data_ptr()]
    ws, n = call.workspace()
    with _on_device(call.device):
        _native.check(entry(*args, ws.data_ptr(), n, call.stream), "policy_loss")
    return PolicyLoss(loss, kl, clipped, logps), saved, grad


# ------------------------------------------------------------ autograd

class _TokenLogps(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, ignore_index):
        call = _Call(logits, labels, ignore_index, sequences=False)
        logps, saved = _logps_forward(call)
        ctx.ignore_index, ctx.desc = ignore_index, call.desc
        ctx.save_for_backward(logits, labels, saved)
        return logps

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        logits, labels, saved = ctx.saved_tensors
        call = _Call.again(ctx.desc, logits, labels, ctx.ignore_index, sequences=False)
        k = call.per_token(grad, "gradient")
        return call.grad(saved, k.data_ptr(), False, 1.0), None, None


class _SequenceLoss(torch.autograd.Function):
    """Both sequence losses: `forward_of` returns the outputs and what the gradient needs; by_row: whether rows
    have coefficients of their own."""

    @staticmethod
    def forward(ctx, logits, labels, cu_seqlens, ignore_index, forward_of, by_row):
        call = _Call(logits, labels, ignore_index, cu_seqlens)
        out, saved = forward_of(call)
        ctx.ignore_index, ctx.desc, ctx.by_row = ignore_index, call.desc, by_row
        ctx.save_for_backward(logits, labels, cu_seqlens, saved)
        ctx.mark_non_differentiable(*out[1:])
        ctx.set_materialize_grads(False)
        return tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, *unused):
        if grad is None:
            return None, None, None, None, None, None
        logits, labels, cu_seqlens, saved = ctx.saved_tensors
        call = _Call.again(ctx.desc, logits, labels, ctx.ignore_index, cu_seqlens)
        k = call.saved_ptrs(saved)[1] if ctx.by_row else None
        return call.grad(saved, k, True, grad), None, None, None, None, None


@_outside_graphs
def token_logps(logits, labels, *, ignore_index=-100):
    """log softmax(logits)[label] of every row, fp32 in the labels' shape (0
    where ignored); differentiable in the logits."""
    return _TokenLogps.apply(logits, labels, ignore_index)


@_outside_graphs
def preference_loss(logits, labels, ref_logps=None, *, cu_seqlens=None, beta=0.1, label_smoothing=0.0, average=False,
                    ignore_index=-100):
    """Preference loss of pairs of sequences, the chosen ones first:

        reward = beta * sum over the sequence's labels of (logp - ref_logp)
        h = reward of the chosen - reward of the rejected
        loss = mean of -(1 - label_smoothing) log sigmoid(h) - label_smoothing log sigmoid(-h)

    average: rewards are divided by the sequence's number of labels (a sequence
    without any has reward 0).  ref_logps: the reference model's token_logps;
    None: zeros."""
    def forward_of(call):
        return _preference_forward(call, ref_logps, beta, label_smoothing, average)
    return PreferenceLoss(*_SequenceLoss.apply(logits, labels, cu_seqlens, ignore_index, forward_of, False))


@_outside_graphs
def preference_loss_and_grad(logits, labels, ref_logps=None, *, cu_seqlens=None, beta=0.1, label_smoothing=0.0,
                             average=False, ignore_index=-100, grad_scale=1.0):
    """(preference_loss(...), gradient of the loss times grad_scale in the logits)."""
    call = _Call(logits, labels, ignore_index, cu_seqlens)
    out, saved = _preference_forward(call, ref_logps, beta, label_smoothing, average)
    return out, call.grad(saved, None, True, grad_scale)


@_outside_graphs
def policy_loss(logits, labels, old_logps, advantages, ref_logps=None, *, cu_seqlens=None, clip_low=0.2, clip_high=0.2,
                kl_coef=0.0, reduction="token", advantages_per=None, ignore_index=-100):
    """Clipped policy loss with a KL term; per labelled token, with q = exp(logp - old_logp), d = ref_logp - logp:

        -min(q A, clamp(q, 1 - clip_low, 1 + clip_high) A) + kl_coef * (exp(d) - d - 1)

    reduction: "token", the mean over all labelled tokens, or "sequence", the mean over the sequences that have
    any of their mean; 0 without any.  advantages: one per token, or one per sequence [N]; advantages_per ("token" or
    "sequence") says which where packed logits have as many rows as sequences (left out there, the call waits for
    cu_seqlens and is refused unless every sequence has one row)."""
    def forward_of(call):
        return _policy_forward(call, old_logps, advantages, ref_logps, clip_low, clip_high, kl_coef, reduction,
                               advantages_per)[:2]
    return PolicyLoss(*_SequenceLoss.apply(logits, labels, cu_seqlens, ignore_index, forward_of, True))


@_outside_graphs
def policy_loss_and_grad(logits, labels, old_logps, advantages, ref_logps=None, *, cu_seqlens=None, clip_low=0.2,
                         clip_high=0.2, kl_coef=0.0, reduction="token", advantages_per=None, ignore_index=-100, grad_scale=1.0):
    """(policy_loss(...), gradient of the loss times grad_scale in the logits)."""
    if grad_scale is None:
        raise ValueError("grad_scale must be a number or one value on the logits' device")
    call = _Call(logits, labels, ignore_index, cu_seqlens)
    out, _, grad = _policy_forward(call, old_logps, advantages, ref_logps, clip_low, clip_high, kl_coef, reduction,
                                   advantages_per, grad_scale)
    return out, grad
