"""Statistics of tokens and distillation from a teacher's likeliest tokens, over logits, on the MI355X.

What a teacher or a sampler answers with, per row of its logits (the
log-probability of a token, the entropy, the likeliest tokens), and the loss that
trains a student against it.  The reference has neither.  Logits, labels,
``cu_seqlens``, ``ignore_index`` and ``grad_scale`` are those of the losses in
gefen.losses: fp32, fp16 or bf16 logits [..., vocab] read in place, one pass over
the rows that count and one write of their gradient, sums in fp32 and float64.
Everything is of softmax(logits / temperature).
"""
from __future__ import annotations

import ctypes
import operator
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from gefen.gefen import _on_device, _outside_graphs
from gefen.kernels import _native
from gefen.losses import _Call, _ptr

_REST = {"bucket": 0, "drop": 1, "normalize": 2}
_MOST_TOP = 128  # likeliest tokens of a row


class TokenStatistics(NamedTuple):
    """log-probability of the label (None without labels) and entropy, fp32 in the leading shape of the logits; ids
    (int64) and log-probabilities (fp32) of the likeliest tokens, [..., top], likeliest first."""
    logps: Optional[torch.Tensor]
    entropy: torch.Tensor
    top_ids: torch.Tensor
    top_logps: torch.Tensor


class DistillationLoss(NamedTuple):
    """loss, mean divergence and mean negative log-probability of the labels (0 with hard_weight 0), 0-dim; the
    divergence of every row (fp32 in the labels' shape, 0 where ignored)."""
    loss: torch.Tensor
    divergence: torch.Tensor
    nll: torch.Tensor
    token_divergence: torch.Tensor


# ------------------------------------------------------------ token statistics

def _scratch(call, kept, n, keep):
    """`kept` fp32 values that the gradient needs (None unless it does) and a workspace of n bytes: tensors, and the
    pointers of both."""
    saved = call.empty(kept) if keep else None
    end = (n + 15) // 16 * 16
    ws = torch.empty(end + (16 if keep else 4 * kept + 16), dtype=torch.uint8, device=call.device)
    at = ws.data_ptr()
    return saved, ws, saved.data_ptr() if keep else at + end, at


def _statistics_forward(call, top, temperature, keep=False):
    """The statistics, and where asked to keep it, what their gradient needs."""
    top, lead = operator.index(top), call.lead
    if not 0 <= top <= min(_MOST_TOP, call.vocab):  # before anything of that size is allocated
        raise ValueError("top must be in [0, {}] but is: {!r}".format(min(_MOST_TOP, call.vocab), top))
    lib = _native.load()
    logps = None if call.labels is None else call.empty(*lead)
    entropy, top_logps = call.empty(*lead), call.empty(*lead, top)
    top_ids = torch.empty(top_logps.shape, dtype=torch.int64, device=call.device)
    n = int(lib.gefenx_token_statistics_workspace_bytes(call.ref, top))
    saved, ws, saved_ptr, ws_ptr = _scratch(call, 4 * call.rows, n, keep)
    with _on_device(call.device):
        _native.check(lib.gefenx_token_statistics(
            call.ref, temperature, top, _ptr(logps), entropy.data_ptr(), top_ids.data_ptr(), top_logps.data_ptr(),
            saved_ptr, ws_ptr, n, call.stream), "token_statistics")
    return (logps, entropy, top_ids, top_logps), saved


class _TokenStatistics(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, top, temperature, ignore_index):
        call = _Call(logits, labels, ignore_index, sequences=False, labelled=False)
        out, saved = _statistics_forward(call, top, temperature, keep=True)
        ctx.top, ctx.temperature, ctx.ignore_index, ctx.desc = operator.index(top), temperature, ignore_index, call.desc
        ctx.save_for_backward(logits, labels, out[2], saved)
        ctx.mark_non_differentiable(out[2])
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, logps, entropy, _, top_logps):
        logits, labels, top_ids, saved = ctx.saved_tensors
        call = _Call.again(ctx.desc, logits, labels, ctx.ignore_index, sequences=False, labelled=False)
        ups = [call.per_token(logps, "gradient"), call.per_token(entropy, "gradient"),
               None if top_logps is None or not ctx.top else top_logps.to(torch.float32).contiguous()]
        out = call.empty_grad()
        with _on_device(call.device):
            _native.check(_native.load().gefenx_token_statistics_grad(
                call.ref, ctx.temperature, ctx.top, saved.data_ptr(), top_ids.data_ptr(), *map(_ptr, ups), out.data_ptr(),
                call.stream), "token_statistics gradient")
        return out, None, None, None, None


@_outside_graphs
def token_statistics(logits, labels=None, *, top=0, temperature=1.0, ignore_index=-100):
    """Per row of logits [..., vocab], of softmax(logits / temperature): the log-probability of the label, the
    entropy, and the `top` (up to 128) likeliest tokens with their log-probabilities, ties by the lowest id, NaN
    before all.  Rows whose label is ignore_index are not read: 0, 0, and ids 0 with log-probability -inf.  Without
    labels every row counts and logps is None.  Differentiable in the logits through the log-probabilities, the
    entropy and the top log-probabilities, in reverse mode."""
    temperature = float(temperature)
    # a tangent goes there too: the function refuses forward mode
    if isinstance(logits, torch.Tensor) and ((logits.requires_grad and torch.is_grad_enabled())
                                             or forward_ad.unpack_dual(logits).tangent is not None):
        return TokenStatistics(*_TokenStatistics.apply(logits, labels, top, temperature, ignore_index))
    call = _Call(logits, labels, ignore_index, sequences=False, labelled=False)
    return TokenStatistics(*_statistics_forward(call, top, temperature)[0])


# ------------------------------------------------------------ distillation

class _Teacher:
    """What a call of the distillation is held to, checked, and its descriptor."""

    def __init__(self, call, ids, logps, temperature, rest, hard_weight, reduction):
        for t, name in ((ids, "teacher_ids"), (logps, "teacher_logps")):
            if not isinstance(t, torch.Tensor):
                raise TypeError("{} must be a tensor".format(name))
            if t.device != call.device or t.dim() != len(call.lead) + 1 or t.shape[:-1] != call.lead:
                raise ValueError("{} must be of shape {} on {}, got {} on {}".format(
                    name, (*call.lead, "tokens"), call.device, tuple(t.shape), t.device))
        if ids.dtype not in (torch.int32, torch.int64) or not logps.is_floating_point() or ids.shape != logps.shape:
            raise ValueError("teacher_ids (int32 or int64) and teacher_logps (floating) must have the same shape, got {} of "
                             "shape {} and {} of shape {}".format(ids.dtype, tuple(ids.shape), logps.dtype, tuple(logps.shape)))
        if rest not in _REST:
            raise ValueError("rest must be 'bucket', 'drop' or 'normalize' but is: {!r}".format(rest))
        if reduction not in ("token", "sequence"):
            raise ValueError("reduction must be 'token' or 'sequence' but is: {!r}".format(reduction))
        self.ids = ids if ids.is_contiguous() else ids.contiguous()
        self.logps = (logps if logps.dtype is torch.float32 and logps.is_contiguous()
                      else logps.detach().to(torch.float32).contiguous())
        self.how = (float(temperature), rest, float(hard_weight), reduction)
        self.desc = _native.Teacher(
            self.ids.data_ptr(), self.logps.data_ptr(), self.how[0], self.how[2], ids.shape[-1], int(ids.dtype is torch.int64),
            _REST[rest], int(reduction == "sequence"))
        self.ref = ctypes.byref(self.desc)


def _distillation_call(logits, labels, ignore_index, cu_seqlens, ids, logps, temperature, rest, hard_weight, reduction):
    call = _Call(logits, labels, ignore_index, cu_seqlens, sequences=reduction == "sequence")
    return call, _Teacher(call, ids, logps, temperature, rest, hard_weight, reduction)


def _distillation_saved(call, at):
    """Pointers of the rows' slopes [rows, 8] and the sequences' weights in what the gradient needs, at `at`."""
    return at, at + 32 * call.desc.rows


def _distillation_forward(call, teacher, grad_scale=None):
    """The loss and what its gradient needs; with a grad_scale the gradient too."""
    lib = _native.load()
    loss, divergence, nll, each = call.empty(), call.empty(), call.empty(), call.empty(*call.lead)
    n = int(lib.gefenx_distillation_workspace_bytes(call.ref, teacher.ref))
    saved, ws, saved_ptr, ws_ptr = _scratch(call, 8 * call.rows + max(call.n_seq, 1), n, grad_scale is None)
    args = [call.ref, teacher.ref, loss.data_ptr(), divergence.data_ptr(), nll.data_ptr(), each.data_ptr(),
            *_distillation_saved(call, saved_ptr)]
    entry, grad = lib.gefenx_distillation_loss, None
    if grad_scale is not None:
        (scale_dev, factor), grad = call.scale(grad_scale), call.empty_grad()
        entry = lib.gefenx_distillation_loss_grad
        args += [_ptr(scale_dev), factor, grad.data_ptr()]
    with _on_device(call.device):
        _native.check(entry(*args, ws_ptr, n, call.stream), "distillation_loss")
    return DistillationLoss(loss, divergence, nll, each), saved, grad


class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, cu_seqlens, ignore_index, ids, logps, how):
        call, teacher = _distillation_call(logits, labels, ignore_index, cu_seqlens, ids, logps, *how)
        out, saved, _ = _distillation_forward(call, teacher)
        ctx.ignore_index, ctx.desc, ctx.how = ignore_index, call.desc, teacher.how
        ctx.save_for_backward(logits, labels, cu_seqlens, teacher.ids, teacher.logps, saved)
        ctx.mark_non_differentiable(*out[1:])
        ctx.set_materialize_grads(False)
        return tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad, *unused):
        if grad is None:
            return (None,) * 7
        logits, labels, cu_seqlens, ids, logps, saved = ctx.saved_tensors
        call = _Call.again(ctx.desc, logits, labels, ctx.ignore_index, cu_seqlens, sequences=ctx.how[3] == "sequence")
        teacher = _Teacher(call, ids, logps, *ctx.how)
        (scale_dev, factor), out = call.scale(grad), call.empty_grad()
        with _on_device(call.device):
            _native.check(_native.load().gefenx_distillation_grad(
                call.ref, teacher.ref, *_distillation_saved(call, saved.data_ptr()), _ptr(scale_dev), factor, out.data_ptr(), call.stream),
                "distillation gradient")
        return (out,) + (None,) * 6


@_outside_graphs
def distillation_loss(logits, labels, teacher_ids, teacher_logps, *, cu_seqlens=None, temperature=1.0, rest="bucket",
                      hard_weight=0.0, reduction="token", ignore_index=-100):
    """Loss of a student's logits against a teacher's likeliest tokens: teacher_ids (int32 or int64) and
    teacher_logps [..., tokens] (up to 512; token_statistics(teacher's logits, top=..., temperature=...) gives them),
    constants.  With p = exp(teacher_logps), P their sum and q = softmax(logits / temperature), per row

        D = sum p (log p - log q), and by `rest`, for the tokens that the teacher does not name,
            "bucket": r log(r / s), r = max(0, 1 - P), s = 1 - sum q: they count as one (no term where the
                      student has no other token)
            "drop": nothing;  "normalize": p / P in the place of p (0 where P = 0)

    and loss = mean of (1 - hard_weight) temperature^2 D - hard_weight log softmax(logits)[label] over the labelled
    rows, or (reduction "sequence") the mean over the sequences that have any of their mean; 0 without any.  An entry of
    log-probability -inf names no token, whatever its id; a token that several entries name is in P and the sum of D with
    each of them, in s once.  With hard_weight 0 labels only say which rows count, with 1
    the teacher gives the divergence alone, whatever it holds."""
    how = (temperature, rest, hard_weight, reduction)
    return DistillationLoss(*_Distillation.apply(logits, labels, cu_seqlens, ignore_index, teacher_ids, teacher_logps, how))


@_outside_graphs
def distillation_loss_and_grad(logits, labels, teacher_ids, teacher_logps, *, cu_seqlens=None, temperature=1.0, rest="bucket",
                               hard_weight=0.0, reduction="token", ignore_index=-100, grad_scale=1.0):
    """(distillation_loss(...), gradient of the loss times grad_scale in the logits)."""
    if grad_scale is None:
        raise ValueError("grad_scale must be a number or one value on the logits' device")
    call, teacher = _distillation_call(logits, labels, ignore_index, cu_seqlens, teacher_ids, teacher_logps, temperature, rest,
                                       hard_weight, reduction)
    out, _, grad = _distillation_forward(call, teacher, grad_scale)
    return out, grad
