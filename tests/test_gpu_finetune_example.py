"""The fine-tuning example runs its losses and optimizers together, and learns as plain torch does."""
import importlib.util
import os
import types

import pytest
import torch

import gefen

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("finetune", os.path.join(ROOT, "examples", "finetune.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


class PlainAdamW(torch.optim.AdamW):
    def __init__(self, params, state_bits=32, max_grad_norm=None, **kw):
        super().__init__(params, **kw)
        self.max_grad_norm = max_grad_norm

    def step(self):
        if self.max_grad_norm is not None:
            torch.nn.utils.clip_grad_norm_([p for g in self.param_groups for p in g["params"]], self.max_grad_norm)
        super().step()


def plain_logps(logits, labels):
    lp = torch.log_softmax(logits.float(), -1).gather(-1, labels.clamp(min=0)[..., None])[..., 0]
    return torch.where(labels == -100, torch.zeros_like(lp), lp)


def plain_preference(logits, labels, ref, beta):
    r = beta * (plain_logps(logits, labels) - ref).sum(1)
    half = r.numel() // 2
    return types.SimpleNamespace(loss=-torch.nn.functional.logsigmoid(r[:half] - r[half:]).mean())


def test_preference_training_follows_plain_torch():
    """The same batches through torch's AdamW in 32 bits and plain losses.  8-bit moments leave each step within some
    tens of percent of the exact one per element (both formats have 3 mantissa bits), without a bias: the loss after
    40 steps stays within a fifth of the exact run's way down."""
    m = example()
    torch.manual_seed(0)
    model = m.Model().to("cuda")
    state = {k: v.clone() for k, v in model.state_dict().items()}
    torch.manual_seed(1)
    losses = m.prefer(model, 40)
    model.load_state_dict(state)
    m.gefen = types.SimpleNamespace(AdamW=PlainAdamW, token_logps=plain_logps, preference_loss=plain_preference)
    torch.manual_seed(1)
    plain = m.prefer(model, 40)
    m.gefen = gefen
    assert abs(losses[0] - plain[0]) < 1e-5
    assert plain[-1] < plain[0] - 0.2
    assert abs(losses[-1] - plain[-1]) < 0.2 * (plain[0] - plain[-1])


def test_policy_training_learns():
    m = example()
    _, rewards = m.main(steps=40)
    # untrained, a quarter of the tokens are rewarded
    assert abs(rewards[0] - 0.25) < 0.1 and rewards[-1] > rewards[0] + 0.05
