"""torch.compile'd callers of the losses and of AdamW.step run them between their graphs, with eager's results."""
import pytest
import torch

import gefen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda", 0)


@pytest.mark.parametrize("which", ["logps", "preference", "policy"])
def test_compiled_losses(dev, which):
    x = torch.randn(4, 16, 500, device=dev, requires_grad=True)
    y = torch.randint(0, 500, (4, 16), device=dev)
    ref, adv = torch.randn(4, 16, device=dev) - 6, torch.randn(4, device=dev)
    fn = {"logps": lambda t: gefen.token_logps(t * 1.5, y).sum(),
          "preference": lambda t: gefen.preference_loss(t * 1.5, y, ref).loss * 2.0,
          "policy": lambda t: gefen.policy_loss(t * 1.5, y, ref, adv, ref, kl_coef=0.1).loss}[which]
    got = []
    for f in (fn, torch.compile(fn, backend="eager")):
        x.grad = None
        loss = f(x)
        loss.backward()
        got.append((loss.detach().clone(), x.grad.clone()))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_compiled_step(dev):
    params = [torch.nn.Parameter(torch.linspace(-1, 1, 300, device=dev)) for _ in range(2)]
    opts = [gefen.AdamW([p], state_bits=8, max_grad_norm=1.0) for p in params]
    steps = [opts[0].step, torch.compile(opts[1].step, backend="eager")]
    for k in range(2):
        for p, step in zip(params, steps):
            p.grad = torch.full((300,), 0.1 + k, device=dev)
            step()
    assert torch.equal(*params) and opts[1].state[params[1]]["step"] == 2 and opts[1].grad_norm is not None
