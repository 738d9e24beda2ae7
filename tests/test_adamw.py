"""AdamW's host side: arguments, layouts, checkpoints, and the 8-bit formats' restatement (no GPU)."""
import copy
import os
import pickle
import subprocess
import sys

import pytest
import torch

import gefen
from gefen.adamw import _dense, _order, _same_layout
import adamw_reference as ref


def one(n=24, **kw):
    p = torch.nn.Parameter(torch.ones(n))
    return p, gefen.AdamW([p], **kw)


@pytest.mark.parametrize("kw", [
    {"lr": -1.0}, {"lr": float("nan")}, {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)}, {"betas": (0.9,)}, {"eps": -1e-8},
    {"weight_decay": -0.1}, {"state_bits": 16}, {"max_grad_norm": 0.0}, {"max_grad_norm": -1.0},
    {"max_grad_norm": float("inf")}, {"max_grad_norm": float("nan")},
])
def test_bad_arguments_are_refused(kw):
    with pytest.raises(ValueError):
        one(**kw)


def test_group_options_are_checked():
    p, opt = one()
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.ones(2))], "state_bits": 4})
    opt.add_param_group({"params": [torch.nn.Parameter(torch.ones(2))], "state_bits": 8, "lr": 1.0})
    assert [g["state_bits"] for g in opt.param_groups] == [32, 8]


def test_host_parameters_are_refused_before_anything_moves():
    p, opt = one()
    p.grad = torch.ones(24)
    with pytest.raises(RuntimeError, match="HIP device"):
        opt.step()
    assert not opt.state and torch.equal(p.detach(), torch.ones(24))


def test_step_without_gradients_and_closure():
    _, opt = one()
    assert opt.step(lambda: 3.0) == 3.0 and not opt.state


def test_named_parameters():
    net = torch.nn.Linear(3, 2)
    opt = gefen.AdamW(net.named_parameters(), state_bits=8)
    assert len(opt.param_groups[0]["params"]) == 2


def test_layouts():
    t = torch.zeros(4, 6)
    assert _order(t) is None and _dense(t)
    assert _order(t.t()) == (1, 0) and _dense(t.t()) and not _same_layout(t.t(), torch.zeros(6, 4))
    assert _same_layout(t.t(), torch.zeros(4, 6).t())
    gap = torch.zeros(4, 9)[:, :6]
    assert _order(gap) == (0, 1) and not _dense(gap)
    assert _dense(torch.zeros(2, 3, 4, 5).to(memory_format=torch.channels_last))
    assert _dense(torch.zeros(5, 1).t()) and _dense(torch.zeros(())) and _dense(torch.zeros(0, 3))
    with pytest.raises(ValueError, match="share memory"):
        _order(torch.zeros(1, 3).expand(4, 3))
    with pytest.raises(ValueError, match="share memory"):
        _order(torch.zeros(20).as_strided((3, 3), (2, 1)))


def state8(n, order=None, **kw):
    b = -(-n // 256)
    got = {"step": 7, "exp_avg": torch.arange(n, dtype=torch.int64).remainder(100).to(torch.uint8).view(torch.float8_e4m3fn),
           "exp_avg_sq": torch.arange(n, dtype=torch.int64).remainder(256).to(torch.uint8),
           "exp_avg_scale": torch.rand(b), "exp_avg_sq_scale": torch.rand(b), "order": order}
    got.update(kw)
    return got


def test_checkpoint_of_8_bits_keeps_its_codes():
    p, opt = one(300, state_bits=8)
    saved = {"state": {0: state8(300)}, "param_groups": opt.state_dict()["param_groups"]}
    opt.load_state_dict(saved)
    got = opt.state[p]
    assert got["step"] == 7 and got["exp_avg"].dtype is torch.float8_e4m3fn
    for k in ("exp_avg", "exp_avg_sq"):
        assert torch.equal(got[k].view(torch.uint8), saved["state"][0][k].view(torch.uint8))
        assert got[k].data_ptr() != saved["state"][0][k].data_ptr()
    again = gefen.AdamW([torch.nn.Parameter(torch.ones(300))], state_bits=8)
    again.load_state_dict(opt.state_dict())
    assert torch.equal(again.state_dict()["state"][0]["exp_avg_sq"], got["exp_avg_sq"])


@pytest.mark.parametrize("change", [
    {"exp_avg": torch.zeros(300)}, {"exp_avg_sq": torch.zeros(299, dtype=torch.uint8)}, {"exp_avg_scale": torch.zeros(3)},
    {"exp_avg_sq_scale": torch.zeros(2, dtype=torch.float16)}, {"exp_avg_sq": None}, {"order": (1, 0)},
])
def test_checkpoint_that_does_not_fit_is_refused_whole(change):
    p, opt = one(300, state_bits=8)
    with pytest.raises(ValueError):
        opt.load_state_dict({"state": {0: state8(300, **change)}, "param_groups": opt.state_dict()["param_groups"]})
    assert not opt.state


def test_checkpoint_of_another_storage_order_is_refused():
    turned = torch.nn.Parameter(torch.ones(4, 6).t())
    opt = gefen.AdamW([turned], state_bits=8)
    groups = opt.state_dict()["param_groups"]
    with pytest.raises(ValueError, match="storage order"):
        opt.load_state_dict({"state": {0: state8(24)}, "param_groups": groups})
    opt.load_state_dict({"state": {0: state8(24, order=[1, 0])}, "param_groups": groups})
    assert opt.state[turned]["order"] == (1, 0)


def test_state_of_8_bits_follows_the_memory_that_is_stepped():
    """A parameter with gaps is stepped in a row-major copy: its state is that of a contiguous parameter, whichever way
    it is turned, and is not taken for that of a dense turned one."""
    rows, turned, dense, flat = (torch.nn.Parameter(t) for t in (
        torch.ones(4, 9)[:, :6], torch.ones(9, 6)[:, :4].t()[:, :6], torch.ones(6, 4).t(), torch.ones(4, 6)))
    states = {}
    for p in (rows, turned, dense, flat):
        opt = gefen.AdamW([p], state_bits=8)
        states[p] = opt._new_state(p, 8)
        opt._check_state(p, states[p], 8)
    assert [states[p]["order"] for p in (rows, turned, dense, flat)] == [None, None, (1, 0), None]
    for p, fits in ((rows, True), (turned, True), (flat, True), (dense, False)):
        opt = gefen.AdamW([p], state_bits=8)
        saved = {"state": {0: states[turned]}, "param_groups": opt.state_dict()["param_groups"]}
        if fits:
            opt.load_state_dict(saved)
            # row-major by its dims, as saved for a parameter with gaps
            opt.load_state_dict(dict(saved, state={0: dict(states[turned], order=(0, 1))}))
        else:
            with pytest.raises(ValueError, match="storage order"):
                opt.load_state_dict(saved)
    opt = gefen.AdamW([turned], state_bits=8)
    with pytest.raises(ValueError, match="storage order"):
        opt.load_state_dict({"state": {0: states[dense]}, "param_groups": opt.state_dict()["param_groups"]})


def test_torch_checkpoint_loads_and_goes_back():
    a = torch.nn.Parameter(torch.ones(5, 3))
    theirs = torch.optim.AdamW([a], lr=0.1)
    a.grad = torch.ones(5, 3)
    theirs.step()
    p = torch.nn.Parameter(torch.ones(5, 3))
    opt = gefen.AdamW([p])
    opt.load_state_dict(theirs.state_dict())
    assert opt.state[p]["step"] == 1 and opt.param_groups[0]["lr"] == 0.1 and opt.param_groups[0]["state_bits"] == 32
    assert torch.equal(opt.state[p]["exp_avg_sq"], theirs.state[a]["exp_avg_sq"])
    back = torch.optim.AdamW([torch.nn.Parameter(torch.ones(5, 3))])
    back.load_state_dict({"state": opt.state_dict()["state"], "param_groups": theirs.state_dict()["param_groups"]})


@pytest.mark.parametrize("kw", [dict(amsgrad=True), dict(maximize=True)])
def test_variants_of_the_formula_are_refused(kw):
    a, b = torch.nn.Parameter(torch.ones(4)), torch.nn.Parameter(torch.ones(4))
    a.grad = torch.ones(4)
    theirs = torch.optim.AdamW([a], **kw)
    theirs.step()
    opt = gefen.AdamW([b])
    with pytest.raises(ValueError, match=next(iter(kw))):
        opt.load_state_dict(theirs.state_dict())
    assert not opt.state and not opt.param_groups[0].get(next(iter(kw)))
    with pytest.raises(ValueError, match=next(iter(kw))):
        gefen.AdamW([dict(params=[b], **kw)])


def test_checkpoint_with_coupled_decay_is_refused():
    a, b = torch.nn.Parameter(torch.ones(4)), torch.nn.Parameter(torch.ones(4))
    a.grad = torch.ones(4)
    theirs = torch.optim.Adam([a], weight_decay=0.1)
    theirs.step()
    opt = gefen.AdamW([b])
    with pytest.raises(ValueError, match="decoupled"):
        opt.load_state_dict(theirs.state_dict())
    theirs.param_groups[0]["weight_decay"] = 0.0  # the same formula either way
    opt.load_state_dict(theirs.state_dict())
    assert opt.state[b]["step"] == 1


def test_groups_keep_their_width_where_a_checkpoint_names_none():
    a, b = torch.nn.Parameter(torch.ones(4)), torch.nn.Parameter(torch.ones(300))
    opt = gefen.AdamW([{"params": [a]}, {"params": [b], "state_bits": 8}])
    groups = [{k: v for k, v in g.items() if k != "state_bits"} for g in opt.state_dict()["param_groups"]]
    opt.load_state_dict({"state": {1: state8(300)}, "param_groups": groups})
    assert [g["state_bits"] for g in opt.param_groups] == [32, 8] and opt.state[b]["step"] == 7


def test_other_groups_are_refused():
    _, opt = one()
    with pytest.raises(ValueError, match="parameter groups"):
        opt.load_state_dict({"state": {}, "param_groups": []})


@pytest.mark.parametrize("bits", [32, 8])
def test_hooks_of_loading_see_what_is_loaded(bits):
    """Pre-hooks get the checkpoint and may replace it, post-hooks find its state in place, none stays behind."""
    p, opt = one(300, state_bits=bits)
    entry = state8(300) if bits == 8 else {"step": 7, "exp_avg": torch.rand(300), "exp_avg_sq": torch.rand(300)}
    saved = {"state": {0: entry}, "param_groups": opt.state_dict()["param_groups"]}
    seen = []

    def later(optimizer, state_dict):
        seen.append(state_dict["state"][0]["step"])
        return dict(state_dict, state={0: dict(state_dict["state"][0], step=9)})
    opt.register_load_state_dict_pre_hook(later)
    opt.register_load_state_dict_pre_hook(lambda optimizer, state_dict: seen.append(state_dict["state"][0]["step"]))
    opt.register_load_state_dict_post_hook(lambda optimizer: seen.append(optimizer.state[p]["step"]), prepend=True)
    opt.register_load_state_dict_post_hook(lambda optimizer: optimizer.state[p].update(step=10))
    for _ in range(2):
        opt.load_state_dict(saved)
        assert seen == [7, 9, 9] and opt.state[p]["step"] == 10 and saved["state"][0]["step"] == 7
        assert opt.param_groups[0]["state_bits"] == bits
        seen.clear()
    bad = dict(saved, state={0: dict(entry, exp_avg=torch.zeros(5))})
    with pytest.raises(ValueError):
        opt.load_state_dict(bad)
    assert seen == [7, 9] and opt.state[p]["step"] == 10
    seen.clear()
    opt.load_state_dict(saved)
    assert seen == [7, 9, 9]


def test_copies_keep_the_options():
    _, opt = one(max_grad_norm=2.0, seed=5)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert other.max_grad_norm == 2.0 and other.seed == 5 and other.grad_norm is None


def test_import_leaves_the_compiler_alone():
    """torch._dynamo, an import of half a second, is for callers who compile."""
    package = os.path.dirname(os.path.dirname(os.path.abspath(gefen.__file__)))
    code = "import sys, gefen; print('torch._dynamo' in sys.modules)"
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, check=True,
                         env=dict(os.environ, PYTHONPATH=package))
    assert out.stdout.strip() == "False"


def test_moments_of_foreign_tensors_are_refused():
    _, opt = one()
    with pytest.raises(ValueError):
        opt.moments([torch.ones(2)])
    assert opt.moments() == [None]


def test_host_state_of_8_bits_is_not_read_on_a_device():
    p, opt = one(300, state_bits=8)
    opt.load_state_dict({"state": {0: state8(300)}, "param_groups": opt.state_dict()["param_groups"]})
    with pytest.raises(RuntimeError, match="HIP device"):
        opt.moments()


# ------------------------------------------------ the formats, by their restatement

def test_v_code_round_trip_and_order():
    c = torch.arange(256, dtype=torch.uint8)
    x = ref.value_v(c, torch.ones(1))
    assert x[0] == 0 and x[255] == 1 and torch.all(x[1:] > x[:-1])
    back, scale = ref.codes_v(x, torch.zeros(256, dtype=torch.int64))
    assert scale.item() == 1.0 and torch.equal(back, c)
    ratio = x[2:] / x[1:-1]
    assert ratio.max() <= 1.125 and ratio.min() > 1.06


def test_v_code_never_loses_a_positive_value():
    v = torch.tensor([1.0, 1e-30, 1e-38, 0.0])
    code, _ = ref.codes_v(v, torch.zeros(4, dtype=torch.int64))
    assert code.tolist() == [255, 1, 1, 0]


def test_v_code_is_unbiased():
    """Over all 2^16 roundings, a value's mean is the value but for the 4 bits below the random ones: 2^-16 of a code."""
    bits = torch.arange(1 << 16, dtype=torch.int64)
    for x in (0.9371, 0.5001, 0.12345, 3e-4):
        v = torch.full((1 << 16,), x)
        v[::256] = 1.0  # the block's scale
        code, scale = ref.codes_v(v, bits)
        got = ref.value_v(code, scale).double()
        keep = torch.ones(1 << 16, dtype=torch.bool)
        keep[::256] = False
        # the 256 roundings left out are spread evenly: they shift the mean by at most 1/256 of a code's 2^-8
        assert abs(got[keep].mean() / torch.tensor(x).double() - 1).item() < 2 ** -14


def test_random_bits_are_spread():
    bits = ref.random16(ref.step_key(1, 0, 1), 4096).double()
    # mean of 4096 uniform values: standard deviation 18919 / 64 = 296
    assert abs(bits.mean().item() - 32767.5) < 5 * 296
    assert not torch.equal(bits, ref.random16(ref.step_key(1, 0, 2), 4096).double())
    assert not torch.equal(bits, ref.random16(ref.step_key(1, 1, 1), 4096).double())
