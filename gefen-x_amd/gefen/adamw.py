"""AdamW on the MI355X: many tensors per launch, moments in 32 or 8 bits.

The plain optimizer beside Gefen's factored one, with torch.optim.AdamW's
arithmetic, param groups and 32-bit state keys (``step``, ``exp_avg``,
``exp_avg_sq``), so checkpoints of torch's class load.  The reference has no
AdamW of its own (its hybrid builds torch's, hybrid.py:546-560).

With ``state_bits=8`` a moment is one byte per element and one fp32 scale per
256 elements: ``exp_avg`` in E4M3, ``exp_avg_sq`` in 5 exponent and 3 mantissa
bits, rounded stochastically from ``seed`` (same seed, same run), because a
step moves it by far less than half a code.  The formats are those of
gefenx_adamw_desc in include/gefenx.h.
"""
from __future__ import annotations

import ctypes
import math
import struct

import torch
from torch.autograd.graph import increment_version

from gefen.gefen import _amp_gate, _amp_native_scaling_required, _on_device, _outside_graphs
from gefen.kernels import _native

BLOCK = 256  # elements per scale of the 8-bit moments

_DESC_STRUCT = struct.Struct("<6QqQ8f2iQ")
_COUNTER_STRUCT = struct.Struct("<3Q4dQ2i")
assert _DESC_STRUCT.size == ctypes.sizeof(_native.AdamWDesc)
assert _COUNTER_STRUCT.size == ctypes.sizeof(_native.AdamWCounter)
_DTYPES = {torch.float32: _native.DT_F32, torch.float16: _native.DT_F16, torch.bfloat16: _native.DT_BF16}
_PLAIN = frozenset((torch.Tensor, torch.nn.Parameter))
_U64 = (1 << 64) - 1
_GOLDEN = 0x9E3779B97F4A7C15
# state keys and dtypes by width
_STATE = {
    32: {"exp_avg": torch.float32, "exp_avg_sq": torch.float32},
    8: {"exp_avg": torch.float8_e4m3fn, "exp_avg_sq": torch.uint8,
        "exp_avg_scale": torch.float32, "exp_avg_sq_scale": torch.float32},
}


def _mix(z: int) -> int:
    """SplitMix64's finalizer, as the kernels draw with."""
    z &= _U64
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9 & _U64
    z = (z ^ (z >> 27)) * 0x94D049BB133111EB & _U64
    return z ^ (z >> 31)


def _pack(rows, form=_DESC_STRUCT) -> bytes:
    """The descriptors of gefenx_adamw_* calls."""
    return b"".join([form.pack(*row) for row in rows])


def _order(t: torch.Tensor):
    """None for a contiguous tensor, else its dims (of size > 1) from the
    largest stride to the smallest; ValueError where elements may overlap."""
    if t.is_contiguous():
        return None
    dims = sorted((d for d in range(t.dim()) if t.shape[d] > 1), key=lambda d: -t.stride(d))
    reach = 1  # elements spanned by the inner dims
    for d in reversed(dims):
        if t.stride(d) < reach:
            raise ValueError("AdamW cannot step a parameter whose elements may share memory (shape {}, strides {})".format(
                tuple(t.shape), t.stride()))
        reach += (t.shape[d] - 1) * t.stride(d)
    return tuple(dims)


def _dense(t: torch.Tensor) -> bool:
    """Whether a tensor without overlap fills one run of memory."""
    return t.is_contiguous() or t.numel() == 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))


def _code_order(p: torch.Tensor):
    """The order of a parameter's 8-bit moments: that of the memory it is stepped in, which for one with gaps is a
    contiguous copy (None, as for a contiguous parameter)."""
    return _order(p) if _dense(p) else None


def _same_layout(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two dense tensors of one shape hold their elements in the same order."""
    if a.is_contiguous() and b.is_contiguous():
        return True
    return all(sa == sb for n, sa, sb in zip(a.shape, a.stride(), b.stride()) if n > 1)


def _plainly_fits(p, state, bits) -> bool:
    """Whether the common state of a contiguous parameter is what _check_state asks for (it costs half as much)."""
    m, v, device = state.get("exp_avg"), state.get("exp_avg_sq"), p.get_device()
    if type(m) is not torch.Tensor or type(v) is not torch.Tensor or m.get_device() != device or v.get_device() != device:
        return False
    if bits == 32:
        return m.dtype is torch.float32 and v.dtype is torch.float32 and m.shape == p.shape and v.shape == p.shape
    ms, vs, n = state.get("exp_avg_scale"), state.get("exp_avg_sq_scale"), p.numel()
    if type(ms) is not torch.Tensor or type(vs) is not torch.Tensor or ms.get_device() != device or vs.get_device() != device:
        return False
    blocks = -(-n // BLOCK)
    return (m.dtype is torch.float8_e4m3fn and v.dtype is torch.uint8 and ms.dtype is torch.float32
            and vs.dtype is torch.float32 and m.numel() == n and v.numel() == n and ms.numel() == blocks
            and vs.numel() == blocks and m.is_contiguous() and v.is_contiguous() and ms.is_contiguous()
            and vs.is_contiguous() and p.is_contiguous() and state.get("order") is None)


def _refuse_variants(group):
    """Options of torch's class, by argument or checkpoint, that would be another formula."""
    for name in ("amsgrad", "maximize"):
        if group.get(name):
            raise ValueError("AdamW has no {} (a parameter group asks for it)".format(name))
    if not group.get("decoupled_weight_decay", True) and float(group["weight_decay"]) != 0.0:
        raise ValueError("AdamW decays weights apart from the gradient; a parameter group asks for "
                         "decoupled_weight_decay=False")


class AdamW(torch.optim.Optimizer):
    """AdamW (decoupled weight decay) over fp32, fp16 or bf16 parameters.

    params, lr, betas, eps, weight_decay: as torch.optim.AdamW (also per
    group).  state_bits: 32 or 8, also per group.  max_grad_norm: gradients
    are scaled by min(1, max_grad_norm / (norm + 1e-6)), norm the 2-norm of
    all of them together, inside the step (``p.grad`` keeps its values); the
    norm is left in ``grad_norm``, a 0-dim device tensor.  seed: of the
    stochastic rounding of 8-bit moments.

    A parameter's elements are stepped in place in the order it is stored in.
    Slices with gaps, and gradients laid out otherwise than their parameter,
    go through a contiguous copy.  Work is enqueued on the current stream; the
    step does not wait for the GPU.  A backward pass through a graph that has
    saved a parameter from before the step raises, as after any write in
    place (a captured step's replays are not seen).

    capturable=True: step counters are 0-dim device tensors and a step can be
    captured into a graph and replayed (each parameter's first step runs
    eagerly; an lr on the device, the parameters', is read at every replay, one
    on the host is what it was at capture).  load_state_dict makes new state:
    graphs captured before it step the old one and are not to be replayed.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32,
                 max_grad_norm=None, seed=0, capturable=False):
        if max_grad_norm is not None and not (float(max_grad_norm) > 0.0 and math.isfinite(float(max_grad_norm))):
            raise ValueError("max_grad_norm must be positive and finite but is: {!r}".format(max_grad_norm))
        self.max_grad_norm = None if max_grad_norm is None else float(max_grad_norm)
        self.seed = int(seed)
        self.capturable = bool(capturable)
        self.grad_norm = None
        self._rows = {}  # capturable: parameter -> device row of what changes from step to step
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits))

    def add_param_group(self, param_group):
        group = dict(self.defaults, **param_group)
        lr, betas, eps, wd = group["lr"], group["betas"], group["eps"], group["weight_decay"]
        if not float(lr) >= 0.0:
            raise ValueError("Invalid learning rate: {}".format(lr))
        if len(betas) != 2 or not all(0.0 <= float(b) < 1.0 for b in betas):
            raise ValueError("betas must be two numbers in [0, 1) but are: {!r}".format(betas))
        if not float(eps) >= 0.0:
            raise ValueError("Invalid epsilon value: {}".format(eps))
        if not float(wd) >= 0.0:
            raise ValueError("Invalid weight_decay value: {}".format(wd))
        if group["state_bits"] not in _STATE:
            raise ValueError("state_bits must be 8 or 32 but is: {!r}".format(group["state_bits"]))
        _refuse_variants(group)
        super().add_param_group(param_group)

    def __getstate__(self):
        return dict(super().__getstate__(), max_grad_norm=self.max_grad_norm, seed=self.seed, grad_norm=self.grad_norm,
                    capturable=self.capturable, _rows={})

    @property
    def _step_supports_amp_scaling(self) -> bool:
        """The GradScaler protocol of Gefen: true fp16 gradients are unscaled here."""
        return _amp_native_scaling_required(self)

    # --------------------------------------------------------------- step

    @staticmethod
    def _refuse_grad(p, g):
        """What is wrong with a gradient that is not plainly the parameter's."""
        if g.layout is not torch.strided:
            raise RuntimeError("AdamW does not support sparse gradients")
        if hasattr(p, "placements") or hasattr(g, "placements"):
            raise RuntimeError("AdamW does not step DTensor parameters")
        if not p.is_cuda or g.device != p.device:
            raise RuntimeError("AdamW steps HIP device parameters with gradients on the same device: parameter "
                               "on {}, gradient on {}".format(p.device, g.device))
        if g.shape != p.shape:
            raise RuntimeError("gradient shape {} does not match parameter shape {}".format(tuple(g.shape), tuple(p.shape)))
        if p.dtype not in _DTYPES:
            raise NotImplementedError("AdamW is not implemented for {}".format(p.dtype))
        if g.dtype is not p.dtype:
            raise RuntimeError("gradient dtype {} does not match parameter dtype {}".format(g.dtype, p.dtype))

    def _checked(self):
        """[(group, [(index, parameter, gradient, state), ...]), ...] of what there is to step; refuses what cannot
        be stepped before anything moves."""
        found, devices, index, known = [], set(), 0, self.state
        for group in self.param_groups:
            bits, members, lr_device = group["state_bits"], [], None
            if self.capturable:
                _, lr_tensor = self._lr_of(group["lr"])
                lr_device = None if lr_tensor is None else lr_tensor.get_device()
            for p in group["params"]:
                index += 1
                g = p.grad
                if g is None:
                    continue
                dtype = p.dtype
                if not (type(g) is torch.Tensor and type(p) in _PLAIN and g.dtype is dtype and dtype in _DTYPES
                        and p.is_cuda and g.is_cuda and g.layout is torch.strided and g.shape == p.shape
                        and g.get_device() == p.get_device()):
                    self._refuse_grad(p, g)
                if not p.is_contiguous():
                    _order(p)
                if lr_device is not None and lr_device != p.get_device():
                    raise ValueError("a device lr is read by the parameters' kernels: it is on device {}, a parameter on "
                                     "{}".format(lr_device, p.device))
                state = known.get(p)
                if state and self.capturable:
                    step = state.get("step")
                    if not (isinstance(step, torch.Tensor) and step.dtype is torch.float32 and step.numel() == 1
                            and step.get_device() == p.get_device()):
                        raise ValueError("AdamW capturable needs the step counter as an fp32 value on {}".format(p.device))
                if state and not _plainly_fits(p, state, bits):
                    self._check_state(p, state, bits)
                devices.add(p.get_device())
                members.append((index, p, g, state))
            if members:
                found.append((group, members))
        if self.max_grad_norm is not None and len(devices) > 1:
            raise RuntimeError("AdamW with max_grad_norm steps parameters of one device, got devices {}".format(sorted(devices)))
        return found

    @staticmethod
    def _check_state(p, state, bits):
        n, device, contiguous = p.numel(), p.get_device(), p.is_contiguous()
        for key, dtype in _STATE[bits].items():
            t = state.get(key)
            if type(t) is not torch.Tensor or t.dtype is not dtype:
                raise ValueError("AdamW with state_bits={} needs {} as {}, got {}".format(
                    bits, key, dtype, t.dtype if isinstance(t, torch.Tensor) else type(t).__name__))
            if bits == 32:
                fits = t.shape == p.shape
            else:
                fits = t.numel() == (-(-n // BLOCK) if dtype is torch.float32 else n) and t.is_contiguous()
            if not fits or t.get_device() != device:
                raise ValueError("AdamW state {} (shape {}, {}) does not belong to a parameter of shape {} on {}".format(
                    key, tuple(t.shape), t.device, tuple(p.shape), p.device))
        if bits == 8:
            order = state.get("order")
            if not (contiguous and order is None) and order != _code_order(p):
                raise ValueError("AdamW's 8-bit state follows the storage order of the parameter it was made for "
                                 "({}); this one is stepped in {}".format(order, _code_order(p)))

    def _counter(self, p, value):
        """A step counter: a number, or under capturable a 0-dim device tensor."""
        return torch.full((), float(value), dtype=torch.float32, device=p.device) if self.capturable else int(value)

    def _new_state(self, p, bits):
        if bits == 32:
            like = p if _dense(p) else p.contiguous()
            return {"step": self._counter(p, 0),
                    "exp_avg": torch.zeros_like(like, dtype=torch.float32, memory_format=torch.preserve_format),
                    "exp_avg_sq": torch.zeros_like(like, dtype=torch.float32, memory_format=torch.preserve_format)}
        blocks, dev = -(-p.numel() // BLOCK), p.device
        return {"step": self._counter(p, 0),
                "exp_avg": torch.zeros(p.numel(), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn),
                "exp_avg_sq": torch.zeros(p.numel(), dtype=torch.uint8, device=dev),
                "exp_avg_scale": torch.zeros(blocks, dtype=torch.float32, device=dev),
                "exp_avg_sq_scale": torch.zeros(blocks, dtype=torch.float32, device=dev), "order": _code_order(p)}

    @_outside_graphs
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        found = self._checked()
        capturing = bool(found) and torch.cuda.is_current_stream_capturing()
        if capturing:
            self._check_capture(found)
        if not _amp_gate(self):
            return loss
        self.grad_norm = None
        batches = {}  # device -> descriptors, counters, parameters to write back, tensors that the launch reads
        stepped = []
        for group, members in found:
            (beta1, beta2), bits, lr_tensor = group["betas"], group["state_bits"], None
            eps, decay, last = float(group["eps"]), float(group["weight_decay"]), None
            if self.capturable:
                lr, lr_tensor = self._lr_of(group["lr"])
            else:
                lr = float(group["lr"])
            wdf, step_size, rbc2 = 1.0 - lr * decay, 0.0, 0.0
            for index, p, grad, state in members:
                if not state:
                    state = self.state[p] = self._new_state(p, bits)
                device = p.get_device()
                if device not in batches:
                    batches[device] = ([], [], [], [])
                rows, counters, back, held = batches[device]
                row, n = 0, p.numel()
                if self.capturable:
                    row = self._row_of(p).data_ptr()
                    counters.append((state["step"].data_ptr(), row, 0 if lr_tensor is None else lr_tensor.data_ptr(), lr, decay,
                                     beta1, beta2, _mix(self.seed + _GOLDEN * index),
                                     _native.DT_F64 if lr_tensor is not None and lr_tensor.dtype is torch.float64
                                     else _native.DT_F32, 0))
                else:
                    state["step"] = t = int(state["step"]) + 1
                    if t != last:
                        step_size, rbc2, last = lr / (1.0 - beta1 ** t), 1.0 / math.sqrt(1.0 - beta2 ** t), t
                if n == 0:
                    continue
                stepped.append(p)
                work, m, v = p, state["exp_avg"], state["exp_avg_sq"]
                if not (p.is_contiguous() and grad.is_contiguous() and m.is_contiguous() and v.is_contiguous()):
                    work, grad, m, v = self._laid_out(p, grad, state, bits, back)
                    held.append((work, grad))
                key = ms = vs = 0
                if bits == 8:
                    ms, vs = state["exp_avg_scale"].data_ptr(), state["exp_avg_sq_scale"].data_ptr()
                    if not row:
                        key = _mix(_mix(self.seed + _GOLDEN * index) + _GOLDEN * t)
                rows.append((work.data_ptr(), grad.data_ptr(), m.data_ptr(), v.data_ptr(), ms, vs, n, key, step_size, wdf,
                             beta1, 1.0 - beta1, beta2, 1.0 - beta2, rbc2, eps, _DTYPES[p.dtype], bits, row))
        # the kernels write behind autograd's back: a graph that has saved a parameter must not go on with its new values
        increment_version(stepped)
        for device, (rows, counters, back, _) in batches.items():
            device = torch.device("cuda", device)
            with _on_device(device):
                self._launch(device, rows, counters)
            for p, work in back:
                p.copy_(work)
        return loss

    def _check_capture(self, found):
        """What a captured step asks for: everything that it keeps exists, and stays where it is."""
        if not self.capturable:
            raise RuntimeError("AdamW.step is captured into a graph with capturable=True only: its bias corrections are "
                               "host values otherwise")
        for group, members in found:
            for _, p, _, state in members:
                if not state or p not in self._rows:
                    raise RuntimeError("AdamW capturable: a parameter's first step runs eagerly, before the capture")
                if group["state_bits"] == 32:
                    moments, dense = (state["exp_avg"], state["exp_avg_sq"]), _dense(p)
                    if not all(_dense(m) and _same_layout(m, p) if dense else m.is_contiguous() for m in moments):
                        raise RuntimeError("AdamW capturable: moments laid out otherwise than their parameter need an eager "
                                           "step before the capture")

    @staticmethod
    def _lr_of(lr):
        """(host value, None), or (0.0, device tensor) where the kernels read it."""
        if not isinstance(lr, torch.Tensor) or not lr.is_cuda:
            return float(lr), None
        if lr.numel() != 1 or lr.dtype not in (torch.float32, torch.float64):
            raise ValueError("a device lr is one fp32 or fp64 value, got {} of shape {}".format(lr.dtype, tuple(lr.shape)))
        return 0.0, lr

    def _row_of(self, p):
        row = self._rows.get(p)
        if row is None or row.get_device() != p.get_device():
            row = self._rows[p] = torch.zeros(3, dtype=torch.int64, device=p.device)
        return row

    @staticmethod
    def _laid_out(p, grad, state, bits, back):
        """Parameter, gradient and moments as runs of memory in one order; a parameter with gaps is stepped in a
        copy that `back` says to write back."""
        work = p
        if not _dense(p):
            work = p.contiguous()
            back.append((p, work))
        if not _same_layout(grad, work) or not _dense(grad):
            grad = torch.empty_like(work).copy_(grad)
        if bits == 32:
            for name in ("exp_avg", "exp_avg_sq"):
                if not _dense(state[name]) or not _same_layout(state[name], work):
                    state[name] = torch.empty_like(work, dtype=torch.float32).copy_(state[name])
        return work, grad, state["exp_avg"], state["exp_avg_sq"]

    def _launch(self, device, rows, counters):
        lib = _native.load()
        descs = _pack(rows)
        stream = torch.cuda.current_stream(device).cuda_stream
        if counters:
            _native.check(lib.gefenx_adamw_advance(_pack(counters, _COUNTER_STRUCT), len(counters), stream), "AdamW counters")
        coef = None
        if self.max_grad_norm is not None:
            bytes_ = int(lib.gefenx_adamw_norm_workspace_bytes(descs, len(rows)))
            ws = torch.empty(bytes_, dtype=torch.uint8, device=device)
            out = torch.empty(2, dtype=torch.float32, device=device)
            coef = out.data_ptr() + 4
            _native.check(lib.gefenx_adamw_norm(descs, len(rows), self.max_grad_norm, coef - 4, ws.data_ptr(), bytes_, stream),
                          "AdamW gradient norm")
            self.grad_norm = out[0]
        _native.check(lib.gefenx_adamw_step(descs, len(rows), coef, stream), "AdamW step")

    # ------------------------------------------------------------ moments

    @torch.no_grad()
    def moments(self, params=None):
        """[(exp_avg, exp_avg_sq), ...] in fp32 for each parameter (default:
        all, in group order), laid out as the state is: with 32 bits the
        state's own tensors, in the parameter's shape; with 8 the values that
        the codes stand for, flat, in the order the parameter is stored in
        (row by row where it has gaps).  None for a parameter that has not
        been stepped."""
        bits_of = {p: group["state_bits"] for group in self.param_groups for p in group["params"]}
        got, batches, known = [], {}, self.state
        for p in bits_of if params is None else params:
            bits = bits_of.get(p)
            if bits is None:
                raise ValueError("moments() of a tensor that this optimizer does not step")
            state = known.get(p)
            if not state:
                got.append(None)
                continue
            if bits == 32:
                got.append((state["exp_avg"], state["exp_avg_sq"]))
                continue
            if not _plainly_fits(p, state, bits):
                self._check_state(p, state, bits)
            m, v = state["exp_avg"], state["exp_avg_sq"]
            if not p.is_cuda:
                raise RuntimeError("AdamW reads 8-bit moments on a HIP device only; the parameter is on {}".format(p.device))
            n = p.numel()
            to_m, to_v = torch.empty_like(m, dtype=torch.float32), torch.empty_like(v, dtype=torch.float32)
            got.append((to_m, to_v))
            if n:
                batches.setdefault(p.get_device(), []).append(
                    (to_m.data_ptr(), to_v.data_ptr(), m.data_ptr(), v.data_ptr(), state["exp_avg_scale"].data_ptr(),
                     state["exp_avg_sq_scale"].data_ptr(), n, 0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, _native.DT_F32, 8, 0))
        for device, rows in batches.items():
            device = torch.device("cuda", device)
            with _on_device(device):
                _native.check(_native.load().gefenx_adamw_moments(
                    _pack(rows), len(rows), torch.cuda.current_stream(device).cuda_stream), "AdamW moments")
        return got

    # --------------------------------------------------------- checkpoint

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """Loads this class's checkpoints, and torch.optim.AdamW's where
        state_bits is 32 (fp32 moments from any floating type; amsgrad and
        maximize are refused).  The state is copied; a mismatch is refused
        before anything changes.  Hooks run as torch's class runs them: what
        pre-hooks return is loaded, post-hooks find it in place."""
        new, widths = {}, []

        def take(_, state_dict):  # after every pre-hook
            got, bits = self._loaded(state_dict)
            new.update(got)
            widths.extend(bits)
            return dict(state_dict, state={})  # torch's class would cast codes

        def install(_):  # before every post-hook
            for group, bits in zip(self.param_groups, widths):
                group["state_bits"] = bits
            self.state.clear()
            self.state.update(new)
        handles = [self.register_load_state_dict_pre_hook(take),
                   self.register_load_state_dict_post_hook(install, prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for handle in handles:
                handle.remove()

    def _loaded(self, state_dict):
        """What a checkpoint holds for this optimizer: ({parameter: state}, width of each group)."""
        groups, saved = self.param_groups, state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in saved]:
            raise ValueError("loaded state dict has other parameter groups than this optimizer")
        new, widths = {}, []
        for group, old in zip(groups, saved):
            bits = old.get("state_bits", group["state_bits"])
            widths.append(bits)
            if bits not in _STATE:
                raise ValueError("state_bits must be 8 or 32 but is: {!r}".format(bits))
            _refuse_variants(old)
            for p, i in zip(group["params"], old["params"]):
                entry = state_dict["state"].get(i)
                if not entry:
                    continue
                state = {"step": self._counter(p, int(entry["step"]))}
                for key, dtype in _STATE[bits].items():
                    t = entry.get(key)
                    if not torch.is_tensor(t):
                        raise ValueError("loaded state has no {} for state_bits={}".format(key, bits))
                    if bits == 32 and t.is_floating_point():
                        t = t.to(dtype)
                    # codes are moved as bytes
                    raw = t.view(torch.uint8) if t.dtype is torch.float8_e4m3fn else t
                    moved = raw.to(p.device, copy=True)
                    state[key] = moved.view(torch.float8_e4m3fn) if t.dtype is torch.float8_e4m3fn else moved
                if bits == 8:
                    # without an order: in that of the parameter that it is loaded for
                    order = entry["order"] if "order" in entry else _code_order(p)
                    # dims in ascending order: row-major by another name
                    state["order"] = None if order is None or list(order) == sorted(order) else tuple(order)
                self._check_state(p, state, bits)
                new[p] = state
        return new, widths
