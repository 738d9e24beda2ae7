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

from gefen.gefen import _amp_gate, _amp_native_scaling_required, _on_device
from gefen.kernels import _native
from gefen.kernels.automatic_gefen_fused import _dtype_code

BLOCK = 256  # elements per scale of the 8-bit moments

_DESC_STRUCT = struct.Struct("<6QqQ8f2i")
assert _DESC_STRUCT.size == ctypes.sizeof(_native.AdamWDesc)
_DTYPES = frozenset((torch.float32, torch.float16, torch.bfloat16))
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


def _order(t: torch.Tensor):
    """None for a contiguous tensor, else its dims (of size > 1) from the
    largest stride to the smallest; ValueError where elements may overlap."""
    if t.is_contiguous():
        return None
    dims = sorted((d for d in range(t.dim()) if t.shape[d] > 1), key=lambda d: -t.stride(d))
    reach = 1  # elements spanned by the inner dims
    for d in reversed(dims):
        if t.stride(d) < reach:
            raise ValueError("AdamW cannot step a parameter whose elements share memory (shape {}, strides {})".format(
                tuple(t.shape), t.stride()))
        reach += (t.shape[d] - 1) * t.stride(d)
    return tuple(dims)


def _dense(t: torch.Tensor) -> bool:
    """Whether a tensor without overlap fills one run of memory."""
    return t.is_contiguous() or t.numel() == 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))


def _same_layout(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two dense tensors of one shape hold their elements in the same order."""
    if a.is_contiguous() and b.is_contiguous():
        return True
    return all(sa == sb for n, sa, sb in zip(a.shape, a.stride(), b.stride()) if n > 1)


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
    step does not wait for the GPU and cannot be captured into a graph (the
    bias corrections are host values).
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32,
                 max_grad_norm=None, seed=0):
        if max_grad_norm is not None and not (float(max_grad_norm) > 0.0 and math.isfinite(float(max_grad_norm))):
            raise ValueError("max_grad_norm must be positive and finite but is: {!r}".format(max_grad_norm))
        self.max_grad_norm = None if max_grad_norm is None else float(max_grad_norm)
        self.seed = int(seed)
        self.grad_norm = None
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
        super().add_param_group(param_group)

    def __getstate__(self):
        return dict(super().__getstate__(), max_grad_norm=self.max_grad_norm, seed=self.seed, grad_norm=self.grad_norm)

    @property
    def _step_supports_amp_scaling(self) -> bool:
        """The GradScaler protocol of Gefen: true fp16 gradients are unscaled here."""
        return _amp_native_scaling_required(self)

    # --------------------------------------------------------------- step

    def _validate_grads(self):
        """Refuse what cannot be stepped before anything moves."""
        devices = set()
        for group in self.param_groups:
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                if g.layout is not torch.strided:
                    raise RuntimeError("AdamW does not support sparse gradients")
                if hasattr(p, "placements") or hasattr(g, "placements"):
                    raise RuntimeError("AdamW does not step DTensor parameters")
                if p.device.type != "cuda" or g.device != p.device:
                    raise RuntimeError("AdamW steps HIP device parameters with gradients on the same device: parameter "
                                       "on {}, gradient on {}".format(p.device, g.device))
                if g.shape != p.shape:
                    raise RuntimeError("gradient shape {} does not match parameter shape {}".format(
                        tuple(g.shape), tuple(p.shape)))
                if p.dtype not in _DTYPES:
                    raise NotImplementedError("AdamW is not implemented for {}".format(p.dtype))
                if g.dtype is not p.dtype:
                    raise RuntimeError("gradient dtype {} does not match parameter dtype {}".format(g.dtype, p.dtype))
                if not p.is_contiguous():
                    _order(p)
                if self.state.get(p):
                    self._check_state(p, self.state[p], group["state_bits"])
                devices.add(p.device)
        if self.max_grad_norm is not None and len(devices) > 1:
            raise RuntimeError("AdamW with max_grad_norm steps parameters of one device, got {}".format(
                sorted(str(d) for d in devices)))

    @staticmethod
    def _check_state(p, state, bits):
        blocks = -(-p.numel() // BLOCK)
        for key, dtype in _STATE[bits].items():
            t = state.get(key)
            if not torch.is_tensor(t) or t.dtype is not dtype:
                raise ValueError("AdamW with state_bits={} needs {} as {}, got {}".format(
                    bits, key, dtype, t.dtype if torch.is_tensor(t) else type(t).__name__))
            if bits == 32:
                fits = t.shape == p.shape
            else:
                fits = t.numel() == (blocks if key.endswith("scale") else p.numel()) and t.is_contiguous()
            if not fits or t.device != p.device:
                raise ValueError("AdamW state {} (shape {}, {}) does not belong to a parameter of shape {} on {}".format(
                    key, tuple(t.shape), t.device, tuple(p.shape), p.device))
        if bits == 8 and state.get("order") != _order(p):
            raise ValueError("AdamW's 8-bit state follows the storage order of the parameter it was made for "
                             "({}); this one is stored as {}".format(state.get("order"), _order(p)))

    def _state_of(self, p, bits):
        state = self.state[p]
        if not state:
            state["step"] = 0
            if bits == 32:
                like = p if _dense(p) else p.contiguous()
                state["exp_avg"] = torch.zeros_like(like, dtype=torch.float32, memory_format=torch.preserve_format)
                state["exp_avg_sq"] = torch.zeros_like(like, dtype=torch.float32, memory_format=torch.preserve_format)
            else:
                blocks = -(-p.numel() // BLOCK)
                state["exp_avg"] = torch.zeros(p.numel(), dtype=torch.uint8, device=p.device).view(torch.float8_e4m3fn)
                state["exp_avg_sq"] = torch.zeros(p.numel(), dtype=torch.uint8, device=p.device)
                state["exp_avg_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
                state["exp_avg_sq_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
                state["order"] = _order(p)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._validate_grads()
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW.step cannot be captured into a graph: its bias corrections are host values")
        if not _amp_gate(self):
            return loss
        self.grad_norm = None
        batches = {}  # device -> descriptors, parameters to write back, tensors that the launch reads
        index = 0
        for group in self.param_groups:
            lr, (beta1, beta2), bits = float(group["lr"]), group["betas"], group["state_bits"]
            eps, wdf = float(group["eps"]), 1.0 - lr * float(group["weight_decay"])
            for p in group["params"]:
                index += 1
                grad = p.grad
                if grad is None:
                    continue
                state = self._state_of(p, bits)
                state["step"] = t = int(state["step"]) + 1
                if p.numel() == 0:
                    continue
                rows, back, held = batches.setdefault(p.device, ([], [], []))
                work = p
                if not _dense(p):
                    work = p.contiguous()
                    back.append((p, work))
                if not _same_layout(grad, work) or not _dense(grad):
                    grad = torch.empty_like(work).copy_(grad)
                m, v = state["exp_avg"], state["exp_avg_sq"]
                key = ms = vs = 0
                if bits == 8:
                    ms, vs = state["exp_avg_scale"].data_ptr(), state["exp_avg_sq_scale"].data_ptr()
                    key = _mix(_mix(self.seed + _GOLDEN * index) + _GOLDEN * t)
                else:
                    for name in ("exp_avg", "exp_avg_sq"):
                        if not _dense(state[name]) or not _same_layout(state[name], work):
                            state[name] = torch.empty_like(work, dtype=torch.float32).copy_(state[name])
                    m, v = state["exp_avg"], state["exp_avg_sq"]
                held.append((work, grad))
                rows.append((work.data_ptr(), grad.data_ptr(), m.data_ptr(), v.data_ptr(), ms, vs, p.numel(), key,
                             lr / (1.0 - beta1 ** t), wdf, beta1, 1.0 - beta1, beta2, 1.0 - beta2,
                             1.0 / math.sqrt(1.0 - beta2 ** t), eps, _dtype_code(p.dtype), bits))
        for device, (rows, back, _) in batches.items():
            with _on_device(device):
                self._launch(device, rows)
            for p, work in back:
                p.copy_(work)
        return loss

    def _launch(self, device, rows):
        lib = _native.load()
        descs = ctypes.create_string_buffer(len(rows) * _DESC_STRUCT.size)
        for i, row in enumerate(rows):
            _DESC_STRUCT.pack_into(descs, i * _DESC_STRUCT.size, *row)
        stream = torch.cuda.current_stream(device).cuda_stream
        coef = None
        if self.max_grad_norm is not None:
            bytes_ = int(lib.gefenx_adamw_norm_workspace_bytes(descs, len(rows)))
            ws = torch.empty(bytes_, dtype=torch.uint8, device=device)
            out = torch.empty(2, dtype=torch.float32, device=device)
            _native.check(lib.gefenx_adamw_norm(descs, len(rows), self.max_grad_norm, out.data_ptr(), ws.data_ptr(),
                                                bytes_, stream), "AdamW gradient norm")
            self.grad_norm = out[0]
            coef = out.data_ptr() + 4
        _native.check(lib.gefenx_adamw_step(descs, len(rows), coef, stream), "AdamW step")

    # ------------------------------------------------------------ moments

    @torch.no_grad()
    def moments(self, params=None):
        """[(exp_avg, exp_avg_sq), ...] in fp32 for each parameter (default:
        all, in group order), laid out as the state is: with 32 bits the
        state's own tensors, in the parameter's shape; with 8 the values that
        the codes stand for, flat, in the order the parameter is stored in.
        None for a parameter that has not been stepped."""
        bits_of = {p: group["state_bits"] for group in self.param_groups for p in group["params"]}
        got, batches = [], {}
        for p in bits_of if params is None else params:
            if p not in bits_of:
                raise ValueError("moments() of a tensor that this optimizer does not step")
            state = self.state.get(p)
            if not state:
                got.append(None)
                continue
            self._check_state(p, state, bits_of[p])
            if bits_of[p] == 32:
                got.append((state["exp_avg"], state["exp_avg_sq"]))
                continue
            m, v = (torch.empty(p.numel(), dtype=torch.float32, device=p.device) for _ in range(2))
            got.append((m, v))
            if p.numel():
                batches.setdefault(p.device, []).append(
                    (m.data_ptr(), v.data_ptr(), state["exp_avg"].data_ptr(), state["exp_avg_sq"].data_ptr(),
                     state["exp_avg_scale"].data_ptr(), state["exp_avg_sq_scale"].data_ptr(), p.numel(), 0,
                     0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0, _native.DT_F32, 8))
        for device, rows in batches.items():
            descs = b"".join(_DESC_STRUCT.pack(*row) for row in rows)
            with _on_device(device):
                _native.check(_native.load().gefenx_adamw_moments(
                    descs, len(rows), torch.cuda.current_stream(device).cuda_stream), "AdamW moments")
        return got

    # --------------------------------------------------------- checkpoint

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """Loads this class's checkpoints, and torch.optim.AdamW's where
        state_bits is 32 (fp32 moments from any floating type).  The state is
        copied; a mismatch is refused before anything changes."""
        groups, saved = self.param_groups, state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in saved]:
            raise ValueError("loaded state dict has other parameter groups than this optimizer")
        new = {}
        for group, old in zip(groups, saved):
            bits = old.get("state_bits", group["state_bits"])
            if bits not in _STATE:
                raise ValueError("state_bits must be 8 or 32 but is: {!r}".format(bits))
            for p, i in zip(group["params"], old["params"]):
                entry = state_dict["state"].get(i)
                if not entry:
                    continue
                state = {"step": int(entry["step"])}
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
                    # without an order: in the storage order of the parameter that it is loaded for
                    order = entry["order"] if "order" in entry else _order(p)
                    state["order"] = None if order is None else tuple(order)
                self._check_state(p, state, bits)
                new[p] = state
        super().load_state_dict({"state": {}, "param_groups": saved})
        for group in self.param_groups:
            group.setdefault("state_bits", self.defaults["state_bits"])
        self.state.clear()
        self.state.update(new)
