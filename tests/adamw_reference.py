"""The AdamW step and its 8-bit state in plain torch on the CPU, for the tests.

`codes_m` / `codes_v` restate the two formats of gefenx_adamw_desc in the fp32
operations that define them (so codes compare for equality); `step64` is the
step's formula in float64.
"""
import torch

BLOCK = 256
TINY = 2.0 ** -126
GOLDEN = 0x9E3779B97F4A7C15
U64 = (1 << 64) - 1


def mix(z):
    z &= U64
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9 & U64
    z = (z ^ (z >> 27)) * 0x94D049BB133111EB & U64
    return z ^ (z >> 31)


def random16(key, n):
    """The 16 random bits of elements 0 .. n - 1, by integer arithmetic."""
    out = []
    for i in range(0, n, 4):
        z = mix(key + GOLDEN * (i // 4 + 1))
        out += [(z >> s) & 0xFFFF for s in (0, 16, 32, 48)]
    return torch.tensor(out[:n], dtype=torch.int64)


def step_key(seed, index, step):
    return mix(mix(seed + GOLDEN * (index + 1)) + GOLDEN * step)


def blocks(flat):
    return torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)


def codes_m(m):
    b = blocks(m)
    amax = b.abs().amax(1)
    scale = torch.where(torch.isfinite(amax), (amax * torch.tensor(1.0 / 448.0)).clamp(min=TINY),
                        torch.full_like(amax, float("nan")))
    code = (b * (1.0 / scale)[:, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return code.view(-1)[:m.numel()], scale


def codes_v(v, bits16):
    b = blocks(v)
    amax = b.amax(1)
    scale = torch.where(torch.isfinite(amax), amax.clamp(min=TINY), torch.full_like(amax, float("nan")))
    x = (b * (1.0 / scale)[:, None]).view(-1)[:v.numel()].contiguous()
    code = ((x.view(torch.int32).long() + (bits16 << 4)) >> 20) - 761
    return torch.where(v == 0, torch.zeros_like(code), code.clamp(1, 255)).to(torch.uint8), scale


def value_m(code, scale):
    return (blocks(code.float()) * scale[:, None]).view(-1)[:code.numel()]


def value_v(code, scale):
    c = code.int()
    x = torch.where(c == 0, torch.zeros_like(c), (c + 761) << 20).view(torch.float32)
    return (blocks(x) * scale[:, None]).view(-1)[:code.numel()]


def moments32(m, v, g, beta1, beta2):
    """The moments in fp32, each operation rounded."""
    f = lambda x: torch.tensor(x, dtype=torch.float32)  # noqa: E731
    return m * f(beta1) + g * f(1 - beta1), v * f(beta2) + (g * g) * f(1 - beta2)


def step64(p, g, m, v, t, lr, beta1, beta2, eps, wd, coef=1.0):
    """(p, m, v) after step t, in float64 from values of any type."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * coef
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    update = lr / (1 - beta1 ** t) * m / ((v / (1 - beta2 ** t)).sqrt() + eps)
    return p * (1 - lr * wd) - update, m, v


def tolerance(p64, update_scale, dtype):
    """Per element: the rounding of p to its type, and for the arithmetic before it 16 fp32 roundings of
    either term (fewer than that many operations produce them)."""
    unit = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    least = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}[dtype]
    return unit * p64.abs() + 16 * 2.0 ** -24 * (p64.abs() + update_scale) + least
