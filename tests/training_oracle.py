"""The operators around the cast in 64 bits, from their definitions, and the
random NVFP4 operands their tests use."""
import math

import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
BLOCK = 128


def half_step(dtype) -> float:
    """Largest relative error of one rounding to nearest."""
    return torch.finfo(dtype).eps / 2


def least_step(dtype) -> float:
    """Spacing of the subnormal numbers."""
    f = torch.finfo(dtype)
    return f.smallest_normal * f.eps


def random_operand(rows, k, seed, amax=3.0):
    """Random codes (all sixteen), finite positive E4M3 scales of several binades, an amax."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (rows, k // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(0x28, 0x60, (rows, k // 16), generator=g, dtype=torch.uint8)
    return codes, scales, torch.tensor([amax], dtype=torch.float32)


def e4m3(scales):
    return scales.view(torch.float8_e4m3fn).double()


def operand_values(codes, scales, amax):
    rows, half = codes.shape
    x = torch.empty(rows, 2 * half, dtype=torch.float64)
    for odd in (0, 1):
        c = (codes >> (4 * odd)) & 15
        x[:, odd::2] = E2M1[(c & 7).long()] * (1.0 - 2.0 * (c >> 3).double())
    x = x * e4m3(scales).repeat_interleave(16, dim=1)
    a = float(amax)
    return x * (1.0 if a == 0 else 1.0 / min(2688.0 / a, torch.finfo(torch.float32).max))


def act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def act_slope(z, name):
    if name == "relu":
        return (z > 0).double()
    if name == "gelu":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z ** 2)
    if name == "silu":
        q = torch.sigmoid(z)
        return q * (1 + z * (1 - q))
    return torch.ones_like(z)


def layernorm(x, gamma, beta, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    y = (x - mean) * rstd * gamma.double()
    if beta is not None:
        y = y + beta.double()
    return y, mean[:, 0], rstd[:, 0]


def layernorm_backward(dy, x, mean, rstd, gamma, residual):
    dy, h = dy.double(), (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    u = dy * gamma.double()
    dx = rstd.double()[:, None] * (u - u.mean(1, keepdim=True) - h * (u * h).mean(1, keepdim=True))
    if residual is not None:
        dx = dx + residual.double()
    return dx, (dy * h).sum(0), dy.sum(0)


def unpack8(codes, scales, moment):
    steps = 8 if moment == "exp_avg" else 16
    c = codes.long()
    sign = torch.ones(c.shape, dtype=torch.float64)
    if moment == "exp_avg":
        sign = 1.0 - 2.0 * (c >> 7).double()
        c = c & 127
    e, f = c // steps, (c % steps).double()
    y = torch.where(e == 0, f / steps * 2.0 ** -6, (1 + f / steps) * 2.0 ** (e.double() - 7))
    s = torch.where(scales == 255, torch.tensor(float("nan"), dtype=torch.float64),
                    2.0 ** (scales.double() - 127))
    s = torch.where(scales == 0, torch.zeros_like(s), s)
    return sign * y * s.repeat_interleave(BLOCK)[:c.numel()]


def philox(seed, offset, index):
    """Philox4x32-10, key = seed, counter = (offset, index), in Python integers."""
    mask = 0xFFFFFFFF
    c = [offset & mask, (offset >> 32) & mask, index & mask, (index >> 32) & mask]
    k = [seed & mask, (seed >> 32) & mask]
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & mask, (p0 >> 32) ^ c[3] ^ k[1], p0 & mask]
        k = [(k[0] + 0x9E3779B9) & mask, (k[1] + 0xBB67AE85) & mask]
    return c


def adamw(p, g, m, v, *, lr, beta1, beta2, eps, step, wd, grad_scale=1.0):
    p, g, m, v = (t.double() for t in (p, g, m, v))
    g = g * grad_scale
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    den = torch.sqrt(v / (1 - beta2 ** step)) + eps
    return (1 - lr * wd) * p - lr / (1 - beta1 ** step) * m / den, m, v
