"""One AdamW step in 64 bits and the 8-bit moments' format, restated with whole tensors.

e4m3 with random rounding: of t = |x| / scale (scale = the block's largest / 448) the multiple of the step
of t's binade (2^(e - 3), at least 2^-9) at or below t + u / 2^16 of that step, u = 16 bits of the hash."""
import math

import torch

BLOCK = 256


def mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def key(place, step, seed):
    k = mix((seed & 0xFFFFFFFF) ^ mix((seed >> 32) ^ mix(step)))
    return mix((k + 0x9E3779B9 * (place + 1)) & 0xFFFFFFFF)


def step64(p, g, m, v, t, lr, betas, eps, weight_decay, scale=1.0):
    p, g, m, v = p.double(), g.double() * scale, m.double(), v.double()
    b1, b2 = betas
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    d = v.sqrt() / math.sqrt(1 - b2 ** t) + eps
    return p - lr * weight_decay * p - lr / (1 - b1 ** t) * m / d, m, v


def sqrt32(x):
    """The fp32 root, rounded once (torch's vectorised CPU root is not always): through 64 bits, where a second
    rounding cannot change it (53 >= 2 * 24 + 2 bits)."""
    return x.double().sqrt().float()


def step32(p, g, m, v, t, lr, betas, eps, weight_decay, scale=None):
    """The kernels' own order of fp32 operations (each product, sum, quotient and root rounded), on the CPU."""
    f = lambda x: torch.tensor(x, dtype=torch.float32)
    b1, b2 = betas
    x = g.float() if scale is None else g.float() * f(scale)
    m = m * f(b1) + x * f(1 - b1)
    v = v * f(b2) + (x * x) * f(1 - b2)
    d = sqrt32(v) * f(1 / math.sqrt(1 - b2 ** t)) + f(eps)
    return p.float() * f(1 - lr * weight_decay) - (m / d) * f(lr / (1 - b1 ** t)), m, v


def blocks(x):
    return torch.nn.functional.pad(x.reshape(-1), (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def decode(q, s, n):
    """The n numbers that (e4m3, scale a block) stand for."""
    return (blocks(q.reshape(-1).float()) * s[:, None]).reshape(-1)[:n]


def encode32(x, u):
    """x [n, BLOCK] fp32 -> (values on the e4m3 grid with their sign, scale), in fp32 as the kernel does."""
    top = x.abs().amax(1, keepdim=True)
    live = top >= 1e-30
    one = torch.full_like(top, 448.0)
    t = (x.abs() * torch.where(live, one / top, torch.zeros_like(top))).clamp(max=448.0)
    step = torch.exp2(torch.frexp(t).exponent.sub(1).clamp(min=-6).double() - 3)
    v = (((t.double() / step) + u.double() / 65536).floor() * step).float()
    return v.clamp(max=448.0) * x.sign(), torch.where(live, top / one, torch.zeros_like(top))[:, 0]


def step8(p, g, m8, ms, r8, rs, t, k, lr, betas, eps, weight_decay, scale=None):
    """The 8-bit step in the kernel's own operations: (p fp32, m8 values, ms, r8 values, rs)."""
    n = p.numel()
    m, r = decode(m8, ms, n), decode(r8, rs, n)
    p1, m1, v1 = step32(p.reshape(-1), g.reshape(-1), m, r * r, t, lr, betas, eps, weight_decay, scale)
    r1 = sqrt32(v1)
    u = mix(torch.arange(-(-n // BLOCK) * BLOCK) ^ k).view(-1, BLOCK)
    mq, mso = encode32(blocks(m1), u & 0xFFFF)
    rq, rso = encode32(blocks(r1), u >> 16)
    rq = torch.where((blocks(r1) > 0) & (rso > 0)[:, None], rq.clamp(min=2.0 ** -9), rq)
    return p1.view(p.shape), mq.reshape(-1)[:n].view(p.shape), mso, rq.reshape(-1)[:n].view(p.shape), rso
