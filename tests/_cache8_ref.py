"""What the 8-bit KV cache holds, from its definition, in 64 bits on the CPU."""
import math

import torch

BLOCK = 64


def _pow2(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantised(x):
    """One block (64, D) of doubles that bf16 holds, as e4m3 with its scale holds them."""
    fin = torch.isfinite(x)
    y = torch.where(fin, x, torch.zeros_like(x))
    top = y.abs().max()
    if top == 0:
        e = torch.zeros((), dtype=torch.int32)
    else:
        m, e = torch.frexp(top / 448)  # top / 448 = m 2^e, 1/2 <= m < 1
        e = (e - (m == 0.5).int()).clamp(min=-100)
    z = y / _pow2(e)
    _, n = torch.frexp(z)
    step = _pow2((n - 1).clamp(min=-6) - 3)
    z = torch.round(z / step) * step * _pow2(e)
    return torch.where(fin, z, torch.full_like(z, math.nan))


def held(x, length):
    """Rows (H, n, D) of one sequence of `length` positions as the cache holds them."""
    y = x[:, :length].to(torch.bfloat16).double()
    for h in range(y.shape[0]):
        for b in range(length // BLOCK):
            s = slice(b * BLOCK, (b + 1) * BLOCK)
            y[h, s] = quantised(y[h, s])
    return y


def attend(q, k, v, scale, window, sinks):
    """q (Hq, T, D) of the last T of the positions of k, v (H, n, D): o and sum p |v|."""
    q = q.double()
    n, T, G = k.shape[1], q.shape[1], q.shape[0] // k.shape[0]
    k, v = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
    i, j = (n - T + torch.arange(T))[:, None], torch.arange(n)[None]
    m = j <= i
    if window:
        m = m & ((i - j < window) | (j < sinks))
    s = (q @ k.transpose(1, 2) * scale).masked_fill(~m, -math.inf)
    lse = torch.logsumexp(s, -1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isneginf(lse), torch.zeros_like(lse), lse))
    p = torch.where(m, p, torch.zeros_like(p))
    if torch.isfinite(v).all():
        return p @ v, p @ v.abs()
    o = torch.zeros(q.shape[0], T, v.shape[2], dtype=torch.float64)
    for x in range(n):
        o += torch.where(m[:, x:x + 1], p[:, :, x:x + 1] * v[:, x:x + 1], torch.zeros((), dtype=torch.float64))
    return o, o.abs()
