"""The sliding-window attention's definition in 64 bits, with the absolute sums that bound
what rounding to bf16 may change. Torch, CPU."""
import math

import torch


def sees(Sq, Sk, window, sinks, kv_len=None, device="cpu"):
    """(B or 1, 1, Sq, Sk)"""
    i, j = torch.arange(Sq, device=device)[:, None], torch.arange(Sk, device=device)[None, :]
    m = ((j <= i) & ((i - j < window) | (j < sinks)))[None, None]
    return m if kv_len is None else m & (j < torch.tensor(kv_len, device=device)[:, None, None, None])


def _masked(x, m):
    return torch.where(m, x, torch.zeros((), dtype=x.dtype, device=x.device))


def _mm(p, x, m):
    """sum_j p_ij x_j over the pairs of m only: 0 times an infinity counts for nothing."""
    if torch.isfinite(x).all():
        return p @ x
    out = torch.zeros(*p.shape[:-1], x.shape[-1], dtype=p.dtype)
    for j in range(x.shape[-2]):
        out += torch.where(m[..., j:j + 1], p[..., j:j + 1] * x[..., j:j + 1, :], torch.zeros((), dtype=p.dtype))
    return out


def fwd(q, k, v, scale, window, sinks, kv_len=None, device="cpu"):
    """o, lse, and sum_j p |v|."""
    q, k, v = (x.detach().to(device).double() for x in (q, k, v))
    G = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    m = sees(q.shape[2], k.shape[2], window, sinks, kv_len, device).expand(q.shape[0], q.shape[1], -1, -1)
    s = (q @ k.transpose(-1, -2) * scale).masked_fill(~m, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = _masked(torch.exp(s - torch.where(torch.isinf(lse) & (lse < 0), torch.zeros_like(lse), lse)[..., None]), m)
    return _mm(p, v, m), lse, _mm(p, v.abs(), m)


def bwd(q, k, v, o, lse, dO, scale, window, sinks, kv_len=None, device="cpu"):
    """(dq, dk, dv), their absolute sums, and the sums with |dO| |v| + |dO| |o| in the place of
    |dS / P|: the difference dP - delta keeps the roundings of both, however small it is."""
    q, k, v, o, lse, dO = (x.detach().to(device).double() for x in (q, k, v, o, lse, dO))
    B, H, Sq, D = q.shape
    Hkv, Sk = k.shape[1:3]
    G = H // Hkv
    kh, vh = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    m = sees(Sq, Sk, window, sinks, kv_len, device).expand(B, H, -1, -1)
    mt = m.transpose(-1, -2)
    lse = lse.view(B, H, Sq, 1)
    s = (q @ kh.transpose(-1, -2) * scale).masked_fill(~m, -math.inf)
    p = _masked(torch.exp(s - torch.where(torch.isinf(lse) & (lse < 0), torch.zeros_like(lse), lse)), m)
    ds = _masked(p * (dO @ vh.transpose(-1, -2) - (dO * o).sum(-1, keepdim=True)), m)
    group = lambda x: x.view(B, Hkv, G, Sk, D).sum(2)  # noqa: E731
    grads = (_mm(ds, kh, m) * scale, group(_mm(ds.transpose(-1, -2), q, mt)) * scale,
             group(_mm(p.transpose(-1, -2), dO, mt)))
    sums = (_mm(ds.abs(), kh.abs(), m) * abs(scale), group(_mm(ds.abs().transpose(-1, -2), q.abs(), mt)) * abs(scale),
            group(_mm(p.transpose(-1, -2), dO.abs(), mt)))
    ns = _masked(p * (dO.abs() @ vh.abs().transpose(-1, -2) + (dO * o).abs().sum(-1, keepdim=True)), m)
    noise = (_mm(ns, kh.abs(), m) * abs(scale), group(_mm(ns.transpose(-1, -2), q.abs(), mt)) * abs(scale),
             torch.zeros_like(k))
    return grads, sums, noise


def check(got, ref, total, what, noise=None):
    """bf16: each weight and the result are rounded once, by at most half a step (2^-8
    relative each), sums are in fp32. fp32: the root of about a thousand roundings.
    noise: dP and delta are sums of up to 128 products in at most 48 + 8 accumulations
    (six piece products of eight 16-element steps, and the pieces' own 2^-25), each off by
    at most 2^-24 of the products' absolute sum: under 2^-18 of it together. A query that
    sees one key has dS = 0 and nothing but that."""
    g = got.detach().cpu().double()
    ref, total = ref.cpu(), total.cpu()
    noise = noise if noise is None else noise.cpu()
    assert g.shape == ref.shape, what
    assert torch.equal(torch.isnan(g), torch.isnan(ref)), f"{what}: NaN in other places"
    ok = torch.isfinite(ref)
    assert torch.equal(g[~ok & ~torch.isnan(ref)], ref[~ok & ~torch.isnan(ref)]), what
    d = (g - ref)[ok].abs()
    if got.dtype == torch.bfloat16:
        # 2^-14: the fp32 exponents and sums beside the two roundings.
        bound = 2.0 ** -8 * (ref.abs() + total)[ok] * (1 + 2.0 ** -6) + 2.0 ** -14 * total[ok] + 1e-38
        if noise is not None:
            bound += 2.0 ** -18 * noise[ok]
        worst = (d / bound).max().item() if d.numel() else 0.0
        print(f"[{what}] bf16 worst {worst:.3f} of the bound", flush=True)
        assert worst <= 1.0, (what, worst)
    else:
        n = torch.linalg.norm(ref[ok]).item()
        off = torch.linalg.norm(d).item()
        bound = 2.0 ** -24 * 32 * n
        if noise is not None:
            bound += 2.0 ** -18 * torch.linalg.norm(noise[ok]).item()
        print(f"[{what}] fp32 rel {off / max(n, 1e-300):.2e}, {off / max(bound, 1e-300):.2f} of the bound", flush=True)
        assert off <= bound, (what, off, bound)
