"""Sliding-window attention with sinks (attn_window_fwd, attn_window_bwd) against its
definition in 64 bits: element types, shared key heads, lengths from one, cross lengths,
padding, rows without keys, infinities in masked places, graphs, streams, refusals."""
import math

import pytest

from tests import _window_ref as ref

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

# B, H, Hkv, Sq, Sk, D, window, sinks, kv_len
CASES = [
    (1, 1, 1, 1, 1, 64, 1, 0, None),
    (2, 4, 2, 33, 33, 64, 7, 3, None),
    (1, 2, 1, 130, 130, 128, 64, 0, None),
    (1, 2, 2, 257, 257, 128, 100, 70, None),
    (2, 3, 1, 200, 200, 64, 1000, 0, None),          # wider than the sequence
    (3, 2, 2, 150, 90, 64, 16, 2, (0, 37, 90)),      # padded, queries past every key
    (2, 2, 1, 150, 90, 128, 16, 0, (20, 90)),        # rows that see nothing
    (1, 2, 1, 40, 300, 128, 25, 4, None),            # keys no query reaches
    (1, 1, 1, 515, 515, 64, 1, 1, None),
    (2, 5, 5, 321, 321, 128, 33, 130, (321, 200)),   # sinks over several blocks
    (4, 16, 4, 256, 256, 64, 40, 5, None),           # 64-row blocks
    (16, 16, 16, 200, 200, 64, 50, 3, (200,) * 15 + (77,)),  # 128-row blocks
    (16, 16, 16, 150, 150, 128, 64, 0, None),
    # Large grids with shared key heads: items over several query heads.
    (8, 64, 32, 300, 300, 64, 40, 5, (300, 1, 64, 128, 129, 200, 299, 0)),
    (4, 64, 32, 260, 300, 128, 100, 140, None),
    (2, 32, 16, 1100, 1100, 64, 128, 4, None),
    (2, 32, 16, 1100, 1100, 128, 70, 32, (1100, 20)),
    (1, 3, 1, 700, 640, 128, 50, 7, None),           # queries past every key but the sinks
]


def _data(c, dtype, seed=0):
    B, H, Hkv, Sq, Sk, D = c[:6]
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(s, generator=g).to(dtype).cuda()  # noqa: E731
    return mk(B, H, Sq, D), mk(B, Hkv, Sk, D), mk(B, Hkv, Sk, D), mk(B, H, Sq, D)


def _len(kv):
    return None if kv is None else torch.tensor(kv, dtype=torch.int32).cuda()


def _check_lse(lse, r, what):
    l = lse.cpu().double().view(r.shape)
    ok = torch.isfinite(r)
    assert torch.equal(l[~ok], r[~ok]), what
    # Scores of fp32 sums of up to 128 products whose absolute values add up to about ten.
    assert ((l - r)[ok].abs() <= 2.0 ** -16 * r[ok].abs().clamp(min=1)).all(), what


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("c", CASES, ids=lambda c: "x".join(map(str, c[:8])))
def test_forward_and_backward(c, dtype):
    from gonn_amd import hip
    window, sinks, kv = c[6:]
    q, k, v, dO = _data(c, dtype)
    scale = 1.0 / math.sqrt(c[5])
    o, lse = hip.attn_window_fwd(q, k, v, window=window, sinks=sinks, kv_len=_len(kv))
    assert o.dtype == dtype and lse.dtype == torch.float32 and lse.shape == (c[0] * c[1], c[3])
    ro, rl, ra = ref.fwd(q, k, v, scale, window, sinks, kv)
    ref.check(o, ro, ra, f"o {c}")
    _check_lse(lse, rl, c)
    grads = hip.attn_window_bwd(q, k, v, o, lse, dO, window=window, sinks=sinks, kv_len=_len(kv))
    rg, rs, rn = ref.bwd(q, k, v, o, lse, dO, scale, window, sinks, kv)
    for name, g, r, s, n in zip(("dq", "dk", "dv"), grads, rg, rs, rn):
        ref.check(g, r, s, f"{name} {c}", n)
    again = hip.attn_window_bwd(q, k, v, o, lse, dO, window=window, sinks=sinks, kv_len=_len(kv))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("c", [(1, 32, 32, 4500, 4500, 64, 70, 4, None), (2, 32, 16, 2700, 2690, 128, 40, 32, (2690, 31))],
                         ids=lambda c: "x".join(map(str, c[:8])))
def test_long_sequences_with_sinks(c, dtype):
    """So many later queries of the sinks that they have items of their own. The reference
    in 64 bits on the GPU."""
    from gonn_amd import hip
    window, sinks, kv = c[6:]
    q, k, v, dO = _data(c, dtype, 13)
    scale = 1.0 / math.sqrt(c[5])
    o, lse = hip.attn_window_fwd(q, k, v, window=window, sinks=sinks, kv_len=_len(kv))
    ro, rl, ra = ref.fwd(q, k, v, scale, window, sinks, kv, "cuda")
    ref.check(o, ro, ra, f"o {c}")
    _check_lse(lse, rl.cpu(), c)
    del ro, rl, ra
    grads = hip.attn_window_bwd(q, k, v, o, lse, dO, window=window, sinks=sinks, kv_len=_len(kv))
    rg, rs, rn = ref.bwd(q, k, v, o, lse, dO, scale, window, sinks, kv, "cuda")
    for name, g, r, s, n in zip(("dq", "dk", "dv"), grads, rg, rs, rn):
        ref.check(g, r, s, f"{name} {c}", n)
    again = hip.attn_window_bwd(q, k, v, o, lse, dO, window=window, sinks=sinks, kv_len=_len(kv))
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_gradients_against_differences():
    """Central differences of sum(O dO) in fp32: step 2^-6, whose own error is of order
    step^2 = 2^-12 of the third derivative and 2^-24 / step of the sum's rounding."""
    from gonn_amd import hip
    c = (1, 4, 2, 50, 50, 64, 9, 2, None)
    q, k, v, dO = _data(c, torch.float32, 3)
    o, lse = hip.attn_window_fwd(q, k, v, window=9, sinks=2)
    grads = hip.attn_window_bwd(q, k, v, o, lse, dO, window=9, sinks=2)
    f = lambda: (hip.attn_window_fwd(q, k, v, window=9, sinks=2)[0].double() * dO.double()).sum().item()  # noqa: E731
    h = 2.0 ** -6
    for x, g in zip((q, k, v), grads):
        d = torch.randn(x.shape, generator=torch.Generator().manual_seed(5)).cuda()
        d /= d.norm()
        x0 = x.clone()
        x.copy_(x0 + h * d)
        up = f()
        x.copy_(x0 - h * d)
        down = f()
        x.copy_(x0)
        want = (g.double() * d.double()).sum().item()
        assert abs((up - down) / (2 * h) - want) <= 2e-3 * max(1.0, g.norm().item() / math.sqrt(g.numel())), (up, down, want)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("big", [False, True])
def test_scales(scale, dtype, big):
    from gonn_amd import hip
    c = (16, 32, 16, 100, 100, 64, 30, 4, None) if big else (1, 2, 1, 100, 100, 64, 30, 4, None)
    q, k, v, dO = _data(c, dtype, 7)
    if scale == 3.0:
        q *= 0.25
    o, lse = hip.attn_window_fwd(q, k, v, window=30, sinks=4, scale=scale)
    ro, rl, ra = ref.fwd(q, k, v, scale, 30, 4)
    ref.check(o, ro, ra, f"o scale {scale}")
    _check_lse(lse, rl, scale)
    grads = hip.attn_window_bwd(q, k, v, o, lse, dO, window=30, sinks=4, scale=scale)
    rg, rs, rn = ref.bwd(q, k, v, o, lse, dO, scale, 30, 4)
    for g, r, s, n in zip(grads, rg, rs, rn):
        ref.check(g, r, s, f"grad scale {scale}", n)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("bad", [math.inf, math.nan], ids=["inf", "nan"])
@pytest.mark.parametrize("S,big", [(70, False), (330, False), (100, True)])
def test_bad_values_reach_only_those_that_see_them(dtype, bad, S, big):
    from gonn_amd import hip
    c = (2, 4, 2, S, S, 64, 20, 3, (S, S - 30))
    if big:  # the kernels of large grids
        c = (32, 16, 8, S, S, 64, 20, 3, (S, S - 30) * 16)
    window, sinks, kv = c[6:]
    scale = 1.0 / 8
    for where in ("v", "k", "q", "dO", "pad"):
        q, k, v, dO = _data(c, dtype, 11)
        x = {"v": v, "k": k, "q": q, "dO": dO, "pad": v}[where]
        if where == "pad":
            k[1, :, S - 30:] = bad
            v[1, :, S - 30:] = bad
        else:
            x[0, 1, 37, 5] = bad
        o, lse = hip.attn_window_fwd(q, k, v, window=window, sinks=sinks, kv_len=_len(kv))
        ro, rl, ra = ref.fwd(q, k, v, scale, window, sinks, kv)
        seen = torch.isfinite(ro).all(-1)
        g = o.cpu().double()
        assert torch.equal(torch.isfinite(g).all(-1), seen), where
        ref.check(torch.where(seen[..., None], o.cpu(), torch.zeros((), dtype=dtype)),
                  torch.where(seen[..., None], ro, torch.zeros((), dtype=torch.float64)),
                  torch.where(seen[..., None], ra, torch.zeros((), dtype=torch.float64)), where)
        # The saved statistics of the clean call, so that only the gradients see the value.
        if where in ("v", "k", "q"):
            continue
        grads = hip.attn_window_bwd(q, k, v, o, lse, dO, window=window, sinks=sinks, kv_len=_len(kv))
        rg, rs, rn = ref.bwd(q, k, v, o, lse, dO, scale, window, sinks, kv)
        for name, a, r, s, n in zip(("dq", "dk", "dv"), grads, rg, rs, rn):
            fine = torch.isfinite(r)
            assert torch.equal(torch.isfinite(a.cpu()).all(-1), fine.all(-1)), (where, name)
            keep = fine.all(-1)[..., None]
            z = torch.zeros((), dtype=torch.float64)
            ref.check(torch.where(keep, a.cpu(), torch.zeros((), dtype=dtype)), torch.where(keep, r, z),
                      torch.where(keep, s, z), f"{where} {name}", torch.where(keep, n, z))


def test_many_bad_rows_finish():
    """A diverged training step: everything NaN in, everything NaN out."""
    from gonn_amd import hip
    c = (1, 2, 1, 300, 300, 128, 64, 4, None)
    q, k, v, dO = (torch.full_like(x, math.nan) for x in _data(c, torch.bfloat16))
    o, lse = hip.attn_window_fwd(q, k, v, window=64, sinks=4)
    assert torch.isnan(o).all() and torch.isnan(lse).all()
    assert all(torch.isnan(g).all() for g in hip.attn_window_bwd(q, k, v, o, lse, dO, window=64, sinks=4))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_graph_and_streams(dtype):
    from gonn_amd import hip
    c = (2, 4, 2, 300, 300, 64, 40, 4, (300, 170))
    q, k, v, dO = _data(c, dtype, 21)
    kv = _len(c[8])

    def step():
        o, lse = hip.attn_window_fwd(q, k, v, window=40, sinks=4, kv_len=kv)
        return (o, lse, *hip.attn_window_bwd(q, k, v, o, lse, dO, window=40, sinks=4, kv_len=kv))

    step()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for gr in graphs:
        with torch.cuda.graph(gr):
            outs.append(step())
    # Larger eager calls in between: the shared workspace grows and moves.
    big = _data((4, 8, 4, 600, 600, 64, 40, 4, None), dtype)
    bo, bl = hip.attn_window_fwd(*big[:3], window=40, sinks=4)
    hip.attn_window_bwd(*big[:3], bo, bl, big[3], window=40, sinks=4)
    for seed in (31, 32, 33):
        for x, y in zip((q, k, v, dO), _data(c, dtype, seed)):
            x.copy_(y)
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        side = [torch.cuda.Stream(), torch.cuda.Stream()]
        for gr, s in zip(graphs, side):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    o, lse = hip.attn_window_fwd(q, k, v, window=40, sinks=4, kv_len=kv, stream=other)
    g = hip.attn_window_bwd(q, k, v, o, lse, dO, window=40, sinks=4, kv_len=kv, stream=other)
    other.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((o, lse, *g), want))


def test_wide_window_is_the_causal_attention():
    """Beside the causal kernels: a window over everything, fp32, the fp32 mode's bar twice."""
    from gonn_amd import hip
    q, k, v, dO = _data((2, 3, 3, 200, 200, 64, 0, 0, None), torch.float32, 41)
    o, lse = hip.attn_window_fwd(q, k, v, window=200)
    co, cl = hip.attn_fwd(q, k, v, causal=True)
    assert (o - co).norm() <= 2.0 ** -18 * co.norm() and (lse - cl).abs().max() <= 2.0 ** -18 * cl.abs().max()
    g = hip.attn_window_bwd(q, k, v, o, lse, dO, window=200)
    for a, b in zip(g, hip.attn_bwd(q, k, v, co, cl, dO, causal=True)):
        assert (a - b).norm() <= 2.0 ** -18 * b.norm()


def test_refusals():
    from gonn_amd import hip
    q, k, v, dO = _data((1, 4, 2, 40, 40, 64, 0, 0, None), torch.bfloat16)
    for kw in ({"window": 0}, {"window": -3}, {"window": 4, "sinks": -1}, {"window": 4, "scale": math.inf}):
        with pytest.raises(hip.GonnHipError):
            hip.attn_window_fwd(q, k, v, **kw)
    with pytest.raises(ValueError):
        hip.attn_window_fwd(q[:, :3].contiguous(), k, v, window=4)  # 3 heads over 2
    with pytest.raises(TypeError):
        hip.attn_window_fwd(q, k.float(), v, window=4)
    with pytest.raises(ValueError):
        hip.attn_window_fwd(q.transpose(1, 2), k, v, window=4)
    with pytest.raises(ValueError):
        hip.attn_window_fwd(q, k, v, window=4, out=torch.empty_like(k))
    with pytest.raises(hip.GonnHipError):  # one byte pair off the alignment
        flat = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")[1:]
        hip.attn_window_fwd(q, k, v, window=4, out=flat.view(q.shape))
    with pytest.raises((ValueError, RuntimeError)):
        hip.attn_window_fwd(q, k.cpu(), v.cpu(), window=4)
    o, lse = hip.attn_window_fwd(q, k, v, window=4)
    with pytest.raises(ValueError):
        hip.attn_window_bwd(q, k, v, o.float(), lse, dO, window=4)
    with pytest.raises(hip.GonnHipError):
        hip.attn_window_bwd(q, k, v, o, lse[:2].contiguous(), dO, window=4)


def test_windows_past_32_bits_are_the_widest():
    from gonn_amd import hip
    q, k, v, dO = _data((1, 2, 1, 90, 90, 64), torch.bfloat16, 31)
    o, lse = hip.attn_window_fwd(q, k, v, window=90)
    want = hip.attn_window_bwd(q, k, v, o, lse, dO, window=90)
    for window, sinks in ((2 ** 31 - 1, 0), (2 ** 32 + 5, 2 ** 32 + 1), (2 ** 63, 2 ** 31 - 1)):
        o2, lse2 = hip.attn_window_fwd(q, k, v, window=window, sinks=sinks)
        assert torch.equal(o2, o) and torch.equal(lse2, lse)
        got = hip.attn_window_bwd(q, k, v, o, lse, dO, window=window, sinks=sinks)
        for a, b in zip(got, want):  # other items, another order of the sums
            assert ((a.double() - b.double()).abs() <= 2.0 ** -6 * b.double().abs() + 2.0 ** -8).all()
    with pytest.raises(hip.GonnHipError):
        hip.attn_window_fwd(q, k, v, window=2 ** 32 + 5, sinks=-2 ** 32)


def test_offsets_past_32_bits():
    """Tensors of more than 2^32 elements: the last head's last rows, which see the last keys
    and the sinks. The reference is the same attention with the rows between left out; it
    holds for the queries whose windows end within what is kept."""
    from gonn_amd import hip
    B, H, S, D, window, sinks, keep, n = 8, 8, 524_353, 128, 100, 3, 512, 256
    assert B * H * S * D > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(3)
    mk = lambda: torch.randn(B, H, S, D, generator=g, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    q, k, v, dO = (mk() for _ in range(4))
    o, lse = hip.attn_window_fwd(q, k, v, window=window, sinks=sinks)
    grads = hip.attn_window_bwd(q, k, v, o, lse, dO, window=window, sinks=sinks)
    part = lambda x: torch.cat([x[-1:, -1:, :64], x[-1:, -1:, S - keep:]], 2).cpu()  # noqa: E731
    last = lambda x: x[..., -n:, :]  # noqa: E731
    scale = 1.0 / math.sqrt(D)
    ro, rl, ra = ref.fwd(part(q), part(k), part(v), scale, window, sinks)
    ref.check(last(part(o)), last(ro), last(ra), "o")
    le = part(lse.view(B, H, S, 1))[..., 0]
    _check_lse(le[..., -n:], rl[..., -n:], "lse")
    rg, rs, rn = ref.bwd(part(q), part(k), part(v), part(o), le, part(dO), scale, window, sinks)
    for name, x, r, s, m in zip(("dq", "dk", "dv"), grads, rg, rs, rn):
        ref.check(last(part(x)), last(r), last(s), name, last(m))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("shape", [(2, 4, 2, 70, 70, 64), (8, 64, 32, 200, 200, 64), (4, 64, 16, 130, 140, 128)],
                         ids=lambda c: "x".join(map(str, c)))
def test_outputs_given_and_neighbours_untouched(shape, dtype):
    """Outputs inside larger tensors: what lies before and behind them stays as it was, and
    rows behind k's and v's last (infinite here) are not read."""
    from gonn_amd import hip
    B, H, Hkv, Sq, Sk, D = shape
    q, k, v, dO = _data(shape, dtype, 41)
    o, lse = hip.attn_window_fwd(q, k, v, window=30, sinks=3)
    assert hip.attn_window_fwd(q, k, v, window=30, sinks=3, lse=False)[1] is None
    want = (o, lse, *hip.attn_window_bwd(q, k, v, o, lse, dO, window=30, sinks=3))
    pad, flag = 256, -7.0  # elements: keeps 16 bytes

    def inside(t, fill=flag):
        big = torch.full((t.numel() + 2 * pad,), fill, dtype=t.dtype, device="cuda")
        x = big[pad:pad + t.numel()].view(t.shape)
        x.copy_(t)
        return big, x

    ins = [inside(t, math.inf) for t in (q, k, v, dO)]
    outs = [inside(torch.zeros_like(t)) for t in want]
    q2, k2, v2, dO2 = (x for _, x in ins)
    o2, lse2, dq, dk, dv = (x for _, x in outs)
    got = hip.attn_window_fwd(q2, k2, v2, window=30, sinks=3, out=o2, lse_out=lse2)
    assert got[0] is o2 and got[1] is lse2
    hip.attn_window_bwd(q2, k2, v2, o2, lse2, dO2, window=30, sinks=3, out=(dq, dk, dv))
    for (big, x), w in zip(outs, want):
        assert torch.equal(x, w)
        assert (big[:pad] == flag).all() and (big[-pad:] == flag).all()
