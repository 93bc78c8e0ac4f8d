"""The 8-bit KV cache (KVCache8) against its definition: what it holds, however it was
appended; attention of one and of several tokens over it; cutting back; graphs; refusals."""
import math

import numpy as np
import pytest

from tests import _cache8_ref as ref
from tests._window_ref import check

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _rows(B, H, T, D, seed, dtype=torch.bfloat16, spread=0.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, H, T, D, generator=g)
    if spread:  # blocks of very different sizes
        x *= torch.exp2(torch.randint(-int(spread), int(spread), (B, H, T // 64 + 1, 1), generator=g).float()) \
            .repeat_interleave(64, 2)[:, :, :T]
    return x.to(dtype)


def _same(got, want):
    got = got.cpu().double()
    return torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("spread", [0, 120])
def test_holds_its_definition(D, dtype, spread):
    from gonn_amd import hip
    B, H, Lmax, lens = 3, 2, 330, [330, 64, 127]
    k, v = (_rows(B, H, Lmax, D, 10 + i, dtype, spread) for i in range(2))
    k[0, 0, 5, 3], k[0, 1, 70, 0], v[0, 0, 200, 7], v[1, 1, 63, 1] = math.nan, math.inf, -math.inf, math.nan
    k[0, 0, 64:128] = 0  # a block of zeros
    v[0, 1, 128:192] *= 2.0 ** -60
    with hip.KVCache8(B, H, Lmax, D) as c:
        c.append(k.cuda(), v.cuda(), counts=lens)
        assert list(c.lengths()) == lens
        rk, rv = c.read(0, Lmax)
        lk, lv = c.read(last=70)
        for b, n in enumerate(lens):
            for x, r, l in ((k, rk, lk), (v, rv, lv)):
                want = ref.held(x[b], n)
                assert _same(r[b, :, :n], want), b
                assert not r[b, :, n:].any()
                m = min(n, 70)
                assert _same(l[b, :, 70 - m:], want[:, n - m:]) and not l[b, :, :70 - m].any()


def test_every_bf16_value_at_a_fixed_scale():
    """All magnitudes up to 448 beside one 448, which fixes the scale at 1."""
    from gonn_amd import hip
    u = torch.arange(0, 0x43e1, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)  # 0 .. 448
    u = torch.cat([u, -u])
    n = (u.numel() + 64 * 127 - 1) // (64 * 127)
    x = torch.zeros(n, 64, 128, dtype=torch.bfloat16)
    x[:, :, 0] = 448
    flat = torch.zeros(n * 64 * 127, dtype=torch.bfloat16)
    flat[:u.numel()] = u
    x[:, :, 1:] = flat.view(n, 64, 127)
    x = x.view(1, 1, n * 64, 128)
    with hip.KVCache8(1, 1, n * 64, 128) as c:
        c.append(x.cuda(), (x * 2.0 ** -20).cuda())
        k, v = c.read(0, n * 64)
    want = ref.held(x[0], n * 64)
    assert _same(k[0], want) and _same(v[0], want * 2.0 ** -20)


@pytest.mark.parametrize("D", [64, 128])
def test_chunks_and_cuts_do_not_show(D):
    from gonn_amd import hip
    B, H, Lmax = 2, 3, 400
    k, v = (_rows(B, H, Lmax, D, 20 + i).cuda() for i in range(2))
    q = _rows(B, H, 1, D, 30)[:, :, 0].contiguous().cuda()
    junk = torch.full((B, H, 90, D), math.nan, dtype=torch.bfloat16, device="cuda")
    with hip.KVCache8(B, H, Lmax, D) as one, hip.KVCache8(B, H, Lmax, D) as many:
        at = 0
        for n in (1, 62, 1, 1, 64, 65, 3, 120, 1, 70):  # closes blocks in every way
            one.reset()
            one.append(k[:, :, :at + n].contiguous(), v[:, :, :at + n].contiguous())
            many.append(k[:, :, at:at + n].contiguous(), v[:, :, at:at + n].contiguous())
            at += n
            # A draft that is dropped again; what it left behind must not show.
            m = min(64, Lmax - at)
            if m:
                many.append(junk[:, :, :m].contiguous(), junk[:, :, :m].contiguous())
                many.truncate([at] * B)
            assert list(many.lengths()) == [at] * B
            for a, b in zip(one.read(0, Lmax), many.read(0, Lmax)):
                assert torch.equal(a, b), (at, n)
            assert torch.equal(one.attend(q), many.attend(q)), at
        # Far back to a block's start, and on from there.
        many.truncate([128, 64])
        many.append(k[:, :, 128:140].contiguous(), v[:, :, 128:140].contiguous(), counts=[12, 0])
        many.append(k[:, :, 64:70].contiguous(), v[:, :, 64:70].contiguous(), counts=[0, 6])
        one.reset()
        one.append(k[:, :, :140].contiguous(), v[:, :, :140].contiguous(), counts=[140, 70])
        for a, b in zip(one.read(0, Lmax), many.read(0, Lmax)):
            assert torch.equal(a, b)


# B, Hq, H, Lmax, D, T, window, sinks, lens
ATTEND = [
    (1, 1, 1, 1, 64, 1, 0, 0, [1]),
    (2, 4, 4, 130, 128, 1, 0, 0, [130, 64]),
    (2, 8, 2, 200, 64, 1, 0, 0, [200, 0]),                # an empty sequence
    (3, 8, 1, 300, 128, 1, 50, 4, [300, 10, 128]),
    (1, 40, 8, 3100, 128, 1, 512, 70, [3099]),
    (2, 6, 2, 700, 64, 5, 0, 0, [700, 3]),                # fewer positions than queries
    (2, 4, 4, 500, 128, 33, 40, 3, [500, 333]),
    (1, 10, 2, 260, 64, 100, 0, 0, [260]),                # rows of several heads in a block
    (2, 4, 1, 600, 128, 130, 64, 0, [600, 191]),
    (1, 2, 2, 129, 128, 129, 1, 0, [129]),
    (40, 4, 2, 150, 64, 1, 0, 0, list(range(40, 80))),
    (2, 4, 2, 1500, 128, 1, 2000, 5, [1500, 1472]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("a", ATTEND, ids=lambda a: "x".join(map(str, a[:8])))
def test_attend(a, dtype):
    from gonn_amd import hip
    B, Hq, H, Lmax, D, T, window, sinks, lens = a
    k, v = (_rows(B, H, Lmax, D, 40 + i) for i in range(2))
    q = _rows(B, Hq, T, D, 50, dtype)
    with hip.KVCache8(B, H, Lmax, D) as c:
        c.append(k.cuda(), v.cuda(), counts=lens)
        o = c.attend((q[:, :, 0].contiguous() if T == 1 else q).cuda(), window=window, sinks=sinks).cpu()
    o = o.view(B, Hq, T, D)
    assert o.dtype == dtype
    ro, ra = [], []
    for b, n in enumerate(lens):
        x, y = ref.attend(q[b], ref.held(k[b], n), ref.held(v[b], n), 1 / math.sqrt(D), window, sinks)
        ro.append(x)
        ra.append(y)
    check(o, torch.stack(ro), torch.stack(ra), f"attend {a[:8]}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("where", [2, 70, 299], ids=["sink", "closed", "open"])
@pytest.mark.parametrize("bad", [math.nan, math.inf], ids=["nan", "inf"])
def test_bad_values_reach_only_those_that_see_them(where, bad, dtype):
    from gonn_amd import hip
    B, Hq, H, n, D, T = 1, 4, 2, 310, 64, 40
    for tensor in ("k", "v"):
        k, v = (_rows(B, H, n, D, 60 + i) for i in range(2))
        (k if tensor == "k" else v)[0, 1, where, 9] = bad
        q = _rows(B, Hq, T, D, 62, dtype)
        for window, sinks in ((30, 2), (30, 3), (0, 0)):
            with hip.KVCache8(B, H, n, D) as c:
                c.append(k.cuda(), v.cuda())
                o = c.attend(q.cuda(), window=window, sinks=sinks).cpu()
            ro, ra = ref.attend(q[0], ref.held(k[0], n), ref.held(v[0], n), 1 / 8, window, sinks)
            fine = torch.isfinite(ro).all(-1)
            assert torch.equal(torch.isfinite(o[0].double()).all(-1), fine), (tensor, window, sinks)
            z = torch.zeros((), dtype=torch.float64)
            keep = fine[..., None]
            ra = ref.attend(q[0], *(torch.nan_to_num(ref.held(x[0], n)) for x in (k, v)), 1 / 8, window, sinks)[1]
            check(torch.where(keep, o[0], z.to(dtype)), torch.where(keep, ro, z), torch.where(keep, ra, z), tensor)


def test_many_sequences():
    """More than one launch's worth of per-sequence numbers."""
    from gonn_amd import hip
    B, H, D = 300, 1, 64
    k, v = (_rows(B, H, 70, D, 70 + i) for i in range(2))
    lens = [i % 71 for i in range(B)]
    with hip.KVCache8(B, H, 96, D) as c:
        c.append(k.cuda(), v.cuda(), counts=lens)
        assert list(c.lengths()) == lens
        rk, rv = c.read(0, 70)
        for b in range(0, B, 7):
            assert _same(rk[b, :, :lens[b]], ref.held(k[b], lens[b]))
        cut = [min(n, 64) for n in lens]
        c.truncate(cut)
        c.append(k[:, :, :5].contiguous().cuda(), v[:, :, :5].contiguous().cuda())
        assert list(c.lengths()) == [n + 5 for n in cut]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
def test_captured_step_is_replayed(dtype):
    """A decoding step in a graph: its replays append at lengths that only the device knows."""
    from gonn_amd import hip
    B, Hq, H, D, Lmax = 2, 8, 2, 128, 260
    k, v = (_rows(B, H, Lmax, D, 80 + i, dtype).cuda() for i in range(2))
    q = _rows(B, Hq, Lmax, D, 82, dtype).cuda()
    with hip.KVCache8(B, H, Lmax, D) as c, hip.KVCache8(B, H, Lmax, D) as eager:
        start = [120, 61]
        for x in (c, eager):
            x.append(k[:, :, :120].contiguous(), v[:, :, :120].contiguous(), counts=start)
        k1, v1, q1 = (x[:, :, :1].contiguous() for x in (k, v, q))
        c.append(k1, v1)
        c.attend(q1, window=100, sinks=4)
        c.truncate(start)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.append(k1, v1)
            o = c.attend(q1, window=100, sinks=4)
            tail = c.read(last=3)
        for t in range(8):
            for x, y in ((k1, k), (v1, v), (q1, q)):
                x.copy_(y[:, :, 130 + t:131 + t])
            eager.append(k1, v1)
            want, wt = eager.attend(q1, window=100, sinks=4), eager.read(last=3)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            n = [s + t + 1 for s in start]
            # One weight and sum apart: the captured call may cut its splits elsewhere.
            err = (o.double() - want.double()).abs().max().item()
            assert err <= (2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -18) * want.abs().max().item()
            assert all(torch.equal(a, b) for a, b in zip(tail, wt))
            assert list(c.lengths()) == n
        c.truncate([120, 64])
        eager.truncate([120, 64])
        for a, b in zip(c.read(0, Lmax), eager.read(0, Lmax)):
            assert torch.equal(a, b)
        # A replay that would pass Lmax leaves that sequence as it is.
        c.append(k[:, :, :139].contiguous(), v[:, :, :139].contiguous(), counts=[139, 0])
        for n in ([260, 65], [260, 66]):
            g.replay()
            assert list(c.lengths()) == n


def test_with_the_window_attention():
    """A prompt through the training kernel, then tokens over the cache: the same attention of
    what the cache holds. Both sides bf16: two roundings of the weights, two of the result."""
    from gonn_amd import hip
    B, Hq, H, S, D, w, s = 2, 8, 2, 320, 128, 90, 4  # whole blocks, so that all keys are as held
    k, v = (_rows(B, H, S, D, 90 + i).cuda() for i in range(2))
    q = _rows(B, Hq, S, D, 92).cuda()
    with hip.KVCache8(B, H, S, D) as c:
        c.append(k, v)
        hk, hv = c.read(0, S)
        o, _ = hip.attn_window_fwd(q, hk, hv, window=w, sinks=s)
        got = c.attend(q[:, :, 100:].contiguous(), window=w, sinks=s)
        _, total = zip(*(ref.attend(q[b, :, 100:].cpu(), hk[b].cpu().double(), hv[b].cpu().double(),
                                    1 / math.sqrt(D), w, s) for b in range(B)))
        err = (got.double() - o[:, :, 100:].double()).abs().cpu()
        bound = 2.0 ** -7 * (o[:, :, 100:].double().abs().cpu() + torch.stack(total)) * 1.05 + 1e-6
        assert (err <= bound).all()


def test_another_stream():
    from gonn_amd import hip
    B, H, D = 2, 2, 64
    k, v = (_rows(B, H, 100, D, 95 + i).cuda() for i in range(2))
    q = _rows(B, H, 1, D, 97).cuda()
    with hip.KVCache8(B, H, 128, D) as c:
        c.append(k, v)
        want = c.attend(q)
        c.reset()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        c.append(k, v, stream=side)
        got = c.attend(q, stream=side)
        side.synchronize()
        assert torch.equal(got, want)


def test_refusals():
    from gonn_amd import hip
    with pytest.raises(hip.GonnHipError):
        hip.KVCache8(1, 1, 64, 80)
    with pytest.raises(hip.GonnHipError):
        hip.KVCache8(0, 1, 64, 64)
    c = hip.KVCache8(2, 2, 300, 64)
    k = _rows(2, 2, 300, 64, 1).cuda()
    q = _rows(2, 4, 1, 64, 2).cuda()
    with pytest.raises(hip.GonnHipError):
        c.append(torch.cat([k, k], 2), torch.cat([k, k], 2))
    with pytest.raises(hip.GonnHipError):
        c.append(k, k, counts=[301, 1])
    with pytest.raises(hip.GonnHipError):
        c.append(k, k, counts=[-1, 1])
    with pytest.raises(ValueError):
        c.append(k, k, counts=[1])
    with pytest.raises(ValueError):
        c.append(k[:, :1].contiguous(), k[:, :1].contiguous())
    with pytest.raises((hip.GonnHipError, TypeError)):
        c.append(k, k.float())
    with pytest.raises((hip.GonnHipError, TypeError)):
        c.append(k.half(), k.half())
    assert list(c.lengths()) == [0, 0]
    c.append(k, k, counts=[300, 200])
    with pytest.raises(hip.GonnHipError):
        c.append(k[:, :, :1].contiguous(), k[:, :, :1].contiguous())
    assert list(c.lengths()) == [300, 200]
    for bad in ([301, 1], [-1, 0], [150, 200], [300, 127]):
        with pytest.raises(hip.GonnHipError):
            c.truncate(bad)
    c.truncate([192, 128])  # as far back as the rows go
    for kw in ({"window": -1}, {"sinks": -1}, {"scale": math.nan}):
        with pytest.raises(hip.GonnHipError):
            c.attend(q, **kw)
    with pytest.raises(ValueError):
        c.attend(q[:, :3].contiguous())
    with pytest.raises(ValueError):
        c.attend(q, out=torch.empty_like(q, dtype=torch.float32))
    with pytest.raises(ValueError):
        c.attend(q.cpu())
    for args, kw in (((), {}), ((0,), {}), ((0, 3), {"last": 2}), ((-1, 3), {})):
        with pytest.raises(ValueError):
            c.read(*args, **kw)
    with pytest.raises(hip.GonnHipError):
        c.read(0, 0)
    c.close()
    with pytest.raises(ValueError):
        c.attend(q)
    with pytest.raises(ValueError):
        c.lengths()


@pytest.mark.parametrize("T", [1, 30, 90, 150])
def test_widest_window_with_rows_ahead_of_the_sequence(T):
    """Queries at positions below zero see nothing, whatever the window, and a window or a
    number of sinks past 32 bits is the widest one."""
    from gonn_amd import hip
    B, Hq, H, D, lens = 2, 2, 1, 64, [40, 20]
    k, v = (_rows(B, H, 64, D, 110 + i) for i in range(2))
    q = _rows(B, Hq, T, D, 112)
    with hip.KVCache8(B, H, 64, D) as c:
        c.append(k.cuda(), v.cuda(), counts=lens)
        want = c.attend(q.cuda())
        for window, sinks in ((2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 40, 2 ** 40), (1, 2 ** 40)):
            assert torch.equal(c.attend(q.cuda(), window=window, sinks=sinks), want), (window, sinks)
        for b, n in enumerate(lens):
            assert not want[b, :, :max(T - n, 0)].any()
            assert want[b, :, max(T - n, 0):].any()


def test_numbers_past_32_bits_are_refused():
    from gonn_amd import hip
    k = _rows(2, 1, 10, 64, 113).cuda()
    with hip.KVCache8(2, 1, 64, 64) as c:
        for call in (lambda: c.append(k, k, counts=[2 ** 32 + 1, 1]), lambda: c.truncate([-2 ** 32, 0]),
                     lambda: c.read(2 ** 32, 1), lambda: hip.KVCache8(1, 1, 2 ** 32 + 64, 64)):
            with pytest.raises(hip.GonnHipError):
                call()
        assert list(c.lengths()) == [0, 0]


def test_captured_refill_of_a_full_cache():
    """What the host knows of the lengths when a graph is captured is not what its replays meet."""
    from gonn_amd import hip
    B, H, D, Lmax = 2, 2, 64, 130
    k, v = (_rows(B, H, Lmax, D, 115 + i).cuda() for i in range(2))
    with hip.KVCache8(B, H, Lmax, D) as c:
        c.append(k, v)
        c.reset()
        c.append(v, k)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.reset()
            c.append(k, v)
            with pytest.raises(hip.GonnHipError):
                c.append(torch.cat([k, k], 2), torch.cat([k, k], 2))  # never fits
            with pytest.raises(hip.GonnHipError):
                c.lengths()  # would wait
            got = c.read(0, Lmax)
        for t in range(3):
            k.copy_(torch.roll(k, 1, 2))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert list(c.lengths()) == [Lmax] * B
            for b in range(B):
                assert _same(got[0][b], ref.held(k[b].cpu(), Lmax)) and _same(got[1][b], ref.held(v[b].cpu(), Lmax))
            c.truncate([64, 0])


def test_offsets_past_32_bits():
    """A head of more than 4e9 codes: every kernel finds the first positions and the last."""
    from gonn_amd import hip
    D, step, n = 128, 1 << 20, (1 << 25) + (1 << 20) - 40
    g = torch.Generator(device="cuda").manual_seed(7)
    rows = torch.randn(1, 1, step, D, generator=g, device="cuda").bfloat16()
    with hip.KVCache8(1, 1, n, D) as c:
        for a in range(0, n, step):
            # The rows of a block of positions, told apart from the others' by their sign and order.
            x = torch.roll(rows, a // step * 97, 2)
            m = min(step, n - a)
            c.append(x[:, :, :m].contiguous(), -x[:, :, :m].contiguous())
        assert list(c.lengths()) == [n]
        a = (n - 1) // step * step
        x = torch.roll(rows, a // step * 97, 2)[:, :, n - a - 200:n - a]
        tail = c.read(last=200)
        lead = (n - 200) % 64  # whole blocks from here on, the open one last
        want = ref.held(x[0].cpu()[:, 64 - lead:], 200 - (64 - lead))
        assert _same(tail[0][0, :, 64 - lead:], want) and _same(tail[1][0, :, 64 - lead:], -want)
        head = c.read(0, 128)
        assert _same(head[0][0], ref.held(rows[0, :, :128].cpu(), 128))
        # Window and sinks: positions of both ends, in each form of the attention.
        held_k = torch.cat([head[0], c.read(last=512)[0]], 2)[0].cpu().double()
        held_v = torch.cat([head[1], c.read(last=512)[1]], 2)[0].cpu().double()
        for T, dtype in ((1, torch.bfloat16), (1, torch.float32), (30, torch.bfloat16), (60, torch.float32),
                         (130, torch.bfloat16), (130, torch.float32)):
            q = _rows(1, 1, T, D, 120, dtype)
            o = c.attend(q.cuda(), window=300, sinks=128).cpu()
            ro, ra = ref.attend(q[0], held_k, held_v, 1 / math.sqrt(D), 300, 128)
            check(o[0], ro, ra, f"{T} queries {dtype}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T", [1, 20, 50, 130])
def test_many_sequences_of_different_lengths(T, dtype):
    """More sequences than lanes, of one split to several, empty ones among them: each has its
    turn, in a call that knows the lengths and in a captured one."""
    from gonn_amd import hip
    B, Hq, H, D, Lmax = 70, 2, 1, 64, 1700
    lens = [(i * 577) % (Lmax + 1) if i % 9 else 0 for i in range(B)]
    lens[5] = Lmax
    k, v = (_rows(B, H, Lmax, D, 130 + i) for i in range(2))
    q = _rows(B, Hq, T, D, 132, dtype)
    with hip.KVCache8(B, H, Lmax, D) as c:
        c.append(k.cuda(), v.cuda(), counts=lens)
        qd = q.cuda()
        o = c.attend(qd, window=900, sinks=70)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            og = c.attend(qd, window=900, sinks=70)
        for _ in range(2):
            og.zero_()
            g.replay()
        torch.cuda.synchronize()
    some = list(range(0, B, 4)) + [5, 63, 65, 69]
    ro, ra = zip(*(ref.attend(q[b], ref.held(k[b], lens[b]), ref.held(v[b], lens[b]), 1 / math.sqrt(D), 900, 70)
                   for b in some))
    for got in (o, og):
        check(torch.stack([got[b].cpu() for b in some]), torch.stack(ro), torch.stack(ra), f"{T} queries")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("T", [1, 25, 60, 140])
def test_outputs_given_and_neighbours_untouched(T, dtype):
    """Outputs inside larger tensors; several splits, so that their join writes them."""
    from gonn_amd import hip
    B, Hq, H, D, n = 2, 2, 2, 64, 1900
    k, v = (_rows(B, H, n, D, 140 + i).cuda() for i in range(2))
    q = _rows(B, Hq, T, D, 142, dtype).cuda()
    pad, flag = 256, -7.0
    with hip.KVCache8(B, H, n, D) as c:
        c.append(k, v)
        want = (c.attend(q), *c.read(3, 500))
        bigs = [torch.full((t.numel() + 2 * pad,), flag, dtype=t.dtype, device="cuda") for t in want]
        o, rk, rv = (b[pad:-pad].view(t.shape) for b, t in zip(bigs, want))
        assert c.attend(q, out=o) is o
        c.read(3, 500, out=(rk, rv))
        for b, x, w in zip(bigs, (o, rk, rv), want):
            assert torch.equal(x, w)
            assert (b[:pad] == flag).all() and (b[-pad:] == flag).all()
