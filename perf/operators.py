"""The windowed attention and the 8-bit KV cache: cases to time and to compare.

Four operators, each in a plain form (elementary torch operations in 32 bits, rounded once
at the end) and through the framework's entry points (`own`):

window_fwd  causal attention over a sliding window with sinks: query i sees key j when
            j <= i, j < kv_len and (i - j < window or j < sinks). O = softmax(scale q k^T) v
            over the keys it sees, and LSE. A query that sees none has O = 0, LSE = -inf.
window_bwd  its gradients from the saved O and LSE: P = exp(s - LSE), dV = P^T dO,
            dS = P (dO v^T - rowsum(dO O)), dQ = scale dS k, dK = scale dS^T q; a key head
            shared by several query heads has the sum of theirs.
append      new positions of a KV cache in 8 bits. Every 64 positions of a head that are
            complete are held in e4m3 with one scale for K and one for V, the smallest power
            of two 2^e, -100 <= e, that brings the largest magnitude to at most 448; the
            positions of the last, incomplete block are held in bf16.
attend      the T newest positions' queries over that cache: query t sees the positions up to
            its own, all of them or those of a window with sinks.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 64  # positions that share a scale
LEAST = -100  # least exponent of a scale


# ---- the cases ----------------------------------------------------------------------------
def _window(name, op, dtype, B, H, Hkv, S, D, window, sinks, shortest):
    return {"name": name, "op": op, "dtype": dtype, "B": B, "H": H, "Hkv": Hkv, "S": S, "D": D, "window": window,
            "sinks": sinks, "shortest": shortest}


def _append(name, dtype, B, Hkv, Lmax, T, D, held, shortest):
    return {"name": name, "op": "append", "dtype": dtype, "B": B, "Hkv": Hkv, "Lmax": Lmax, "T": T, "D": D, "held": held,
            "shortest": shortest}


def _attend(name, dtype, B, H, Hkv, Lmax, T, D, window, sinks, shortest):
    return {"name": name, "op": "attend", "dtype": dtype, "B": B, "H": H, "Hkv": Hkv, "Lmax": Lmax, "T": T, "D": D,
            "window": window, "sinks": sinks, "shortest": shortest}


def listed():
    return [
        # One short sequence batch of a small layer: the latency of a call.
        _window("fwd small bf16", "window_fwd", "bfloat16", 2, 4, 4, 128, 64, 64, 4, 128),
        # An encoder-sized layer in fp32, sequences padded to 1024.
        _window("fwd padded fp32", "window_fwd", "float32", 8, 12, 12, 1024, 64, 256, 4, 700),
        # A long training sequence, every head with keys of its own.
        _window("fwd long bf16", "window_fwd", "bfloat16", 2, 16, 16, 8192, 128, 1024, 4, 8192),
        # A short odd length with shared key heads and no sinks: one training micro-batch.
        _window("bwd odd shared bf16", "window_bwd", "bfloat16", 1, 8, 2, 777, 128, 128, 0, 777),
        # fp32 gradients of padded sequences of an odd length.
        _window("bwd padded fp32", "window_bwd", "float32", 4, 12, 12, 1021, 64, 200, 5, 600),
        # The long training sequence's backward, four query heads to a key head.
        _window("bwd long shared bf16", "window_bwd", "bfloat16", 2, 16, 4, 8192, 128, 1024, 4, 8192),
        # Prompts of several lengths enter an empty cache in one call.
        _append("append prompts bf16", "bfloat16", 8, 8, 4096, 4096, 128, 0, 1500),
        # A chunk of fp32 rows follows what the cache holds.
        _append("append chunk fp32", "float32", 4, 12, 2048, 50, 64, 1900, 1000),
        # One decoding step's rows of a large batch.
        _append("append step bf16", "bfloat16", 64, 32, 8192, 1, 128, 8191, 512),
        # One decoding step of a large batch over everything cached.
        _attend("decode batch bf16", "bfloat16", 64, 32, 32, 8192, 1, 128, 0, 0, 512),
        # One sequence's decoding step over a window, shared key heads: latency.
        _attend("decode window fp32", "float32", 1, 32, 8, 1500, 1, 128, 512, 4, 1500),
        # A prompt's next chunk over a long cache.
        _attend("chunk bf16", "bfloat16", 4, 32, 8, 4096, 256, 128, 0, 0, 2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case: sizes over the listed ranges, and no dearer than the largest of its operator."""
    op = rng.choice(["window_fwd", "window_bwd", "append", "attend"])
    dtype = rng.choice(["bfloat16", "float32"])
    D = rng.choice([64, 128])
    Hkv = rng.choice([1, 2, 3, 4, 8])
    G = rng.choice([1, 1, 2, 4, 5])
    if op.startswith("window"):
        # A query that sees one key has dS = 0 and gradients of nothing but rounding.
        bwd = op == "window_bwd"
        S = _log(rng, 8 if bwd else 1, 8192)
        B = max(1, min(_log(rng, 1, 16), 4 * 8192 // S))
        H = Hkv * G
        while B * H > 1 and B * H * S * S > (1 << 31) // (2 if dtype == "float32" else 1):
            B, H, Hkv = (B - 1, H, Hkv) if B > 1 else (1, H // Hkv, 1) if Hkv > 1 else (1, 1, 1)
        return {"op": op, "dtype": dtype, "B": B, "H": H, "Hkv": Hkv, "S": S, "D": D, "window": _log(rng, 4 if bwd else 1, 2048),
                "sinks": rng.choice([0, 0, 1, 4, rng.randint(2, 130)]), "shortest": S if rng.random() < 0.5 else rng.randint(1, S)}
    Lmax = _log(rng, 64, 8192)
    B = max(1, min(_log(rng, 1, 64), (64 * 32 * 8192) // (Lmax * Hkv * 4)))
    if op == "append":
        if rng.random() < 0.5:  # into an empty cache
            T = rng.randint(1, Lmax)
            return {"op": op, "dtype": dtype, "B": B, "Hkv": Hkv, "Lmax": Lmax, "T": T, "D": D, "held": 0,
                    "shortest": rng.randint(1, T)}
        T = _log(rng, 1, BLOCK)
        held = rng.randint(0, Lmax - T)
        return {"op": op, "dtype": dtype, "B": B, "Hkv": Hkv, "Lmax": Lmax, "T": T, "D": D, "held": held,
                "shortest": rng.randint(0, held)}
    T = 1 if rng.random() < 0.5 else min(_log(rng, 2, 300), Lmax)
    B = max(1, min(B, (1 << 28) // (Hkv * G * T * Lmax)))
    return {"op": op, "dtype": dtype, "B": B, "H": Hkv * G, "Hkv": Hkv, "Lmax": Lmax, "T": T, "D": D,
            "window": rng.choice([0, _log(rng, 1, 4096)]), "sinks": rng.choice([0, 4, rng.randint(1, 100)]),
            "shortest": rng.randint(T, Lmax)}


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, evenly spread and not in order."""
    v = [lo + (hi - lo) * i // (n - 1) for i in range(n)] if n > 1 else [hi]
    return v[::2] + v[1::2]


# ---- inputs -------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, dtype, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _keys(g, dtype, *shape):
    """Rows whose channels differ in size, as keys' do."""
    size = torch.exp(0.5 * torch.randn((1, shape[1], 1, shape[-1]), generator=g, device="cuda"))
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * size).to(dtype)


def _scale(case):
    return 1.0 / math.sqrt(case["D"])


def _kv_len(case):
    if case["shortest"] == case["S"]:
        return None
    return torch.tensor(_spread(case["shortest"], case["S"], case["B"]), dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    dtype = getattr(torch, case["dtype"])
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    st = {"case": case}
    if case["op"].startswith("window"):
        H, S = case["H"], case["S"]
        st["q"], st["k"], st["v"] = _rows(g, dtype, B, H, S, D), _keys(g, dtype, B, Hkv, S, D), _rows(g, dtype, B, Hkv, S, D)
        st["kv_len"] = _kv_len(case)
        if case["op"] == "window_bwd":  # what the forward saved
            o, lse = _window_fwd(st)
            st["o"], st["lse"], st["dO"] = o, lse, _rows(g, dtype, B, H, S, D)
        return st
    T, Lmax = case["T"], case["Lmax"]
    if case["op"] == "append":
        st["base"] = _spread(case["shortest"], case["held"], B) if case["held"] else [0] * B
        st["counts"] = [T] * B if case["held"] else _spread(case["shortest"], T, B)
        st["k"], st["v"] = _keys(g, dtype, B, Hkv, T, D), _rows(g, dtype, B, Hkv, T, D)
        lens, most = st["base"], case["held"]
    else:
        st["q"] = _rows(g, dtype, B, case["H"], T, D)
        lens = _spread(case["shortest"], Lmax, B)
        most = Lmax
    k, v = _keys(g, torch.bfloat16, B, Hkv, most, D), _rows(g, torch.bfloat16, B, Hkv, most, D)
    if own:
        from gonn_amd import hip
        st["cache"] = hip.KVCache8(B, Hkv, Lmax, D)
        if most:
            st["cache"].append(k, v, counts=lens)
    else:
        st["lens"] = torch.tensor(lens, dtype=torch.int64, device="cuda")
        st["counts"] = torch.tensor(st["counts"], dtype=torch.int64, device="cuda") if "counts" in st else None
        st["k8"], st["v8"] = _held(k, st["lens"]), _held(v, st["lens"])
    return st


# ---- plain forms --------------------------------------------------------------------------
def _sees(case, kv_len):
    """(B or 1, 1, S, S): whether query i sees key j."""
    S = case["S"]
    i = torch.arange(S, device="cuda")[:, None]
    j = torch.arange(S, device="cuda")[None, :]
    sees = ((j <= i) & ((i - j < case["window"]) | (j < case["sinks"])))[None, None]
    return sees if kv_len is None else sees & (j < kv_len[:, None, None, None])


def _heads(x, H):
    """Key heads as the query heads read them, in 32 bits."""
    return x.float().repeat_interleave(H // x.shape[1], 1)


def _softmax(s):
    """Weights and log-sum-exp of masked scores; a row of -inf has weights 0."""
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isinf(m), torch.zeros_like(m), m))
    l = e.sum(-1, keepdim=True)
    lse = torch.where(l > 0, m + torch.log(l), torch.full_like(m, -math.inf))
    return e / torch.where(l > 0, l, torch.ones_like(l)), lse[..., 0]


def _window_fwd(st):
    case, q = st["case"], st["q"]
    k, v = _heads(st["k"], case["H"]), _heads(st["v"], case["H"])
    s = torch.matmul(q.float() * _scale(case), k.transpose(-1, -2))
    s = s.masked_fill(~_sees(case, st["kv_len"]), -math.inf)
    p, lse = _softmax(s)
    return torch.matmul(p, v).to(q.dtype), lse.reshape(-1, case["S"])


def _window_bwd(st):
    case, q = st["case"], st["q"].float()
    B, H, Hkv, S, D = case["B"], case["H"], case["Hkv"], case["S"], case["D"]
    k, v, dO = _heads(st["k"], H), _heads(st["v"], H), st["dO"].float()
    lse = st["lse"].view(B, H, S, 1)
    lse = torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)
    p = torch.exp(torch.matmul(q * _scale(case), k.transpose(-1, -2)) - lse)
    p = p.masked_fill(~_sees(case, st["kv_len"]), 0.0)
    dv = torch.matmul(p.transpose(-1, -2), dO)
    ds = p * (torch.matmul(dO, v.transpose(-1, -2)) - (dO * st["o"].float()).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k) * _scale(case)
    dk = torch.matmul(ds.transpose(-1, -2), q) * _scale(case)
    dk, dv = (x.view(B, Hkv, H // Hkv, S, D).sum(2) for x in (dk, dv))
    return tuple(x.to(st["q"].dtype) for x in (dq, dk, dv))


def _quantise(x):
    """Blocks (..., 64, D) in 8 bits: e4m3 codes and the scale, a power of two."""
    x = x.float()
    mant, e = torch.frexp(x.abs().amax((-1, -2)))
    e = torch.where(mant <= 0.875, e - 9, e - 8).clamp(min=LEAST)  # 448 = 0.875 * 2^9
    e = torch.where(mant == 0, torch.zeros_like(e), e)
    scale = ((e + 127).int() << 23).view(torch.float32)  # 2^e
    return (x / scale[..., None, None]).to(torch.float8_e4m3fn), scale


def _values(codes, scale):
    return codes.float() * scale[..., None, None]


def _blocks(x):
    """(B, H, T, D) as whole blocks (B, H, n, 64, D), padded with zeros."""
    B, H, T, D = x.shape
    n = T // BLOCK + 1
    out = torch.zeros((B, H, n * BLOCK, D), dtype=torch.bfloat16, device=x.device)
    out[:, :, :T] = x
    return out.view(B, H, n, BLOCK, D)


def _held(x, lens):
    """What a cache of these rows holds: codes and scales of every block, and the open block's rows."""
    x = _blocks(x)
    open_block = (lens // BLOCK)[:, None, None, None, None].expand(-1, x.shape[1], 1, BLOCK, x.shape[4])
    tail = torch.gather(x, 2, open_block)[:, :, 0]
    return (*_quantise(x), tail)


def _append_empty(x, counts):
    """Rows of an empty cache after x was appended, as it holds them; zeros past the end."""
    b = _blocks(x)
    B, H, n, _, D = b.shape
    at = torch.arange(n * BLOCK, device="cuda").view(n, BLOCK)
    c = counts[:, None, None]
    closed, there = at < c // BLOCK * BLOCK, at < c
    out = torch.where(closed[:, None, :, :, None], _values(*_quantise(b)), b.float() * there[:, None, :, :, None])
    return out.view(B, H, n * BLOCK, D)[:, :, :x.shape[2]].to(torch.bfloat16)


def _append_more(x, held, lens):
    """The last 64 positions (zeros before the first) after up to 64 rows were appended."""
    codes, scale, tail = held
    B, H, _, D = tail.shape
    T = x.shape[2]
    o = lens % BLOCK
    j = torch.arange(2 * BLOCK, device="cuda")[None]
    # The open block's rows, then the new ones.
    from_new = (j - o[:, None]).clamp(0, T - 1)[:, None, :, None].expand(B, H, -1, D)
    from_tail = j.clamp(max=BLOCK - 1)[:, None, :, None].expand(B, H, -1, D)
    rows = torch.where((j < o[:, None])[:, None, :, None], torch.gather(tail, 2, from_tail),
                       torch.gather(x.to(torch.bfloat16), 2, from_new)).float()
    n = o + T
    closed = _values(*_quantise(rows[:, :, :BLOCK]))
    rows[:, :, :BLOCK] = torch.where((n >= BLOCK)[:, None, None, None], closed, rows[:, :, :BLOCK])
    before = (lens // BLOCK - 1).clamp(min=0)
    pick = before[:, None, None, None, None].expand(B, H, 1, BLOCK, D)
    prev = torch.gather(codes.view(torch.uint8), 2, pick).view(torch.float8_e4m3fn)[:, :, 0]
    prev = _values(prev, torch.gather(scale, 2, before[:, None, None].expand(B, H, 1))[:, :, 0])
    prev = prev * (lens >= BLOCK)[:, None, None, None]
    # Position n - 64 + i from the open block's first; negative ones are the block's before it.
    idx = (n[:, None] + torch.arange(BLOCK, device="cuda")[None])[:, None, :, None].expand(B, H, -1, D)
    there = (lens[:, None] + T - BLOCK + torch.arange(BLOCK, device="cuda")[None]) >= 0
    out = torch.gather(torch.cat([prev, rows], 2), 2, idx)
    return (out * there[:, None, :, None]).to(torch.bfloat16)


def _cached(held, lens, Lmax):
    """The cache's rows (B, H, Lmax, D) in 32 bits."""
    codes, scale, tail = held
    B, H, n, _, D = codes.shape
    is_open = torch.arange(n, device="cuda") == lens[:, None] // BLOCK
    x = torch.where(is_open[:, None, :, None, None], tail.float()[:, :, None], _values(codes, scale))
    return x.view(B, H, n * BLOCK, D)[:, :, :Lmax]


def _attended(case, lens):
    """(B, 1, T, Lmax): whether query t sees position j."""
    T = case["T"]
    i = lens[:, None] - T + torch.arange(T, device="cuda")[None]
    i, j = i[:, None, :, None], torch.arange(case["Lmax"], device="cuda")
    sees = j <= i
    return sees & ((i - j < case["window"]) | (j < case["sinks"])) if case["window"] else sees


def _attend_plain(st):
    case, q = st["case"], st["q"]
    B, H, Hkv, T, D = case["B"], case["H"], case["Hkv"], case["T"], case["D"]
    k, v = _cached(st["k8"], st["lens"], case["Lmax"]), _cached(st["v8"], st["lens"], case["Lmax"])
    s = torch.matmul((q.float() * _scale(case)).view(B, Hkv, -1, D), k.transpose(-1, -2))
    s = s.view(B, H, T, -1).masked_fill(~_attended(case, st["lens"]), -math.inf)
    p, _ = _softmax(s)
    return torch.matmul(p.view(B, Hkv, (H // Hkv) * T, -1), v).view(B, H, T, D).to(q.dtype)


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "window_fwd":
        return _window_fwd(state)
    if case["op"] == "window_bwd":
        return _window_bwd(state)
    if case["op"] == "attend":
        return _attend_plain(state)
    if case["held"]:
        return _append_more(state["k"], state["k8"], state["lens"]), _append_more(state["v"], state["v8"], state["lens"])
    return _append_empty(state["k"], state["counts"]), _append_empty(state["v"], state["counts"])


def _run_own(case, st):
    from gonn_amd import hip
    if case["op"] == "window_fwd":
        return hip.attn_window_fwd(st["q"], st["k"], st["v"], window=case["window"], sinks=case["sinks"], kv_len=st["kv_len"])
    if case["op"] == "window_bwd":
        return hip.attn_window_bwd(st["q"], st["k"], st["v"], st["o"], st["lse"], st["dO"], window=case["window"],
                                   sinks=case["sinks"], kv_len=st["kv_len"])
    cache = st["cache"]
    if case["op"] == "attend":
        return cache.attend(st["q"], window=case["window"], sinks=case["sinks"])
    if case["held"]:  # a step whose positions are dropped again, as a rejected draft's are
        cache.truncate(st["base"])
        cache.append(st["k"], st["v"])
        return cache.read(last=BLOCK)
    cache.reset()
    cache.append(st["k"], st["v"], counts=st["counts"])
    return cache.read(0, case["T"])


# ---- what a pass cannot do without --------------------------------------------------------
def _pairs(n, first, window, sinks, length):
    """Query-key pairs, and keys that some query sees, of queries first .. first + n - 1 over `length` keys."""
    i = np.arange(first, first + n, dtype=np.int64)
    hi = np.minimum(i + 1, length).clip(min=0)
    lo = np.minimum((i - window + 1).clip(min=0), hi) if window else np.zeros_like(i)
    pairs = int((hi - lo + np.minimum(sinks, lo)).sum())
    keys = int(hi[-1] - lo[0] + min(sinks, lo[0])) if n else 0
    return pairs, keys


def work(case):
    size = 2 if case["dtype"] == "bfloat16" else 4
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    if case["op"].startswith("window"):
        H, S = case["H"], case["S"]
        lens = _spread(case["shortest"], S, B) if case["shortest"] < S else [S] * B
        seen = [_pairs(S, 0, case["window"], case["sinks"], n) for n in lens]
        pairs, keys = sum(p for p, _ in seen) * H, sum(k for _, k in seen) * Hkv
        if case["op"] == "window_fwd":
            return {"bytes": (2 * B * H * S + 2 * keys) * D * size + B * H * S * 4, "flops": 4 * D * pairs}
        return {"bytes": (4 * B * H * S + 2 * keys + 2 * B * Hkv * S) * D * size + B * H * S * 4, "flops": 10 * D * pairs}
    T = case["T"]
    if case["op"] == "append":
        rows = B * T if case["held"] else sum(_spread(case["shortest"], T, B))
        out = B * (BLOCK if case["held"] else T)
        return {"bytes": 2 * Hkv * D * (rows * (size + 1) + out * 2), "flops": 2 * rows * Hkv * D}
    H = case["H"]
    seen = [_pairs(T, n - T, case["window"], case["sinks"], n) for n in _spread(case["shortest"], case["Lmax"], B)]
    pairs, keys = sum(p for p, _ in seen) * H, sum(k for _, k in seen) * Hkv
    return {"bytes": 2 * keys * D + 2 * B * H * T * D * size, "flops": 4 * D * pairs}


# ---- from the definition, in 64 bits ------------------------------------------------------
def _grid(x):
    """Doubles on the e4m3 grid: to nearest, ties to even (|x| <= 448)."""
    _, e = torch.frexp(x)
    step = _power64((e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _power64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _stored(x, length):
    """(H, n, D) rows of one sequence as the cache holds them once it has `length` of them."""
    y = x[:, :length].double()
    whole = length // BLOCK * BLOCK
    if whole:
        b = y[:, :whole].reshape(y.shape[0], -1, BLOCK, y.shape[2])
        top = b.abs().amax((2, 3), keepdim=True)
        mant, e = torch.frexp(torch.where(top > 0, top, torch.full_like(top, 448.0)) / 448)
        unit = _power64((e - (mant == 0.5).int()).clamp(min=LEAST))  # 2^ceil(log2(top / 448))
        y[:, :whole] = (_grid(b / unit) * unit).reshape(y.shape[0], whole, -1)
    return y


def _attend64(q, k, v, i, j, window, sinks, scale):
    """Attention of the queries at positions i over the keys at positions j (H, n, D), in 64 bits: o, lse, weights."""
    s = torch.matmul(q * scale, k.transpose(1, 2))
    d = i[:, None] - j[None, :]
    ok = d >= 0
    if window:
        ok = ok & ((d < window) | (j < sinks)[None, :])
    s = torch.where(ok, s, torch.full_like(s, -math.inf))
    lse = torch.logsumexp(s, -1)
    p = torch.where(ok, torch.exp(s - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[..., None]), torch.zeros_like(s))
    return torch.matmul(p, v), lse, p


def exact(case, seed):
    g = _gen(seed)
    dtype = getattr(torch, case["dtype"])
    B, Hkv, D, scale = case["B"], case["Hkv"], case["D"], _scale(case)
    if case["op"].startswith("window"):
        H, S = case["H"], case["S"]
        G = H // Hkv
        st = {"case": case}
        st["q"], st["k"], st["v"] = _rows(g, dtype, B, H, S, D), _keys(g, dtype, B, Hkv, S, D), _rows(g, dtype, B, Hkv, S, D)
        st["kv_len"] = _kv_len(case)
        lens = [S] * B if st["kv_len"] is None else st["kv_len"].tolist()
        bwd = case["op"] == "window_bwd"
        if bwd:
            o_in, lse_in = _window_fwd(st)
            dO_in = _rows(g, dtype, B, H, S, D)
        at = torch.arange(S, device="cuda")
        fwd_o, fwd_l = [], []
        dq = torch.zeros((B, H, S, D), dtype=torch.float64, device="cuda")
        dk, dv = (torch.zeros((B, Hkv, S, D), dtype=torch.float64, device="cuda") for _ in range(2))
        for b, n in enumerate(lens):
            for h in range(H):
                q = st["q"][b, h][None].double()
                k, v = st["k"][b, h // G, :n][None].double(), st["v"][b, h // G, :n][None].double()
                o, lse, p = _attend64(q, k, v, at, at[:n], case["window"], case["sinks"], scale)
                if not bwd:
                    fwd_o.append(o)
                    fwd_l.append(lse)
                    continue
                # From the saved statistics, which the call is given.
                saved = lse_in.view(B, H, S)[b, h].double()
                p = p * torch.exp(torch.where(torch.isinf(saved), torch.zeros_like(saved), lse[0] - saved))[None, :, None]
                dO, o_s = dO_in[b, h].double(), o_in[b, h].double()
                ds = p[0] * (dO @ v[0].T - (dO * o_s).sum(-1, keepdim=True))
                dq[b, h] = ds @ k[0] * scale
                dk[b, h // G, :n] += ds.T @ q[0] * scale
                dv[b, h // G, :n] += p[0].T @ dO
        if bwd:
            return dq, dk, dv
        return torch.cat(fwd_o).view(B, H, S, D), torch.cat(fwd_l).view(B * H, S)
    T, Lmax = case["T"], case["Lmax"]
    if case["op"] == "append":
        base = _spread(case["shortest"], case["held"], B) if case["held"] else [0] * B
        counts = [T] * B if case["held"] else _spread(case["shortest"], T, B)
        new = _keys(g, dtype, B, Hkv, T, D), _rows(g, dtype, B, Hkv, T, D)
        old = _keys(g, torch.bfloat16, B, Hkv, case["held"], D), _rows(g, torch.bfloat16, B, Hkv, case["held"], D)
        shown = BLOCK if case["held"] else T
        outs = []
        for x, was in zip(new, old):
            out = torch.zeros((B, Hkv, shown, D), dtype=torch.float64, device="cuda")
            for b in range(B):
                # Only the blocks that are shown, so that long caches stay quick.
                end = base[b] + counts[b]
                first = max(0, end - BLOCK) // BLOCK * BLOCK if case["held"] else 0
                rows = torch.cat([was[b, :, first:base[b]].to(torch.bfloat16),
                                  x[b, :, max(0, first - base[b]):counts[b]].to(torch.bfloat16)], 1)
                y = _stored(rows, end - first)
                if case["held"]:
                    y = y[:, -min(BLOCK, end):]
                    out[b, :, BLOCK - y.shape[1]:] = y
                else:
                    out[b, :, :end] = y
            outs.append(out)
        return tuple(outs)
    H = case["H"]
    G = H // Hkv
    q = _rows(g, dtype, B, H, T, D)
    k, v = _keys(g, torch.bfloat16, B, Hkv, Lmax, D), _rows(g, torch.bfloat16, B, Hkv, Lmax, D)
    out = torch.zeros((B, H, T, D), dtype=torch.float64, device="cuda")
    for b, n in enumerate(_spread(case["shortest"], Lmax, B)):
        kb, vb = (_stored(x[b], n).repeat_interleave(G, 0) for x in (k, v))
        at = torch.arange(n, device="cuda")
        out[b] = _attend64(q[b].double(), kb, vb, at[n - T:], at, case["window"], case["sinks"], scale)[0]
    return out
