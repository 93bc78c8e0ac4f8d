// attn_window_bwd.hip -- sliding-window attention with sinks: the backward.
//
// With P_ij = exp(s_ij - LSE_i) over the pairs that attn_window.h's mask keeps:
//   delta_i = dO_i . O_i      dS_ij = P_ij (dO_i . v_j - delta_i)
//   dQ_i = scale sum_j dS_ij k_j    dK_j = scale sum_i dS_ij q_i    dV_j = sum_i P_ij dO_i
// and the queries of every head that shares a key head add up in its dK and dV.
//
//   dQ     a wave owns 32 queries (Q and dO in registers), the key tiles of its
//          two runs stream through LDS; it forms delta first and stores it.
//   dK/dV  a wave owns 32 keys; the query tiles of its band, and of every later
//          query where the block holds sinks, stream for each query head. These
//          (head, stage) steps are cut into items of about equal length, one per
//          workgroup, so that the sinks' blocks, which all queries read, and small
//          grids fill the device; blocks of several items leave fp32 partials that
//          a second kernel adds in order. No atomics: results are deterministic.
#include <algorithm>

#include "attn_window.h"

namespace gonn {

namespace {

// LSE in log2 units, as the offset of P; a row without keys (-inf) gets P = 0.
GONN_DEV float lse_log2(float lse) { return lse == -INFINITY ? INFINITY : lse * kLog2e; }

// S and dP of one 32 x 32 tile on the fp32 instruction from global memory: rows
// ra (of ka, va) in registers' order, columns the lane's own rows of qa and oa.
template <int D, typename T>
GONN_DEV void plain_products(const T* a1, const T* b1, const T* a2, const T* b2, int g, f32x16& s,
                             f32x16& dp) {
    constexpr int HD = D / 2;
    s = dp = f32x16{};
#pragma unroll 4
    for (int i = 0; i < HD; i++) {
        s = mfma_f32(to_float(a1[g * HD + i]), to_float(b1[g * HD + i]), s);
        dp = mfma_f32(to_float(a2[g * HD + i]), to_float(b2[g * HD + i]), dp);
    }
}

// dQ of a wave's 32 queries in plain fp32 products, for results that are not finite
// (see window_fwd_plain), 32 channels at a time.
template <int D, typename T>
GONN_DEV void window_dq_plain(const WindowParams& p, int bh, int bk, int kl, const Band& band,
                              int qw, float lq, float dl) {
    const int lane = threadIdx.x & 63, g = lane >> 5, ln = lane & 31, qi = qw + ln;
    const T* Kg = (const T*)p.k + (size_t)bk * p.Sk * D;
    const T* Vg = (const T*)p.v + (size_t)bk * p.Sk * D;
    const size_t row = ((size_t)bh * p.Sq + (qi < p.Sq ? qi : p.Sq - 1)) * D;
    KeyStages ks;
    ks.init(qw, qw + 32 < p.Sq ? qw + 32 : p.Sq, kl, 32, band);
#pragma unroll 1
    for (int t = 0; t < D / 32; t++) {
        f32x16 acc = f32x16{};
#pragma unroll 1
        for (int st = 0; st < ks.count(); st++) {
            const int kb = ks.stage(st) * 32;
            const size_t kr = (size_t)(kb + ln < kl ? kb + ln : kl - 1) * D;
            f32x16 s, dp;
            plain_products<D>(Kg + kr, (const T*)p.q + row, Vg + kr, (const T*)p.dO + row, g, s, dp);
            for (int r = 0; r < 16; r++) {
                const int key = kb + 8 * (r >> 2) + 4 * g + (r & 3);
                const float pv = fast_exp2(__builtin_fmaf(s[r], p.scale_log2, -lq));
                s[r] = key < kl && band.sees(qi, key) ? pv * (dp[r] - dl) : 0.f;
            }
#pragma unroll 1
            for (int x = 0; x < 32; x++) {
                const int r = x >> 1, h = x & 1, key = kb + 8 * (r >> 2) + 4 * h + (r & 3);
                const float w = weight_of(s, r, h, g);
                if (key >= kl) continue;  // uniform
                add_row32(acc, w, Kg + (size_t)key * D + 32 * t, g, band.sees(qi, key));
            }
        }
        if (qi < p.Sq)
            for (int rq = 0; rq < 4; rq++) {
                f32x4 v;
                for (int i = 0; i < 4; i++) v[i] = acc[rq * 4 + i] * p.scale;
                store4<T>((T*)p.dq + row + 32 * t + 8 * rq + 4 * g, v);
            }
    }
}

}  // namespace

template <int D, typename T, int WB, int NBUF, int OCC>
__global__ __launch_bounds__(256, OCC) void window_dq_kernel(WindowParams p) {
    constexpr int NS = 4 / WB, BM = WB * 32, BN = NS * 32, NP = kPlanes<T>;
    constexpr int NKS = D / 16, NDT = D / 32;
    typedef RowStage<D, NS, T> Stage;
    constexpr uint32_t STAGE = NS * Stage::TILE, RED = (NS - 1) * WB * NDT * 4096;
    __shared__ __attribute__((aligned(16))) char smem[NBUF * STAGE > RED ? NBUF * STAGE : RED];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wb = wave % WB, ws = wave / WB, g = lane >> 5, ln = lane & 31;
    int bh, qb;
    map_block(blockIdx.x, (p.Sq + BM - 1) / BM, p.B * p.H, true, bh, qb);
    const int b = bh / p.H, h = bh - b * p.H, bk = b * p.Hkv + h / (p.H / p.Hkv);
    const int q0 = qb * BM, qw = q0 + wb * 32, qi = qw + ln, kl = window_keys(p, b);
    const Band band{p.window, p.sinks};
    KeyStages ks;
    ks.init(q0, q0 + BM < p.Sq ? q0 + BM : p.Sq, kl, BN, band);
    const int nst = ks.count();
    const T* Kg = (const T*)p.k + (size_t)bk * p.Sk * D;
    const T* Vg = (const T*)p.v + (size_t)bk * p.Sk * D;

    Stage in;
    in.init(tid);
    if (nst > 0) in.load(Kg, Vg, ks.stage(0) * BN, kl);
    const size_t qr = ((size_t)bh * p.Sq + (qi < p.Sq ? qi : p.Sq - 1));
    const T* qrow = (const T*)p.q + qr * D;
    const T* grow = (const T*)p.dO + qr * D;
    const T* orow = (const T*)p.o_in + qr * D;
    Frag<NP> qf[NKS], of[NKS];
    load_row_frags<D>(qrow, g, true, qf);
    float dl = 0.f;
    for (int k = 0; k < NKS; k++) {
        Raw8<T> x, y;
        x.load(grow + k * 16 + g * 8);
        y.load(orow + k * 16 + g * 8);
        of[k] = x.frag();
        for (int e = 0; e < 8; e++) dl = __builtin_fmaf(x.f(e), y.f(e), dl);
    }
    dl = pair_sum32(dl);
    const float lq = lse_log2(p.lse_in[qr]);
    if (ws == 0 && g == 0 && qi < p.Sp) {
        const size_t x = (size_t)bh * p.Sp + qi;
        p.lse2[x] = qi < p.Sq ? lq : INFINITY;
        p.delta[x] = qi < p.Sq ? dl : 0.f;
    }
    SplitTile<D> tl;
    tl.init(lane);

    f32x16 acc[NDT];
    for (int t = 0; t < NDT; t++) acc[t] = f32x16{};
    const float c2 = p.scale_log2;
    auto compute = [&](int st, int buf) {
        const int kb = ks.stage(st) * BN + ws * 32;
        if (kb >= kl || !band.any(qw, qw + 31, kb, kb + 31)) return;  // wave-uniform
        char* tile = smem + buf * STAGE + ws * Stage::TILE;
        f32x16 s = f32x16{}, dp = f32x16{};
        for (int k = 0; k < NKS; k++) {
            s = mfma_n(tile_row<D, NP>(tl, tile, 0, k), qf[k], s);
            dp = mfma_n(tile_row<D, NP>(tl, tile, 1, k), of[k], dp);
        }
        const bool part = kb + 32 > kl || !band.all(qw, qw + 31, kb, kb + 31);
        Frag<NP> df[2];
        for (int k = 0; k < 2; k++) {
            float d[8];
            for (int j = 0; j < 8; j++) {
                const int r = 8 * k + j;
                d[j] = fast_exp2(__builtin_fmaf(s[r], c2, -lq)) * (dp[r] - dl);
                if (part) {
                    const int key = kb + 8 * (r >> 2) + 4 * g + (r & 3);
                    d[j] = key < kl && band.sees(qi, key) ? d[j] : 0.f;
                }
            }
            df[k] = to_frag<NP>(d);
        }
        for (int k = 0; k < 2; k++)
            for (int t = 0; t < NDT; t++)
                acc[t] = mfma_n(tile_col<D, NP>(tl, tile, 0, k, t), df[k], acc[t]);
    };
    if (nst > 0) in.store(smem, tid);
    __syncthreads();
    for (int st = 0; st < nst; st++) {
        const int buf = NBUF == 2 ? st & 1 : 0;
        if (st + 1 < nst) in.load(Kg, Vg, ks.stage(st + 1) * BN, kl);
        compute(st, buf);
        if (NBUF == 1) __syncthreads();
        if (st + 1 < nst) in.store(smem + (NBUF == 2 ? buf ^ 1 : 0) * STAGE, tid);
        __syncthreads();
    }
    if (!merge_stream<NDT, WB, NS>(acc, smem, wb, ws, lane, NS)) return;
    {
        bool bad = false;
        SplitCheck chk;
        for (int t = 0; t < NDT; t++)
            for (int r = 0; r < 16; r++) {
                if constexpr (NP == 3) chk.add(acc[t][r]);
                else bad |= nonfinite(acc[t][r]);
            }
        if constexpr (NP == 3) bad = chk.plain();
        if (__builtin_amdgcn_ballot_w64(bad && qi < p.Sq)) {
            window_dq_plain<D, T>(p, bh, bk, kl, band, qw, lq, dl);
            return;
        }
    }
    if (qi >= p.Sq) return;
    T* out = (T*)p.dq + qr * D;
    for (int t = 0; t < NDT; t++)
        for (int rq = 0; rq < 4; rq++) {
            f32x4 v;
            for (int i = 0; i < 4; i++) v[i] = acc[t][rq * 4 + i] * p.scale;
            store4<T>(out + t * 32 + rq * 8 + g * 4, v);
        }
}

namespace {

// The steps of a key block: query stages [st0, st0 + nst) of BQ rows for each of
// the G query heads of its key head.
struct BlockSteps {
    int st0, nst;
    GONN_DEV void init(int k0, int BK, int BQ, int Sq, int kl, const Band& m) {
        st0 = k0 / BQ;
        int end = Sq;  // one past the last query that sees one of the keys
        if (k0 >= m.sinks && Sq - k0 > BK - 1 + m.window) end = k0 + BK - 1 + m.window;
        nst = k0 < kl && k0 < Sq ? (end + BQ - 1) / BQ - st0 : 0;
    }
};

// One workgroup's share of the dK/dV grid: chunk c of key block kb of slice bk.
struct DkdvItem {
    int bk, slot, kb, c, per, b, hk, G, kl;
    GONN_DEV void init(const WindowParams& p) {
        // Slots of a slice: the sinks' blocks first, per_sink items each.
        map_block(blockIdx.x, p.slots, p.B * p.Hkv, false, bk, slot);
        const int sink_slots = p.sink_blocks * p.per_sink;
        const bool sink = slot < sink_slots;
        per = sink ? p.per_sink : p.per_block;
        const int i0 = sink ? slot : slot - sink_slots;
        kb = (sink ? 0 : p.sink_blocks) + i0 / per;
        c = i0 % per;
        b = bk / p.Hkv;
        hk = bk - b * p.Hkv;
        G = p.H / p.Hkv;
        kl = window_keys(p, b);
    }
};
// dV and dK of key kj (row kj - k0 of the block), channels d .. d + 3: the gradients,
// or one item's unscaled sums. live: the key takes part.
template <int D, typename T>
GONN_DEV void write_dkdv(const WindowParams& p, const DkdvItem& it, int BK, int kj, int k0, int d,
                         f32x4 dv, f32x4 dk, bool live) {
    if (!live) dv = dk = f32x4{};
    if (it.per > 1) {
        float* part = p.part + (((size_t)it.bk * p.slots + it.slot) * 2 * BK + kj - k0) * D + d;
        *(f32x4*)part = dv;
        *(f32x4*)(part + (size_t)BK * D) = dk;
    } else {
        const size_t x = ((size_t)it.bk * p.Sk + kj) * D + d;
        store4<T>((T*)p.dv + x, dv);
        store4<T>((T*)p.dk + x, dk * p.scale);
    }
}

// dV and dK of a wave's 32 keys over steps [s0, s1), plain fp32 products, 32 channels
// at a time.
template <int D, typename T>
GONN_DEV void window_dkdv_plain(const WindowParams& p, const DkdvItem& it, const BlockSteps& bs,
                                int BK, int BQ, int s0, int s1, const Band& band, int kw) {
    const int lane = threadIdx.x & 63, g = lane >> 5, ln = lane & 31, kj = kw + ln;
    const size_t kr = ((size_t)it.bk * p.Sk + (kj < p.Sk ? kj : p.Sk - 1)) * D;
    const T *krow = (const T*)p.k + kr, *vrow = (const T*)p.v + kr;
#pragma unroll 1
    for (int t = 0; t < D / 32; t++) {
        f32x16 dv = f32x16{}, dk = f32x16{};
#pragma unroll 1
        for (int st = s0; st < s1; st++) {
            const size_t bh = (size_t)it.b * p.H + it.hk * it.G + st / bs.nst, base = bh * p.Sq;
#pragma unroll 1
            for (int off = 0; off < BQ; off += 32) {
                const int q0 = (bs.st0 + st % bs.nst) * BQ + off;
                if (q0 >= p.Sq || !band.any(q0, q0 + 31, kw, kw + 31)) continue;
                const size_t qr = (base + (q0 + ln < p.Sq ? q0 + ln : p.Sq - 1)) * D;
                f32x16 s, dp;
                plain_products<D>((const T*)p.q + qr, krow, (const T*)p.dO + qr, vrow, g, s, dp);
                for (int r = 0; r < 16; r++) {
                    const int q = q0 + 8 * (r >> 2) + 4 * g + (r & 3), qc = q < p.Sq ? q : p.Sq - 1;
                    const bool on = q < p.Sq && kj < it.kl && band.sees(q, kj);
                    const float pv = fast_exp2(__builtin_fmaf(s[r], p.scale_log2, -p.lse2[bh * p.Sp + qc]));
                    s[r] = on ? pv : 0.f;
                    dp[r] = on ? pv * (dp[r] - p.delta[bh * p.Sp + qc]) : 0.f;
                }
#pragma unroll 1
                for (int x = 0; x < 32; x++) {
                    const int r = x >> 1, h = x & 1, q = q0 + 8 * (r >> 2) + 4 * h + (r & 3);
                    const float wp = weight_of(s, r, h, g), wd = weight_of(dp, r, h, g);
                    if (q >= p.Sq) continue;  // uniform
                    const bool on = kj < it.kl && band.sees(q, kj);
                    add_row32(dv, wp, (const T*)p.dO + (base + q) * D + 32 * t, g, on);
                    add_row32(dk, wd, (const T*)p.q + (base + q) * D + 32 * t, g, on);
                }
            }
        }
        if (kj < p.Sk)
            for (int rq = 0; rq < 4; rq++) {
                f32x4 x, y;
                for (int i = 0; i < 4; i++) {
                    x[i] = dv[rq * 4 + i];
                    y[i] = dk[rq * 4 + i];
                }
                write_dkdv<D, T>(p, it, BK, kj, kw / BK * BK, 32 * t + 8 * rq + 4 * g, x, y, kj < it.kl);
            }
    }
}

}  // namespace

template <int D, typename T, int WB, int NBUF, int OCC>
__global__ __launch_bounds__(256, OCC) void window_dkdv_kernel(WindowParams p) {
    constexpr int NS = 4 / WB, BK = WB * 32, BQ = NS * 32, NP = kPlanes<T>;
    constexpr int NKS = D / 16, NDT = D / 32;
    typedef RowStage<D, NS, T> Stage;
    constexpr uint32_t STAGE = NS * Stage::TILE, RED = (NS - 1) * WB * 2 * NDT * 4096;
    __shared__ __attribute__((aligned(16))) char smem[NBUF * STAGE > RED ? NBUF * STAGE : RED];
    __shared__ __attribute__((aligned(16))) float sld[NBUF][2][BQ];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wb = wave % WB, ws = wave / WB, g = lane >> 5, ln = lane & 31;
    DkdvItem it;
    it.init(p);
    const int bk = it.bk, b = it.b, hk = it.hk, G = it.G, kl = it.kl, per = it.per;
    const int k0 = it.kb * BK, kw = k0 + wb * 32, kj = kw + ln;
    const Band band{p.window, p.sinks};
    BlockSteps bs;
    bs.init(k0, BK, BQ, p.Sq, kl, band);
    const int s0 = it.c * p.chunk;
    int s1 = bs.nst * G;
    s1 = per > 1 && s1 - s0 > p.chunk ? s0 + p.chunk : s1;
    if (per > 1 && s0 >= s1) return;  // no such item: nothing is read from its slot

    Stage in;
    in.init(tid);
    float rl = 0.f, rd = 0.f;
    auto gload = [&](int st) {
        const size_t bh = (size_t)b * p.H + hk * G + st / bs.nst;
        const int q0 = (bs.st0 + st % bs.nst) * BQ;
        in.load((const T*)p.q + bh * p.Sq * D, (const T*)p.dO + bh * p.Sq * D, q0, p.Sq);
        if (tid < BQ) {
            const int q = q0 + tid;
            rl = q < p.Sp ? p.lse2[bh * p.Sp + q] : INFINITY;
            rd = q < p.Sp ? p.delta[bh * p.Sp + q] : 0.f;
        }
    };
    auto sstore = [&](int buf) {
        in.store(smem + buf * STAGE, tid);
        if (tid < BQ) {
            sld[buf][0][tid] = rl;
            sld[buf][1][tid] = rd;
        }
    };
    if (s0 < s1) gload(s0);
    const size_t kr = ((size_t)bk * p.Sk + (kj < p.Sk ? kj : p.Sk - 1)) * D;
    const T *krow = (const T*)p.k + kr, *vrow = (const T*)p.v + kr;
    Frag<NP> kf[NKS], vf[NKS];
    load_row_frags<D>(krow, g, kj < kl, kf);
    load_row_frags<D>(vrow, g, kj < kl, vf);
    SplitTile<D> tl;
    tl.init(lane);
    f32x16 acc[2 * NDT];  // dV^T tiles, then dK^T tiles
    for (int t = 0; t < 2 * NDT; t++) acc[t] = f32x16{};
    const float c2 = p.scale_log2;

    auto compute = [&](int st, int buf) {
        const int q0 = (bs.st0 + st % bs.nst) * BQ + ws * 32;
        if (q0 >= p.Sq || !band.any(q0, q0 + 31, kw, kw + 31)) return;  // wave-uniform
        char* tile = smem + buf * STAGE + ws * Stage::TILE;
        f32x16 s = f32x16{}, dp = f32x16{};
        for (int k = 0; k < NKS; k++) s = mfma_n(tile_row<D, NP>(tl, tile, 0, k), kf[k], s);
        for (int k = 0; k < NKS; k++) dp = mfma_n(tile_row<D, NP>(tl, tile, 1, k), vf[k], dp);
        const bool part = kw + 32 > kl || !band.all(q0, q0 + 31, kw, kw + 31);
        Frag<NP> pf[2], df[2];
        for (int k = 0; k < 2; k++) {
            float e[8], d[8];
            for (int j4 = 0; j4 < 2; j4++) {
                const int qr = 16 * k + 8 * j4 + 4 * g;
                const f32x4 L = *(const f32x4*)&sld[buf][0][ws * 32 + qr];
                const f32x4 Dl = *(const f32x4*)&sld[buf][1][ws * 32 + qr];
                for (int j = 0; j < 4; j++) {
                    const int r = 8 * k + 4 * j4 + j;
                    float pv = fast_exp2(__builtin_fmaf(s[r], c2, -L[j]));
                    float dv = pv * (dp[r] - Dl[j]);
                    if (part) {
                        const bool on = kj < kl && band.sees(q0 + qr + j, kj);
                        pv = on ? pv : 0.f;
                        dv = on ? dv : 0.f;
                    }
                    e[4 * j4 + j] = pv;
                    d[4 * j4 + j] = dv;
                }
            }
            pf[k] = to_frag<NP>(e);
            df[k] = to_frag<NP>(d);
        }
        for (int k = 0; k < 2; k++)
            for (int t = 0; t < NDT; t++)
                acc[t] = mfma_n(tile_col<D, NP>(tl, tile, 1, k, t), pf[k], acc[t]);
        for (int k = 0; k < 2; k++)
            for (int t = 0; t < NDT; t++)
                acc[NDT + t] = mfma_n(tile_col<D, NP>(tl, tile, 0, k, t), df[k], acc[NDT + t]);
    };
    if (s0 < s1) sstore(0);
    __syncthreads();
    for (int st = s0; st < s1; st++) {
        const int buf = NBUF == 2 ? (st - s0) & 1 : 0;
        if (st + 1 < s1) gload(st + 1);
        compute(st, buf);
        if (NBUF == 1) __syncthreads();
        if (st + 1 < s1) sstore(NBUF == 2 ? buf ^ 1 : 0);
        __syncthreads();
    }
    if (!merge_stream<2 * NDT, WB, NS>(acc, smem, wb, ws, lane, NS)) return;
    {
        bool bad = false;
        SplitCheck chk;
        for (int t = 0; t < 2 * NDT; t++)
            for (int r = 0; r < 16; r++) {
                if constexpr (NP == 3) chk.add(acc[t][r]);
                else bad |= nonfinite(acc[t][r]);
            }
        if constexpr (NP == 3) bad = chk.plain();
        if (__builtin_amdgcn_ballot_w64(bad && kj < kl)) {
            window_dkdv_plain<D, T>(p, it, bs, BK, BQ, s0, s1, band, kw);
            return;
        }
    }
    if (kj >= p.Sk) return;
    for (int t = 0; t < NDT; t++)
        for (int rq = 0; rq < 4; rq++) {
            f32x4 x, y;
            for (int i = 0; i < 4; i++) {
                x[i] = acc[t][rq * 4 + i];
                y[i] = acc[NDT + t][rq * 4 + i];
            }
            write_dkdv<D, T>(p, it, BK, kj, k0, t * 32 + rq * 8 + g * 4, x, y, kj < kl);
        }
}

// dK and dV of the blocks of several items: their partials in order. Four
// elements a thread; blocks [0, nb) of each slice.
template <int D, typename T>
__global__ __launch_bounds__(256) void window_join_kernel(WindowParams p, int BK, int BQ, int nb,
                                                          size_t n) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int d = (int)(i % (D / 4)) * 4;
    size_t r = i / (D / 4);
    const int w = (int)(r & 1);
    r >>= 1;
    const int row = (int)(r % BK);
    r /= BK;
    const int kb = (int)(r % nb), bk = (int)(r / nb), b = bk / p.Hkv, kj = kb * BK + row;
    if (kj >= p.Sk) return;
    const bool sink = kb < p.sink_blocks;
    const int per = sink ? p.per_sink : p.per_block;
    if (per == 1) return;  // written by its item
    const int slot = sink ? kb * per : p.sink_blocks * p.per_sink + (kb - p.sink_blocks) * per;
    int kl = p.kv_len ? p.kv_len[b] : p.Sk;
    kl = kl < 0 ? 0 : (kl > p.Sk ? p.Sk : kl);
    BlockSteps bs;
    bs.init(kb * BK, BK, BQ, p.Sq, kl, {p.window, p.sinks});
    const int cnt = (bs.nst * (p.H / p.Hkv) + p.chunk - 1) / p.chunk;
    const float* src = p.part + (((size_t)bk * p.slots + slot) * 2 * BK + w * BK + row) * D + d;
    f32x4 sum = f32x4{};
    for (int c = 0; c < cnt; c++) sum += *(const f32x4*)(src + (size_t)c * 2 * BK * D);
    if (w) sum *= p.scale;
    store4<T>((T*)(w ? p.dk : p.dv) + ((size_t)bk * p.Sk + kj) * D + d, sum);
}

namespace {

// Shape of the dK/dV grid.
struct DkdvShape {
    int BK, BQ;
};
DkdvShape dkdv_shape(const WindowParams& p, int is_bf16) {
    const long long cus = device_cus();
    const long long b128 = (long long)((p.Sk + 127) / 128) * p.B * p.Hkv;
    if (b128 >= cus && is_bf16) return {128, 32};
    return {64, 64};
}

template <int D, typename T, int WB, int NBUF, int OCC>
void run_dkdv(const WindowParams& p, hipStream_t s) {
    const unsigned grid = (unsigned)p.slots * (unsigned)(p.B * p.Hkv);
    window_dkdv_kernel<D, T, WB, NBUF, OCC><<<grid, 256, 0, s>>>(p);
    const int BK = WB * 32, BQ = 4 / WB * 32, nkb = (p.Sk + BK - 1) / BK;
    const int nb = p.per_block > 1 ? nkb : (p.per_sink > 1 ? p.sink_blocks : 0);
    if (!nb) return;
    const size_t n = (size_t)p.B * p.Hkv * nb * BK * 2 * (D / 4);
    window_join_kernel<D, T><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(p, BK, BQ, nb, n);
}

template <int D, typename T>
void run_window_bwd(const WindowParams& p, hipStream_t s) {
    const long long cus = device_cus(), BH = (long long)p.B * p.H;
    const long long b128 = (long long)((p.Sq + 127) / 128) * BH;
    const unsigned g128 = (unsigned)b128, g64 = (unsigned)((p.Sq + 63) / 64 * BH);
    const DkdvShape sh = dkdv_shape(p, sizeof(T) == 2);
    if constexpr (sizeof(T) == 2) {
        if (b128 >= 2 * cus) window_dq_kernel<D, T, 4, 2, 2><<<g128, 256, 0, s>>>(p);
        else window_dq_kernel<D, T, 2, 2, 1><<<g64, 256, 0, s>>>(p);
        if (sh.BK == 128) run_dkdv<D, T, 4, 2, 1>(p, s);
        else run_dkdv<D, T, 2, 2, 1>(p, s);
    } else {
        window_dq_kernel<D, T, 2, 1, 1><<<g64, 256, 0, s>>>(p);
        run_dkdv<D, T, 2, 1, 1>(p, s);
    }
}

}  // namespace

size_t plan_window_bwd(WindowParams& p, int D, int is_bf16) {
    const DkdvShape sh = dkdv_shape(p, is_bf16);
    const long long slices = (long long)p.B * p.Hkv, G = p.H / p.Hkv, want = 2 * device_cus();
    const int nkb = (p.Sk + sh.BK - 1) / sh.BK;
    const long long all = G * ((p.Sq + sh.BQ - 1) / sh.BQ);
    const long long band = std::min<long long>(
        all, G * (((long long)sh.BK - 1 + p.window + sh.BQ - 1) / sh.BQ + 1));
    p.sink_blocks = std::min(nkb, (p.sinks + sh.BK - 1) / sh.BK);
    // Items as long as a block's band, shorter where that leaves the device
    // without work, but no shorter than 4 stages.
    const long long items = slices * nkb;
    long long chunk = band;
    if (items < want) chunk = std::max<long long>(4, (band * items + want - 1) / want);
    chunk = std::min(chunk, all);
    p.chunk = (int)chunk;
    p.per_block = (int)((band + chunk - 1) / chunk);
    p.per_sink = (int)((all + chunk - 1) / chunk);
    p.slots = p.sink_blocks * p.per_sink + (nkb - p.sink_blocks) * p.per_block;
    const size_t part = p.per_block > 1 || (p.sink_blocks && p.per_sink > 1)
                            ? (size_t)slices * p.slots * 2 * sh.BK * D * sizeof(float)
                            : 0;
    return part;
}

hipError_t launch_window_bwd(const WindowParams& p, int D, int is_bf16, hipStream_t s) {
    if (D == 64) {
        if (is_bf16) run_window_bwd<64, bf16>(p, s);
        else run_window_bwd<64, float>(p, s);
    } else if (D == 128) {
        if (is_bf16) run_window_bwd<128, bf16>(p, s);
        else run_window_bwd<128, float>(p, s);
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace gonn
