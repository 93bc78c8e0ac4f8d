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
//
// S and dP are formed in both kernels: seven products for the five of the formulas.
// Writing dS for the first kernel to read would spare two of them, about 120 us of the
// 563 below, for a second buffer the size of the visible pairs.
//
// Bound: the matrix cores. 2 x 16 heads over 4, 8192 queries, window 1024, 4 sinks, D
// 128, bf16: 563 us, 573 TFLOP/s of the five products; dQ 237 (820 of its three), dK/dV
// 292 and the sinks' items 32 (797 of the four), join 14. Matrix pipe busy 0.34 and 0.39
// of the cycles at 2.4 GHz, about 5.5 and 4.3 VALU instructions per MFMA; dK/dV runs one
// wave per SIMD with 252 registers beside 256 accumulators. fp32, 4 x 12 x 1021, window
// 200, D 64: 118 us (dQ 54, dK/dV 63), 42 TFLOP/s in six products each. 8 heads over 2 x
// 777, window 128, D 128, bf16: 34 us, three short kernels in a row.
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
    constexpr int NP = kPlanes<T>, NS = 4 / WB, BM = WB * 32;
    // Tiles of a stage per wave: two where four waves share a tile, which halves the barriers.
    constexpr int KT = NP == 1 && NS == 1 ? 2 : 1, NT = NS * KT, BN = NT * 32;
    constexpr int NKS = D / 16, NDT = D / 32;
    typedef RowStage<D, NT, T> Stage;
    constexpr uint32_t STAGE = NT * Stage::TILE, RED = (NS - 1) * WB * NDT * 4096;
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

    static_assert(!Stage::DIRECT || NBUF == 2, "loads to LDS need the other buffer");
    const uint32_t lds = lds_addr(smem);
    Stage in;
    in.init(tid);
    if (nst > 0) {
        if constexpr (Stage::DIRECT) in.load(Kg, Vg, ks.stage(0) * BN, kl, lds, wave);
        else in.load(Kg, Vg, ks.stage(0) * BN, kl);
    }
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
    auto compute = [&](int st, int buf, int x) {
        const int kb = ks.stage(st) * BN + (ws * KT + x) * 32;
        if (kb >= kl || !band.any(qw, qw + 31, kb, kb + 31)) return;  // wave-uniform
        char* tile = smem + buf * STAGE + (ws * KT + x) * Stage::TILE;
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
    if constexpr (Stage::DIRECT) {
        for (int st = 0; st < nst; st++) {
            GONN_VMCNT(0);
            __syncthreads();  // stage st has landed, and its buffer's last reader is past it
            if (st + 1 < nst)
                in.load(Kg, Vg, ks.stage(st + 1) * BN, kl, lds + (uint32_t)((st + 1) & 1) * STAGE, wave);
            for (int x = 0; x < KT; x++) compute(st, st & 1, x);
        }
        if (NS > 1) __syncthreads();  // the merge reuses the stages
    } else {
        if (nst > 0) in.store(smem, tid);
        __syncthreads();
        for (int st = 0; st < nst; st++) {
            const int buf = NBUF == 2 ? st & 1 : 0;
            if (st + 1 < nst) in.load(Kg, Vg, ks.stage(st + 1) * BN, kl);
            compute(st, buf, 0);
            if (NBUF == 1) __syncthreads();
            if (st + 1 < nst) in.store(smem + (NBUF == 2 ? buf ^ 1 : 0) * STAGE, tid);
            __syncthreads();
        }
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

// Keys of the tail's items, of which the sinks are the first (32; 64 where the stages
// of four waves along the queries do not fit in LDS), and query rows per stage.
constexpr int tail_keys(int D, bool f32) { return f32 && D == 128 ? 64 : 32; }
constexpr int tail_rows(int D, bool f32) { return 4096 / tail_keys(D, f32); }

// The steps of a key block: nst query stages of BQ rows, from q0 on, for each of the G
// query heads of its key head.
struct BlockSteps {
    int q0, nst;
    GONN_DEV void init(const WindowParams& p, int k0, int BK, int BQ, int kl, bool tail) {
        if (tail) {  // the sinks' later queries
            q0 = p.tail_q0;
            nst = k0 < kl ? (p.Sq - q0 + BQ - 1) / BQ : 0;
            return;
        }
        q0 = k0 / BQ * BQ;
        int end = p.Sq;  // one past the last query that sees one of the keys
        if ((k0 >= p.sinks || p.per_tail) && p.Sq - k0 > BK - 1 + p.window) end = k0 + BK - 1 + p.window;
        nst = k0 < kl && k0 < p.Sq ? (end - q0 + BQ - 1) / BQ : 0;
    }
};

// One workgroup's share of a dK/dV grid: chunk c of key block kb of slice bk.
struct DkdvItem {
    int bk, kb, c, b, hk, G, kl;
    float* part;  // its partial, (2, BK, D), or null: it writes the gradients
    GONN_DEV void init(const WindowParams& p, int BK, int D, bool tail) {
        const int slots = tail ? p.per_tail : p.slots;
        int slot;
        map_block(blockIdx.x, slots, p.B * p.Hkv, false, bk, slot);
        b = bk / p.Hkv;
        hk = bk - b * p.Hkv;
        G = p.H / p.Hkv;
        kl = window_keys(p, b);
        const size_t at = ((size_t)bk * slots + slot) * 2 * BK * D;
        if (tail) {
            kb = 0;
            c = slot;
            part = p.part_tail + at;
            return;
        }
        // Slots of a slice: the sinks' blocks first, per_sink items each.
        const int sink_slots = p.sink_blocks * p.per_sink;
        const bool sink = slot < sink_slots;
        const int per = sink ? p.per_sink : p.per_block, i0 = sink ? slot : slot - sink_slots;
        kb = (sink ? 0 : p.sink_blocks) + i0 / per;
        c = i0 % per;
        part = per > 1 || (p.per_tail && kb == 0) ? p.part + at : nullptr;
    }
};
// dV and dK of key kj (row kj - k0 of the block), channels d .. d + 3: the gradients,
// or one item's unscaled sums. live: the key takes part.
template <int D, typename T>
GONN_DEV void write_dkdv(const WindowParams& p, const DkdvItem& it, int BK, int kj, int d, f32x4 dv,
                         f32x4 dk, bool live) {
    if (!live) dv = dk = f32x4{};
    if (it.part) {
        float* part = it.part + (size_t)(kj - it.kb * BK) * D + d;
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
                const int q0 = bs.q0 + st % bs.nst * BQ + off;
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
                write_dkdv<D, T>(p, it, BK, kj, 32 * t + 8 * rq + 4 * g, x, y, kj < it.kl);
            }
    }
}

}  // namespace

// TAIL: the items of the sinks' later queries.
template <int D, typename T, int WB, int NBUF, int OCC, bool TAIL = false>
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
    it.init(p, BK, D, TAIL);
    const int bk = it.bk, b = it.b, hk = it.hk, G = it.G, kl = it.kl;
    const int k0 = it.kb * BK, kw = k0 + wb * 32, kj = kw + ln;
    const Band band{p.window, p.sinks};
    BlockSteps bs;
    bs.init(p, k0, BK, BQ, kl, TAIL);
    const int chunk = TAIL ? p.tail_chunk : p.chunk, s0 = it.c * chunk;
    const int s1 = bs.nst * G - s0 > chunk ? s0 + chunk : bs.nst * G;
    if (it.part && s0 >= s1) return;  // no such item: nothing is read from its slot

    static_assert(!Stage::DIRECT || NBUF == 2, "loads to LDS need the other buffer");
    const uint32_t lds = lds_addr(smem);
    Stage in;
    in.init(tid);
    float rl = 0.f, rd = 0.f;
    // Step st: its rows (to buffer buf of LDS, or to registers), its L and D to registers.
    auto gload = [&](int st, int buf) {
        const size_t bh = (size_t)b * p.H + hk * G + st / bs.nst;
        const int q0 = bs.q0 + st % bs.nst * BQ;
        const T *Qg = (const T*)p.q + bh * p.Sq * D, *dOg = (const T*)p.dO + bh * p.Sq * D;
        if constexpr (Stage::DIRECT) in.load(Qg, dOg, q0, p.Sq, lds + buf * STAGE, wave);
        else in.load(Qg, dOg, q0, p.Sq);
        if (tid < BQ) {
            const int q = q0 + tid;
            rl = q < p.Sp ? p.lse2[bh * p.Sp + q] : INFINITY;
            rd = q < p.Sp ? p.delta[bh * p.Sp + q] : 0.f;
        }
    };
    auto sstore = [&](int buf) {
        if constexpr (!Stage::DIRECT) in.store(smem + buf * STAGE, tid);
        if (tid < BQ) {
            sld[buf][0][tid] = rl;
            sld[buf][1][tid] = rd;
        }
    };
    if (s0 < s1) gload(s0, 0);
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
        const int q0 = bs.q0 + st % bs.nst * BQ + ws * 32;
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
    if constexpr (Stage::DIRECT) {
        for (int st = s0; st < s1; st++) {
            const int buf = (st - s0) & 1;
            sstore(buf);
            GONN_VMCNT(0);
            __syncthreads();  // step st has landed, and its buffer's last reader is past it
            if (st + 1 < s1) gload(st + 1, buf ^ 1);
            compute(st, buf);
        }
        if (NS > 1) __syncthreads();  // the merge reuses the stages
    } else {
        if (s0 < s1) sstore(0);
        __syncthreads();
        for (int st = s0; st < s1; st++) {
            const int buf = NBUF == 2 ? (st - s0) & 1 : 0;
            if (st + 1 < s1) gload(st + 1, 0);
            compute(st, buf);
            if (NBUF == 1) __syncthreads();
            if (st + 1 < s1) sstore(NBUF == 2 ? buf ^ 1 : 0);
            __syncthreads();
        }
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
            write_dkdv<D, T>(p, it, BK, kj, t * 32 + rq * 8 + g * 4, x, y, kj < kl);
        }
}

// ---------------------------------------------------------------------------
// bf16 dK/dV of large grids: 128 keys per workgroup (32 per wave, K and V in
// registers), query tiles of 64 in four-slot LDS rings filled straight from memory,
// one wave per SIMD, in the hand-ordered three-stage pipeline of attn_bwd.hip. Step
// i issues, without dependences between them,
//   MFMA  S(i+1) = Q K^T, dP(i+1) = dO V^T
//   VALU  P(i) = exp2(S c2 - LSE log2e), dS(i) = P (dP - delta), packed to bf16
//   MFMA  dV^T += dO^T P(i-1), dK^T += Q^T dS(i-1)
// over the query heads and tiles of its item in turn. Slot e issues the LDS read of
// MFMA e + 3, MFMA e, a tile load and the VALU work mapped to it. Masked scores are
// set to -inf between steps, on tiles that cross the window's or the causal edge. S
// and dP have VGPR accumulators and K and V lie in AGPRs (inline asm, whose wait
// states the kernel provides itself: three s_nop 7 that the accumulators pass
// through behind each step's last such MFMA).
// ---------------------------------------------------------------------------
GONN_DEV void mfma_vacc0(f32x16& d, bf16x8 a, bf16x8 b) {
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(d) : "v"(a), "a"(b));
}
GONN_DEV void mfma_vacc(f32x16& d, bf16x8 a, bf16x8 b) {
    asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(d) : "v"(a), "a"(b));
}

template <int D>
__global__ __launch_bounds__(256, 1) void window_dkdv_pipe_kernel(WindowParams p) {
    constexpr int BK = 128, BQ = 64, NKS = D / 16, NDT = D / 32;
    constexpr int RTILE = BQ * D;  // elements of a Q or dO tile
    constexpr uint32_t RTB = RTILE * 2;
    constexpr int NRI = RTILE / 8 / 256, NSLOT = 4;
    __shared__ __attribute__((aligned(16))) bf16 sQ[NSLOT * RTILE];
    __shared__ __attribute__((aligned(16))) bf16 sdO[NSLOT * RTILE];
    __shared__ __attribute__((aligned(16))) float sLD[2][2 * BQ];  // lse2, then delta

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 5, ln = lane & 31;
    DkdvItem it;
    it.init(p, BK, D, false);
    const int k0 = it.kb * BK, kw = k0 + wave * 32, kj = kw + ln, kl = it.kl;
    const Band band{p.window, p.sinks};
    BlockSteps bs;
    bs.init(p, k0, BK, BQ, kl, false);
    const int s0 = it.c * p.chunk;
    int nq = bs.nst * it.G - s0;
    nq = nq > p.chunk ? p.chunk : nq;
    if (nq <= 0) {  // no such item, or no query sees the block
        if (it.part) return;
        for (int i = tid; i < BK * D / 4; i += 256) {
            const int r = i / (D / 4);
            if (k0 + r < p.Sk)
                write_dkdv<D, bf16>(p, it, BK, k0 + r, i % (D / 4) * 4, f32x4{}, f32x4{}, false);
        }
        return;
    }

    bf16x8 kf[NKS], vf[NKS];
    {
        const size_t kr = ((size_t)it.bk * p.Sk + (kj < p.Sk ? kj : p.Sk - 1)) * D;
        const bf16 *krow = (const bf16*)p.k + kr + g * 8, *vrow = (const bf16*)p.v + kr + g * 8;
        // The scale's sign goes into K here, so that -inf masks stay -inf.
        const uint32_t flip = p.sign < 0.f ? 0x80008000u : 0u, keep = p.sign != 0.f ? ~0u : 0u;
        for (int ks = 0; ks < NKS; ks++) {
            u32x4 a = u32x4{}, c = u32x4{};
            if (kj < kl) {
                a = *(const u32x4*)(krow + ks * 16);
                c = *(const u32x4*)(vrow + ks * 16);
            }
            for (int e = 0; e < 4; e++) a[e] = (a[e] ^ flip) & keep;
            kf[ks] = __builtin_bit_cast(bf16x8, a);
            vf[ks] = __builtin_bit_cast(bf16x8, c);
        }
    }
    for (int ks = 0; ks < NKS; ks++) {  // into AGPRs, then wait states
        asm volatile("s_nop 4" : "+a"(kf[ks]));
        asm volatile("s_nop 4" : "+a"(vf[ks]));
    }
    asm volatile("s_nop 7");

    // Step s of the item: query tile qt of head hh. One cursor per pipeline stage.
    struct Cursor {
        int hh, qt;
    };
    const int st0 = bs.q0 / BQ, stE = st0 + bs.nst;
    auto next = [&](Cursor c) {
        c.qt++;
        if (c.qt == stE) {
            c.qt = st0;
            c.hh++;
        }
        return c;
    };
    const int Sq = p.Sq, Sp = p.Sp;
    const size_t h0 = (size_t)it.b * p.H + it.hk * it.G;
    const bf16* Qg = (const bf16*)p.q + h0 * Sq * D;
    const bf16* dOg = (const bf16*)p.dO + h0 * Sq * D;
    // One resource over the key head's query heads: rows past a head's last are the
    // next head's, or zeros, and lse2 = +inf gives them no weight.
    const uint32_t bytes = (uint32_t)it.G * Sq * D * 2, lbytes = (uint32_t)it.G * Sp * 4;
    const brsrc rq = make_rsrc(Qg, bytes), rdo = make_rsrc(dOg, bytes);
    const brsrc rl = make_rsrc(p.lse2 + h0 * Sp, lbytes), rd = make_rsrc(p.delta + h0 * Sp, lbytes);
    uint32_t roff[NRI];
    for (int i = 0; i < NRI; i++) {
        int r, c;
        slab_chunk(i * 256 + tid, BQ, r, c);
        roff[i] = (uint32_t)((r * D + c * 8) * 2);
    }
    const uint32_t lq = lds_addr(sQ) + wave * 1024, ldo = lds_addr(sdO) + wave * 1024;
    auto dma_row = [&](uint32_t so, int slot, int j, uint32_t on) {
        const int i = j % NRI;
        dma16_if(j < NRI ? rq : rdo, (j < NRI ? lq : ldo) + slot * RTB + i * 4096, roff[i], so, on);
    };
    auto row_off = [&](Cursor c) { return (uint32_t)((c.hh * Sq + c.qt * BQ) * D) * 2u; };
    auto dma_ld = [&](Cursor c, int slot) {
        if (wave == 0) {
            const uint32_t dl = lds_addr(sLD) + slot * 2 * BQ * 4, so = (uint32_t)(c.hh * Sp + c.qt * BQ) * 4u;
            if (lane < 16) dma16(rl, dl, (lane & 15) * 16, so);
            else if (lane < 32) dma16(rd, dl, (lane & 15) * 16, so);
        }
    };

    // Operand reads (bytes from a slot's start), as in attn_bwd.hip.
    const int hs = slab_swz(ln);
    const uint32_t ra0 = (uint32_t)(ln * 64 + ((0 + g) ^ hs) * 16);
    const uint32_t ra1 = (uint32_t)(ln * 64 + ((2 + g) ^ hs) * 16);
    const int s16 = lane & 15;
    const int tcx = 2 * ((ln >> 4) & 1) + ((s16 >> 1) & 1);
    const uint32_t ta0 = (uint32_t)((4 * g + (s16 >> 2)) * 64 + (tcx ^ g) * 16 + 8 * (s16 & 1));
    const uint32_t ta1 =
        (uint32_t)((8 + 4 * g + (s16 >> 2)) * 64 + (tcx ^ (2 + g)) * 16 + 8 * (s16 & 1));
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    typedef __attribute__((address_space(3))) char lds_char;
    lds_char* const tQ = (lds_char*)sQ;
    lds_char* const tdO = (lds_char*)sdO;
    const char* cQ = (const char*)sQ;
    const char* cdO = (const char*)sdO;
    auto rowa = [&](int kk, int mt) {
        return (uint32_t)(((kk >> 1) * BQ + mt * 32) * 64) + ((kk & 1) ? ra1 : ra0);
    };

    f32x16 dvacc[NDT], dkacc[NDT];
    for (int t = 0; t < NDT; t++) dvacc[t] = dkacc[t] = f32x16{};
    const float c2 = p.c2;
    u32x4 pp[4], pd[4];  // P and dS of the tile dV/dK consume next
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

    // Scores of query tile qt that this lane's key is not seen by, to -inf.
    auto mask = [&](int qt, f32x16* s) {
        const int q0 = qt * BQ;
        if (kw + 32 <= kl && band.all(q0, q0 + BQ - 1, kw, kw + 31)) return;  // wave-uniform
        // Query 8 (r / 4) + r % 4 + 32 mt of the lane group: from lo on, and below hi.
        const int lo = kj < kl ? kj - q0 - 4 * g : BQ;
        const int hi = kj < p.sinks ? BQ : lo + p.window;
        for (int mt = 0; mt < 2; mt++)
            for (int r = 0; r < 16; r++) {
                const int c = mt * 32 + 8 * (r >> 2) + (r & 3);
                s[mt][r] = c < lo || c >= hi ? -INFINITY : s[mt][r];
            }
    };
    // One pipeline step. sA <- S(i+1), dA <- dP(i+1); sB, dB = S(i), dP(i). c1, c2q:
    // the cursors of tiles i + 1 and i + 2.
    auto step = [&](auto ha_tag, auto hb_tag, auto hc_tag, int i, Cursor c1, Cursor c2q, f32x16* sA,
                    f32x16* dA, f32x16* sB, f32x16* dB) __attribute__((always_inline)) {
        constexpr bool HA = decltype(ha_tag)::value;  // S/dP of tile i+1
        constexpr bool HB = decltype(hb_tag)::value;  // P/dS of tile i
        constexpr bool HC = decltype(hc_tag)::value;  // dV/dK of tile i-1
        const uint32_t dr = HA && i + 2 < nq;
        if (HA) dma_ld(c1, (i + 1) & 1);
        const uint32_t so2 = row_off(c2q);
        const uint32_t rsl = (uint32_t)((i + 1) & 3) * RTB;  // tile i+1 (S, dP)
        const uint32_t tsl = (uint32_t)((i + 3) & 3) * RTB;  // tile i-1 (dV, dK)
        const uint32_t nsl = (uint32_t)((i + 2) & 3);        // slot of tile i+2
        const int lsl = i & 1;

        constexpr int HCn = HC ? 2 * NDT : 0, HAn = HA ? NKS : 0;
        constexpr int GW = HCn + HAn;  // MFMAs per 16-query k-step group
        constexpr int NM = 4 * GW, LA = 3, NO = 4;
        constexpr int NDMA = 2 * NRI, SPAN = 16 < NM ? 16 : NM;
        constexpr int DS = SPAN / NDMA > 0 ? SPAN / NDMA : 1;
        bf16x8 opr[NO];
        auto fetch = [&](auto E) {
            constexpr int e = decltype(E)::value, ks = e / GW, w = e % GW;
            if constexpr (w < HCn) {
                constexpr int t = w % NDT;
                lds_char* const base = (w < NDT ? tdO : tQ) + tsl + (t * BQ + 16 * ks) * 64;
                const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(base + ta0));
                const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(base + ta1));
                const s4 b8[2] = {lo, hi};
                opr[e % NO] = __builtin_bit_cast(bf16x8, b8);
            } else {
                constexpr int u = w - HCn, kk = ks * (NKS / 4) + u / 4, mt = u & 1;
                const char* base = ((u & 2) ? cdO : cQ) + rsl;
                opr[e % NO] = *(const bf16x8*)(base + rowa(kk, mt));
            }
        };
        auto issue = [&](auto E) {
            constexpr int e = decltype(E)::value, ks = e / GW, w = e % GW;
            if constexpr (w < HCn) {
                constexpr int t = w % NDT;
                if constexpr (w < NDT)
                    dvacc[t] = mfma_bf16(opr[e % NO], __builtin_bit_cast(bf16x8, pp[ks]), dvacc[t]);
                else
                    dkacc[t] = mfma_bf16(opr[e % NO], __builtin_bit_cast(bf16x8, pd[ks]), dkacc[t]);
            } else {
                constexpr int u = w - HCn, kk = ks * (NKS / 4) + u / 4, mt = u & 1;
                f32x16& acc = (u & 2) ? dA[mt] : sA[mt];
                const bf16x8& b = (u & 2) ? vf[kk] : kf[kk];
                if constexpr (kk == 0) mfma_vacc0(acc, opr[e % NO], b);
                else mfma_vacc(acc, opr[e % NO], b);
            }
        };
        // VALU of tile i in 8 groups (registers 4 j4 .. of sB/dB[mt]) of five
        // micro-ops; group k fills words of k-step k / 2 behind its dV/dK MFMAs.
        f32x4 uL[8], uD[8];
        float ue[8][4];
        auto ub = [](int k, int st) {
            int b0 = (k >> 1) * GW + (HCn ? HCn - 1 : 0) + 2 * (k & 1);
            const int off[5] = {-5, -3, -2, 0, 1};
            const int s = b0 + off[st];
            return s < 0 ? 0 : s;
        };
        auto uop = [&](auto K, auto ST) {
            constexpr int k = decltype(K)::value, st = decltype(ST)::value;
            constexpr int mt = k >> 2, j4 = k & 3, ks = k >> 1, w0 = (j4 & 1) * 2;
            if constexpr (st == 0) {
                uL[k] = *(const f32x4*)&sLD[lsl][mt * 32 + 8 * j4 + 4 * g];
                uD[k] = *(const f32x4*)&sLD[lsl][BQ + mt * 32 + 8 * j4 + 4 * g];
            } else if constexpr (st <= 2) {
                constexpr int e0 = (st - 1) * 2;
                for (int e = e0; e < e0 + 2; e++) {
                    ue[k][e] = fast_exp2(__builtin_fmaf(sB[mt][4 * j4 + e], c2, -uL[k][e]));
                    pin(ue[k][e]);
                }
            } else {
                constexpr int e0 = (st - 3) * 2;
                const float d0 = ue[k][e0] * (dB[mt][4 * j4 + e0] - uD[k][e0]);
                const float d1 = ue[k][e0 + 1] * (dB[mt][4 * j4 + e0 + 1] - uD[k][e0 + 1]);
                const bf16x2 pr = {to_bf16(ue[k][e0]), to_bf16(ue[k][e0 + 1])};
                const bf16x2 dr2 = {to_bf16(d0), to_bf16(d1)};
                pp[ks][w0 + e0 / 2] = __builtin_bit_cast(uint32_t, pr);
                pd[ks][w0 + e0 / 2] = __builtin_bit_cast(uint32_t, dr2);
                pin(pp[ks][w0 + e0 / 2]);
                pin(pd[ks][w0 + e0 / 2]);
            }
        };
        auto uops_at = [&](auto E) {
            constexpr int e = decltype(E)::value;
            if constexpr (HB) {
                static_for<5>([&](auto ST) {
                    static_for<8>([&](auto K) {
                        constexpr int at = ub(decltype(K)::value, decltype(ST)::value);
                        if constexpr (e < NM ? at == e : at >= NM) uop(K, ST);
                    });
                });
            }
        };
        static_for<LA>([&](auto E) {
            if constexpr (decltype(E)::value < NM) fetch(E);
        });
        static_for<NM>([&](auto E) {
            constexpr int e = decltype(E)::value;
            if constexpr (e + LA < NM) fetch(std::integral_constant<int, e + LA>{});
            issue(E);
            if constexpr (e >= 1 && (e - 1) % DS == 0 && (e - 1) / DS < NDMA)
                dma_row(so2, nsl, (e - 1) / DS, dr);
            uops_at(E);
            __builtin_amdgcn_sched_barrier(0);
        });
        static_for<NDMA>([&](auto Dd) {
            constexpr int d = decltype(Dd)::value;
            if constexpr (NM == 0 || 1 + d * DS >= NM) dma_row(so2, nsl, d, dr);
        });
        uops_at(std::integral_constant<int, NM>{});
        if constexpr (HA)
            asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7"
                         : "+v"(sA[0]), "+v"(sA[1]), "+v"(dA[0]), "+v"(dA[1]));
        GONN_VMCNT(0);
        __syncthreads();
        if constexpr (HA) mask(c1.qt, sA);
    };
    using Yes = std::integral_constant<bool, true>;
    using No = std::integral_constant<bool, false>;

    // Prologue: tiles 0, 1 and L/D of tile 0; S/dP of tile 0.
    Cursor c0{s0 / bs.nst, st0 + s0 % bs.nst};
    Cursor ca = next(c0), cb = next(ca);
    for (int j = 0; j < 2 * NRI; j++) dma_row(row_off(c0), 0, j, 1);
    for (int j = 0; j < 2 * NRI; j++) dma_row(row_off(ca), 1, j, nq > 1);
    dma_ld(c0, 0);
    GONN_VMCNT(0);
    __syncthreads();
    f32x16 sX[2], dX[2], sY[2], dY[2];
    for (int kk = 0; kk < NKS; kk++)
        for (int mt = 0; mt < 2; mt++) {
            const bf16x8 aq = *(const bf16x8*)(cQ + rowa(kk, mt));
            const bf16x8 ad = *(const bf16x8*)(cdO + rowa(kk, mt));
            if (kk == 0) {
                mfma_vacc0(sX[mt], aq, kf[kk]);
                mfma_vacc0(dX[mt], ad, vf[kk]);
            } else {
                mfma_vacc(sX[mt], aq, kf[kk]);
                mfma_vacc(dX[mt], ad, vf[kk]);
            }
        }
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" : "+v"(sX[0]), "+v"(sX[1]), "+v"(dX[0]), "+v"(dX[1]));
    mask(c0.qt, sX);

    // Steps 0 .. nq, the full ones in pairs (see attn_bwd.hip).
    auto advance = [&] {
        ca = cb;
        cb = next(cb);
    };
    if (nq == 1) {
        step(No{}, Yes{}, No{}, 0, ca, cb, sY, dY, sX, dX);
        step(No{}, No{}, Yes{}, 1, ca, cb, sX, dX, sY, dY);
    } else {
        step(Yes{}, Yes{}, No{}, 0, ca, cb, sY, dY, sX, dX);
        advance();
        int i = 1;
        if ((nq - 2) & 1) {
            step(Yes{}, Yes{}, Yes{}, 1, ca, cb, sX, dX, sY, dY);
            advance();
            for (int mt = 0; mt < 2; mt++) {
                sY[mt] = sX[mt];
                dY[mt] = dX[mt];
            }
            i = 2;
        }
        for (; i < nq - 1; i += 2) {
            step(Yes{}, Yes{}, Yes{}, i, ca, cb, sX, dX, sY, dY);
            advance();
            step(Yes{}, Yes{}, Yes{}, i + 1, ca, cb, sY, dY, sX, dX);
            advance();
        }
        step(No{}, Yes{}, Yes{}, nq - 1, ca, cb, sX, dX, sY, dY);
        step(No{}, No{}, Yes{}, nq, ca, cb, sY, dY, sX, dX);
    }

    bool bad = false;
    for (int t = 0; t < NDT; t++)
        for (int r = 0; r < 16; r++) bad |= nonfinite(dvacc[t][r]) || nonfinite(dkacc[t][r]);
    if (__builtin_amdgcn_ballot_w64(bad && kj < kl)) {
        window_dkdv_plain<D, bf16>(p, it, bs, BK, BQ, s0, s0 + nq, band, kw);
        return;
    }
    if (kj >= p.Sk) return;
    for (int t = 0; t < NDT; t++)
        for (int rq4 = 0; rq4 < 4; rq4++) {
            f32x4 x, y;
            for (int k = 0; k < 4; k++) {
                x[k] = dvacc[t][rq4 * 4 + k];
                y[k] = dkacc[t][rq4 * 4 + k];
            }
            write_dkdv<D, bf16>(p, it, BK, kj, t * 32 + rq4 * 8 + g * 4, x, y, kj < kl);
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
    const bool sink = kb < p.sink_blocks, tail = p.per_tail && kb == 0;
    const int per = sink ? p.per_sink : p.per_block;
    if (per == 1 && !tail) return;  // written by its item
    const int slot = sink ? kb * per : p.sink_blocks * p.per_sink + (kb - p.sink_blocks) * per;
    int kl = p.kv_len ? p.kv_len[b] : p.Sk;
    kl = kl < 0 ? 0 : (kl > p.Sk ? p.Sk : kl);
    const int G = p.H / p.Hkv;
    BlockSteps bs;
    bs.init(p, kb * BK, BK, BQ, kl, false);
    const int cnt = (bs.nst * G + p.chunk - 1) / p.chunk;
    const float* src = p.part + (((size_t)bk * p.slots + slot) * 2 * BK + w * BK + row) * D + d;
    f32x4 sum = f32x4{};
    for (int c = 0; c < cnt; c++) sum += *(const f32x4*)(src + (size_t)c * 2 * BK * D);
    constexpr int TK = tail_keys(D, sizeof(T) == 4);
    if (tail && row < TK) {
        bs.init(p, 0, TK, tail_rows(D, sizeof(T) == 4), kl, true);
        const int n = (bs.nst * G + p.tail_chunk - 1) / p.tail_chunk;
        src = p.part_tail + (((size_t)bk * p.per_tail) * 2 * TK + w * TK + row) * D + d;
        for (int c = 0; c < n; c++) sum += *(const f32x4*)(src + (size_t)c * 2 * TK * D);
    }
    if (w) sum *= p.scale;
    store4<T>((T*)(w ? p.dk : p.dv) + ((size_t)bk * p.Sk + kj) * D + d, sum);
}

namespace {

// Shape of the dK/dV grid.
struct DkdvShape {
    int BK, BQ;
};
DkdvShape dkdv_shape(const WindowParams& p, int D, int is_bf16) {
    const long long cus = device_cus();
    const long long b128 = (long long)((p.Sk + 127) / 128) * p.B * p.Hkv;
    // The 128-key kernel reads a key head's queries with 32-bit offsets.
    const bool near = (double)(p.H / p.Hkv) * p.Sp * D * 2 < 4.0e9;
    if (b128 >= cus && is_bf16 && near) return {128, 64};
    // fp32, us: D 64 64 keys and two waves per SIMD (the sizes of the forward's note: 99;
    // 61; 25; one wave 147; 78; 25; 128 keys 104; -; 25). D 128: 128 keys 560; 44, 64
    // keys 671; 49.
    if (!is_bf16 && D == 128) return {128, 32};
    return {64, 64};
}

template <int D, typename T>
void run_dkdv(const WindowParams& p, int BK, int BQ, hipStream_t s) {
    const unsigned grid = (unsigned)p.slots * (unsigned)(p.B * p.Hkv);
    if constexpr (sizeof(T) == 2) {
        if (BK == 128) window_dkdv_pipe_kernel<D><<<grid, 256, 0, s>>>(p);
        else window_dkdv_kernel<D, T, 2, 2, D == 64 ? 2 : 1><<<grid, 256, 0, s>>>(p);
    } else {
        window_dkdv_kernel<D, T, D == 64 ? 2 : 4, 1, D == 64 ? 2 : 1><<<grid, 256, 0, s>>>(p);
    }
    if (p.per_tail)
        window_dkdv_kernel<D, T, tail_keys(D, sizeof(T) == 4) / 32, sizeof(T) == 2 ? 2 : 1, 1, true>
            <<<(unsigned)p.per_tail * (unsigned)(p.B * p.Hkv), 256, 0, s>>>(p);
    const int nkb = (p.Sk + BK - 1) / BK;
    const int nb = p.per_block > 1 ? nkb : p.per_tail ? 1 : p.per_sink > 1 ? p.sink_blocks : 0;
    if (!nb) return;
    const size_t n = (size_t)p.B * p.Hkv * nb * BK * 2 * (D / 4);
    window_join_kernel<D, T><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(p, BK, BQ, nb, n);
}

template <int D, typename T>
void run_window_bwd(const WindowParams& p, hipStream_t s) {
    const long long cus = device_cus(), BH = (long long)p.B * p.H;
    const long long b128 = (long long)((p.Sq + 127) / 128) * BH;
    const unsigned g128 = (unsigned)b128, g64 = (unsigned)((p.Sq + 63) / 64 * BH);
    const DkdvShape sh = dkdv_shape(p, D, sizeof(T) == 2);
    if constexpr (sizeof(T) == 2) {
        if (b128 >= 2 * cus) window_dq_kernel<D, T, 4, 2, 2><<<g128, 256, 0, s>>>(p);
        else window_dq_kernel<D, T, 2, 2, 2><<<g64, 256, 0, s>>>(p);
    } else {
        // fp32, us, 128 and 64 rows: D 64, the forward's sizes: 91, 87; 50, 55; 36, 25; 2 x
        // 16 x 4096, window 1024: 277, 292. D 128: 439, 494; 67, 45.
        if constexpr (D == 64) {
            if (b128 >= cus) window_dq_kernel<D, T, 4, 2, 2><<<g128, 256, 0, s>>>(p);
            else window_dq_kernel<D, T, 2, 1, 2><<<g64, 256, 0, s>>>(p);
        } else {
            if (b128 >= cus) window_dq_kernel<D, T, 4, 2, 1><<<g128, 256, 0, s>>>(p);
            else window_dq_kernel<D, T, 2, 1, 1><<<g64, 256, 0, s>>>(p);
        }
    }
    run_dkdv<D, T>(p, sh.BK, sh.BQ, s);
}

}  // namespace

WindowParts plan_window_bwd(WindowParams& p, int D, int is_bf16) {
    const DkdvShape sh = dkdv_shape(p, D, is_bf16);
    const long long slices = (long long)p.B * p.Hkv, G = p.H / p.Hkv, want = 2 * device_cus();
    const int nkb = (p.Sk + sh.BK - 1) / sh.BK;
    const long long all = G * ((p.Sq + sh.BQ - 1) / sh.BQ);
    const long long stages = ((long long)sh.BK - 1 + p.window + sh.BQ - 1) / sh.BQ;
    const long long band = std::min<long long>(all, G * (stages + 1));
    // Sinks are read by every later query. Up to 32 of them (one tile) have those
    // queries in items of 32 keys and four waves along the queries, in a kernel of its
    // own, where that takes many steps off the first one (its 15 us pay from 4 to 8
    // steps per CU on); else their blocks have all queries and more items.
    const long long tail_q0 = stages * sh.BQ;
    p.per_tail = 0;
    p.sink_blocks = std::min(nkb, (p.sinks + sh.BK - 1) / sh.BK);
    if (p.sinks > 0 && p.sinks <= 32 && tail_q0 < p.Sq &&
        slices * (all - band) >= (is_bf16 ? 4 : 2) * want) {
        p.sink_blocks = 0;
        p.tail_q0 = (int)tail_q0;
        const int rows = tail_rows(D, !is_bf16);
        const long long steps = G * ((p.Sq - tail_q0 + rows - 1) / rows);
        p.tail_chunk = (int)std::max<long long>(2, (steps * slices + want / 2 - 1) / (want / 2));
        p.per_tail = (int)((steps + p.tail_chunk - 1) / p.tail_chunk);
    }
    // Items as long as a block's band, shorter where that leaves workgroup slots (one
    // per CU with 128 bf16 keys, else two) without work, but no shorter than two
    // stages: the sum of the partials costs 4 to 15 us (8 heads over 2, 777, D 128: two
    // stages 19 + 5 us, four 22 + 4, eight 31 + 4).
    const long long items = slices * nkb, fill = is_bf16 && sh.BK == 128 ? want / 2 : want;
    long long chunk = band;
    if (items < fill) chunk = std::max<long long>(2, (band * items + fill - 1) / fill);
    chunk = std::min(chunk, all);
    p.chunk = (int)chunk;
    p.per_block = (int)((band + chunk - 1) / chunk);
    p.per_sink = (int)((all + chunk - 1) / chunk);
    p.slots = p.sink_blocks * p.per_sink + (nkb - p.sink_blocks) * p.per_block;
    WindowParts n{0, (size_t)slices * p.per_tail * 2 * tail_keys(D, !is_bf16) * D};
    if (p.per_block > 1 || (p.sink_blocks && p.per_sink > 1) || p.per_tail)
        n.part = (size_t)slices * p.slots * 2 * sh.BK * D;
    return n;
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
