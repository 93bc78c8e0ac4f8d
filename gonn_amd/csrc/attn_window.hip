// attn_window.hip -- sliding-window attention with sinks: the forward.
//
// O = softmax(scale Q K^T) V over the keys that a query sees (attn_window.h), and
// LSE. A workgroup is 4 wave64s: WQ along the queries (32 rows each), 4 / WQ along
// the keys. A stage is one 32-key sub-tile per key wave, loaded as it lies one
// stage ahead: bf16 straight to LDS, fp32 through registers as operand planes. S^T =
// K Q^T gives every lane one query; P feeds O^T += V^T P^T from registers, V^T read
// from the row-major tile with ds_read_b64_tr_b16. Key waves merge through LDS.
// Only the tiles that some row of the wave sees are formed, and only the border ones
// are masked, so the work follows the window and not the length.
//
// Large bf16 grids (two workgroups of 128 queries per CU and more) run the
// hand-ordered pipeline of attn_fwd.hip's kernel over the two runs of keys.
//
// Bound: the matrix cores. 2 x 16 heads, 8192 queries, window 1024, 4 sinks, D 128,
// bf16: 173 us, 744 TFLOP/s over the visible pairs (matrix pipe busy 0.34 of the
// cycles at 2.4 GHz; 7 VALU instructions per MFMA, of which the softmax; the border
// tiles, two in 18, count half); with the window as wide as the sequence 1071 to 1088.
// fp32, 8 x 12 x 1024, window 256, D 64: 54 us, 97 TFLOP/s in six products each. 2 x 4
// x 128, D 64: 6 us on the device, the call 13.
#include "attn_window.h"

namespace gonn {

namespace {

// O of four channels and LSE of a row.
template <int D, typename T>
GONN_DEV void write_row(const WindowParams& p, size_t row, int d, f32x4 v, float m, float l) {
    v *= l == 0.f ? 0.f : 1.f / l;
    store4<T>((T*)p.o + row * D + d, v);
    // In double: m and log2 l may be large and cancel.
    if (p.lse && d == 0) {
        const int ex = __builtin_amdgcn_frexp_expf(l);
        const float lm = fast_log2(__builtin_amdgcn_frexp_mantf(l));
        p.lse[row] = l == 0.f ? -INFINITY : (float)(((double)m + (double)ex + lm) * kLn2d);
    }
}

// A wave's 32 rows in plain fp32 products from global memory, for rows whose result
// is not finite (or, in fp32, outside the split's range): a masked key's weight of 0
// would make NaN of an infinite V, so P V is added with a select per key. 32 channels
// at a time, each time from the scores on: few registers beside the kernels'.
template <int D, typename T>
GONN_DEV void window_fwd_plain(const WindowParams& p, int bh, int bk, int kl, const Band& band,
                               int qw) {
    constexpr int HD = D / 2;
    const int lane = threadIdx.x & 63, g = lane >> 5, ln = lane & 31, qi = qw + ln;
    const T* Kg = (const T*)p.k + (size_t)bk * p.Sk * D;
    const T* Vg = (const T*)p.v + (size_t)bk * p.Sk * D;
    const size_t row = (size_t)bh * p.Sq + (qi < p.Sq ? qi : p.Sq - 1);
    const T* qrow = (const T*)p.q + row * D + g * HD;
    KeyStages ks;
    ks.init(qw, qw + 32 < p.Sq ? qw + 32 : p.Sq, kl, 32, band);
#pragma unroll 1
    for (int t = 0; t < D / 32; t++) {
        f32x16 o = f32x16{};
        float m = -INFINITY, l = 0.f;
#pragma unroll 1
        for (int st = 0; st < ks.count(); st++) {
            const int kb = ks.stage(st) * 32;
            const T* krow = Kg + (size_t)(kb + ln < kl ? kb + ln : kl - 1) * D + g * HD;
            f32x16 s = f32x16{};
#pragma unroll 4
            for (int i = 0; i < HD; i++) s = mfma_f32(to_float(krow[i]), to_float(qrow[i]), s);
            float mx = -INFINITY;
            for (int r = 0; r < 16; r++) {
                const int key = kb + 8 * (r >> 2) + 4 * g + (r & 3);
                s[r] = key < kl && band.sees(qi, key) ? s[r] * p.scale_log2 : -INFINITY;
                // A NaN score has to make the row NaN: fmaxf would drop it.
                mx = s[r] != s[r] ? s[r] : fmaxf(mx, s[r]);
            }
            mx = pair_max32(mx);
            const float mnew = fmaxf(m, mx), mref = mnew == -INFINITY ? 0.f : mnew;
            const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - mref);
            float rs = 0.f;
            for (int r = 0; r < 16; r++) {
                s[r] = fast_exp2(s[r] - mref);
                rs += s[r];
            }
            l = l * alpha + rs;
            m = mnew;
            o *= alpha;
#pragma unroll 1
            for (int x = 0; x < 32; x++) {
                const int r = x >> 1, h = x & 1, key = kb + 8 * (r >> 2) + 4 * h + (r & 3);
                const float w = weight_of(s, r, h, g);
                if (key >= kl) continue;  // uniform
                add_row32(o, w, Vg + (size_t)key * D + 32 * t, g, band.sees(qi, key));
            }
        }
        l = pair_sum32(l);
        if (qi < p.Sq)
            for (int rq = 0; rq < 4; rq++)
                write_row<D, T>(p, row, 32 * t + 8 * rq + 4 * g,
                                f32x4{o[4 * rq], o[4 * rq + 1], o[4 * rq + 2], o[4 * rq + 3]}, m, l);
    }
}

}  // namespace

template <int D, typename T, int WQ, int NBUF, int OCC>
__global__ __launch_bounds__(256, OCC) void window_fwd_kernel(WindowParams p) {
    constexpr int WK = 4 / WQ, BM = WQ * 32, BN = WK * 32, NP = kPlanes<T>;
    constexpr int NKS = D / 16, NDT = D / 32;
    typedef RowStage<D, WK, T> Stage;
    constexpr uint32_t STAGE = WK * Stage::TILE;
    constexpr int NE = 16 * NDT + 2;
    constexpr uint32_t RED = (WK - 1) * WQ * NE * 256;
    __shared__ __attribute__((aligned(16))) char smem[NBUF * STAGE > RED ? NBUF * STAGE : RED];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wq = wave % WQ, wk = wave / WQ, g = lane >> 5, ln = lane & 31;
    const int nqb = (p.Sq + BM - 1) / BM;
    int bh, qb;
    map_block(blockIdx.x, nqb, p.B * p.H, true, bh, qb);
    const int b = bh / p.H, h = bh - b * p.H, bk = b * p.Hkv + h / (p.H / p.Hkv);
    const int q0 = qb * BM, qw = q0 + wq * 32, qi = qw + ln, kl = window_keys(p, b);
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
    const T* qrow = (const T*)p.q + ((size_t)bh * p.Sq + (qi < p.Sq ? qi : p.Sq - 1)) * D;
    Frag<NP> qf[NKS];
    load_row_frags<D>(qrow, g, true, qf);
    SplitTile<D> tl;
    tl.init(lane);

    f32x16 oacc[NDT];
    for (int t = 0; t < NDT; t++) oacc[t] = f32x16{};
    float m = -INFINITY, l = 0.f;
    const float c2 = p.scale_log2;

    auto compute = [&](int st, int buf) {
        const int kb = ks.stage(st) * BN + wk * 32;
        if (kb >= kl || !band.any(qw, qw + 31, kb, kb + 31)) return;  // wave-uniform
        char* tile = smem + buf * STAGE + wk * Stage::TILE;
        f32x16 s = f32x16{};
        for (int k = 0; k < NKS; k++) s = mfma_n(tile_row<D, NP>(tl, tile, 0, k), qf[k], s);
        s *= c2;
        pin_before_branch(s);
        if (kb + 32 > kl || !band.all(qw, qw + 31, kb, kb + 31))
            for (int r = 0; r < 16; r++) {
                const int key = kb + 8 * (r >> 2) + 4 * g + (r & 3);
                s[r] = key < kl && band.sees(qi, key) ? s[r] : -INFINITY;
            }
        float mx = fmaxf(s[0], s[1]);
        for (int r = 2; r < 16; r++) mx = fmaxf(mx, s[r]);
        mx = pair_max32(mx);
        // The offset moves by more than 2^8 at a time (P stays below 2^8).
        const bool need = mx > m && (m == -INFINITY || mx - m > 8.f);
        if (__builtin_amdgcn_ballot_w64(need)) {
            const float mn = need ? mx : m;
            const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - mn);
            m = mn;
            l *= alpha;
            for (int t = 0; t < NDT; t++) oacc[t] *= alpha;
        }
        const float mref = m == -INFINITY ? 0.f : m;
        float rs[4] = {0.f, 0.f, 0.f, 0.f};
        Frag<NP> pf[2];
        for (int k = 0; k < 2; k++) {
            float e[8];
            for (int j = 0; j < 8; j++) {
                e[j] = fast_exp2(s[8 * k + j] - mref);
                rs[j & 3] += e[j];
            }
            pf[k] = to_frag<NP>(e);
        }
        l += (rs[0] + rs[1]) + (rs[2] + rs[3]);
        for (int k = 0; k < 2; k++)
            for (int t = 0; t < NDT; t++)
                oacc[t] = mfma_n(tile_col<D, NP>(tl, tile, 1, k, t), pf[k], oacc[t]);
    };
    if constexpr (Stage::DIRECT) {
        for (int st = 0; st < nst; st++) {
            GONN_VMCNT(0);
            __syncthreads();  // stage st has landed, and its buffer's last reader is past it
            if (st + 1 < nst)
                in.load(Kg, Vg, ks.stage(st + 1) * BN, kl, lds + (uint32_t)((st + 1) & 1) * STAGE, wave);
            compute(st, st & 1);
        }
    } else {
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
    }

    // Key waves > 0 leave (o, m, l) in LDS, key wave 0 merges in order.
    auto merge = [&](float& l) {
        if constexpr (WK > 1) {
            __syncthreads();  // every wave is past its last tile
            float* red = (float*)smem;
            if (wk > 0) {
                float* d = red + ((wk - 1) * WQ + wq) * NE * 64 + lane;
                for (int t = 0; t < NDT; t++)
                    for (int r = 0; r < 16; r++) d[(t * 16 + r) * 64] = oacc[t][r];
                d[(NE - 2) * 64] = m;
                d[(NE - 1) * 64] = l;
            }
            __syncthreads();
            if (wk > 0) return;
            for (int w = 1; w < WK; w++) {
                const float* d = red + ((w - 1) * WQ + wq) * NE * 64 + lane;
                const float m2 = d[(NE - 2) * 64], l2 = d[(NE - 1) * 64];
                const float M = fmaxf(m, m2), Mr = M == -INFINITY ? 0.f : M;
                const float a = fast_exp2(m - Mr), c = fast_exp2(m2 - Mr);
                l = l * a + l2 * c;
                for (int t = 0; t < NDT; t++)
                    for (int r = 0; r < 16; r++)
                        oacc[t][r] = oacc[t][r] * a + d[(t * 16 + r) * 64] * c;
                m = M;
            }
        }
    };
    float lt = pair_sum32(l);
    merge(lt);
    if (wk > 0) return;
    bool bad = nonfinite(lt);
    SplitCheck chk;
    for (int t = 0; t < NDT; t++)
        for (int r = 0; r < 16; r++) {
            if constexpr (NP == 3) chk.add(oacc[t][r]);
            else bad |= nonfinite(oacc[t][r]);
        }
    if constexpr (NP == 3) bad |= chk.plain();
    if (__builtin_amdgcn_ballot_w64(bad && qi < p.Sq)) {
        window_fwd_plain<D, T>(p, bh, bk, kl, band, qw);
        return;
    }
    if (qi >= p.Sq) return;
    const size_t row = (size_t)bh * p.Sq + qi;
    for (int t = 0; t < NDT; t++)
        for (int rq = 0; rq < 4; rq++)
            write_row<D, T>(p, row, t * 32 + rq * 8 + g * 4,
                            f32x4{oacc[t][rq * 4], oacc[t][rq * 4 + 1], oacc[t][rq * 4 + 2],
                                  oacc[t][rq * 4 + 3]}, m, lt);
}

// ---------------------------------------------------------------------------
// bf16 forward of large grids: the three-stage pipeline of attn_fwd.hip (4 waves, 128
// query rows, 64-key tiles) on the two runs of tiles. Step t issues
//   MFMA  O^T += V(t)^T P(t)
//   MFMA  S^T(t+2) = K(t+2) Q^T
//   VALU  P(t+1) = exp2(S^T(t+1) c2 - mc), packed to bf16, and its row sums
// K and V tiles go straight from memory to two-slot LDS rings, row-major (V^T is read
// with ds_read_b64_tr_b16, so nothing is packed beforehand). Scores stay unscaled and
// exact; P is exact for any offset mc, which only has to keep it bounded: a tile whose
// row sum exceeds 2^14, or a row that has seen nothing yet, takes a rare branch that
// moves mc to the tile's maximum. Rows sum the unrounded P, so that LSE keeps fp32
// accuracy. The scale's sign goes into Q.
// ---------------------------------------------------------------------------
constexpr float kSumBound = 16384.f, kLazyLog2 = 8.f;

template <int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void window_fwd_pipe_kernel(WindowParams p) {
    constexpr int NW = 4, BM = NW * 32, BN = 64, NT = NW * 64;
    constexpr int NKS = D / 16, NDT = D / 32;
    constexpr uint32_t TB = BN * D * 2;  // bytes of a K or V tile
    constexpr int KLEAD = 3, VLEAD = 1;
    __shared__ __attribute__((aligned(16))) bf16 sKb[2 * BN * D];
    __shared__ __attribute__((aligned(16))) bf16 sVb[2 * BN * D];

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 5, ln = lane & 31;
    int bh, qb;
    map_block(blockIdx.x, (p.Sq + BM - 1) / BM, p.B * p.H, true, bh, qb);
    const int b = bh / p.H, h = bh - b * p.H, bk = b * p.Hkv + h / (p.H / p.Hkv);
    const int Sq = p.Sq, q0 = qb * BM, qw = q0 + wave * 32, qi = qw + ln, kl = window_keys(p, b);
    const Band band{p.window, p.sinks};
    KeyStages ks_;
    ks_.init(q0, q0 + BM < Sq ? q0 + BM : Sq, kl, BN, band);
    const int ntiles = ks_.count();
    if (ntiles == 0) {  // uniform: no row sees a key
        for (int i = tid; i < BM * D / 4; i += NT) {
            const int r = i / (D / 4);
            if (q0 + r < Sq)
                write_row<D, bf16>(p, (size_t)bh * Sq + q0 + r, i % (D / 4) * 4, f32x4{}, 0.f, 0.f);
        }
        return;
    }
    const float c2 = p.c2;

    bf16x8 qf[NKS];
    auto load_q = [&]() {
        const bf16* qrow = (const bf16*)p.q + ((size_t)bh * Sq + (qi < Sq ? qi : Sq - 1)) * D + g * 8;
        const uint32_t flip = p.sign < 0.f ? 0x80008000u : 0u, keep = p.sign != 0.f ? ~0u : 0u;
        for (int ks = 0; ks < NKS; ks++) {
            u32x4 a = *(const u32x4*)(qrow + ks * 16);
            for (int e = 0; e < 4; e++) a[e] = (a[e] ^ flip) & keep;
            qf[ks] = __builtin_bit_cast(bf16x8, a);
        }
    };

    // Tile loads: instruction i of thread tid fills 16-byte position i * NT + tid.
    constexpr int NI = BN * D / 8 / NT;  // loads of a tile
    uint32_t toff[NI];
    for (int i = 0; i < NI; i++) {
        int r, c;
        slab_chunk(i * NT + tid, BN, r, c);
        toff[i] = (uint32_t)((r * D + c * 8) * 2);
    }
    // Keys at and past kl read as zeros.
    const brsrc krs = make_rsrc((const bf16*)p.k + (size_t)bk * p.Sk * D, (uint32_t)kl * D * 2);
    const brsrc vrs = make_rsrc((const bf16*)p.v + (size_t)bk * p.Sk * D, (uint32_t)kl * D * 2);
    const uint32_t kl0 = lds_addr(sKb) + wave * 1024, vl0 = lds_addr(sVb) + wave * 1024;
    auto clamped = [&](int t) { return (uint32_t)ks_.stage(t < ntiles ? t : ntiles - 1) * TB; };
    auto dma = [&](brsrc rs, uint32_t base, uint32_t so) {
        for (int i = 0; i < NI; i++) dma16(rs, base + i * NT * 16, toff[i], so);
    };

    const int hs = slab_swz(ln);
    const uint32_t qa0 = (uint32_t)(ln * 64 + ((0 + g) ^ hs) * 16);
    const uint32_t qa1 = (uint32_t)(ln * 64 + ((2 + g) ^ hs) * 16);
    const int s16 = lane & 15, tcx = 2 * ((ln >> 4) & 1) + ((s16 >> 1) & 1);
    const uint32_t ta0 = (uint32_t)((4 * g + (s16 >> 2)) * 64 + (tcx ^ g) * 16 + 8 * (s16 & 1));
    const uint32_t ta1 =
        (uint32_t)((8 + 4 * g + (s16 >> 2)) * 64 + (tcx ^ (2 + g)) * 16 + 8 * (s16 & 1));
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds_s4;
    typedef __attribute__((address_space(3))) char lds_char;
    const char* sKc = (const char*)sKb;
    lds_char* const sVc = (lds_char*)sVb;
    auto kfrag = [&](const char* tile, int ks, int mt) {
        return *(const bf16x8*)(tile + ((ks & 1) ? qa1 : qa0) + ((ks >> 1) * BN + mt * 32) * 64);
    };
    auto vfrag = [&](uint32_t base, int ks, int dt) {
        lds_char* const x = sVc + base + (dt * BN + 16 * ks) * 64;
        const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(x + ta0));
        const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(x + ta1));
        const s4 b8[2] = {lo, hi};
        return __builtin_bit_cast(bf16x8, b8);
    };

    f32x16 oacc[NDT];
    for (int dt = 0; dt < NDT; dt++) oacc[dt] = f32x16{};
    float mc = 0.f, l = 0.f, alpha = 1.f;

    // Scores of tile t that this lane's row does not see, to -inf (c2 > 0).
    auto mask = [&](int t, f32x16* s) {
        const int kb = ks_.stage(t) * BN;
        if (kb + BN <= kl && band.all(qw, qw + 31, kb, kb + BN - 1)) return;  // wave-uniform
        // Key 32 mt + 8 (r / 4) + r % 4 of the lane group: up to hi, and past lo or below sk.
        const int base = kb + 4 * g, hi = (qi < kl - 1 ? qi : kl - 1) - base;
        const int lo = qi - p.window - base, sk = p.sinks - base;
        for (int mt = 0; mt < 2; mt++)
            for (int r = 0; r < 16; r++) {
                const int c = mt * 32 + 8 * (r >> 2) + (r & 3);
                s[mt][r] = c > hi || (c <= lo && c >= sk) ? -INFINITY : s[mt][r];
            }
    };
    // Maximum of a tile's scaled scores over the row.
    auto tile_max = [&](const f32x16* s) {
        float m0 = -INFINITY;
        for (int mt = 0; mt < 2; mt++)
            for (int r = 0; r < 16; r++) m0 = fmaxf(m0, s[mt][r]);
        return pair_max32(m0) * c2;
    };
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    auto p_tile = [&](const f32x16* s, u32x4* pk) {
        float part[4] = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < 16; k++) {
            const int mt = k >> 3, r = (k & 7) * 2;
            const float a = fast_exp2(__builtin_fmaf(s[mt][r], c2, -mc));
            const float c = fast_exp2(__builtin_fmaf(s[mt][r + 1], c2, -mc));
            part[k & 3] += a + c;
            const bf16x2 pr = {to_bf16(a), to_bf16(c)};
            pk[k >> 2][k & 3] = __builtin_bit_cast(uint32_t, pr);
        }
        return (part[0] + part[1]) + (part[2] + part[3]);
    };
    u32x4 pp[4];  // P of the tile PV consumes next

    // One step, scheduled by hand as in attn_fwd.hip. TAIL: 0 a full step; 1 the
    // next-to-last (no S^T(t+2)); 2 the last (no P(t+1) either).
    auto step = [&](int t, f32x16* sA, f32x16* sB, auto TAILC) __attribute__((always_inline)) {
        constexpr int TAIL = decltype(TAILC)::value;
        const uint32_t kso = clamped(t + KLEAD), vso = clamped(t + VLEAD);
        const int kslot = (t + KLEAD) & 1, vslot = (t + 1) & 1;
        if constexpr (TAIL < 2) mask(t + 1, sB);
        const uint32_t vb = (uint32_t)(t & 1) * TB;
        const char* kt = sKc + (uint32_t)(t & 1) * TB;

        constexpr int SKS = NKS / 4, GW = NDT + 2 * SKS, NM = 4 * GW, NU = 16, LA = 3;
        constexpr int NDMA = 2 * NI, DS = 2;
        static_assert(DS * NDMA <= NM, "the step's tile loads fit in its slots");
        bf16x8 opr[4];
        auto fetch = [&](auto E) {
            constexpr int e = decltype(E)::value, j = e / GW, w = e % GW;
            if constexpr (w < NDT) opr[e & 3] = vfrag(vb, j, w);
            else if constexpr (TAIL == 0)
                opr[e & 3] = kfrag(kt, SKS * j + ((w - NDT) >> 1), (w - NDT) & 1);
        };
        auto issue = [&](auto E) {
            constexpr int e = decltype(E)::value, j = e / GW, w = e % GW;
            if constexpr (w < NDT) {
                oacc[w] = mfma_bf16(opr[e & 3], __builtin_bit_cast(bf16x8, pp[j]), oacc[w]);
            } else if constexpr (TAIL == 0) {
                constexpr int kk = SKS * j + ((w - NDT) >> 1), mt = (w - NDT) & 1;
                sA[mt] = mfma_bf16(opr[e & 3], qf[kk], kk == 0 ? f32x16{} : sA[mt]);
            }
        };
        auto dma_slot = [&](auto E) {
            constexpr int e = decltype(E)::value;
            constexpr int d0 = TAIL == 0 ? 0 : (TAIL == 1 ? NI : NDMA);
            if constexpr (e % DS == 0 && e / DS < NDMA && e / DS >= d0) {
                constexpr int d = e / DS;
                dma_set_m0(d < NI ? kl0 + kslot * TB + d * NT * 16 : vl0 + vslot * TB + (d - NI) * NT * 16);
            }
            if constexpr (e >= 1 && (e - 1) % DS == 0 && (e - 1) / DS < NDMA && (e - 1) / DS >= d0) {
                constexpr int d = (e - 1) / DS;
                if constexpr (d < NI) dma16_m0(krs, toff[d], kso);
                else dma16_m0(vrs, toff[d - NI], vso);
            }
        };
        float part[4] = {0.f, 0.f, 0.f, 0.f};
        auto uslot = [](int k) { return (k >> 2) * GW + NDT + (k & 3); };
        float ub[16][2];
        auto uop = [&](auto U, auto S) {
            constexpr int k = decltype(U)::value, stage = decltype(S)::value;
            constexpr int mt = k >> 3, r = (k & 7) * 2;
            if constexpr (stage == 0) {
                ub[k][0] = fast_exp2(__builtin_fmaf(sB[mt][r], c2, -mc));
                ub[k][1] = fast_exp2(__builtin_fmaf(sB[mt][r + 1], c2, -mc));
                pin(ub[k][0]);
                pin(ub[k][1]);
            } else {
                part[k & 3] += ub[k][0] + ub[k][1];
                const bf16x2 pr = {to_bf16(ub[k][0]), to_bf16(ub[k][1])};
                pp[k >> 2][k & 3] = __builtin_bit_cast(uint32_t, pr);
                pin(pp[k >> 2][k & 3]);
                pin(part[k & 3]);
            }
        };
        auto uops_at = [&](auto E) {
            constexpr int e = decltype(E)::value;
            if constexpr (TAIL == 2) return;
            static_for<2>([&](auto S) {
                static_for<NU>([&](auto U) {
                    constexpr int at = uslot(decltype(U)::value) - 2 + 2 * decltype(S)::value;
                    if constexpr (e < NM ? at == e : at >= NM) uop(U, S);
                });
            });
        };
        __builtin_amdgcn_s_setprio(1);
        static_for<LA>([&](auto E) { fetch(E); });
        static_for<NM>([&](auto E) {
            constexpr int e = decltype(E)::value;
            if constexpr (e + LA < NM) fetch(std::integral_constant<int, e + LA>{});
            issue(E);
            dma_slot(E);
            uops_at(E);
            __builtin_amdgcn_sched_barrier(0);
        });
        uops_at(std::integral_constant<int, NM>{});
        __builtin_amdgcn_s_setprio(0);
        float ts = (part[0] + part[1]) + (part[2] + part[3]);
        alpha = 1.f;
        if (TAIL < 2 && __builtin_amdgcn_ballot_w64(!(ts <= kSumBound) || l == 0.f)) {
            const float mx = tile_max(sB);
            const bool empty = pair_sum32(l) == 0.f;
            const float mn = mx > -INFINITY && (empty || mx - mc > kLazyLog2) ? mx : mc;
            alpha = empty ? 0.f : fast_exp2(mc - mn);
            mc = mn;
            ts = p_tile(sB, pp);
        }
        l = l * alpha + ts;
        GONN_VMCNT(0);
        __syncthreads();
        if (__builtin_amdgcn_ballot_w64(alpha != 1.f))
            for (int dt = 0; dt < NDT; dt++) oacc[dt] *= alpha;
    };

    // Prologue: S^T(0) -> P(0), S^T(1); K(0) is staged in V slot 1.
    f32x16 s0[2], s1[2];
    auto qk_tile = [&](const char* tile, f32x16* s) {
        s[0] = s[1] = f32x16{};
        for (int ks = 0; ks < NKS; ks++)
            for (int mt = 0; mt < 2; mt++) s[mt] = mfma_bf16(kfrag(tile, ks, mt), qf[ks], s[mt]);
    };
    dma(krs, vl0 + TB, clamped(0));
    dma(krs, kl0 + TB, clamped(1));
    dma(krs, kl0, clamped(2));
    dma(vrs, vl0, clamped(0));
    load_q();
    GONN_VMCNT(0);
    __syncthreads();
    qk_tile((const char*)sVb + TB, s0);
    qk_tile(sKc + TB, s1);
    settle_before_branch(s0[0], s0[1]);
    settle_before_branch(s1[0], s1[1]);
    mask(0, s0);
    mc = tile_max(s0);
    if (!(mc > -INFINITY)) mc = 0.f;  // nothing seen yet: no offset
    l = p_tile(s0, pp);
    __syncthreads();  // K(0) and K(1) read by every wave

    {
        const std::integral_constant<int, 0> full;
        const std::integral_constant<int, 1> tail1;
        const std::integral_constant<int, 2> tail2;
        const int nfull = ntiles - 2;
        int t = 0;
        for (; t + 1 < nfull; t += 2) {
            step(t, s0, s1, full);
            step(t + 1, s1, s0, full);
        }
        if (t < nfull) step(t++, s0, s1, full);
        if (ntiles >= 2) {
            if (t & 1)
                for (int mt = 0; mt < 2; mt++) {
                    const f32x16 x = s0[mt];
                    s0[mt] = s1[mt];
                    s1[mt] = x;
                }
            step(t, s0, s1, tail1);
        }
        step(ntiles - 1, s1, s0, tail2);
    }
    GONN_VMCNT(0);  // loads in flight write this workgroup's LDS

    const float lt = pair_sum32(l);
    bool bad = nonfinite(lt);
    for (int t = 0; t < NDT; t++)
        for (int r = 0; r < 16; r++) bad |= nonfinite(oacc[t][r]);
    if (__builtin_amdgcn_ballot_w64(bad && qi < Sq)) {
        window_fwd_plain<D, bf16>(p, bh, bk, kl, band, qw);
        return;
    }
    if (qi >= Sq) return;
    const size_t row = (size_t)bh * Sq + qi;
    for (int t = 0; t < NDT; t++)
        for (int rq = 0; rq < 4; rq++)
            write_row<D, bf16>(p, row, t * 32 + rq * 8 + g * 4,
                               f32x4{oacc[t][rq * 4], oacc[t][rq * 4 + 1], oacc[t][rq * 4 + 2],
                                     oacc[t][rq * 4 + 3]}, mc, lt);
}

namespace {

template <int D, typename T, int WQ, int NBUF, int OCC>
void run_window_fwd(const WindowParams& p, hipStream_t s) {
    const unsigned grid = (unsigned)((p.Sq + WQ * 32 - 1) / (WQ * 32)) * (unsigned)(p.B * p.H);
    window_fwd_kernel<D, T, WQ, NBUF, OCC><<<grid, 256, 0, s>>>(p);
}

// bf16: the pipeline from two workgroups of 128 rows per CU, else 64 rows where that gives
// every CU one, else 32 rows and four key waves: a small grid is bound by its longest
// workgroup. fp32: figures below.
template <int D, typename T>
void pick_window_fwd(const WindowParams& p, hipStream_t s) {
    const long long cus = device_cus(), BH = (long long)p.B * p.H;
    const long long b128 = (long long)((p.Sq + 127) / 128) * BH;
    const long long b64 = (long long)((p.Sq + 63) / 64) * BH;
    if constexpr (sizeof(T) == 2) {
        if (b128 >= 2 * cus) window_fwd_pipe_kernel<D><<<(unsigned)b128, 256, 0, s>>>(p);
        else if (b64 >= cus) run_window_fwd<D, T, 2, 2, 2>(p, s);
        else run_window_fwd<D, T, 1, 2, 1>(p, s);
    } else {
        // fp32, us: B 8, H 12, S 1024, window 256, D 64: 128 rows 57, 64 rows 73; 4 x 12 x
        // 1021, window 200: 40 and 41; 8 heads x 1000: 30 and 19; D 128: 4 x 16 over 8,
        // 2048, window 512: 217 and 346; 8 x 1000: 47 and 32.
        if constexpr (D == 64) {
            if (b128 >= cus) run_window_fwd<D, T, 4, 2, 3>(p, s);
            else run_window_fwd<D, T, 2, 1, 2>(p, s);
        } else {
            if (b128 >= cus) run_window_fwd<D, T, 4, 1, 2>(p, s);
            else run_window_fwd<D, T, 2, 1, 1>(p, s);
        }
    }
}

}  // namespace

hipError_t launch_window_fwd(const WindowParams& p, int D, int is_bf16, hipStream_t s) {
    if (D == 64) {
        if (is_bf16) pick_window_fwd<64, bf16>(p, s);
        else pick_window_fwd<64, float>(p, s);
    } else if (D == 128) {
        if (is_bf16) pick_window_fwd<128, bf16>(p, s);
        else pick_window_fwd<128, float>(p, s);
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace gonn
