// attn_window.hip -- sliding-window attention with sinks: the forward.
//
// O = softmax(scale Q K^T) V over the keys that a query sees (attn_window.h), and
// LSE. A workgroup is 4 wave64s: WQ along the queries (32 rows each), 4 / WQ along
// the keys. A stage is one 32-key sub-tile per key wave, loaded as it lies one
// stage ahead and stored in LDS as operand planes. S^T = K Q^T gives every lane
// one query; P feeds O^T += V^T P^T from registers, V^T read from the row-major
// tile with ds_read_b64_tr_b16. Key waves merge through LDS.
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

    Stage in;
    in.init(tid);
    if (nst > 0) in.load(Kg, Vg, ks.stage(0) * BN, kl);
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

    // Key waves > 0 leave (o, m, l) in LDS, key wave 0 merges in order.
    auto merge = [&](float& l) {
        if constexpr (WK > 1) {
            __syncthreads();
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

namespace {

template <int D, typename T, int WQ, int NBUF, int OCC>
void run_window_fwd(const WindowParams& p, hipStream_t s) {
    const unsigned grid = (unsigned)((p.Sq + WQ * 32 - 1) / (WQ * 32)) * (unsigned)(p.B * p.H);
    window_fwd_kernel<D, T, WQ, NBUF, OCC><<<grid, 256, 0, s>>>(p);
}

template <int D, typename T>
void pick_window_fwd(const WindowParams& p, hipStream_t s) {
    const long long cus = device_cus(), BH = (long long)p.B * p.H;
    const long long b128 = (long long)((p.Sq + 127) / 128) * BH;
    const long long b64 = (long long)((p.Sq + 63) / 64) * BH;
    if constexpr (sizeof(T) == 2) {
        if (b128 >= 2 * cus) run_window_fwd<D, T, 4, 2, 2>(p, s);
        else if (b64 >= cus) run_window_fwd<D, T, 2, 2, 2>(p, s);
        else run_window_fwd<D, T, 1, 2, 1>(p, s);
    } else {
        if (b128 >= 2 * cus) run_window_fwd<D, T, 4, 1, 2>(p, s);
        else run_window_fwd<D, T, 2, 1, 1>(p, s);
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
