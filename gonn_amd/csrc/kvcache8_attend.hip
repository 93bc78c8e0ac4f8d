// kvcache8_attend.hip -- attention over the 8-bit KV cache.
//
// The T newest positions' queries, Hq / H query heads to a key head: R = (Hq / H) T
// rows read the same keys. Row r is query t = r % T at position len - T + t and sees
// the positions up to its own, or those of a window with sinks.
//
// A workgroup is 4 wave64s: WQ along the rows (32 each), 4 / WQ along the keys. A
// wave takes whole 64-position blocks of its split. K (row-major) and V
// (transposed) are matrix operands as they lie in the cache, so they go from memory
// to registers without LDS: 16 bytes a lane, turned to bf16 with the block's scale
// in one instruction per two values. S^T = K q^T gives each lane one row; the
// cache rows are taken in the order that leaves a lane 16 consecutive positions,
// which are also the 16 bytes of V^T that it loads for O^T += V^T P^T. Keys and
// values are exact in bf16; a bf16 row has one product per term and its weights
// are rounded to bf16 once, an fp32 row has q and P in three pieces. Key waves
// merge through LDS, splits through the combine kernel.
//
// Three forms. Up to 16 rows, a decoding step: 16 x 16 tiles (attend8_few_kernel),
// bound by the cache's bytes: 64 sequences of 512 to 8192 positions, 32 heads, D 128,
// 2.28 GB in 356 us, 6.4 TB/s; 8192 each 6.55. Up to 64 rows, and fp32 rows: 32 x 32
// tiles from registers. More bf16 rows: blocks turned to bf16 once per 128 rows, in LDS
// (attend8_pipe_kernel), bound by the matrix cores: 4 x 256 rows over 8 heads of 4
// sequences of 2048 to 4096 positions, D 128, 76 us (650 TFLOP/s; 71 and the combine's
// 10, one round of workgroups); 8 x 4096 rows over 65536 positions 1137 TFLOP/s.
#include <type_traits>

#include "common.h"
#include "kvcache8.h"

namespace gonn {

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Eight codes as bf16, times the scale (a power of two: exact).
GONN_DEV bf16x8 decode8(uint32_t lo, uint32_t hi, float scale) {
    bf16x8 r;
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, scale, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, scale, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, scale, true);
    const uint32_t w[4] = {__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
                           __builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, d)};
    __builtin_memcpy(&r, w, 16);
    return r;
}

// The visible blocks of a workgroup's rows: ns from block 0 (sinks), nw from w0 on.
struct Blocks8 {
    int ns, w0, nw;
    // Rows at positions i0 .. i1 (i1 < len).
    GONN_DEV void init(int i0, int i1, int window, int sinks) {
        const int hi = i1 + 1;  // 0 or less: nothing
        const int lo = window > 0 && i0 - window + 1 > 0 ? i0 - window + 1 : 0;
        const int end = hi > 0 ? (hi + kBlk8 - 1) / kBlk8 : 0;
        w0 = lo / kBlk8;
        w0 = w0 < end ? w0 : end;
        nw = end - w0;
        const int sk = sinks < hi ? sinks : hi;
        ns = sk > 0 ? (sk + kBlk8 - 1) / kBlk8 : 0;
        ns = ns < w0 ? ns : w0;
    }
    GONN_DEV int count() const { return ns + nw; }
    GONN_DEV int block(int i) const { return i < ns ? i : i - ns + w0; }
};

// First and last query of rows r0 .. r1.
GONN_DEV void query_span(int r0, int r1, int T, int& t0, int& t1) {
    t0 = r0 % T;
    t1 = r1 % T;
    if (r0 / T != r1 / T) {
        t0 = 0;
        t1 = T - 1;
    }
}

// Splits of nv blocks, no more than the launch has (a replayed graph's cache may
// have grown: they are longer then).
GONN_DEV int splits8(const Attend8& a, int nv) {
    const int ns = (nv + a.split - 1) / a.split;
    return ns < a.nsplit ? ns : a.nsplit;
}

// Split and head of the workgroup whose turn is `us`, for rows of queries t0 .. t1. Long
// splits: of every 64 sequences those with the longest ones first. A workgroup streams 64
// blocks for about 80 us, and one that starts last leaves the device idle for as long.
// With the later splits, which only long sequences have, ahead of the first ones, short
// sequences are left for the end. (2048 heads, 512 to 8192 positions, D 128, one row: 390
// us in the order of the sequences, in splits of 64 blocks; 356 this way, in splits of 128.)
// Splits of less than 32 blocks, 40 us, are taken as they come: finding the order is then
// no small part of them (2048 heads, window 512: 70 us; ordered, by a loop over the
// lanes, 75; window 100 37 and 42).
struct Turn8 {
    int sp, len;  // split; the sequence's length
    size_t bh;    // its row of heads
};
GONN_DEV Turn8 turn_of(const Attend8& a, int us, int t0, int t1, int lane) {
    const Cache8& c = a.c;
    const int BH = c.B * c.H, order = us / BH, at = us - order * BH, place = at / c.H;
    int b = place, len = 0;
    if (a.split >= 32) {
        const int g0 = place & ~63;
        int key = -1;
        if (g0 + lane < c.B) {
            len = c.len[g0 + lane];
            len = len < c.Lmax ? len : c.Lmax;
            Blocks8 bs;
            bs.init(len - a.T + t0, len - a.T + t1, a.window, a.sinks);
            const int nv = bs.count(), ns = splits8(a, nv);
            key = (ns ? (nv + ns - 1) / ns : 0) * 64 + 63 - lane;  // all different; under 2^31
        }
        int before = 0;
#pragma unroll
        for (int j = 0; j < 64; j++) before += __builtin_amdgcn_readlane(key, j) > key ? 1 : 0;
        const uint64_t hit = __builtin_amdgcn_ballot_w64(key >= 0 && before == (place & 63));
        b = __builtin_amdgcn_readfirstlane(__builtin_ctzll(hit));
        len = __builtin_amdgcn_readlane(len, b);
        b += g0;
    } else {
        len = c.len[b];
        len = __builtin_amdgcn_readfirstlane(len < c.Lmax ? len : c.Lmax);
    }
    b = __builtin_amdgcn_readfirstlane(b);
    return {__builtin_amdgcn_readfirstlane(a.nsplit - 1 - order), len,
            (size_t)b * c.H + __builtin_amdgcn_readfirstlane(at - place * c.H)};
}

GONN_DEV bool sees8(int i, int j, int window, int sinks) {
    return j <= i && (window == 0 || i - j < window || j < sinks);
}

// The q operand of eight channels, and eight weights as one.
template <int NP>
GONN_DEV void pieces(const float* x, bf16x8* f) {
    if constexpr (NP == 1) f[0] = pack8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
    else {
        const bf16x8x3 s = split3(x);
        f[0] = s.h;
        f[1] = s.m;
        f[2] = s.l;
    }
}
template <int NP, typename T>
GONN_DEV void load_q(const T* p, bf16x8* f) {
    if constexpr (NP == 1) f[0] = *(const bf16x8*)p;
    else {
        const f32x4 u = *(const f32x4*)p, v = *(const f32x4*)(p + 4);
        const float y[8] = {u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
        pieces<NP>(y, f);
    }
}
GONN_DEV f32x4 mfma_bf16_16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// Over the four lanes 16 apart.
GONN_DEV float quad_max(float x) {
    const uint32_t u = __float_as_uint(x);
    auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return pair_max32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
GONN_DEV float quad_sum(float x) { return pair_sum32(pair_sum16(x)); }

// Channels d .. d + 3 of a row's result: o, or one split's part of it.
template <int D, typename T>
GONN_DEV void write_row4(const Attend8& a, size_t row, int sp, int d, f32x4 v, float m, float l) {
    if (a.nsplit > 1) {
        *(f32x4*)(a.part_o + (row * a.nsplit + sp) * D + d) = v;
        if (d == 0) {
            // A NaN row has no maximum; a finite one keeps its weight non-zero.
            a.part_ml[(row * a.nsplit + sp) * 2 + 0] = l != l ? 0.f : m;
            a.part_ml[(row * a.nsplit + sp) * 2 + 1] = l;
        }
        return;
    }
    v *= l == 0.f ? 0.f : 1.f / l;
    if constexpr (sizeof(T) == 4) *(f32x4*)((float*)a.o + row * D + d) = v;
    else {
        typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
        *(bf16x4*)((bf16*)a.o + row * D + d) =
            bf16x4{to_bf16(v[0]), to_bf16(v[1]), to_bf16(v[2]), to_bf16(v[3])};
    }
}

// One element of the cache, for the plain path.
GONN_DEV float element8(const Cache8& c, size_t bh, int len, int key, int d, bool v) {
    const int blk = key / kBlk8, r = key % kBlk8;
    if (blk < len / kBlk8) {
        const size_t at = bh * c.nblk + blk;
        const uint8_t x = v ? c.v8[(at * c.D + d) * kBlk8 + r] : c.k8[(at * kBlk8 + r) * c.D + d];
        const auto f = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, false);
        return f[0] * (v ? c.vs[at] : c.ks[at]);
    }
    return bf16_to_f32(v ? c.vt[((bh * 2 + (blk & 1)) * c.D + d) * kBlk8 + r]
                         : c.kt[((bh * 2 + (blk & 1)) * kBlk8 + r) * c.D + d]);
}

template <typename T>
GONN_DEV float float_of(T x) {
    if constexpr (sizeof(T) == 4) return x;
    else return bf16_to_f32(__builtin_bit_cast(uint16_t, x));
}

// One wave's 32 rows in plain fp32 products, for results that are not finite: a
// masked position's weight of 0 would make NaN of a value that is. 32 channels at a
// time (few registers beside the kernels'), each time from the scores on.
template <int D, typename T>
GONN_DEV void attend8_plain(const Attend8& a, size_t bh, int len, const T* qrow, const Blocks8& bs,
                            int b0, int b1, int pi, size_t row, int sp, bool live) {
    constexpr int HD = D / 2;
    const int lane = threadIdx.x & 63, g = lane >> 5, ln = lane & 31;
#pragma unroll 1
    for (int t = 0; t < D / 32; t++) {
        f32x16 o = f32x16{};
        float m = -INFINITY, l = 0.f;
#pragma unroll 1
        for (int x = 2 * b0; x < 2 * b1; x++) {
            const int kb = bs.block(x >> 1) * kBlk8 + 32 * (x & 1);
            if (kb >= len) continue;
            const int kr = kb + ln < len ? kb + ln : len - 1;
            f32x16 s = f32x16{};
#pragma unroll 1
            for (int i = 0; i < HD; i++)
                s = mfma_f32(element8(a.c, bh, len, kr, g * HD + i, false), float_of(qrow[g * HD + i]), s);
            float mx = -INFINITY;
            for (int r = 0; r < 16; r++) {
                const int key = kb + 8 * (r >> 2) + 4 * g + (r & 3);
                s[r] = key < len && sees8(pi, key, a.window, a.sinks) ? s[r] * a.scale_log2 : -INFINITY;
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
            for (int y = 0; y < 32; y++) {
                const int r = y >> 1, h = y & 1, key = kb + 8 * (r >> 2) + 4 * h + (r & 3);
                float w = 0.f;
                for (int i = 0; i < 16; i++) w = i == r ? s[i] : w;
                const float other = __shfl_xor(w, 32);
                w = h == g ? w : other;
                if (key >= len) continue;  // uniform
                const bool on = sees8(pi, key, a.window, a.sinks);
                for (int e = 0; e < 16; e++) {
                    const float v = element8(a.c, bh, len, key, 32 * t + 8 * (e >> 2) + 4 * g + (e & 3), true);
                    o[e] = on ? __builtin_fmaf(w, v, o[e]) : o[e];
                }
            }
        }
        l = pair_sum32(l);
        if (live)
            for (int rq = 0; rq < 4; rq++)
                write_row4<D, T>(a, row, sp, t * 32 + rq * 8 + g * 4,
                                 f32x4{o[rq * 4], o[rq * 4 + 1], o[rq * 4 + 2], o[rq * 4 + 3]}, m, l);
    }
}

}  // namespace

template <int D, typename T, int WQ>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attend8_kernel(Attend8 a) {
    constexpr int WK = 4 / WQ, BM = WQ * 32, NP = sizeof(T) == 4 ? 3 : 1;
    constexpr int NJ = D / 32, NDT = D / 32;  // 32-element steps of a row, channel tiles
    constexpr int NE = 16 * NDT + 2;
    __shared__ float red[WK > 1 ? (WK - 1) * WQ * NE * 64 : 1];
    __shared__ int again;

    const Cache8& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wq = wave % WQ, wk = wave / WQ, g = lane >> 5, ln = lane & 31;
    const int T_ = a.T, R = a.Hq / c.H * T_, nrb = (R + BM - 1) / BM, BH = c.B * c.H;
    int us, rb;
    map_block(blockIdx.x, nrb, BH * a.nsplit, true, us, rb, 1, true);
    const int r0 = rb * BM, r1 = r0 + BM < R ? r0 + BM : R;
    int t0, t1;
    query_span(r0, r1 - 1, T_, t0, t1);
    const Turn8 turn = turn_of(a, us, t0, t1, lane);
    const int sp = turn.sp, len = turn.len;
    const size_t bh = turn.bh;
    Blocks8 bs;
    bs.init(len - T_ + t0, len - T_ + t1, a.window, a.sinks);
    const int nv = bs.count(), ns = splits8(a, nv);
    if (sp >= ns && sp > 0) return;  // uniform; split 0 writes also where there is nothing to see
    const int b0 = ns ? (int)((long long)sp * nv / ns) : 0;
    const int b1 = ns ? (int)((long long)(sp + 1) * nv / ns) : 0;

    // This wave's rows, this lane's, and the positions that they stand for.
    const int rw = r0 + wq * 32, ri = rw + ln, rc = ri < R ? ri : R - 1;
    const int pi = len - T_ + rc % T_;
    const int re = rw + 31 < R ? rw + 31 : R - 1;
    int wt0 = 0, wt1 = 0;
    if (rw < R) query_span(rw, re, T_, wt0, wt1);
    const int pw0 = len - T_ + wt0, pw1 = len - T_ + wt1;
    const T* qrow = (const T*)a.q + ((size_t)bh * R + rc) * D;
    // q operand of step (j, x): elements 32 j + 16 g + 8 x .. +7.
    bf16x8 qf[NJ * 2][NP];
    for (int j = 0; j < NJ; j++)
        for (int x = 0; x < 2; x++) load_q<NP>(qrow + 32 * j + 16 * g + 8 * x, qf[2 * j + x]);
    // Cache row of operand row ln: accumulator register r of half g is then
    // position 16 g + r of the 32-position tile.
    const int krow = 16 * ((ln >> 2) & 1) + 4 * (ln >> 3) + (ln & 3);
    const int closed = len / kBlk8;

    f32x16 oacc[NDT];
    for (int t = 0; t < NDT; t++) oacc[t] = f32x16{};
    float m = -INFINITY, l = 0.f;
    if (tid == 0) again = 0;

    u32x4 kr[2][NJ], vr[2][NDT];
    auto load_k = [&](int blk) {
        const uint8_t* p = c.k8 + (bh * c.nblk + blk) * kBlk8 * D + krow * D + 16 * g;
        for (int u = 0; u < 2; u++)
            for (int j = 0; j < NJ; j++) kr[u][j] = *(const u32x4*)(p + u * 32 * D + 32 * j);
    };
    auto load_v = [&](int blk) {
        const uint8_t* p = c.v8 + (bh * c.nblk + blk) * kBlk8 * D + ln * kBlk8 + 16 * g;
        for (int u = 0; u < 2; u++)
            for (int t = 0; t < NDT; t++) vr[u][t] = *(const u32x4*)(p + t * 32 * kBlk8 + 32 * u);
    };
    // Scores of tile u of block blk, masked; kf(j, x) is the operand of step (j, x).
    auto scores = [&](int blk, int u, auto kf) {
        f32x16 s = f32x16{}, s2 = f32x16{};
        for (int j = 0; j < NJ; j++)
            for (int x = 0; x < 2; x++) {
                const bf16x8 k = kf(j, x);
                if constexpr (NP == 3) {
                    s2 = mfma_bf16(k, qf[2 * j + x][2], s2);
                    s2 = mfma_bf16(k, qf[2 * j + x][1], s2);
                }
                s = mfma_bf16(k, qf[2 * j + x][0], s);
            }
        if constexpr (NP == 3) s += s2;
        s *= a.scale_log2;
        pin_before_branch(s);
        const int k0 = blk * kBlk8 + 32 * u;
        const bool all = k0 + 31 <= pw0 && (a.window == 0 || pw1 - k0 < a.window || k0 + 31 < a.sinks);
        if (!all)
            for (int r = 0; r < 16; r++)
                s[r] = sees8(pi, k0 + 16 * g + r, a.window, a.sinks) ? s[r] : -INFINITY;
        return s;
    };
    // P and the running statistics; pf[u][x] is the operand of positions 8 x .. of tile u.
    auto weights = [&](f32x16* s, bf16x8 (*pf)[2][NP]) {
        float mx = -INFINITY;
        for (int u = 0; u < 2; u++)
            for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[u][r]);
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
        for (int u = 0; u < 2; u++)
            for (int x = 0; x < 2; x++) {
                float e[8];
                for (int j = 0; j < 8; j++) {
                    e[j] = fast_exp2(s[u][8 * x + j] - mref);
                    rs[j & 3] += e[j];
                }
                pieces<NP>(e, pf[u][x]);
            }
        l += (rs[0] + rs[1]) + (rs[2] + rs[3]);
    };
    auto accumulate = [&](bf16x8 (*pf)[2][NP], auto vf) {
        for (int t = 0; t < NDT; t++) {
            if constexpr (NP == 1) {
                for (int u = 0; u < 2; u++)
                    for (int x = 0; x < 2; x++) oacc[t] = mfma_bf16(vf(t, u, x), pf[u][x][0], oacc[t]);
            } else {
                // A block's V^T P^T on its own, the small pieces first, added once.
                bf16x8 v[2][2];
                f32x16 y = f32x16{};
                for (int u = 0; u < 2; u++)
                    for (int x = 0; x < 2; x++) v[u][x] = vf(t, u, x);
                for (int n = NP - 1; n >= 0; n--)
                    for (int u = 0; u < 2; u++)
                        for (int x = 0; x < 2; x++) y = mfma_bf16(v[u][x], pf[u][x][n], y);
                oacc[t] += y;
                pin_before_branch(oacc[t]);
            }
        }
    };

    const bool live = rw < R;
    // This wave's blocks: b0 + wk, b0 + wk + WK, ...; the open one is the last of all.
    int bi = b0 + wk;
    const int open_at = b1 > b0 && bs.block(b1 - 1) == closed ? b1 - 1 : b1;  // closed ones end here
    if (live && bi < open_at) {
        load_k(bs.block(bi));
        load_v(bs.block(bi));
        for (; bi < open_at; bi += WK) {
            const int blk = bs.block(bi), nx = bi + WK < open_at ? bs.block(bi + WK) : -1;
            const float ksc = c.ks[bh * c.nblk + blk], vsc = c.vs[bh * c.nblk + blk];
            f32x16 s[2];
            for (int u = 0; u < 2; u++)
                s[u] = scores(blk, u, [&](int j, int x) {
                    return decode8(kr[u][j][2 * x], kr[u][j][2 * x + 1], ksc);
                });
            if (nx >= 0) load_k(nx);
            bf16x8 pf[2][2][NP];
            weights(s, pf);
            accumulate(pf, [&](int t, int u, int x) {
                return decode8(vr[u][t][2 * x], vr[u][t][2 * x + 1], vsc);
            });
            if (nx >= 0) load_v(nx);
        }
    }
    if (live && open_at < b1 && (open_at - b0) % WK == wk) {
        // The open block, bf16; positions past the last are no one's values.
        const uint16_t* kp = c.kt + ((bh * 2 + (closed & 1)) * kBlk8 + krow) * D + 16 * g;
        const uint16_t* vp = c.vt + ((bh * 2 + (closed & 1)) * D + ln) * kBlk8 + 16 * g;
        const int n = len - closed * kBlk8;
        f32x16 s[2];
        for (int u = 0; u < 2; u++)
            s[u] = scores(closed, u, [&](int j, int x) {
                return *(const bf16x8*)(kp + u * 32 * D + 32 * j + 8 * x);
            });
        bf16x8 pf[2][2][NP];
        weights(s, pf);
        accumulate(pf, [&](int t, int u, int x) {
            u16x8 v = *(const u16x8*)(vp + (size_t)t * 32 * kBlk8 + 32 * u + 8 * x);
            for (int e = 0; e < 8; e++) v[e] = 32 * u + 16 * g + 8 * x + e < n ? v[e] : (uint16_t)0;
            return __builtin_bit_cast(bf16x8, v);
        });
    }

    auto merge = [&](float& l) {
        if constexpr (WK > 1) {
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
                const float x = fast_exp2(m - Mr), y = fast_exp2(m2 - Mr);
                l = l * x + l2 * y;
                for (int t = 0; t < NDT; t++)
                    for (int r = 0; r < 16; r++) oacc[t][r] = oacc[t][r] * x + d[(t * 16 + r) * 64] * y;
                m = M;
            }
        }
    };
    float lt = pair_sum32(l);
    merge(lt);
    if (wk == 0) {
        bool bad = nonfinite(lt);
        for (int t = 0; t < NDT; t++)
            for (int r = 0; r < 16; r++) bad |= nonfinite(oacc[t][r]);
        if (__builtin_amdgcn_ballot_w64(bad && ri < R) && lane == 0) again = 1;
    }
    __syncthreads();
    if (wk > 0) return;
    const size_t row = (size_t)bh * R + ri;
    if (again) {  // uniform
        attend8_plain<D>(a, bh, len, qrow, bs, b0, b1, pi, row, sp, ri < R);
        return;
    }
    if (ri >= R) return;
    for (int t = 0; t < NDT; t++)
        for (int rq = 0; rq < 4; rq++)
            write_row4<D, T>(a, row, sp, t * 32 + rq * 8 + g * 4,
                             f32x4{oacc[t][rq * 4], oacc[t][rq * 4 + 1], oacc[t][rq * 4 + 2], oacc[t][rq * 4 + 3]},
                             m, lt);
}

// Up to 16 rows (a decoding step, with up to 16 query heads to a key head): the
// same scheme on v_mfma_f32_16x16x32_bf16, four key waves. It costs half the
// products, weights and accumulators of a 32-row tile, and reads whole runs: an
// operand of V^T is 16 channels x 64 bytes, 1 KB in a row.
//
// Bound: the cache stream. Lane l of a wave holds row n = l % 16 and quarter g = l /
// 16 of the keys: position 16 g + 4 u + r of the block in register r of tile u.
template <int D, typename T>
__global__ __launch_bounds__(256, 2) void attend8_few_kernel(Attend8 a) {
    constexpr int WK = 4, NP = sizeof(T) == 4 ? 3 : 1, NJ = D / 64, ND = D / 16;
    constexpr int NE = 4 * ND + 2;
    __shared__ float red[(WK - 1) * NE * 64];
    __shared__ int again;

    const Cache8& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wk = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, n = lane & 15;
    const int T_ = a.T, R = a.Hq / c.H * T_, BH = c.B * c.H;
    int t0, t1;
    query_span(0, R - 1, T_, t0, t1);
    const Turn8 turn = turn_of(a, blockIdx.x, t0, t1, lane);
    const int sp = turn.sp, len = turn.len;
    const size_t bh = turn.bh;
    Blocks8 bs;
    bs.init(len - T_ + t0, len - T_ + t1, a.window, a.sinks);
    const int nv = bs.count(), ns = splits8(a, nv);
    if (sp >= ns && sp > 0) return;  // uniform; split 0 writes also where there is nothing to see
    const int b0 = ns ? (int)((long long)sp * nv / ns) : 0;
    const int b1 = ns ? (int)((long long)(sp + 1) * nv / ns) : 0;
    const int closed = len / kBlk8;
    const int open_at = b1 > b0 && bs.block(b1 - 1) == closed ? b1 - 1 : b1;

    // Block's operands: tile u's K rows, 64 jj + 16 g .. of their channels; V^T rows
    // 16 t + n, positions 16 g ...
    const int krow = 16 * (n >> 2) + (n & 3);
    u32x4 kr[4][NJ], vr[ND];
    float ksc = 0.f, vsc = 0.f;
    auto load_k = [&](int blk) {
        const uint8_t* p = c.k8 + ((bh * c.nblk + blk) * kBlk8 + krow) * D + 16 * g;
        for (int u = 0; u < 4; u++)
            for (int j = 0; j < NJ; j++)
                kr[u][j] = __builtin_nontemporal_load((const u32x4*)(p + 4 * u * D + 64 * j));
        ksc = c.ks[bh * c.nblk + blk];
    };
    auto load_v = [&](int blk) {
        const uint8_t* p = c.v8 + ((bh * c.nblk + blk) * D + n) * kBlk8 + 16 * g;
        for (int t = 0; t < ND; t++)
            vr[t] = __builtin_nontemporal_load((const u32x4*)(p + t * 16 * kBlk8));
        vsc = c.vs[bh * c.nblk + blk];
    };
    int bi = b0 + wk;
    if (bi < open_at) {
        load_k(bs.block(bi));
        load_v(bs.block(bi));
    }
    const int rc = n < R ? n : R - 1, pi = len - T_ + rc % T_;
    const int pw0 = len - T_ + t0, pw1 = len - T_ + t1;
    const T* qrow = (const T*)a.q + ((size_t)bh * R + rc) * D;
    bf16x8 qf[2 * NJ][NP];
    for (int j = 0; j < NJ; j++)
        for (int x = 0; x < 2; x++) load_q<NP>(qrow + 64 * j + 16 * g + 8 * x, qf[2 * j + x]);
    if (tid == 0) again = 0;

    f32x4 oacc[ND];
    for (int t = 0; t < ND; t++) oacc[t] = f32x4{};
    float m = -INFINITY, l = 0.f;

    // A whole block: kf(u, jj, x) and vf(t, w) give the operands.
    auto block = [&](int blk, auto kf, auto vf, auto next_k, auto next_v) {
        f32x4 s[4];
        for (int u = 0; u < 4; u++) {
            f32x4 x0 = f32x4{}, x1 = f32x4{};
            for (int j = 0; j < NJ; j++)
                for (int x = 0; x < 2; x++) {
                    const bf16x8 k = kf(u, j, x);
                    if constexpr (NP == 3) {
                        x1 = mfma_bf16_16(k, qf[2 * j + x][2], x1);
                        x1 = mfma_bf16_16(k, qf[2 * j + x][1], x1);
                    }
                    x0 = mfma_bf16_16(k, qf[2 * j + x][0], x0);
                }
            if constexpr (NP == 3) x0 += x1;
            s[u] = x0 * a.scale_log2;
        }
        for (int u = 0; u < 4; u++) pin_before_branch(s[u]);
        next_k();
        const int k0 = blk * kBlk8;
        if (!(k0 + 63 <= pw0 && (a.window == 0 || pw1 - k0 < a.window || k0 + 63 < a.sinks)))
            for (int u = 0; u < 4; u++)
                for (int r = 0; r < 4; r++)
                    s[u][r] = sees8(pi, k0 + 16 * g + 4 * u + r, a.window, a.sinks) ? s[u][r] : -INFINITY;
        float mx = -INFINITY;
        for (int u = 0; u < 4; u++)
            for (int r = 0; r < 4; r++) mx = fmaxf(mx, s[u][r]);
        mx = quad_max(mx);
        const bool need = mx > m && (m == -INFINITY || mx - m > 8.f);
        if (__builtin_amdgcn_ballot_w64(need)) {
            const float mn = need ? mx : m;
            const float alpha = m == -INFINITY ? 0.f : fast_exp2(m - mn);
            m = mn;
            l *= alpha;
            for (int t = 0; t < ND; t++) oacc[t] *= alpha;
        }
        const float mref = m == -INFINITY ? 0.f : m;
        float rs[4] = {0.f, 0.f, 0.f, 0.f};
        bf16x8 pf[2][NP];  // positions 16 g + 8 w ..
        for (int w = 0; w < 2; w++) {
            float e[8];
            for (int i = 0; i < 8; i++) {
                e[i] = fast_exp2(s[2 * w + (i >> 2)][i & 3] - mref);
                rs[i & 3] += e[i];
            }
            pieces<NP>(e, pf[w]);
        }
        l += (rs[0] + rs[1]) + (rs[2] + rs[3]);
        for (int t = 0; t < ND; t++) {
            if constexpr (NP == 1) {
                for (int w = 0; w < 2; w++) oacc[t] = mfma_bf16_16(vf(t, w), pf[w][0], oacc[t]);
            } else {
                f32x4 y = f32x4{};
                const bf16x8 v[2] = {vf(t, 0), vf(t, 1)};
                for (int i = NP - 1; i >= 0; i--)
                    for (int w = 0; w < 2; w++) y = mfma_bf16_16(v[w], pf[w][i], y);
                oacc[t] += y;
            }
        }
        for (int t = 0; t < ND; t++) pin_before_branch(oacc[t]);
        next_v();
    };
    for (; bi < open_at; bi += WK) {
        const int blk = bs.block(bi), nx = bi + WK < open_at ? bs.block(bi + WK) : blk;
        const float k1 = ksc, v1 = vsc;
        block(
            blk, [&](int u, int j, int x) { return decode8(kr[u][j][2 * x], kr[u][j][2 * x + 1], k1); },
            [&](int t, int w) { return decode8(vr[t][2 * w], vr[t][2 * w + 1], v1); },
            [&] { load_k(nx); }, [&] { load_v(nx); });
    }
    if (open_at < b1 && (open_at - b0) % WK == wk) {
        // The open block, bf16; positions past the last are no one's values.
        const uint16_t* kp = c.kt + ((bh * 2 + (closed & 1)) * kBlk8 + krow) * D + 16 * g;
        const uint16_t* vp = c.vt + ((bh * 2 + (closed & 1)) * D + n) * kBlk8 + 16 * g;
        const int left = len - closed * kBlk8 - 16 * g;
        block(
            closed,
            [&](int u, int j, int x) { return *(const bf16x8*)(kp + 4 * u * D + 64 * j + 8 * x); },
            [&](int t, int w) {
                u16x8 v = *(const u16x8*)(vp + (size_t)t * 16 * kBlk8 + 8 * w);
                for (int e = 0; e < 8; e++) v[e] = 8 * w + e < left ? v[e] : (uint16_t)0;
                return __builtin_bit_cast(bf16x8, v);
            },
            [] {}, [] {});
    }

    float lt = quad_sum(l);
    __syncthreads();
    if (wk > 0) {
        float* d = red + (wk - 1) * NE * 64 + lane;
        for (int t = 0; t < ND; t++)
            for (int r = 0; r < 4; r++) d[(t * 4 + r) * 64] = oacc[t][r];
        d[(NE - 2) * 64] = m;
        d[(NE - 1) * 64] = lt;
    }
    __syncthreads();
    if (wk == 0) {
        for (int w = 1; w < WK; w++) {
            const float* d = red + (w - 1) * NE * 64 + lane;
            const float m2 = d[(NE - 2) * 64], l2 = d[(NE - 1) * 64];
            const float M = fmaxf(m, m2), Mr = M == -INFINITY ? 0.f : M;
            const float x = fast_exp2(m - Mr), y = fast_exp2(m2 - Mr);
            lt = lt * x + l2 * y;
            for (int t = 0; t < ND; t++)
                for (int r = 0; r < 4; r++) oacc[t][r] = oacc[t][r] * x + d[(t * 4 + r) * 64] * y;
            m = M;
        }
        bool bad = nonfinite(lt);
        for (int t = 0; t < ND; t++)
            for (int r = 0; r < 4; r++) bad |= nonfinite(oacc[t][r]);
        if (__builtin_amdgcn_ballot_w64(bad && n < R) && lane == 0) again = 1;
    }
    __syncthreads();
    if (wk > 0) return;
    const size_t row = (size_t)bh * R;
    if (again) {  // uniform: one wave, the 32-row form
        const int ln = lane & 31, ri = ln < R ? ln : R - 1;
        attend8_plain<D>(a, bh, len, (const T*)a.q + (row + ri) * D, bs, b0, b1, len - T_ + ri % T_,
                         row + ln, sp, ln < R);
        return;
    }
    if (n >= R) return;
    for (int t = 0; t < ND; t++) write_row4<D, T>(a, row + n, sp, t * 16 + 4 * g, oacc[t], m, lt);
}

// ---------------------------------------------------------------------------
// Many bf16 rows (a prompt's next chunk): bound by the matrix cores, so the blocks are
// turned to bf16 once for the workgroup's 128 rows and the three-stage pipeline of
// window_fwd_pipe_kernel (attn_window.hip) runs on them. A thread loads its share of
// a block (K(t+4), V(t+2)) into registers one step ahead, and in the next step's slots
// turns it to bf16 and writes it to the two-slot LDS rings: K row-major, V transposed
// as it lies, each 16 positions in the order of P's registers. The open block comes
// last, straight from the ring to registers.
// ---------------------------------------------------------------------------
constexpr float kSumBound8 = 16384.f, kLazy8 = 8.f;

template <int D>
__global__ __launch_bounds__(256, 2) void attend8_pipe_kernel(Attend8 a) {
    constexpr int BM = 128, BN = 64, NKS = D / 16, NDT = D / 32, NPC = D / 64;
    constexpr uint32_t TB = BN * D * 2;  // bytes of a K or V tile
    constexpr int KLEAD = 3, VLEAD = 1;
    __shared__ __attribute__((aligned(16))) bf16 sKb[2 * BN * D];
    __shared__ __attribute__((aligned(16))) bf16 sVb[2 * BN * D];

    const Cache8& c = a.c;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 5, ln = lane & 31;
    const int T_ = a.T, R = a.Hq / c.H * T_, nrb = (R + BM - 1) / BM, BH = c.B * c.H;
    int us, rb;
    map_block(blockIdx.x, nrb, BH * a.nsplit, true, us, rb, 1, true);
    const int r0 = rb * BM, r1 = r0 + BM < R ? r0 + BM : R;
    int t0, t1;
    query_span(r0, r1 - 1, T_, t0, t1);
    const Turn8 turn = turn_of(a, us, t0, t1, lane);
    const int sp = turn.sp, len = turn.len;
    const size_t bh = turn.bh;
    Blocks8 bs;
    bs.init(len - T_ + t0, len - T_ + t1, a.window, a.sinks);
    const int nv = bs.count(), ns = splits8(a, nv);
    if (sp >= ns && sp > 0) return;  // uniform; split 0 writes also where there is nothing to see
    const int b0 = ns ? (int)((long long)sp * nv / ns) : 0;
    const int b1 = ns ? (int)((long long)(sp + 1) * nv / ns) : 0;
    const int closed = len / kBlk8;
    const bool open = b1 > b0 && bs.block(b1 - 1) == closed;
    const int ntiles = b1 - b0 - (open ? 1 : 0);

    // This wave's rows, this lane's, and the positions that they stand for.
    const int rw = r0 + wave * 32, ri = rw + ln, rc = ri < R ? ri : R - 1, pi = len - T_ + rc % T_;
    int wt0 = 0, wt1 = 0;
    if (rw < R) query_span(rw, rw + 31 < R ? rw + 31 : R - 1, T_, wt0, wt1);
    const int pw0 = len - T_ + wt0, pw1 = len - T_ + wt1;
    const float c2 = a.c2;
    const bf16* qrow = (const bf16*)a.q + ((size_t)bh * R + rc) * D;
    bf16x8 qf[NKS];
    auto load_q = [&](int d) {  // eight channels, times the scale's sign
        const uint32_t flip = a.sign < 0.f ? 0x80008000u : 0u, keep = a.sign != 0.f ? ~0u : 0u;
        u32x4 x = *(const u32x4*)(qrow + d);
        for (int e = 0; e < 4; e++) x[e] = (x[e] ^ flip) & keep;
        return __builtin_bit_cast(bf16x8, x);
    };

    // This thread's pieces of a block, 16 codes each: keys 16 wave + lane % 16, channels
    // 16 (lane / 16 + 4 i) ..; channels 16 (wave + 4 i) + lane % 16, positions 16 (lane /
    // 16) ... LDS: slabs as in common.h, K of 64 rows, V^T of D.
    const int pr = lane & 15, pc = lane >> 4;
    u32x4 kst[NPC], vst[NPC];
    float ksc = 1.f, vsc = 1.f;
    auto blk_of = [&](int t) { return bs.block(b0 + (t < ntiles ? t : ntiles - 1)); };
    const uint32_t head = (uint32_t)c.nblk * kBlk8 * D;  // bytes of a head's codes
    const brsrc krs = make_rsrc(c.k8 + bh * head, head), vrs = make_rsrc(c.v8 + bh * head, head);
    const uint32_t kvo = (uint32_t)((16 * wave + pr) * D + 16 * pc), vvo = (uint32_t)((16 * wave + pr) * kBlk8 + 16 * pc);
    auto load_k = [&](int t, int i) {
        kst[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(krs, kvo + 64 * i, (uint32_t)blk_of(t) * kBlk8 * D, 0));
    };
    auto load_v = [&](int t, int i) {
        vst[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(vrs, vvo + 64 * i * kBlk8, (uint32_t)blk_of(t) * kBlk8 * D, 0));
    };
    auto slot_pos = [&](int rows, int row, int chunk) {
        return (uint32_t)((((chunk >> 2) * rows + row) * 4 + ((chunk & 3) ^ slab_swz(row))) * 16);
    };
    const uint32_t kp0 = slot_pos(BN, 16 * wave + pr, 2 * pc), kp1 = slot_pos(BN, 16 * wave + pr, 2 * pc + 1);
    const uint32_t vp0 = slot_pos(D, 16 * wave + pr, 2 * pc), vp1 = slot_pos(D, 16 * wave + pr, 2 * pc + 1);
    // Half x of piece i: eight codes to bf16 and to LDS.
    auto put_k = [&](char* tile, int i, int x) {
        *(bf16x8*)(tile + (x ? kp1 : kp0) + i * 2 * BN * 64) = decode8(kst[i][2 * x], kst[i][2 * x + 1], ksc);
    };
    auto put_v = [&](char* tile, int i, int x) {  // positions {0..3, 8..11} and {4..7, 12..15}
        *(bf16x8*)(tile + (x ? vp1 : vp0) + i * 64 * 64) = decode8(vst[i][x], vst[i][x + 2], vsc);
    };
    const int hs = slab_swz(ln);
    const uint32_t qa0 = (uint32_t)(ln * 64 + ((0 + g) ^ hs) * 16);
    const uint32_t qa1 = (uint32_t)(ln * 64 + ((2 + g) ^ hs) * 16);
    char *const sKc = (char*)sKb, *const sVc = (char*)sVb;
    auto kfrag = [&](const char* tile, int ks, int mt) {
        return *(const bf16x8*)(tile + ((ks & 1) ? qa1 : qa0) + ((ks >> 1) * BN + mt * 32) * 64);
    };
    auto vfrag = [&](uint32_t base, int ks, int dt) {
        return *(const bf16x8*)(sVc + base + ((ks & 1) ? qa1 : qa0) + ((ks >> 1) * D + dt * 32) * 64);
    };

    f32x16 oacc[NDT];
    for (int dt = 0; dt < NDT; dt++) oacc[dt] = f32x16{};
    float mc = 0.f, l = 0.f, alpha = 1.f;

    // Scores of block blk that this lane's row does not see, to -inf (c2 > 0).
    auto mask_blk = [&](int blk, f32x16* s, auto key_of) {
        const int kb = blk * kBlk8;
        if (kb + 63 <= pw0 && (a.window == 0 || pw1 - kb < a.window || kb + 63 < a.sinks)) return;
        const int hi = pi - kb, lo = a.window ? hi - a.window : -1, sk = a.sinks - kb;
        for (int mt = 0; mt < 2; mt++)
            for (int r = 0; r < 16; r++) {
                const int x = key_of(mt, r);
                s[mt][r] = x > hi || (x <= lo && x >= sk) ? -INFINITY : s[mt][r];
            }
    };
    auto mask = [&](int t, f32x16* s) {
        mask_blk(blk_of(t), s, [&](int mt, int r) { return mt * 32 + 8 * (r >> 2) + 4 * g + (r & 3); });
    };
    // Maximum of a tile's scaled scores over the row.
    auto tile_max = [&](const f32x16* s) {
        float m0 = -INFINITY;
        for (int mt = 0; mt < 2; mt++)
            for (int r = 0; r < 16; r++) m0 = fmaxf(m0, s[mt][r]);
        return pair_max32(m0) * c2;
    };
    auto p_tile = [&](const f32x16* s, u32x4* pk) {
        float part[4] = {0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < 16; k++) {
            const int mt = k >> 3, r = (k & 7) * 2;
            const float x = fast_exp2(__builtin_fmaf(s[mt][r], c2, -mc));
            const float y = fast_exp2(__builtin_fmaf(s[mt][r + 1], c2, -mc));
            part[k & 3] += x + y;
            const bf16x2 pr2 = {to_bf16(x), to_bf16(y)};
            pk[k >> 2][k & 3] = __builtin_bit_cast(uint32_t, pr2);
        }
        return (part[0] + part[1]) + (part[2] + part[3]);
    };
    // Moves the offset to the tile's maximum where the row has seen nothing yet or the
    // tile exceeds it by far; alpha is what that scales l and O by.
    auto move_offset = [&](const f32x16* s) {
        const float mx = tile_max(s);
        const bool empty = pair_sum32(l) == 0.f;
        const float mn = mx > -INFINITY && (empty || mx - mc > kLazy8) ? mx : mc;
        alpha = empty ? 0.f : fast_exp2(mc - mn);
        mc = mn;
    };
    u32x4 pp[4];  // P of the tile PV consumes next

    // One step, scheduled by hand as in attn_window.hip. TAIL: 0 a full step; 1 the
    // next-to-last (no S^T(t+2)); 2 the last (no P(t+1) either).
    auto step = [&](int t, f32x16* sA, f32x16* sB, auto TAILC) __attribute__((always_inline)) {
        constexpr int TAIL = decltype(TAILC)::value;
        char *const ktile = sKc + ((t + KLEAD) & 1) * TB, *const vtile = sVc + ((t + VLEAD) & 1) * TB;
        const float kn = c.ks[bh * c.nblk + blk_of(t + KLEAD + 1)], vn = c.vs[bh * c.nblk + blk_of(t + VLEAD + 1)];
        if constexpr (TAIL < 2) mask(t + 1, sB);
        const uint32_t vb = (uint32_t)(t & 1) * TB;
        const char* kt = sKc + (uint32_t)(t & 1) * TB;

        constexpr int SKS = NKS / 4, GW = NDT + 2 * SKS, NM = 4 * GW, NU = 16, LA = 3;
        constexpr int NPUT = 4 * NPC, DS = NM / NPUT < 2 ? NM / NPUT : 2;  // half pieces: K's, then V's
        static_assert(DS * NPUT <= NM, "the step's tile writes fit in its slots");
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
        auto put_slot = [&](auto E) {
            constexpr int e = decltype(E)::value, d = e / DS;
            // Tail steps write no K tile (TAIL >= 1) and no V tile (TAIL 2).
            if constexpr (e % DS == 0 && d < NPUT && d >= (TAIL == 0 ? 0 : TAIL == 1 ? NPUT / 2 : NPUT)) {
                constexpr int i = d % (2 * NPC) / 2, x = d % 2;
                if constexpr (d < 2 * NPC) {
                    put_k(ktile, i, x);
                    if constexpr (x == 1) load_k(t + KLEAD + 1, i);
                } else {
                    put_v(vtile, i, x);
                    if constexpr (x == 1) load_v(t + VLEAD + 1, i);
                }
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
            put_slot(E);
            uops_at(E);
            __builtin_amdgcn_sched_barrier(0);
        });
        uops_at(std::integral_constant<int, NM>{});
        __builtin_amdgcn_s_setprio(0);
        float ts = (part[0] + part[1]) + (part[2] + part[3]);
        alpha = 1.f;
        if (TAIL < 2 && __builtin_amdgcn_ballot_w64(!(ts <= kSumBound8) || l == 0.f)) {
            move_offset(sB);
            ts = p_tile(sB, pp);
        }
        l = l * alpha + ts;
        ksc = kn;
        vsc = vn;
        __syncthreads();
        if (__builtin_amdgcn_ballot_w64(alpha != 1.f))
            for (int dt = 0; dt < NDT; dt++) oacc[dt] *= alpha;
    };

    if (ntiles > 0) {
        // Prologue: S^T(0) -> P(0), S^T(1); K(0) is staged in V slot 1.
        f32x16 s0[2], s1[2];
        auto qk_tile = [&](const char* tile, f32x16* s) {
            s[0] = s[1] = f32x16{};
            for (int ks = 0; ks < NKS; ks++)
                for (int mt = 0; mt < 2; mt++) s[mt] = mfma_bf16(kfrag(tile, ks, mt), qf[ks], s[mt]);
        };
        auto fill_k = [&](int t, char* tile) {
            ksc = c.ks[bh * c.nblk + blk_of(t)];
            for (int i = 0; i < NPC; i++) load_k(t, i);
            for (int i = 0; i < NPC; i++)
                for (int x = 0; x < 2; x++) put_k(tile, i, x);
        };
        fill_k(0, sVc + TB);
        fill_k(1, sKc + TB);
        fill_k(2, sKc);
        vsc = c.vs[bh * c.nblk + blk_of(0)];
        for (int i = 0; i < NPC; i++) load_v(0, i);
        for (int i = 0; i < NPC; i++)
            for (int x = 0; x < 2; x++) put_v(sVc, i, x);
        for (int i = 0; i < NPC; i++) {  // what step 0 puts
            load_k(KLEAD, i);
            load_v(VLEAD, i);
        }
        ksc = c.ks[bh * c.nblk + blk_of(KLEAD)];
        vsc = c.vs[bh * c.nblk + blk_of(VLEAD)];
        for (int ks = 0; ks < NKS; ks++) qf[ks] = load_q(ks * 16 + g * 8);
        __syncthreads();
        qk_tile(sVc + TB, s0);
        qk_tile(sKc + TB, s1);
        settle_before_branch(s0[0], s0[1]);
        settle_before_branch(s1[0], s1[1]);
        mask(0, s0);
        mc = tile_max(s0);
        if (!(mc > -INFINITY)) mc = 0.f;  // nothing seen yet: no offset
        l = p_tile(s0, pp);
        __syncthreads();  // K(0) and K(1) read by every wave

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
    if (open && rw < R) {
        // The open block, bf16, with the operands of attend8_kernel: register r of tile u
        // is position 32 u + 16 g + r. Positions past the last are no one's values.
        const int krow = 16 * ((ln >> 2) & 1) + 4 * (ln >> 3) + (ln & 3), n = len - closed * kBlk8;
        const uint16_t* kp = c.kt + ((bh * 2 + (closed & 1)) * kBlk8 + krow) * D + 16 * g;
        const uint16_t* vp = c.vt + ((bh * 2 + (closed & 1)) * D + ln) * kBlk8 + 16 * g;
        f32x16 s[2];
        s[0] = s[1] = f32x16{};
        for (int u = 0; u < 2; u++)
            for (int j = 0; j < D / 32; j++)
                for (int x = 0; x < 2; x++)
                    s[u] = mfma_bf16(*(const bf16x8*)(kp + u * 32 * D + 32 * j + 8 * x),
                                     load_q(32 * j + 16 * g + 8 * x), s[u]);
        settle_before_branch(s[0], s[1]);
        mask_blk(closed, s, [&](int u, int r) { return 32 * u + 16 * g + r; });
        alpha = 1.f;
        move_offset(s);
        const float ts = p_tile(s, pp);
        l = l * alpha + ts;
        for (int t = 0; t < NDT; t++) {
            oacc[t] *= alpha;
            for (int u = 0; u < 2; u++)
                for (int x = 0; x < 2; x++) {
                    u16x8 v = *(const u16x8*)(vp + (size_t)t * 32 * kBlk8 + 32 * u + 8 * x);
                    for (int e = 0; e < 8; e++) v[e] = 32 * u + 16 * g + 8 * x + e < n ? v[e] : (uint16_t)0;
                    oacc[t] = mfma_bf16(__builtin_bit_cast(bf16x8, v), __builtin_bit_cast(bf16x8, pp[2 * u + x]), oacc[t]);
                }
        }
    }

    const float lt = pair_sum32(l);
    bool bad = nonfinite(lt);
    for (int t = 0; t < NDT; t++)
        for (int r = 0; r < 16; r++) bad |= nonfinite(oacc[t][r]);
    const size_t row = (size_t)bh * R + ri;
    if (__builtin_amdgcn_ballot_w64(bad && ri < R)) {
        attend8_plain<D>(a, bh, len, qrow, bs, b0, b1, pi, row, sp, ri < R);
        return;
    }
    if (ri >= R) return;
    // A row that saw nothing has no offset (its share of a combine is nothing).
    const float m = lt == 0.f ? -INFINITY : mc;
    for (int t = 0; t < NDT; t++)
        for (int rq = 0; rq < 4; rq++)
            write_row4<D, bf16>(a, row, sp, t * 32 + rq * 8 + g * 4,
                                f32x4{oacc[t][rq * 4], oacc[t][rq * 4 + 1], oacc[t][rq * 4 + 2], oacc[t][rq * 4 + 3]},
                                m, lt);
}

// Splits joined: a thread takes four channels of a row, 16 bytes of each split (a
// workgroup per row took 31 us for 32768 rows of 4 splits). A split in which the row
// saw nothing has m = -inf and counts for nothing.
template <int D, typename T>
__global__ __launch_bounds__(256) void attend8_combine_kernel(Attend8 a, unsigned rows) {
    const unsigned row = (blockIdx.x * 256 + threadIdx.x) / (D / 4);
    if (row >= rows) return;
    const int d = threadIdx.x % (D / 4) * 4, R = a.Hq / a.c.H * a.T;
    const int bh = (int)(row / (unsigned)R), r = (int)(row - (unsigned)bh * R);
    int len = a.c.len[bh / a.c.H];
    len = len < a.c.Lmax ? len : a.c.Lmax;
    // The row's workgroup and its splits, as the kernels above cut them.
    const int r0 = r / a.rows * a.rows, r1 = r0 + a.rows < R ? r0 + a.rows : R;
    int t0, t1;
    query_span(r0, r1 - 1, a.T, t0, t1);
    Blocks8 bs;
    bs.init(len - a.T + t0, len - a.T + t1, a.window, a.sinks);
    int ns = splits8(a, bs.count());
    ns = ns < 1 ? 1 : ns;
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2* ml = (const f32x2*)a.part_ml + (size_t)row * a.nsplit;
    const float* po = a.part_o + (size_t)row * a.nsplit * D + d;
    float M = -INFINITY;
    for (int i = 0; i < ns; i++) M = fmaxf(M, ml[i][0]);
    float L = 0.f;
    f32x4 O = f32x4{};
    for (int i = 0; i < ns; i++) {
        const f32x2 x = ml[i];
        const float w = x[0] == -INFINITY ? 0.f : fast_exp2(x[0] - M);
        L = __builtin_fmaf(w, x[1], L);
        const f32x4 v = *(const f32x4*)(po + (size_t)i * D);
        for (int e = 0; e < 4; e++) O[e] = __builtin_fmaf(w, v[e], O[e]);
    }
    for (int e = 0; e < 4; e++) O[e] = L == 0.f ? 0.f : O[e] / L;
    if constexpr (sizeof(T) == 4) *(f32x4*)((float*)a.o + (size_t)row * D + d) = O;
    else {
        typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
        *(bf16x4*)((bf16*)a.o + (size_t)row * D + d) =
            bf16x4{to_bf16(O[0]), to_bf16(O[1]), to_bf16(O[2]), to_bf16(O[3])};
    }
}

namespace {

template <int D, typename T>
void run_attend8(const Attend8& a, hipStream_t s) {
    const int R = a.Hq / a.c.H * a.T;
    const unsigned rows = (unsigned)(a.c.B * a.c.H) * (unsigned)R;
    const unsigned grid = (unsigned)((R + a.rows - 1) / a.rows) * (unsigned)(a.c.B * a.c.H) * (unsigned)a.nsplit;
    if (a.rows == 16) attend8_few_kernel<D, T><<<grid, 256, 0, s>>>(a);
    else if (a.rows == 32) attend8_kernel<D, T, 1><<<grid, 256, 0, s>>>(a);
    else if (a.rows == 128 && sizeof(T) == 2 && (double)a.c.nblk * kBlk8 * D < 4.0e9) {  // 32-bit offsets
        if constexpr (sizeof(T) == 2) attend8_pipe_kernel<D><<<grid, 256, 0, s>>>(a);
    } else if (a.rows == 64) attend8_kernel<D, T, 2><<<grid, 256, 0, s>>>(a);
    else attend8_kernel<D, T, 4><<<grid, 256, 0, s>>>(a);
    if (a.nsplit > 1)
        attend8_combine_kernel<D, T><<<(rows + 1024 / D - 1) / (1024 / D), 256, 0, s>>>(a, rows);
}

}  // namespace

hipError_t launch_attend8(const Attend8& a, int is_bf16, hipStream_t s) {
    if (a.c.D == 128) {
        if (is_bf16) run_attend8<128, bf16>(a, s);
        else run_attend8<128, float>(a, s);
    } else if (a.c.D == 64) {
        if (is_bf16) run_attend8<64, bf16>(a, s);
        else run_attend8<64, float>(a, s);
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace gonn
