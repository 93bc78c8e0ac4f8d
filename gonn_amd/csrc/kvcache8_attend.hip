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

GONN_DEV bool sees8(int i, int j, int window, int sinks) {
    return j <= i && (window == 0 || i - j < window || j < sinks);
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

// The wave's 32 rows in plain fp32 products, for results that are not finite: a
// masked position's weight of 0 would make NaN of a value that is.
template <int D, typename T>
GONN_DEV void attend8_plain(const Attend8& a, size_t bh, int len, const T* qrow, const Blocks8& bs,
                            int b0, int b1, int step, int pi, f32x16* oacc, float& m, float& l) {
    constexpr int HD = D / 2, NDT = D / 32;
    const int lane = threadIdx.x & 63, g = lane >> 5, ln = lane & 31;
    for (int t = 0; t < NDT; t++) oacc[t] = f32x16{};
    m = -INFINITY;
    l = 0.f;
#pragma unroll 1
    for (int bi = b0; bi < b1; bi += step)
#pragma unroll 1
        for (int kb = bs.block(bi) * kBlk8, u = 0; u < 2; u++, kb += 32) {
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
            for (int t = 0; t < NDT; t++) oacc[t] *= alpha;
#pragma unroll 1
            for (int x = 0; x < 32; x++) {
                const int r = x >> 1, h = x & 1, key = kb + 8 * (r >> 2) + 4 * h + (r & 3);
                float w = 0.f;
                for (int i = 0; i < 16; i++) w = i == r ? s[i] : w;
                const float other = __shfl_xor(w, 32);
                w = h == g ? w : other;
                if (key >= len) continue;  // uniform
                const bool on = sees8(pi, key, a.window, a.sinks);
                for (int t = 0; t < NDT; t++)
                    for (int e = 0; e < 16; e++) {
                        const float v = element8(a.c, bh, len, key, 32 * t + 8 * (e >> 2) + 4 * g + (e & 3), true);
                        oacc[t][e] = on ? __builtin_fmaf(w, v, oacc[t][e]) : oacc[t][e];
                    }
            }
        }
    l = pair_sum32(l);
}

}  // namespace

template <int D, typename T, int WQ>
__global__ __launch_bounds__(256, 1) void attend8_kernel(Attend8 a) {
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
    // All first splits before the second ones, which short sequences do not have.
    int us, rb;
    map_block(blockIdx.x, nrb, BH * a.nsplit, true, us, rb, 1, true);
    const int sp = __builtin_amdgcn_readfirstlane(us / BH), bhi = us - sp * BH, b = bhi / c.H;
    const size_t bh = bhi;
    int len = c.len[b];
    len = __builtin_amdgcn_readfirstlane(len < c.Lmax ? len : c.Lmax);
    const int r0 = rb * BM, r1 = r0 + BM < R ? r0 + BM : R;
    int t0, t1;
    query_span(r0, r1 - 1, T_, t0, t1);
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
        for (int x = 0; x < 2; x++) {
            const T* p = qrow + 32 * j + 16 * g + 8 * x;
            if constexpr (NP == 1) qf[2 * j + x][0] = *(const bf16x8*)p;
            else {
                const f32x4 u = *(const f32x4*)p, v = *(const f32x4*)(p + 4);
                const float y[8] = {u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
                const bf16x8x3 s = split3(y);
                qf[2 * j + x][0] = s.h;
                qf[2 * j + x][1] = s.m;
                qf[2 * j + x][2] = s.l;
            }
        }
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
                if constexpr (NP == 1) {
                    pf[u][x][0] = pack8(e[0], e[1], e[2], e[3], e[4], e[5], e[6], e[7]);
                } else {
                    const bf16x8x3 p = split3(e);
                    pf[u][x][0] = p.h;
                    pf[u][x][1] = p.m;
                    pf[u][x][2] = p.l;
                }
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
            __syncthreads();
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
    if (again) {  // uniform
        attend8_plain<D>(a, bh, len, qrow, bs, b0 + wk, b1, WK, pi, oacc, m, lt);
        merge(lt);
    }
    if (wk > 0 || ri >= R) return;
    const size_t row = (size_t)bh * R + ri;
    const bool whole = a.nsplit == 1;
    const float inv = whole ? (lt == 0.f ? 0.f : 1.f / lt) : 1.f;
    for (int t = 0; t < NDT; t++)
        for (int rq = 0; rq < 4; rq++) {
            f32x4 v;
            for (int i = 0; i < 4; i++) v[i] = oacc[t][rq * 4 + i] * inv;
            const int d = t * 32 + rq * 8 + g * 4;
            if (!whole) *(f32x4*)(a.part_o + (row * a.nsplit + sp) * D + d) = v;
            else if constexpr (NP == 3) *(f32x4*)((float*)a.o + row * D + d) = v;
            else {
                typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
                *(bf16x4*)((bf16*)a.o + row * D + d) =
                    bf16x4{to_bf16(v[0]), to_bf16(v[1]), to_bf16(v[2]), to_bf16(v[3])};
            }
        }
    if (!whole && g == 0) {
        // A NaN row has no maximum; a finite one keeps its weight non-zero.
        a.part_ml[(row * a.nsplit + sp) * 2 + 0] = lt != lt ? 0.f : m;
        a.part_ml[(row * a.nsplit + sp) * 2 + 1] = lt;
    }
}

// Splits of one row joined: one workgroup of D threads per row. A split in which
// the row saw nothing has m = -inf and counts for nothing.
template <int D, typename T>
__global__ __launch_bounds__(D) void attend8_combine_kernel(Attend8 a) {
    const size_t row = blockIdx.x;
    const int R = a.Hq / a.c.H * a.T, tid = threadIdx.x;
    const int bh = (int)(row / R), r = (int)(row - (size_t)bh * R);
    int len = a.c.len[bh / a.c.H];
    len = len < a.c.Lmax ? len : a.c.Lmax;
    // The row's workgroup and its splits, as the kernel above cuts them.
    const int r0 = r / a.rows * a.rows, r1 = r0 + a.rows < R ? r0 + a.rows : R;
    int t0, t1;
    query_span(r0, r1 - 1, a.T, t0, t1);
    Blocks8 bs;
    bs.init(len - a.T + t0, len - a.T + t1, a.window, a.sinks);
    int ns = splits8(a, bs.count());
    ns = ns < 1 ? 1 : ns;
    const float* ml = a.part_ml + row * a.nsplit * 2;
    const float* po = a.part_o + row * a.nsplit * D;
    float M = -INFINITY;
    for (int i = 0; i < ns; i++) M = fmaxf(M, ml[2 * i]);
    float L = 0.f, O = 0.f;
    for (int i = 0; i < ns; i++) {
        const float w = ml[2 * i] == -INFINITY ? 0.f : fast_exp2(ml[2 * i] - M);
        L = __builtin_fmaf(w, ml[2 * i + 1], L);
        O = __builtin_fmaf(w, po[(size_t)i * D + tid], O);
    }
    const float o = L == 0.f ? 0.f : O / L;
    if constexpr (sizeof(T) == 4) ((float*)a.o)[row * D + tid] = o;
    else ((bf16*)a.o)[row * D + tid] = to_bf16(o);
}

namespace {

template <int D, typename T>
void run_attend8(const Attend8& a, hipStream_t s) {
    const int R = a.Hq / a.c.H * a.T;
    const unsigned rows = (unsigned)(a.c.B * a.c.H) * (unsigned)R;
    const unsigned grid = (unsigned)((R + a.rows - 1) / a.rows) * (unsigned)(a.c.B * a.c.H) * (unsigned)a.nsplit;
    if (a.rows == 32) attend8_kernel<D, T, 1><<<grid, 256, 0, s>>>(a);
    else if (a.rows == 64) attend8_kernel<D, T, 2><<<grid, 256, 0, s>>>(a);
    else attend8_kernel<D, T, 4><<<grid, 256, 0, s>>>(a);
    if (a.nsplit > 1) attend8_combine_kernel<D, T><<<rows, D, 0, s>>>(a);
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
