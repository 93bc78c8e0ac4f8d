// attn_window.h -- shared parts of the sliding-window attention kernels.
//
// The mask: query i sees key j when j <= i, j < kv_len and (i - j < window or
// j < sinks). A block of queries therefore reads two runs of keys, the first
// `sinks` ones and its window, and a block of keys is read by the queries of its
// band (and, where it holds sinks, by every later query).
//
// Two element types, in = out: bf16 (one plane of operands, products exact,
// sums in fp32) and fp32 (three bf16 planes, six products per product, fp32
// accuracy: split3 in common.h).
#pragma once
#include "attn_f32_split.h"

namespace gonn {

// ---- the mask on runs of keys and queries ----
struct Band {
    int window, sinks;
    GONN_DEV bool sees(int i, int j) const { return j <= i && (i - j < window || j < sinks); }
    // Some pair of queries [i0, i1] and keys [j0, j1] (inclusive, both orders).
    GONN_DEV bool any(int i0, int i1, int j0, int j1) const {
        return j0 <= i1 && (i0 - j1 < window || j0 < sinks);
    }
    // Every pair.
    GONN_DEV bool all(int i0, int i1, int j0, int j1) const {
        return j1 <= i0 && (i1 - j0 < window || j1 < sinks);
    }
};

// Key stages of BN keys that queries [q0, q1) read: ns of them from key 0 (the
// sinks), then nw from stage w0 on. kl: the keys that take part.
struct KeyStages {
    int ns, w0, nw;
    GONN_DEV void init(int q0, int q1, int kl, int BN, const Band& m) {
        const int hi = q1 < kl ? q1 : kl;
        const int lo = m.window <= q0 ? q0 - m.window + 1 : 0;
        const int end = (hi + BN - 1) / BN;
        w0 = lo / BN;
        w0 = w0 < end ? w0 : end;
        nw = end - w0;
        const int sk = m.sinks < hi ? m.sinks : hi;
        ns = (sk + BN - 1) / BN;
        ns = ns < w0 ? ns : w0;
    }
    GONN_DEV int count() const { return ns + nw; }
    GONN_DEV int stage(int st) const { return st < ns ? st : st - ns + w0; }
};

GONN_DEV int window_keys(const WindowParams& p, int b) {
    if (!p.kv_len) return p.Sk;
    int l = p.kv_len[b];
    l = l < 0 ? 0 : (l > p.Sk ? p.Sk : l);
    return __builtin_amdgcn_readfirstlane(l);
}

// ---- element types ----
template <typename T>
constexpr int kPlanes = sizeof(T) == 4 ? 3 : 1;
template <int NP>
struct Frag {
    bf16x8 p[NP];
};
GONN_DEV f32x16 mfma_n(const Frag<1>& a, const Frag<1>& b, f32x16 c) {
    return mfma_bf16(a.p[0], b.p[0], c);
}
GONN_DEV f32x16 mfma_n(const Frag<3>& a, const Frag<3>& b, f32x16 c) {
    return mfma_split3({a.p[0], a.p[1], a.p[2]}, {b.p[0], b.p[1], b.p[2]}, c);
}
template <int NP>
GONN_DEV Frag<NP> to_frag(const float* x) {
    if constexpr (NP == 1) return {{pack8(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7])}};
    else {
        const bf16x8x3 t = split3(x);
        return {{t.h, t.m, t.l}};
    }
}
template <typename T>
GONN_DEV float to_float(T x) {
    if constexpr (sizeof(T) == 4) return x;
    else return bf16_to_f32(__builtin_bit_cast(uint16_t, x));
}
// Eight elements as they lie in memory (16-byte aligned).
template <typename T>
struct Raw8 {
    u32x4 r[sizeof(T) * 8 / 16];
    GONN_DEV void load(const T* p) {
        for (unsigned i = 0; i < sizeof(T) * 8 / 16; i++) r[i] = ((const u32x4*)p)[i];
    }
    GONN_DEV void zero() {
        for (unsigned i = 0; i < sizeof(T) * 8 / 16; i++) r[i] = u32x4{};
    }
    GONN_DEV float f(int e) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(r[e >> 2][e & 3]);
        else return __uint_as_float((e & 1) ? r[0][e >> 1] & 0xffff0000u : r[0][e >> 1] << 16);
    }
    GONN_DEV Frag<kPlanes<T>> frag() const {
        if constexpr (sizeof(T) == 2) return {{__builtin_bit_cast(bf16x8, r[0])}};
        else {
            float x[8];
            for (int e = 0; e < 8; e++) x[e] = f(e);
            return to_frag<3>(x);
        }
    }
};
// Elements 16 ks + 8 g .. +7 of a row, every ks: an operand with one row per lane.
template <int D, typename T>
GONN_DEV void load_row_frags(const T* row, int g, bool live, Frag<kPlanes<T>>* f) {
    for (int ks = 0; ks < D / 16; ks++) {
        Raw8<T> x;
        if (live) x.load(row + ks * 16 + g * 8);
        else x.zero();
        f[ks] = x.frag();
    }
}
// Four consecutive elements.
template <typename T>
GONN_DEV void store4(T* p, f32x4 v) {
    if constexpr (sizeof(T) == 4) *(f32x4*)p = v;
    else {
        typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
        *(bf16x4*)p = bf16x4{to_bf16(v[0]), to_bf16(v[1]), to_bf16(v[2]), to_bf16(v[3])};
    }
}

// The streamed side of a stage: NT tiles of 32 rows of two tensors, in LDS as operand
// planes (SplitTile's layout: the first tensor's planes, then the second's). Rows at and
// past n are zeros.
template <int D, int NT, typename T>
struct RowStage;
// fp32: loaded one stage ahead into registers, split and stored.
template <int D, int NT>
struct RowStage<D, NT, float> {
    typedef float T;
    static constexpr bool DIRECT = false;
    static constexpr int NP = 3, NCH = 32 * D / 8, CH = NT * NCH / 256;
    static constexpr uint32_t PB = 32 * D * 2, TILE = 2 * NP * PB;
    Raw8<T> r[CH][2];
    int row[CH], col[CH];
    GONN_DEV void init(int tid) {
        for (int i = 0; i < CH; i++) {
            int rr, c;
            const int pos = i * 256 + tid;
            slab_chunk(pos % NCH, 32, rr, c);
            row[i] = pos / NCH * 32 + rr;
            col[i] = c * 8;
        }
    }
    GONN_DEV void load(const T* a, const T* b, int row0, int n) {
        for (int i = 0; i < CH; i++) {
            const int x = row0 + row[i];
            if (x < n) {
                r[i][0].load(a + (size_t)x * D + col[i]);
                r[i][1].load(b + (size_t)x * D + col[i]);
            } else {
                r[i][0].zero();
                r[i][1].zero();
            }
        }
    }
    GONN_DEV void store(char* stage, int tid) const {
        for (int i = 0; i < CH; i++) {
            const int pos = i * 256 + tid;
            char* dst = stage + pos / NCH * TILE + pos % NCH * 16;
            for (int w = 0; w < 2; w++) {
                const Frag<NP> f = r[i][w].frag();
                for (int j = 0; j < NP; j++) *(bf16x8*)(dst + (NP * w + j) * PB) = f.p[j];
            }
        }
    }
};
// bf16: straight from memory to LDS (one plane each), so that the load of the next stage
// needs no registers and its store none of the wave's time. Complete behind GONN_VMCNT(0) and a barrier; one barrier a stage instead
// of the two that a store from registers takes. dQ of 2 x 16 heads, 8192 queries, window
// 1024: 277 us through registers, 236 us this way. row0 < n, and n rows below 4 GB.
template <int D, int NT>
struct RowStage<D, NT, bf16> {
    static constexpr bool DIRECT = true;
    static constexpr int NCH = 32 * D / 8, CH = NT * NCH / 256;
    static constexpr uint32_t PB = 32 * D * 2, TILE = 2 * PB;
    uint32_t off[CH];
    GONN_DEV void init(int tid) {
        for (int i = 0; i < CH; i++) {
            int rr, c;
            const int pos = i * 256 + tid;
            slab_chunk(pos % NCH, 32, rr, c);
            off[i] = (uint32_t)((pos / NCH * 32 + rr) * D + c * 8) * 2;
        }
    }
    // Rows row0 .. of a and b, which have n rows, to the LDS stage at byte address lds.
    GONN_DEV void load(const bf16* a, const bf16* b, int row0, int n, uint32_t lds, int wave) const {
        const brsrc ra = make_rsrc(a, (uint32_t)n * D * 2), rb = make_rsrc(b, (uint32_t)n * D * 2);
        for (int i = 0; i < CH; i++) {
            const uint32_t dst = lds + i * 256 / NCH * TILE + i * 256 % NCH * 16 + wave * 1024;
            dma16(ra, dst, off[i], (uint32_t)row0 * D * 2);
            dma16(rb, dst + PB, off[i], (uint32_t)row0 * D * 2);
        }
    }
};
template <int D, int NP>
GONN_DEV Frag<NP> tile_row(const SplitTile<D>& tl, const char* tile, int w, int ks) {
    Frag<NP> f;
    for (int j = 0; j < NP; j++) f.p[j] = tl.row1(tile + (NP * w + j) * SplitTile<D>::PB, ks);
    return f;
}
template <int D, int NP>
GONN_DEV Frag<NP> tile_col(const SplitTile<D>& tl, char* tile, int w, int ks, int t) {
    Frag<NP> f;
    for (int j = 0; j < NP; j++) f.p[j] = tl.col1(tile + (NP * w + j) * SplitTile<D>::PB, ks, t);
    return f;
}

// acc[r] += w * row[8 (r / 4) + 4 g + r % 4] where on, untouched where not: a product
// that an infinity or a NaN in a masked place cannot reach.
template <typename T>
GONN_DEV void add_row32(f32x16& acc, float w, const T* row, int g, bool on) {
#pragma unroll
    for (int r = 0; r < 16; r++) {
        const float x = to_float(row[8 * (r >> 2) + 4 * g + (r & 3)]);
        acc[r] = on ? __builtin_fmaf(w, x, acc[r]) : acc[r];
    }
}
// Weight r of the 32 that a wave holds per column (16 in each half): key or
// query row 8 (r / 4) + 4 h + r % 4.
GONN_DEV float weight_of(const f32x16& w, int r, int h, int g) {
    float x = 0.f;
    for (int i = 0; i < 16; i++) x = i == r ? w[i] : x;
    const float other = __shfl_xor(x, 32);
    return h == g ? x : other;
}

}  // namespace gonn
