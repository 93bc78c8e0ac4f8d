// kvcache8.hip -- the 8-bit KV cache: append, truncate and read (layout: kvcache8.h).
//
// Append: one workgroup per (sequence, head) and block that the new rows touch. It
// closes the block when they complete it: the 64 rows (older ones from the ring)
// go to LDS, K's and V's largest magnitudes give the scales, the codes are written
// as they lie (K) and transposed (V). Rows of the last two blocks also go to the
// ring; those of the half that the first block's workgroup reads are written by that
// workgroup, behind its reads. A sequence's length is advanced on the device by the
// last of its workgroups, so a captured append can be replayed.
//
// All of it is bound by memory. 8 x 8 heads, prompts of 1500 to 4096 rows, D 128, bf16:
// append 35 us (93 MB read, 49 written), read 26 (47 read, 134 written). One row to each
// of 64 x 32 heads: append 13 us, a workgroup per head and 40 ns of it per update of a
// sequence's counter; read of the open blocks 22 (74 MB read, 67 written).
#include "common.h"
#include "kvcache8.h"

namespace gonn {

namespace {

GONN_DEV int seq_number(const Seqs8& s, int i) { return s.use ? s.n[i] : s.all; }

// 2^e of a block with this largest magnitude (a bf16 value, finite).
GONN_DEV float block_scale(float top) {
    const uint32_t u = __float_as_uint(top);
    if (u == 0) return 1.f;
    // top = 1.f 2^(E - 127); 448 = 1.75 2^8.
    int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = e < kLeastExp8 ? kLeastExp8 : e;
    return __uint_as_float((uint32_t)(e + 127) << 23);
}
// e4m3 holds no infinity: one is stored as NaN, so that it is not hidden.
GONN_DEV float finite_or_nan(float x) {
    return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u ? __uint_as_float(0x7fc00000u) : x;
}
GONN_DEV uint32_t codes4(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(finite_or_nan(a), finite_or_nan(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(finite_or_nan(c), finite_or_nan(d), r, true);
}
// Eight rows' elements as bf16.
template <typename T>
GONN_DEV u16x8 bf16_of(const T* p) {
    if constexpr (sizeof(T) == 2) return *(const u16x8*)p;
    else {
        const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
        return __builtin_bit_cast(u16x8, pack8(a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]));
    }
}
GONN_DEV float magnitude(uint16_t h) {  // 0 for infinities and NaN
    const uint32_t m = h & 0x7fffu;
    return m >= 0x7f80u ? 0.f : __uint_as_float(m << 16);
}
GONN_DEV float wave_max(float x) {
    for (int i = 32; i > 0; i >>= 1) x = fmaxf(x, __shfl_xor(x, i));
    return x;
}

}  // namespace

template <int D, typename T>
__global__ __launch_bounds__(256) void append8_kernel(Cache8 c, const T* __restrict__ ksrc,
                                                      const T* __restrict__ vsrc, int T_, int nb,
                                                      Seqs8 cnt) {
    constexpr int CPR = D / 8, NCH = kBlk8 * CPR, PT = NCH / 256;  // 8-element chunks
    constexpr int VS = kBlk8 + 4;  // row stride of the transposed tile, in elements
    __shared__ __attribute__((aligned(16))) uint16_t vtile[D * VS];
    __shared__ float red[2][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int i = blockIdx.x % nb, u = blockIdx.x / nb, bi = u / c.H, h = u - bi * c.H;
    const int b = cnt.b0 + bi;
    const size_t bh = (size_t)b * c.H + h;
    const int pos = c.len[b];
    int n = seq_number(cnt, bi);
    n = pos + n <= c.Lmax ? n : 0;  // the host refuses such calls; a replayed graph may get here
    const int end = pos + n, first = pos / kBlk8, open = end / kBlk8;
    // Blocks first + i, and in the first one's workgroup the later block that takes its
    // half of the ring (the open one or the one before it), for its ring rows only.
    const int other = open - ((open ^ first) & 1);
    for (int pass = 0; pass < (i == 0 && other > first ? 2 : 1); pass++) {
        const int blk = pass ? other : first + i, base = blk * kBlk8;
        const int p0 = pos > base ? pos : base, p1 = end < base + kBlk8 ? end : base + kBlk8;
        if (p0 >= p1) continue;  // uniform
        const bool closing = !pass && end >= base + kBlk8;
        const bool keep = blk >= open - 1 && (pass || blk == first || ((blk ^ first) & 1));
        __syncthreads();  // the LDS tile is free
        uint16_t* kring = c.kt + (bh * 2 + (blk & 1)) * kBlk8 * D;
        uint16_t* vring = c.vt + (bh * 2 + (blk & 1)) * D * kBlk8;
        u16x8 kx[PT];
        float km = 0.f, vm = 0.f;
        for (int j = 0; j < PT; j++) {
            const int ch = j * 256 + tid, r = ch / CPR, d = ch % CPR * 8, p = base + r;
            if (p >= p0 && p < p1) {
                const size_t src = (bh * T_ + (p - pos)) * D + d;
                kx[j] = bf16_of(ksrc + src);
                const u16x8 v = bf16_of(vsrc + src);
                for (int e = 0; e < 8; e++) vtile[(d + e) * VS + r] = v[e];
                if (keep) *(u16x8*)(kring + (size_t)r * D + d) = kx[j];
            } else if (closing) {  // an older row, from the ring
                kx[j] = *(const u16x8*)(kring + (size_t)r * D + d);
            }
        }
        if (closing && p0 > base) {  // older values, eight positions of a channel at a time
            const int old = p0 - base;
            for (int ch = tid; ch < D * 8; ch += 256) {
                const int d = ch >> 3, r = (ch & 7) * 8;
                if (r >= old) continue;
                const u16x8 v = *(const u16x8*)(vring + ch * 8);
                for (int e = 0; e < 8; e++)
                    if (r + e < old) vtile[d * VS + r + e] = v[e];
            }
        }
        __syncthreads();
        if (keep) {
            if (p1 - p0 == 1) {
                if (tid < D) vring[(size_t)tid * kBlk8 + p0 - base] = vtile[tid * VS + p0 - base];
            } else {
                for (int ch = tid; ch < D * 16; ch += 256) {
                    const int d = ch >> 4, r = (ch & 15) * 4, a = base + r;
                    if (a >= p0 && a + 4 <= p1)
                        *(uint64_t*)(vring + (size_t)d * kBlk8 + r) = *(const uint64_t*)(vtile + d * VS + r);
                    else
                        for (int e = 0; e < 4; e++)
                            if (a + e >= p0 && a + e < p1) vring[(size_t)d * kBlk8 + r + e] = vtile[d * VS + r + e];
                }
            }
        }
        if (closing) {
            for (int j = 0; j < PT; j++)
                for (int e = 0; e < 8; e++) km = fmaxf(km, magnitude(kx[j][e]));
            // V pieces of 16 positions of one channel.
            constexpr int NV = D * 4, PV = NV / 256;
            for (int j = 0; j < PV; j++) {
                const int ch = j * 256 + tid;
                const uint16_t* x = vtile + (ch >> 2) * VS + (ch & 3) * 16;
                for (int e = 0; e < 16; e++) vm = fmaxf(vm, magnitude(x[e]));
            }
            km = wave_max(km);
            vm = wave_max(vm);
            if (lane == 0) {
                red[0][wave] = km;
                red[1][wave] = vm;
            }
            __syncthreads();
            const float ks = block_scale(fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3])));
            const float vs = block_scale(fmaxf(fmaxf(red[1][0], red[1][1]), fmaxf(red[1][2], red[1][3])));
            // 2^-e exactly: e lies between -100 and 120.
            const float ki = __uint_as_float((254u << 23) - __float_as_uint(ks));
            const float vi = __uint_as_float((254u << 23) - __float_as_uint(vs));
            const size_t at = bh * c.nblk + blk;
            if (tid == 0) {
                c.ks[at] = ks;
                c.vs[at] = vs;
            }
            for (int j = 0; j < PT; j++) {
                const int ch = j * 256 + tid;
                float x[8];
                for (int e = 0; e < 8; e++) x[e] = bf16_to_f32(kx[j][e]) * ki;
                const uint64_t w = (uint64_t)codes4(x[0], x[1], x[2], x[3]) |
                                   (uint64_t)codes4(x[4], x[5], x[6], x[7]) << 32;
                *(uint64_t*)(c.k8 + at * kBlk8 * D + (size_t)ch * 8) = w;
            }
            for (int j = 0; j < PV; j++) {
                const int ch = j * 256 + tid;
                const uint16_t* x = vtile + (ch >> 2) * VS + (ch & 3) * 16;
                u32x4 w;
                for (int e = 0; e < 4; e++)
                    w[e] = codes4(bf16_to_f32(x[4 * e]) * vi, bf16_to_f32(x[4 * e + 1]) * vi,
                                  bf16_to_f32(x[4 * e + 2]) * vi, bf16_to_f32(x[4 * e + 3]) * vi);
                *(u32x4*)(c.v8 + at * kBlk8 * D + (size_t)ch * 16) = w;
            }
        }
    }
    // The length was read above (the branches waited for it); the last of the
    // sequence's workgroups to say so advances it. One counter, and one cache line,
    // per sequence: updates of one address take about 40 ns each, 2048 on one 84 us.
    __syncthreads();
    unsigned* ticket = c.ticket + (size_t)b * kTicketStep8;
    if (tid == 0 && atomicAdd(ticket, 1u) == (unsigned)(c.H * nb) - 1) {
        c.len[b] = end;
        if ((open - 1) * kBlk8 > c.lo[b]) c.lo[b] = (open - 1) * kBlk8;
        *ticket = 0;
    }
}

__global__ __launch_bounds__(256) void truncate8_kernel(Cache8 c, Seqs8 s) {
    const int i = threadIdx.x;
    if (i >= s.nb) return;
    const int b = s.b0 + i, l = c.len[b], lo = c.lo[b];
    int n = seq_number(s, i);
    if (n >= l) return;
    if (n < lo) {  // the host refuses what is no block's start; a replayed graph may get here
        n = n / kBlk8 * kBlk8;
        c.lo[b] = n;
    }
    c.len[b] = n;
}

template <int D>
__global__ __launch_bounds__(256) void read8_kernel(Cache8 c, uint16_t* __restrict__ ko,
                                                    uint16_t* __restrict__ vo, int start, int count,
                                                    int nb) {
    constexpr int VS = kBlk8 + 4;
    constexpr int CPR = D / 8;
    __shared__ __attribute__((aligned(16))) uint16_t tile[D * VS];  // V as bf16, transposed
    const int tid = threadIdx.x, j = blockIdx.x % nb;
    const size_t bh = blockIdx.x / nb;
    const int len = c.len[bh / c.H], s0 = start < 0 ? len - count : start;
    const int blk = (s0 >= 0 ? s0 / kBlk8 : -((kBlk8 - 1 - s0) / kBlk8)) + j, base = blk * kBlk8;
    if (base >= s0 + count) return;
    const bool closed = blk >= 0 && blk < len / kBlk8, open = blk >= 0 && blk == len / kBlk8;
    const size_t at = bh * c.nblk + (closed ? blk : 0);
    const uint16_t* kring = c.kt + (bh * 2 + (blk & 1)) * kBlk8 * D;
    const uint16_t* vring = c.vt + (bh * 2 + (blk & 1)) * D * kBlk8;
    const float ks = closed ? c.ks[at] : 1.f, vs = closed ? c.vs[at] : 1.f;
    for (int ch = tid; ch < D * 4; ch += 256) {  // 16 positions of one channel
        const int d = ch >> 2, r = (ch & 3) * 16;
        uint16_t* dst = tile + d * VS + r;
        if (closed) {
            const u32x4 w = *(const u32x4*)(c.v8 + at * kBlk8 * D + (size_t)ch * 16);
            for (int e = 0; e < 4; e++) {
                typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
                const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[e], vs, false);
                const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[e], vs, true);
                *(uint32_t*)(dst + 4 * e) = __builtin_bit_cast(uint32_t, a);
                *(uint32_t*)(dst + 4 * e + 2) = __builtin_bit_cast(uint32_t, b);
            }
        } else if (open) {
            for (int e = 0; e < 4; e++)
                *(uint64_t*)(dst + 4 * e) = *(const uint64_t*)(vring + (size_t)d * kBlk8 + r + 4 * e);
        }
    }
    __syncthreads();
    for (int ch = tid; ch < 16 * CPR; ch += 256) {  // 4 rows of 8 channels
        const int r0 = ch / CPR * 4, d = ch % CPR * 8;
        uint64_t col[8];
        for (int e = 0; e < 8; e++) col[e] = *(const uint64_t*)(tile + (d + e) * VS + r0);
        for (int x = 0; x < 4; x++) {
            const int p = base + r0 + x;
            if (p < s0 || p >= s0 + count) continue;
            u16x8 kv = u16x8{}, vv = u16x8{};
            if (p >= 0 && p < len) {
                for (int e = 0; e < 8; e++) vv[e] = (uint16_t)(col[e] >> (16 * x));
                if (closed) {
                    const uint64_t w = *(const uint64_t*)(c.k8 + (at * kBlk8 + r0 + x) * D + d);
                    for (int e = 0; e < 4; e++) {
                        const int word = (int)(w >> (32 * (e >> 1)));
                        const auto y = e & 1 ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, ks, true)
                                             : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, ks, false);
                        const uint32_t z = __builtin_bit_cast(uint32_t, y);
                        kv[2 * e] = (uint16_t)z;
                        kv[2 * e + 1] = (uint16_t)(z >> 16);
                    }
                } else {
                    kv = *(const u16x8*)(kring + (size_t)(r0 + x) * D + d);
                }
            }
            const size_t o = (bh * count + (p - s0)) * D + d;
            *(u16x8*)(ko + o) = kv;
            *(u16x8*)(vo + o) = vv;
        }
    }
}

namespace {

template <int D, typename T>
void run_append8(const Cache8& c, const void* k, const void* v, int rows, const Seqs8& cnt,
                 hipStream_t s) {
    const int nb = (rows + 2 * kBlk8 - 2) / kBlk8;  // blocks that `rows` positions can touch
    const unsigned grid = (unsigned)cnt.nb * (unsigned)c.H * (unsigned)nb;
    append8_kernel<D, T><<<grid, 256, 0, s>>>(c, (const T*)k, (const T*)v, rows, nb, cnt);
}

}  // namespace

hipError_t launch_append8(const Cache8& c, const void* k, const void* v, int src_bf16, int T,
                          const Seqs8& cnt, hipStream_t s) {
    if (c.D == 128) {
        if (src_bf16) run_append8<128, bf16>(c, k, v, T, cnt, s);
        else run_append8<128, float>(c, k, v, T, cnt, s);
    } else if (c.D == 64) {
        if (src_bf16) run_append8<64, bf16>(c, k, v, T, cnt, s);
        else run_append8<64, float>(c, k, v, T, cnt, s);
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_truncate8(const Cache8& c, const Seqs8& n, hipStream_t s) {
    truncate8_kernel<<<1, kSeqs8, 0, s>>>(c, n);
    return hipGetLastError();
}

hipError_t launch_read8(const Cache8& c, void* k, void* v, int start, int count, hipStream_t s) {
    const int nb = (count + 2 * kBlk8 - 2) / kBlk8;
    const unsigned grid = (unsigned)c.B * (unsigned)c.H * (unsigned)nb;
    if (c.D == 128) read8_kernel<128><<<grid, 256, 0, s>>>(c, (uint16_t*)k, (uint16_t*)v, start, count, nb);
    else if (c.D == 64) read8_kernel<64><<<grid, 256, 0, s>>>(c, (uint16_t*)k, (uint16_t*)v, start, count, nb);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace gonn
