// kvcache8.h -- layout of the 8-bit KV cache, shared by its kernels and the C ABI.
//
// Positions come in blocks of 64. The closed ones (all 64 positions appended) are
// e4m3 codes with one scale for K and one for V, the smallest power of two 2^e,
// e >= -100, that brings the block's largest finite magnitude to at most 448, so
// that scaling is exact and a value is rounded once. K is row-major, V transposed:
// both are matrix operands as they lie. The open block is bf16, in the half
// (block & 1) of a two-block ring, which also keeps the block before it in bf16,
// so that a cache can be cut back across the block's start and be what it was.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace gonn {

constexpr int kBlk8 = 64;           // positions per block
constexpr int kLeastExp8 = -100;    // least exponent of a scale
constexpr int kTicketStep8 = 32;    // counters of different sequences: 128 bytes apart
constexpr int kSeqs8 = 256;         // sequences per append or truncate launch

struct Cache8 {
    uint8_t* k8;   // (B*H, nblk, 64, D)
    uint8_t* v8;   // (B*H, nblk, D, 64)
    float* ks;     // (B*H, nblk)
    float* vs;
    uint16_t* kt;  // (B*H, 128, D) bf16: position p at row p % 128
    uint16_t* vt;  // (B*H, 2, D, 64) bf16: position p at (p / 64 % 2, :, p % 64)
    int* len;      // [B]
    int* lo;       // [B] first position whose bf16 row the ring still holds
    unsigned* ticket;  // (B, kTicketStep8) workgroups of a running append that have read len
    int B, H, Lmax, D, nblk;
};

// Per-sequence numbers of one launch, by value: no copy, nothing to keep alive.
struct Seqs8 {
    int b0, nb;          // sequences b0 .. b0 + nb - 1
    int use;             // n[] holds their numbers, else `all` for each
    int all;
    int n[kSeqs8];
};

hipError_t launch_append8(const Cache8& c, const void* k, const void* v, int src_bf16, int T,
                          const Seqs8& cnt, hipStream_t s);
// len = min(len, n); see gonn_hip_kvcache8_truncate.
hipError_t launch_truncate8(const Cache8& c, const Seqs8& n, hipStream_t s);
// Rows [start, start + count) of every sequence, or its last `count` (start < 0),
// as bf16 (B,H,count,D).
hipError_t launch_read8(const Cache8& c, void* k, void* v, int start, int count, hipStream_t s);

struct Attend8 {
    Cache8 c;
    const void* q;  // (B, Hq, T, D), bf16 or f32; o alike
    void* o;
    float* part_o;   // (B*Hq*T, nsplit, D) unnormalised
    float* part_ml;  // (B*Hq*T, nsplit, 2) maximum and sum, log2 units
    int Hq, T, window, sinks;  // window 0: every position
    int split, nsplit;         // blocks per split, splits at most
    int rows;                  // rows (heads x queries) per workgroup: 16, 32, 64 or 128
    float scale_log2;
    float c2, sign;  // the same with the sign apart (WindowParams)
};
hipError_t launch_attend8(const Attend8& a, int is_bf16, hipStream_t s);

}  // namespace gonn
