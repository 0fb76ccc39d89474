// What the attention kernels over a KV cache share (kv_attention.hip, page_attention.hip): operands as pairs of f16 values,
// direct loads into LDS, values that are not finite. kv_attention.hip's head has the mathematics.
#pragma once

#include "kv_ops.h"
#include "wave.h"

namespace {

constexpr int D = 128, KB = 32;                // head dim; keys a block
constexpr int K_CHUNKS = 512, TILE = 1024;     // 16-byte chunks of a block's K, of its K and V
constexpr float P_SHIFT = 10.0f, P_ROOM = 5.0f; // log2 of the largest p when m moves; its growth before m must move
constexpr float LOG2E = 1.4426950408889634f;
constexpr float M_NONE = -3.0e38f;             // m before the first key: finite, so that s − m is never ∞ − ∞

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));
typedef int int2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));
typedef uint16_t ushort2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

// 4 bytes a lane from base + off to LDS bytes lds + 4·lane (as lds_load16)
__device__ __forceinline__ void lds_load4(const void *base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(base)
                 : "memory", "m0");
}
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// v, as a value the compiler does not know: what is computed from it stays where it is used (a rare path's addresses and
// offsets, moved out of the loop, would take registers from the loop)
__device__ __forceinline__ int here(int v) {
    asm volatile("" : "+v"(v));
    return v;
}
// this wave's LDS reads have their values
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// partial sums between workgroups: in the L2 of the XCD that they share (workgroup-scope stores, read by agent-scope loads
// that find the L2's lines), or through the coherence point
__device__ __forceinline__ void put64(void *p, float a, float b, bool xl) {
    const uint64_t v = (uint64_t)__float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32;
    if (xl) __hip_atomic_store((uint64_t *)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    else __hip_atomic_store((uint64_t *)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get64(const void *p) {
    const uint64_t v = __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// the lowest n bits (none for n ≤ 0, all from 32 on)
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? ~0u : (1u << max(n, 0)) - 1; }

// the blocks of the keys 0 … last (−1: none; last + 32 passes 31 bits)
__host__ __device__ __forceinline__ int blocks_to(int last) { return (int)(((uint32_t)last + KB) / KB); }
// a wave's blocks of a tile: the first `whole` all of its rows see the whole of, the first `any` one of them sees. last0, last1: the
// last keys that its first and its last row see; a wave without rows has no blocks (with those that a row would have, it made all
// products of a tile for nobody: 48 chunks of 21 rows of two heads over 4000 keys 216 µs for 182, over q8_0 rows 213 for 175)
struct WaveBlocks {
    int whole, any;
};
__host__ __device__ __forceinline__ WaveBlocks wave_blocks(bool has_rows, int last0, int last1) {
    return has_rows ? WaveBlocks{(last0 + 1) / KB, blocks_to(last1)} : WaveBlocks{0, 0};
}

// p − (float)h for the low (0) or high (1) half of h: one mixed-precision fma
template <int HI> __device__ __forceinline__ float minus_half(float p, uint32_t h) {
    float r;
    if constexpr (HI) asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(p));
    else asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(p));
    return r;
}
// two values as a pair of f16 values each
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const half2_t h = __builtin_convertvector((float2_t{a, b}), half2_t);
    __builtin_memcpy(&hi, &h, 4);
    const half2_t r = __builtin_convertvector((float2_t{minus_half<0>(a, hi), minus_half<1>(b, hi)}), half2_t);
    __builtin_memcpy(&lo, &r, 4);
}

// a row's q as f32: the lane's 8 dims of each of N steps, those of step 0 at qrow. PAIRED (N = 8): two steps are 16 dims in a row
template <int N, bool PAIRED = false> __device__ __forceinline__ void q_load(const float *qrow, float (&x)[N][8]) {
    auto dim = [](int ks) { return N == 4 ? 64 * (ks >> 1) + 8 * (ks & 1) : PAIRED ? 32 * (ks >> 1) + 8 * (ks & 1) : D / N * ks; };
#pragma unroll
    for (int ks = 0; ks < N; ks++) {
        const float4 a0 = *reinterpret_cast<const float4 *>(qrow + dim(ks));
        const float4 a1 = *reinterpret_cast<const float4 *>(qrow + dim(ks) + 4);
        x[ks][0] = a0.x, x[ks][1] = a0.y, x[ks][2] = a0.z, x[ks][3] = a0.w;
        x[ks][4] = a1.x, x[ks][5] = a1.y, x[ks][6] = a1.z, x[ks][7] = a1.w;
    }
}
// q·scale as f16 pairs, the B operand of N steps, of `G` lanes that hold the row; the factor of its scores
template <int N, int G> __device__ __forceinline__ float q_split(float (&x)[N][8], float scale, half8 (&qh)[N], half8 (&ql)[N]) {
    float top = 0.0f;
#pragma unroll
    for (int ks = 0; ks < N; ks++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            x[ks][e] *= scale;
            top = fmaxf(top, fabsf(x[ks][e]));
        }
    if constexpr (G == 16) top = group_max<8>(top, threadIdx.x & 63);  // 16 lanes in a row
    if constexpr (G == 4) top = pair_max<16>(top);                     // every 16th lane
    if constexpr (G <= 4) top = pair_max<32>(top);                     // every 32nd
    // (a row of nothing but tiny values: its scores are 0 to f32 either way, and the factor stays a normal number)
    const int ex = max(__builtin_amdgcn_frexp_expf(top), -100);
    const float up = ldexpf(1.0f, 10 - ex);
#pragma unroll
    for (int ks = 0; ks < N; ks++) {
        uint32_t h[4], r[4];
#pragma unroll
        for (int e = 0; e < 4; e++) split2(x[ks][2 * e] * up, x[ks][2 * e + 1] * up, h[e], r[e]);
        __builtin_memcpy(&qh[ks], h, 16);
        __builtin_memcpy(&ql[ks], r, 16);
    }
    return ldexpf(LOG2E, ex - 10);
}
// both
template <int N, int G> __device__ __forceinline__ float q_pairs(const float *qrow, float scale, half8 (&qh)[N], half8 (&ql)[N]) {
    float x[N][8];
    q_load(qrow, x);
    return q_split<N, G>(x, scale, qh, ql);
}

// values of V that are not finite, in blocks that not every row sees (0·∞ is NaN on the matrix cores, in rows too that do
// not see them): taken as 0 in the product, and NaN put in afterwards where a row does see one, by a product of ones
__device__ __forceinline__ half8 finite(half8 v) {
    uint32_t w[4];
    __builtin_memcpy(w, &v, 16);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const uint32_t b = ((w[e] & 0x7C007C00u) + 0x04000400u) & 0x80008000u;  // a half whose exponent is all ones
        w[e] &= ~((b >> 15) * 0xFFFFu);
    }
    __builtin_memcpy(&v, w, 16);
    return v;
}
// the largest |v| so far, as bits by halves; whether a lane of the wave has met one that is not finite
__device__ __forceinline__ void largest(half8 v, uint32_t &top) {
    ushort2_t t;
    uint32_t w[4];
    __builtin_memcpy(w, &v, 16);
    __builtin_memcpy(&t, &top, 4);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        ushort2_t x;
        w[e] &= 0x7FFF7FFFu;
        __builtin_memcpy(&x, &w[e], 4);
        t = __builtin_elementwise_max(t, x);
    }
    __builtin_memcpy(&top, &t, 4);
}
__device__ __forceinline__ bool any_not_finite(uint32_t top) {
    return __builtin_amdgcn_ballot_w64((((top & 0x7C007C00u) + 0x04000400u) & 0x80008000u) != 0) != 0;
}
// of two scales of a q8_0 cache one that may make such a value: NaN, or 512 and past (of the quant −128, which is not written
// here but may stand in a cache made elsewhere, −128·512 is f16's −∞; 511.75, the number before, gives −65504)
__device__ __forceinline__ bool scale_past(uint32_t d) { return (d & 0x7FFFu) > 0x5FFFu || (d >> 16 & 0x7FFFu) > 0x5FFFu; }
__device__ __forceinline__ half8 ones_of_not_finite(half8 v) {
    uint32_t w[4];
    __builtin_memcpy(w, &v, 16);
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = ((((w[e] & 0x7C007C00u) + 0x04000400u) & 0x80008000u) >> 15) * 0x3C00u;
    __builtin_memcpy(&v, w, 16);
    return v;
}
// o's sums of the rows that see one: NaN. seen: the lane's 16 keys (bits 0 … 3, 8 … 11, 16 …, 24 …);
// vread(u, ss): V's operand of tile u, step ss
template <typename F> __device__ __forceinline__ void put_nan(f32x16 (&o)[4], uint32_t seen, F vread) {
    half8 ind[2];
#pragma unroll
    for (int ss = 0; ss < 2; ss++) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; e++)
            w[e] = ((seen >> (16 * ss + 4 * (e & 2) + 2 * (e & 1))) & 1) * 0x3C00u |
                   ((seen >> (16 * ss + 4 * (e & 2) + 2 * (e & 1) + 1)) & 1) * 0x3C000000u;
        __builtin_memcpy(&ind[ss], w, 16);
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
        f32x16 t = __builtin_amdgcn_mfma_f32_32x32x16_f16(ones_of_not_finite(vread(u, 0)), ind[0], f32x16{}, 0, 0, 0);
        t = __builtin_amdgcn_mfma_f32_32x32x16_f16(ones_of_not_finite(vread(u, 1)), ind[1], t, 0, 0, 0);
#pragma unroll
        for (int x = 0; x < 16; x++) o[u][x] = t[x] > 0.0f ? NAN : o[u][x];
        __builtin_amdgcn_sched_barrier(0);
    }
}

}  // namespace
