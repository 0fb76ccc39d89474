// Attention over a layer's KV cache of f16 or q8_0 rows: of a drafted tree of tokens, and with a sliding window and a few
// first keys that stay visible. Head dim 128, any number of q heads to a KV head.
//
//   out[t][h] = Σ_j p_j·v_j / Σ_j p_j,  p_j = e^(scale·q·k_j − m)  over the keys j that query t sees (zeros if none)
//
// The q heads of a KV head share its keys, so a KV head's queries are rows (t, head of the group), packed: row r is query
// r / group. A workgroup takes 32·WR rows and a run of key blocks of 32; its four waves are WR row tiles by KP = 4 / WR
// parts of the blocks, whose sums are merged through LDS. Where the rows are few, the blocks are also split over
// workgroups, whose sums a second launch joins.
//
// On the f16 matrix cores (v_mfma_f32_32x32x16_f16) with f32-grade operands: q and p are pairs of f16 values, 22 bits; K
// and V are f16 (a q8_0 element stands for f16(q·d): rounded once, 2^-11 of it, beside the block's own step of 2^-8 of its
// largest); all sums are f32.
//   q        x = q·scale is rounded to f32 once, and a row is held times 2^(10 − e), e the exponent of its largest, so that
//            the pair neither overflows nor loses bits whatever the row's size; a score is s·c, c = log2(e)·2^(e − 10);
//   scores   Sᵀ = K·(qh + ql)ᵀ: lane 32·hf + c holds row c's scores of keys 8(i / 4) + 4hf + i % 4, i < 16;
//   softmax  p = 2^((s − m)·c + 3): the difference first, so p is right for scores of any size. m, the row's reference, is
//            moved to the largest score only when some p would pass 2^8 (O and l are rescaled then); the 3 leaves room
//            below, and drops out with l, which carries it too;
//   values   Oᵀ += Vᵀ·(ph + pl)ᵀ, V by transposing LDS reads, p straight from the lane's registers.
// A key that a row does not see is as if it were not there, whatever the cache holds in it: its score becomes −∞ after the
// product, and where a block that not every row sees holds a value of V that is not finite (0·∞ is NaN on the matrix
// cores), its products are summed one by one, with those that are not seen left out.
#include <algorithm>
#include <type_traits>

#include "kv_ops.h"
#include "wave.h"

namespace {

constexpr int D = 128, KB = 32;                // head dim; keys a block
constexpr int K_CHUNKS = 512, TILE = 1024;     // 16-byte chunks of a block's K, of its K and V
constexpr float P_SHIFT = 3.0f, P_ROOM = 5.0f; // log2 of the largest p when m moves; its growth before m must move
constexpr float LOG2E = 1.4426950408889634f;
constexpr float M_NONE = -3.0e38f;             // m before the first key: finite, so that s − m is never ∞ − ∞
constexpr int MAX_SPLIT = 64, TICKET = 32;     // parts of a row group's blocks; words between tickets (128 bytes)

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));
typedef int int2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

struct Args {
    const float *q;
    size_t q_stride;
    float *out;
    HtrKvPlanes kv;
    int n, n_head, group;
    float scale;
    int n_past;                // tree: the committed keys
    int pos0, window, n_sink;  // window
    int n_rg, n_split;         // row groups, parts of a row group's key blocks
    float *part;               // [n_kv·n_rg·n_split][32] rows of partial sums o[128], and each row's (m, l)
    uint64_t *part_ml;
    uint32_t *tickets;         // [n_kv·n_rg], TICKET words apart: zero, self-resetting
};
struct TreeMask {
    uint64_t of[HTR_TREE_MAX];
};

// int8 quants → f16(q·d) (as kv_cache.hip's read-back)
__device__ __forceinline__ half2_t dequant2(uint32_t w, uint32_t sel, half2_t d) {
    const uint32_t p = __builtin_amdgcn_perm(0x64646464u, w, sel);
    half2_t h;
    __builtin_memcpy(&h, &p, 4);
    return (h - half2_t{(_Float16)1152.0f, (_Float16)1152.0f}) * d;
}
__device__ __forceinline__ half8 dequant8(uint32_t q0, uint32_t q1, half2_t d) {
    const uint32_t a = q0 ^ 0x80808080u, b = q1 ^ 0x80808080u;
    half2_t r[4] = {dequant2(a, 0x07010700u, d), dequant2(a, 0x07030702u, d), dequant2(b, 0x07010700u, d),
                    dequant2(b, 0x07030702u, d)};
    half8 o;
    __builtin_memcpy(&o, r, 16);
    return o;
}

// the same with a scale a value
__device__ __forceinline__ half8 dequant8(uint32_t q0, uint32_t q1, half8 d) {
    const uint32_t a = q0 ^ 0x80808080u, b = q1 ^ 0x80808080u;
    half2_t r[4] = {dequant2(a, 0x07010700u, half2_t{d[0], d[1]}), dequant2(a, 0x07030702u, half2_t{d[2], d[3]}),
                    dequant2(b, 0x07010700u, half2_t{d[4], d[5]}), dequant2(b, 0x07030702u, half2_t{d[6], d[7]})};
    half8 o;
    __builtin_memcpy(&o, r, 16);
    return o;
}

// 4 bytes a lane from base + off to LDS bytes lds + 4·lane (as lds_load16)
__device__ __forceinline__ void lds_load4(const void *base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(base)
                 : "memory", "m0");
}
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// this wave's LDS reads have their values
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// partial sums between workgroups, through the coherence point
__device__ __forceinline__ void put64(void *p, float a, float b) {
    const uint64_t v = (uint64_t)__float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32;
    __hip_atomic_store((uint64_t *)p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get64(const void *p) {
    const uint64_t v = __hip_atomic_load((const uint64_t *)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// the key blocks that some row of queries ta … tb sees: the blocks 0 … first − 1, then from … to − 1
struct Blocks {
    int first, from, to;
    __device__ __forceinline__ int count() const { return first + max(0, to - from); }
    __device__ __forceinline__ int at(int i) const { return i < first ? i : from + (i - first); }
};
template <bool TREE> __device__ __forceinline__ Blocks blocks_of(const Args &a, int ta, int tb) {
    if constexpr (TREE) {
        return Blocks{0, 0, (a.n_past + a.n + KB - 1) / KB};
    } else {
        const int pa = a.pos0 + ta, pb = a.pos0 + tb, to = pb / KB + 1;
        const int first = min((min(a.n_sink, pb + 1) + KB - 1) / KB, to), lo = a.window > pa ? 0 : (pa - a.window + 1) / KB;
        return Blocks{first, max(first, lo), to};
    }
}

// one lane's row: query t, its head, and the keys it sees; and what every row of its wave's tile of 32 sees
template <bool TREE> struct Row {
    int r, t, head, pos, tile_a, tile_b;
    uint64_t mask;
    __device__ __forceinline__ Row(const Args &a, const TreeMask &tree, int kvh, int r0, int c) {
        const int last = a.n * a.group - 1, rc = min(r0 + c, last);
        r = r0 + c, t = rc / a.group, head = kvh * a.group + rc % a.group, pos = a.pos0 + t;
        tile_a = min(r0, last) / a.group, tile_b = min(r0 + 31, last) / a.group;
        mask = 0;
        if constexpr (TREE) mask = tree.of[t];
    }
    __device__ __forceinline__ bool sees(const Args &a, int key) const {
        if constexpr (TREE) {
            const unsigned j = (unsigned)(key - a.n_past);
            return key < a.n_past || (j < 64u && ((mask >> j) & 1) != 0);
        } else {
            return key <= pos && (key < a.n_sink || key > pos - a.window);
        }
    }
    __device__ __forceinline__ bool all_see(const Args &a, int k0) const {
        if constexpr (TREE) return k0 + KB <= a.n_past;
        else return k0 + KB - 1 <= a.pos0 + tile_a && (k0 + KB <= a.n_sink || k0 > a.pos0 + tile_b - a.window);
    }
};

// a row's q·scale as f16 pairs, the B operand of step ks = dims 16ks + 8hf … + 7; the factor of its scores
__device__ __forceinline__ float q_pairs(const float *qrow, float scale, half8 (&qh)[8], half8 (&ql)[8]) {
    float x[8][8], top = 0.0f;
#pragma unroll
    for (int ks = 0; ks < 8; ks++) {
        const float4 a0 = *reinterpret_cast<const float4 *>(qrow + 16 * ks);
        const float4 a1 = *reinterpret_cast<const float4 *>(qrow + 16 * ks + 4);
        x[ks][0] = a0.x, x[ks][1] = a0.y, x[ks][2] = a0.z, x[ks][3] = a0.w;
        x[ks][4] = a1.x, x[ks][5] = a1.y, x[ks][6] = a1.z, x[ks][7] = a1.w;
    }
#pragma unroll
    for (int ks = 0; ks < 8; ks++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            x[ks][e] *= scale;
            top = fmaxf(top, fabsf(x[ks][e]));
        }
    // (a row of nothing but tiny values: its scores are 0 to f32 either way, and the factor stays a normal number)
    const int ex = max(__builtin_amdgcn_frexp_expf(pair_max<32>(top)), -100);
    const float up = ldexpf(1.0f, 10 - ex);
#pragma unroll
    for (int ks = 0; ks < 8; ks++)
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float y = x[ks][e] * up;
            const _Float16 hi = (_Float16)y;
            qh[ks][e] = hi;
            ql[ks][e] = (_Float16)(y - (float)hi);
        }
    return ldexpf(LOG2E, ex - 10);
}

// ---- few rows: the blocks split over workgroups ----------------------------------------------------------------------------
//
// A workgroup takes 32 rows, each of its four waves every fourth block of its part. A wave loads its own blocks straight
// into LDS of its own, so the waves wait for nobody until their sums are merged; f16 blocks with one buffer for K and one
// for V, each filled again as soon as it is read (K under the softmax and the values, V under the next scores), q8_0 blocks,
// half the size, with two, raw: a fragment's 8 quants become f16 in the registers of the one wave that uses them (7 VALU
// instructions an operand register; V's by a transposing read of bytes).
//   f16   K and V [32 keys][16 chunks of 16 bytes], row r's chunk c at 16r + (c ^ r % 16), V's at 16r + (c ^ 2(r % 8));
//   q8_0  K and V [32 keys][8 chunks], row r's chunk c at 8r + (c ^ r / 2 % 8); their scales [32 keys][4]; V's once more
//         as [dims / 32][key / 16][hf][8], the order of an operand's slots.
// Reads of 16 (32) lanes then fall on different bank groups.
constexpr int QT = 256 + 256 + 16 + 16;  // 16-byte chunks of a q8_0 buffer: K, V, K scales, V scales

template <bool Q8, bool TREE> __global__ __launch_bounds__(256, 2) void k_kv_attn_split(Args a, TreeMask tree) {
    constexpr int WAVE = Q8 ? 2 * QT + 16 : TILE;  // chunks of a wave's LDS
    __shared__ __attribute__((aligned(16))) uint4_t s_kv[4][WAVE];
    __shared__ float s_p[4][KB / 2][KB];  // weights, where they are summed one by one
    __shared__ float s_ml[4][2][KB];
    __shared__ float s_c[KB];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hf = lane >> 5, c = lane & 31;
    const int kvh = blockIdx.x % a.kv.n_kv, rest = blockIdx.x / a.kv.n_kv;
    const int split = rest % a.n_split, rg = rest / a.n_split;
    const int rows = a.n * a.group, r0 = rg * KB;
    const int n_keys = TREE ? a.n_past + a.n : a.pos0 + a.n;
    const Blocks blk = blocks_of<TREE>(a, r0 / a.group, min(r0 + KB - 1, rows - 1) / a.group);
    const int nb = blk.count(), i0 = (int)((int64_t)nb * split / a.n_split), i1 = (int)((int64_t)nb * (split + 1) / a.n_split);
    const size_t head0 = (size_t)kvh * a.kv.n_ctx;

    uint4_t *tile = s_kv[wave];
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4_t *)tile;
    const uint32_t kx = 16 * ((lane & 15) ^ (lane >> 4)), vx = 16 * ((lane & 15) ^ (2 * (lane >> 4)));
    const uint32_t bx = 16 * ((lane & 7) ^ (lane >> 4));
    // block i's K or V (f16), or all of it into buffer b (q8_0); rows past the last key are the last key's, and are masked
    auto load = [&](int i, bool is_v) {
        const int k0 = KB * blk.at(i);
        const char *base = (const char *)(is_v ? a.kv.v : a.kv.k) + (head0 + k0) * (2 * D);
        const uint32_t last = min(n_keys - 1 - k0, KB - 1);
#pragma unroll
        for (int u = 0; u < 8; u++)
            lds_load16(base, 2 * D * min((uint32_t)(4 * u + (lane >> 4)), last) + (is_v ? vx ^ (128 * (u & 1)) : kx ^ (64 * (u & 3))),
                       lds + 16 * ((is_v ? K_CHUNKS : 0) + 64 * u));
    };
    auto load_q8 = [&](int i, int b) {
        const int k0 = KB * blk.at(i);
        const size_t row = head0 + k0;
        const uint32_t last = min(n_keys - 1 - k0, KB - 1), to = lds + 16 * QT * b;
        lds_load4(a.kv.kd + row * 4, 8 * min((uint32_t)lane >> 1, last) + 4 * (lane & 1), to + 16 * 512);
        lds_load4(a.kv.vd + row * 4, 8 * min((uint32_t)lane >> 1, last) + 4 * (lane & 1), to + 16 * 528);
#pragma unroll
        for (int u = 0; u < 8; u++)
            lds_load16((const char *)(u < 4 ? a.kv.k : a.kv.v) + row * D,
                       D * min((uint32_t)(8 * (u & 3) + (lane >> 3)), last) + (bx ^ (64 * (u & 1))), to + 16 * 64 * u);
    };
    int i = i0 + wave;
    if (i < i1) {
        if constexpr (Q8) {
            load_q8(i, 0);
        } else {
            load(i, false);
            load(i, true);
        }
    }

    const Row<TREE> row(a, tree, kvh, r0, c);
    half8 qh[8], ql[8];
    const float sc = q_pairs(a.q + (size_t)row.t * a.q_stride + (size_t)row.head * D + 8 * hf, a.scale, qh, ql);

    // the lane's places in a block: K step ks is key c, dims 16ks + 8hf …; V tile u, step ss, slots 8hf … + 7 are the keys
    // 16ss + 4hf … + 3, then 16ss + 8 + 4hf … + 3 (the lane's scores 8ss …) of dims 32u + 16(lane / 16 % 2) …
    const int vrow = Q8 ? 8 * ((lane >> 3) & 1) + 4 * hf + ((lane >> 1) & 3) : 4 * hf + ((lane & 15) >> 2);
    int va[4];
#pragma unroll
    for (int u = 0; u < 4; u++)
        va[u] = Q8 ? 16 * (256 + 8 * vrow + ((2 * u + ((lane >> 4) & 1)) ^ (vrow >> 1))) + 8 * (lane & 1)
                   : 16 * (K_CHUNKS + 16 * vrow + ((4 * u + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ (2 * vrow))) + 8 * (lane & 1);

    f32x16 o[4];
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
        for (int x = 0; x < 16; x++) o[u][x] = 0.0f;
    float m = M_NONE, l = 0.0f;

    for (int b = 0; i < i1; i += 4, b ^= Q8) {
        const bool more = i + 4 < i1;
        uint4_t *buf = tile + (Q8 ? QT * b : 0);
        if constexpr (Q8) {
            if (more) {
                wait_reads();  // of the other buffer, a block ago
                load_q8(i + 4, b ^ 1);
                wait_loads<10>();
            } else {
                wait_loads<0>();
            }
        } else {
            wait_loads<8>();  // K; V is still on its way
        }
        f32x16 s;
        if constexpr (Q8) {
            // V's scales into the order of the operands' slots
            const uint32_t d2 = reinterpret_cast<const uint32_t *>(buf + 528)[lane];
            uint16_t *vt = reinterpret_cast<uint16_t *>(tile + 2 * QT);
            const int key = lane >> 1, at = 16 * (key >> 4) + 8 * ((key >> 2) & 1) + 4 * ((key >> 3) & 1) + (key & 3);
            vt[32 * (2 * (lane & 1)) + at] = (uint16_t)d2;
            vt[32 * (2 * (lane & 1) + 1) + at] = (uint16_t)(d2 >> 16);
            const uint2_t dk = reinterpret_cast<const uint2_t *>(buf + 512)[c];
            half2_t d4[2];
            __builtin_memcpy(d4, &dk, 8);
#pragma unroll
            for (int ks = 0; ks < 8; ks++) {
                const uint2_t w = *reinterpret_cast<const uint2_t *>((const char *)(buf + 8 * c + (ks ^ ((c >> 1) & 7))) + 8 * hf);
                const _Float16 d = d4[ks >> 2][(ks >> 1) & 1];
                const half8 f = dequant8(w[0], w[1], half2_t{d, d});
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, qh[ks], ks ? s : f32x16{}, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, ql[ks], s, 0, 0, 0);
            }
        } else {
            half8 f[4];
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int ks = 0; ks < 4; ks++) f[ks] = *reinterpret_cast<const half8 *>(buf + 16 * c + ((8 * h + 2 * ks + hf) ^ (c & 15)));
                if (h == 1) {
                    wait_reads();
                    if (more) load(i + 4, false);
                }
#pragma unroll
                for (int ks = 0; ks < 4; ks++) {
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[ks], qh[4 * h + ks], h || ks ? s : f32x16{}, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[ks], ql[4 * h + ks], s, 0, 0, 0);
                }
            }
        }
        const int k0 = KB * blk.at(i);
        const bool full = row.all_see(a, k0);
        uint32_t seen = 0xffffu;
        if (!full) {
            seen = 0;
#pragma unroll
            for (int x = 0; x < 16; x++) {
                const bool v = row.sees(a, k0 + 8 * (x >> 2) + 4 * hf + (x & 3));
                seen |= (uint32_t)v << x;
                s[x] = v ? s[x] : -INFINITY;
            }
        }
        float mx = s[0];
#pragma unroll
        for (int x = 1; x < 16; x++) mx = fmaxf(mx, s[x]);
        mx = pair_max<32>(mx);
        if (__builtin_amdgcn_ballot_w64((mx - m) * sc > P_ROOM)) {
            const float to = fmaxf(m, mx), corr = __builtin_amdgcn_exp2f((m - to) * sc);
            m = to;
            l *= corr;
#pragma unroll
            for (int u = 0; u < 4; u++) o[u] *= corr;
        }
        float ls = 0.0f;
        half8 ph[2], pl[2];
#pragma unroll
        for (int x = 0; x < 16; x++) {
            s[x] = __builtin_amdgcn_exp2f(fmaf(s[x] - m, sc, P_SHIFT));  // not seen: 2^(−∞) = 0
            ls += s[x];
            const _Float16 hi = (_Float16)s[x];
            ph[x >> 3][x & 7] = hi;
            pl[x >> 3][x & 7] = (_Float16)(s[x] - (float)hi);
        }
        l += ls;
        if constexpr (!Q8) {  // V
            if (more) wait_loads<8>();
            else wait_loads<0>();
        }
        bool odd = false;  // a value of V that is not finite (or a scale that may make one)
        if (!full) {
            uint32_t any = 0;
            if constexpr (Q8) {
                const uint32_t w = reinterpret_cast<const uint32_t *>(buf + 528)[lane];
                any = (w & 0x7FFFu) > 0x6007u || (w >> 16 & 0x7FFFu) > 0x6007u;  // past 515.5
            } else {
#pragma unroll 2
                for (int u = 0; u < 8; u++) {
                    const uint4_t w = buf[K_CHUNKS + 64 * u + lane];
#pragma unroll
                    for (int e = 0; e < 4; e++) any |= (w[e] & 0x7C00u) == 0x7C00u || (w[e] & 0x7C000000u) == 0x7C000000u;
                }
            }
            odd = __builtin_amdgcn_ballot_w64(any != 0) != 0;
        }
        if (!odd) {
#pragma unroll
            for (int ss = 0; ss < 2; ss++)
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    half8 v;
                    if constexpr (Q8) {
                        const auto *p = (const __attribute__((address_space(3))) char *)buf + va[u] + 16 * 128 * ss;
                        const int2_t w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) int2_t *)p);
                        const half8 d = *reinterpret_cast<const half8 *>(tile + 2 * QT + 4 * u + 2 * ss + hf);
                        v = dequant8((uint32_t)w[0], (uint32_t)w[1], d);
                    } else {
                        const auto *p = (const __attribute__((address_space(3))) char *)buf + va[u] + 256 * 16 * ss;
                        const fp16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)p);
                        const fp16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)(p + 256 * 8));
                        __builtin_memcpy(&v, &lo, 8);
                        __builtin_memcpy((char *)&v + 8, &up, 8);
                    }
                    o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[ss], o[u], 0, 0, 0);
                    o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl[ss], o[u], 0, 0, 0);
                }
        } else {
            // 16 keys' weights to LDS (−1: not seen), then key by key; the lane sums row c's dims 32u + 8(x / 4) + 4hf + x % 4
#pragma unroll 1
            for (int half = 0; half < 2; half++) {
#pragma unroll
                for (int x = 0; x < 8; x++)
                    s_p[wave][8 * (x >> 2) + 4 * hf + (x & 3)][c] = (seen >> (8 * half + x)) & 1 ? (half ? s[8 + x] : s[x]) : -1.0f;
                wait_reads();
#pragma unroll 1
                for (int k = 0; k < KB / 2; k++) {
                    const int key = KB / 2 * half + k;
                    const float p = s_p[wave][k][c];
                    const bool v = !(p < 0.0f);
#pragma unroll
                    for (int u = 0; u < 4; u++)
#pragma unroll
                        for (int x = 0; x < 16; x++) {
                            const int dim = 32 * u + 8 * (x >> 2) + 4 * hf + (x & 3);
                            float w;
                            if constexpr (Q8) {
                                const int8_t q = reinterpret_cast<const int8_t *>(buf + 256 + 8 * key + ((dim >> 4) ^ ((key >> 1) & 7)))[dim & 15];
                                w = (float)((_Float16)(float)q * reinterpret_cast<const _Float16 *>(buf + 528)[4 * key + u]);
                            } else {
                                w = (float)reinterpret_cast<const _Float16 *>(buf + K_CHUNKS + 16 * key + ((dim >> 3) ^ (2 * (key & 7))))[dim & 7];
                            }
                            o[u][x] = v ? fmaf(p, w, o[u][x]) : o[u][x];
                            if ((x & 3) == 3) __builtin_amdgcn_sched_barrier(0);  // (few values in registers at once)
                        }
                }
                wait_reads();
            }
        }
        if constexpr (!Q8) {
            wait_reads();
            if (more) load(i + 4, true);
        }
    }
    l = pair_sum<32>(l);

    // the waves' sums through LDS (each its own tile's place): wave u finishes dims 32u … of every row
    wait_reads();
    float4 *so = reinterpret_cast<float4 *>(tile);
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
        for (int x = 0; x < 4; x++)
            so[(4 * u + x) * 64 + lane] = make_float4(o[u][4 * x], o[u][4 * x + 1], o[u][4 * x + 2], o[u][4 * x + 3]);
    if (hf == 0) s_ml[wave][0][c] = m, s_ml[wave][1][c] = l;
    if (wave == 0 && hf == 0) s_c[c] = sc;
    __syncthreads();
    m = fmaxf(fmaxf(s_ml[0][0][c], s_ml[1][0][c]), fmaxf(s_ml[2][0][c], s_ml[3][0][c]));
    l = 0.0f;
    float4 v[4];
#pragma unroll
    for (int x = 0; x < 4; x++) v[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const float w = __builtin_amdgcn_exp2f((s_ml[p][0][c] - m) * sc);
        l = fmaf(s_ml[p][1][c], w, l);
        const float4 *from = reinterpret_cast<const float4 *>(s_kv[p]) + 4 * 64 * wave + lane;
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const float4 y = from[64 * x];
            v[x].x = fmaf(y.x, w, v[x].x), v[x].y = fmaf(y.y, w, v[x].y);
            v[x].z = fmaf(y.z, w, v[x].z), v[x].w = fmaf(y.w, w, v[x].w);
        }
    }
    if (a.n_split == 1) {
        if (row.r >= rows) return;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key seen: zeros
        float *orow = a.out + ((size_t)row.t * a.n_head + row.head) * D + 32 * wave + 4 * hf;
#pragma unroll
        for (int x = 0; x < 4; x++)
            *reinterpret_cast<float4 *>(orow + 8 * x) = make_float4(v[x].x * inv, v[x].y * inv, v[x].z * inv, v[x].w * inv);
        return;
    }

    // the part's sums to memory; the last workgroup of the row group to get there joins them
    const size_t g0 = ((size_t)kvh * a.n_rg + rg) * a.n_split * KB;  // the row group's first row of partial sums
    if (row.r < rows) {
        const size_t pr = g0 + (size_t)split * KB + c;
        float *prow = a.part + pr * D + 32 * wave + 4 * hf;
#pragma unroll
        for (int x = 0; x < 4; x++) {
            put64(prow + 8 * x, v[x].x, v[x].y);
            put64(prow + 8 * x + 2, v[x].z, v[x].w);
        }
        if (wave == 0 && hf == 0) put64(a.part_ml + pr, m, l);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this thread's stores are performed
    __syncthreads();
    uint32_t *ticket = a.tickets + TICKET * ((size_t)kvh * a.n_rg + rg);
    if (tid == 0)
        s_last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(a.n_split - 1);
    __syncthreads();
    if (!s_last) return;
    const int nr = min(KB, rows - r0), ns = a.n_split;
    float2 *s_w = reinterpret_cast<float2 *>(&s_kv[0][0]);  // [row][part]: (m, l), then (weight, l)
    for (int id = tid; id < KB * MAX_SPLIT; id += 256) {
        const int r = id / MAX_SPLIT, p = id % MAX_SPLIT;
        if (r < nr && p < ns) s_w[id] = get64(a.part_ml + g0 + (size_t)p * KB + r);
    }
    __syncthreads();
    {
        const int r = tid >> 3, p0 = tid & 7;
        float top = M_NONE, sum = 0.0f;
        if (r < nr)
            for (int p = p0; p < ns; p += 8) top = fmaxf(top, s_w[MAX_SPLIT * r + p].x);
        top = group_max<4>(top, lane);
        if (r < nr)
            for (int p = p0; p < ns; p += 8) {
                const float2 ml = s_w[MAX_SPLIT * r + p];
                const float w = __builtin_amdgcn_exp2f((ml.x - top) * s_c[r]);
                sum = fmaf(ml.y, w, sum);
                s_w[MAX_SPLIT * r + p].x = w;
            }
        sum = group_sum<4>(sum, lane);
        if (p0 == 0) s_ml[0][0][r] = sum == 0.0f ? 0.0f : 1.0f / sum;
    }
    __syncthreads();
    // 32 threads of 4 dims a row; rows fewer than 8: a row's parts to 2, 4 or 8 such groups
    const int gr = tid >> 5, d4 = tid & 31, lg = nr > 4 ? 3 : nr > 2 ? 2 : nr > 1 ? 1 : 0, groups = 8 >> lg;
    float4 *s_g = reinterpret_cast<float4 *>(s_w + KB * MAX_SPLIT);
    for (int rb = 0; rb < nr; rb += 1 << lg) {
        const int r = min(rb + (gr & ((1 << lg) - 1)), nr - 1), g = gr >> lg;
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const float *from = a.part + (g0 + r) * D + 4 * d4;
        for (int p = g; p < ns; p += 8 * groups) {
            float2 in[8][2];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float *at = from + (size_t)min(p + e * groups, ns - 1) * (KB * D);
                in[e][0] = get64(at), in[e][1] = get64(at + 2);
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float w = p + e * groups < ns ? s_w[MAX_SPLIT * r + p + e * groups].x : 0.0f;
                y.x = fmaf(in[e][0].x, w, y.x), y.y = fmaf(in[e][0].y, w, y.y);
                y.z = fmaf(in[e][1].x, w, y.z), y.w = fmaf(in[e][1].y, w, y.w);
            }
        }
        if (groups > 1) {
            s_g[tid] = y;
            __syncthreads();
            if (g == 0)
                for (int e = 1; e < groups; e++) {
                    const float4 z = s_g[tid + 32 * (e << lg)];
                    y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
                }
        }
        if (g == 0 && rb + (gr & ((1 << lg) - 1)) < nr) {
            const float inv = s_ml[0][0][r];
            const int t = (r0 + r) / a.group, head = kvh * a.group + (r0 + r) % a.group;
            *reinterpret_cast<float4 *>(a.out + ((size_t)t * a.n_head + head) * D + 4 * d4) =
                make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
        }
    }
    if (tid == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
}

// ---- many rows ---------------------------------------------------------------------------------------------------------------

template <bool Q8, bool TREE, int WR>
__global__ __launch_bounds__(256) void k_kv_attn(Args a, TreeMask tree) {
    constexpr int KP = 4 / WR;
    __shared__ __attribute__((aligned(16))) uint4_t s_kv[KP][TILE];  // K, then V
    __shared__ float s_p[4][KB][KB];                                 // the weights, where they are summed one by one
    __shared__ float s_ml[4][2][KB];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hf = lane >> 5, c = lane & 31, rt = wave % WR, kp = wave / WR;
    const int kvh = blockIdx.x % a.kv.n_kv, rest = blockIdx.x / a.kv.n_kv;
    const int split = rest % a.n_split, rg = a.n_rg - 1 - rest / a.n_split;
    const int rows = a.n * a.group, r0 = rg * 32 * WR, r = r0 + 32 * rt + c, rc = min(r, rows - 1);
    const int t = rc / a.group, head = kvh * a.group + rc % a.group;
    const int n_keys = TREE ? a.n_past + a.n : a.pos0 + a.n;

    // the row's keys, and those that every row of the wave's tile sees
    const int qpos = a.pos0 + t;
    uint64_t mask = 0;
    if constexpr (TREE) mask = tree.of[t];
    const int tile_a = min(r0 + 32 * rt, rows - 1) / a.group, tile_b = min(r0 + 32 * rt + 31, rows - 1) / a.group;
    auto all_see = [&](int k0) {
        if constexpr (TREE) return k0 + KB <= a.n_past;
        else return k0 + KB - 1 <= a.pos0 + tile_a && (k0 + KB <= a.n_sink || k0 > a.pos0 + tile_b - a.window);
    };
    auto sees = [&](int key) {
        if constexpr (TREE) {
            const unsigned j = (unsigned)(key - a.n_past);
            return key < a.n_past || (j < 64u && ((mask >> j) & 1) != 0);
        } else {
            return key <= qpos && (key < a.n_sink || key > qpos - a.window);
        }
    };

    const Blocks blk = blocks_of<TREE>(a, r0 / a.group, min(r0 + 32 * WR - 1, rows - 1) / a.group);
    const int nb = blk.count(), i0 = (int)((int64_t)nb * split / a.n_split), i1 = (int)((int64_t)nb * (split + 1) / a.n_split);

    // q·scale as f16 pairs: B operand of step ks = dims 16ks + 8hf … + 7 of row c
    half8 qh[8], ql[8];
    float sc;
    {
        const float *qrow = a.q + (size_t)t * a.q_stride + (size_t)head * D + 8 * hf;
        float x[8][8], top = 0.0f;
#pragma unroll
        for (int ks = 0; ks < 8; ks++) {
            const float4 a0 = *reinterpret_cast<const float4 *>(qrow + 16 * ks);
            const float4 a1 = *reinterpret_cast<const float4 *>(qrow + 16 * ks + 4);
            x[ks][0] = a0.x, x[ks][1] = a0.y, x[ks][2] = a0.z, x[ks][3] = a0.w;
            x[ks][4] = a1.x, x[ks][5] = a1.y, x[ks][6] = a1.z, x[ks][7] = a1.w;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[ks][e] *= a.scale;
                top = fmaxf(top, fabsf(x[ks][e]));
            }
        }
        // (a row of nothing but tiny values: its scores are 0 to f32 either way, and c stays a normal number)
        const int ex = max(__builtin_amdgcn_frexp_expf(pair_max<32>(top)), -100);
        sc = ldexpf(LOG2E, ex - 10);
#pragma unroll
        for (int ks = 0; ks < 8; ks++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float y = ldexpf(x[ks][e], 10 - ex);
                const _Float16 hi = (_Float16)y;
                qh[ks][e] = hi;
                ql[ks][e] = (_Float16)(y - (float)hi);
            }
    }
    // the lane's fragment slots in a block (K row r's 16-byte chunk c is at 16r + (c ^ r % 16), V's at 16r + (c ^ 2(r % 8)):
    // the reads of 16 lanes fall on different bank groups): K step ks (key c, dims 16ks + 8hf …), V tile u (16-lane group:
    // dims 32u + 16(lane / 16 % 2) …, keys 4hf + (lane % 16) / 4 of each group of 8)
    int ka[8], va[4];
#pragma unroll
    for (int ks = 0; ks < 8; ks++) ka[ks] = 16 * c + ((2 * ks + hf) ^ (c & 15));
    const int vrow = 4 * hf + ((lane & 15) >> 2);
#pragma unroll
    for (int u = 0; u < 4; u++)
        va[u] = 16 * (K_CHUNKS + 16 * vrow + ((4 * u + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ (2 * vrow))) + 8 * (lane & 1);

    f32x16 o[4];
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[u][i] = 0.0f;
    float m = M_NONE, l = 0.0f;

    const int n_stage = (i1 - i0 + KP - 1) / KP;
    const int lt = rt * 64 + lane;  // the thread among those that load the part's block
    for (int st = 0; st < n_stage; st++) {
        const int i = i0 + st * KP + kp;
        const bool live = i < i1;
        const int k0 = KB * blk.at(min(i, i1 - 1));
        // K and V → LDS (rows past the last key are the last key's, and are masked)
        if constexpr (Q8) {
#pragma unroll
            for (int u = 0; u < 8 / WR; u++) {
                const int id = lt + 64 * WR * u, is_v = id >> 8, row = (id >> 3) & 31, ch = id & 7;
                const size_t at = (size_t)kvh * a.kv.n_ctx + min(k0 + row, n_keys - 1);
                const uint4_t w = *reinterpret_cast<const uint4_t *>((const char *)(is_v ? a.kv.v : a.kv.k) + at * D + 16 * ch);
                const uint16_t db = (is_v ? a.kv.vd : a.kv.kd)[at * 4 + (ch >> 1)];
                _Float16 d;
                __builtin_memcpy(&d, &db, 2);
                const int sw = is_v ? 2 * (row & 7) : row & 15;
                uint4_t *to = s_kv[kp] + (is_v ? K_CHUNKS : 0) + 16 * row;
                *reinterpret_cast<half8 *>(to + ((2 * ch) ^ sw)) = dequant8(w[0], w[1], half2_t{d, d});
                *reinterpret_cast<half8 *>(to + ((2 * ch + 1) ^ sw)) = dequant8(w[2], w[3], half2_t{d, d});
            }
        } else {
#pragma unroll
            for (int u = 0; u < 16 / WR; u++) {
                const int id = lt + 64 * WR * u, is_v = id >> 9, row = (id >> 4) & 31, ch = id & 15;
                const size_t at = (size_t)kvh * a.kv.n_ctx + min(k0 + row, n_keys - 1);
                const uint4_t w = *reinterpret_cast<const uint4_t *>((const char *)(is_v ? a.kv.v : a.kv.k) + at * (2 * D) + 16 * ch);
                s_kv[kp][(is_v ? K_CHUNKS : 0) + 16 * row + (ch ^ (is_v ? 2 * (row & 7) : row & 15))] = w;
            }
        }
        __syncthreads();
        if (live) {
            f32x16 s;
#pragma unroll
            for (int ks = 0; ks < 8; ks++) {
                const half8 f = *reinterpret_cast<const half8 *>(s_kv[kp] + ka[ks]);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, qh[ks], ks ? s : f32x16{}, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, ql[ks], s, 0, 0, 0);
            }
            const bool full = all_see(k0);
            uint32_t seen = 0xffffu;
            if (!full) {
                seen = 0;
#pragma unroll
                for (int x = 0; x < 16; x++) {
                    const bool v = sees(k0 + 8 * (x >> 2) + 4 * hf + (x & 3));
                    seen |= (uint32_t)v << x;
                    s[x] = v ? s[x] : -INFINITY;
                }
            }
            float mx = s[0];
#pragma unroll
            for (int x = 1; x < 16; x++) mx = fmaxf(mx, s[x]);
            mx = pair_max<32>(mx);
            if (__builtin_amdgcn_ballot_w64((mx - m) * sc > P_ROOM)) {
                const float to = fmaxf(m, mx), corr = __builtin_amdgcn_exp2f((m - to) * sc);
                m = to;
                l *= corr;
#pragma unroll
                for (int u = 0; u < 4; u++) o[u] *= corr;
            }
            float ls = 0.0f;
#pragma unroll
            for (int x = 0; x < 16; x++) {
                s[x] = __builtin_amdgcn_exp2f(fmaf(s[x] - m, sc, P_SHIFT));  // not seen: 2^(−∞) = 0
                ls += s[x];
            }
            l += ls;
            bool odd = false;
            if (!full) {
                uint32_t any = 0;
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    const uint4_t w = s_kv[kp][K_CHUNKS + 64 * u + lane];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        any |= (w[e] & 0x7C00u) == 0x7C00u;
                        any |= (w[e] & 0x7C000000u) == 0x7C000000u;
                    }
                }
                odd = __builtin_amdgcn_ballot_w64(any != 0) != 0;
            }
            if (!odd) {
                half8 ph[2], pl[2];
#pragma unroll
                for (int x = 0; x < 16; x++) {
                    const _Float16 hi = (_Float16)s[x];
                    ph[x >> 3][x & 7] = hi;
                    pl[x >> 3][x & 7] = (_Float16)(s[x] - (float)hi);
                }
                const auto *vb = (const __attribute__((address_space(3))) char *)s_kv[kp];
#pragma unroll
                for (int ss = 0; ss < 2; ss++)
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        // slots 8hf … + 7 are keys 16ss + 4hf … + 3, then 16ss + 8 + 4hf … + 3: the lane's scores 8ss …
                        const auto *p = vb + va[u] + 256 * 16 * ss;
                        const fp16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)p);
                        const fp16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)(p + 256 * 8));
                        half8 v;
                        __builtin_memcpy(&v, &lo, 8);
                        __builtin_memcpy((char *)&v + 8, &up, 8);
                        o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[ss], o[u], 0, 0, 0);
                        o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl[ss], o[u], 0, 0, 0);
                    }
            } else {
                // the weights to LDS (−1: not seen), then key by key; lane 32hf + c sums row c's dims 32u + 8(x / 4) + 4hf + x % 4
#pragma unroll
                for (int x = 0; x < 16; x++)
                    s_p[wave][8 * (x >> 2) + 4 * hf + (x & 3)][c] = (seen >> x) & 1 ? s[x] : -1.0f;
                __builtin_amdgcn_wave_barrier();
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                const _Float16 *vt = reinterpret_cast<const _Float16 *>(s_kv[kp] + K_CHUNKS);
#pragma unroll 1
                for (int key = 0; key < KB; key++) {
                    const float p = s_p[wave][key][c];
                    const bool v = !(p < 0.0f);
#pragma unroll
                    for (int u = 0; u < 4; u++)
#pragma unroll
                        for (int x = 0; x < 16; x++) {
                            const int dim = 32 * u + 8 * (x >> 2) + 4 * hf + (x & 3);
                            const float w = (float)vt[8 * (16 * key + ((dim >> 3) ^ (2 * (key & 7)))) + (dim & 7)];
                            o[u][x] = v ? fmaf(p, w, o[u][x]) : o[u][x];
                        }
                }
            }
        }
        __syncthreads();
    }
    l = pair_sum<32>(l);

    // the parts' sums through LDS, tile by tile of 32 dims: wave (rt, kp) leaves its tile u, then every wave adds its share
    // (8 / KP … of the tile's dims) of its row tile's rows
    if constexpr (KP > 1) {
        if (hf == 0) s_ml[wave][0][c] = m, s_ml[wave][1][c] = l;
        __syncthreads();
        float w[KP], lsum = 0.0f, top = M_NONE;
#pragma unroll
        for (int p = 0; p < KP; p++) top = fmaxf(top, s_ml[p * WR + rt][0][c]);
#pragma unroll
        for (int p = 0; p < KP; p++) {
            w[p] = __builtin_amdgcn_exp2f((s_ml[p * WR + rt][0][c] - top) * sc);
            lsum = fmaf(s_ml[p * WR + rt][1][c], w[p], lsum);
        }
        m = top, l = lsum;
        const float mine = w[kp];
        float *s_o = reinterpret_cast<float *>(&s_kv[0][0]);  // [wave][register][lane], one dim tile at a time
#pragma unroll
        for (int u = 0; u < 4; u++) {
#pragma unroll
            for (int x = 0; x < 16; x++) s_o[(wave * 16 + x) * 64 + lane] = o[u][x] * mine;
            __syncthreads();
#pragma unroll
            for (int x = 0; x < 16; x++) {
                float v = 0.0f;
#pragma unroll
                for (int p = 0; p < KP; p++) v += s_o[((p * WR + rt) * 16 + x) * 64 + lane];
                o[u][x] = v;
            }
            __syncthreads();
        }
    }
    if (kp != 0 || r >= rows) return;
    {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key seen: zeros
        float *orow = a.out + ((size_t)t * a.n_head + head) * D + 4 * hf;
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int x = 0; x < 4; x++)
                *reinterpret_cast<float4 *>(orow + 32 * u + 8 * x) =
                    make_float4(o[u][4 * x] * inv, o[u][4 * x + 1] * inv, o[u][4 * x + 2] * inv, o[u][4 * x + 3] * inv);
    }
}

template <bool TREE> int launch(htr_device *dev, Args &a, const TreeMask &tree, int max_blocks) {
    const int rows = a.n * a.group;
    const int64_t groups = (int64_t)((rows + KB - 1) / KB) * a.kv.n_kv;
    if (groups >= 2 * dev->n_cu) {
        constexpr int WR = 4;
        a.n_rg = (rows + KB * WR - 1) / (KB * WR), a.n_split = 1;
        const int64_t wide = (int64_t)a.n_rg * a.kv.n_kv;
        if (wide > INT32_MAX) return htr_fail("attention: %d rows of %d KV heads", rows, a.kv.n_kv);
        if (a.kv.q8) hipLaunchKernelGGL((k_kv_attn<true, TREE, WR>), dim3((unsigned)wide), dim3(256), 0, dev->stream, a, tree);
        else hipLaunchKernelGGL((k_kv_attn<false, TREE, WR>), dim3((unsigned)wide), dim3(256), 0, dev->stream, a, tree);
        return htr_launched(dev, "k_kv_attn");
    }
    a.n_rg = (rows + KB - 1) / KB;
    // two workgroups a CU, no more parts than a wave has blocks
    a.n_split = (int)std::max<int64_t>(1, std::min<int64_t>({2 * dev->n_cu / groups, (max_blocks + 3) / 4, MAX_SPLIT}));
    if (a.n_split > 1) {
        void *p;
        HTR_TRY(htr_scratch(dev, SCR_KV_TICKET, (size_t)2 * dev->n_cu * TICKET * 4, &p));
        a.tickets = (uint32_t *)p;
        HTR_TRY(htr_scratch(dev, SCR_KV_ATTN, (size_t)2 * dev->n_cu * KB * (D + 2) * 4, &p));
        a.part = (float *)p;
        a.part_ml = (uint64_t *)(a.part + (size_t)2 * dev->n_cu * KB * D);
    }
    const dim3 g((unsigned)(groups * a.n_split)), b(256);
    if (a.kv.q8) hipLaunchKernelGGL((k_kv_attn_split<true, TREE>), g, b, 0, dev->stream, a, tree);
    else hipLaunchKernelGGL((k_kv_attn_split<false, TREE>), g, b, 0, dev->stream, a, tree);
    return htr_launched(dev, "k_kv_attn_split");
}

int check_rows(const char *me, const float *d_q, size_t q_stride, const htr_kv *kv, int n_head, float *d_out, int64_t n) {
    if (!d_q || !d_out) return htr_fail("%s: null argument", me);
    if (n_head < 1 || n_head % kv->n_kv) return htr_fail("%s: %d q heads on %d KV heads", me, n_head, kv->n_kv);
    const size_t qd = (size_t)n_head * D;
    if (q_stride < qd || (q_stride & 3))
        return htr_fail("%s: rows %zu floats apart (a multiple of 4, at least %zu)", me, q_stride, qd);
    if (((uintptr_t)d_q | (uintptr_t)d_out) & 15) return htr_fail("%s: pointers must be 16-byte aligned", me);
    if (n * (n_head / kv->n_kv) > (1 << 30)) return htr_fail("%s: %lld queries of %d heads", me, (long long)n, n_head);
    const uintptr_t q0 = (uintptr_t)d_q, q1 = q0 + 4 * (q_stride * (n - 1) + qd), o0 = (uintptr_t)d_out, o1 = o0 + 4 * qd * n;
    if (q0 < o1 && o0 < q1) return htr_fail("%s: the output overlaps the queries", me);
    return 0;
}

}  // namespace

// ---- ABI -----------------------------------------------------------------------------------------------------------------

extern "C" int htr_tree_attention(htr_device *dev, const float *d_q, size_t q_stride, int n, const uint64_t *h_mask,
                                  int n_past, const htr_kv *kv, int n_head, float scale, float *d_out) {
    const char *me = "htr_tree_attention";
    Args a{};
    HTR_TRY(htr_kv_check(me, kv, &a.kv));
    if (n < 1 || n > HTR_TREE_MAX) return htr_fail("%s: %d nodes (1 … %d)", me, n, HTR_TREE_MAX);
    if (n_past < 0 || n_past > kv->n_ctx - n)
        return htr_fail("%s: %d keys and %d nodes in a %d-row cache", me, n_past, n, kv->n_ctx);
    HTR_TRY(check_rows(me, d_q, q_stride, kv, n_head, d_out, n));
    TreeMask tree{};
    const uint64_t all = n == 64 ? ~0ull : (1ull << n) - 1;
    for (int t = 0; t < n; t++) {
        tree.of[t] = h_mask ? h_mask[t] : (t == 63 ? ~0ull : (2ull << t) - 1);
        if (tree.of[t] & ~all)
            return htr_fail("%s: node %d's mask 0x%llx has bits past the %d nodes", me, t, (unsigned long long)tree.of[t], n);
    }
    HTR_TRY(htr_check_alive(dev));
    const HtrOnDevice on(dev);
    a.q = d_q, a.q_stride = q_stride, a.out = d_out, a.n = n, a.n_head = n_head, a.group = n_head / kv->n_kv;
    a.scale = scale, a.n_past = n_past;
    return launch<true>(dev, a, tree, (n_past + n + KB - 1) / KB);
}

extern "C" int htr_window_attention(htr_device *dev, const float *d_q, size_t q_stride, int n_q, int pos0, int window,
                                    int n_sink, const htr_kv *kv, int n_head, float scale, float *d_out) {
    const char *me = "htr_window_attention";
    Args a{};
    HTR_TRY(htr_kv_check(me, kv, &a.kv));
    if (n_q < 1 || pos0 < 0 || pos0 > kv->n_ctx - n_q)
        return htr_fail("%s: %d queries from position %d in a %d-row cache", me, n_q, pos0, kv->n_ctx);
    if (window < 1 || n_sink < 0) return htr_fail("%s: a window of %d keys and %d first ones", me, window, n_sink);
    HTR_TRY(check_rows(me, d_q, q_stride, kv, n_head, d_out, n_q));
    HTR_TRY(htr_check_alive(dev));
    const HtrOnDevice on(dev);
    a.q = d_q, a.q_stride = q_stride, a.out = d_out, a.n = n_q, a.n_head = n_head, a.group = n_head / kv->n_kv;
    a.scale = scale, a.pos0 = pos0, a.window = window, a.n_sink = n_sink;
    // the most blocks that a tile of 32 rows sees
    const int64_t n_keys = pos0 + n_q, span = std::min<int64_t>(n_keys, (int64_t)window + std::min(n_sink, pos0 + n_q) + 96);
    return launch<false>(dev, a, TreeMask{}, (int)((span + KB - 1) / KB));
}
