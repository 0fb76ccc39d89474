// Attention over a layer's KV cache of f16 or q8_0 rows: of a drafted tree of tokens, and with a sliding window and a few
// first keys that stay visible. Head dim 128, any number of q heads to a KV head.
//
//   out[t][h] = Σ_j p_j·v_j / Σ_j p_j,  p_j = e^(scale·q·k_j − m)  over the keys j that query t sees (zeros if none)
//
// The q heads of a KV head share its keys, so a KV head's queries are rows (t, head of the group), packed: row r is query
// r / group. Up to 16 rows: workgroups of 16 rows and a part of the keys, which share every key (k_kv_attn_few); more:
// workgroups of 32 rows and a part of the keys, whose waves take blocks of their own (k_kv_attn_split); many: workgroups of
// 64 rows and all their keys (k_kv_attn). Parts are joined by the last workgroup that is there, or by a second launch.
//
// On the f16 matrix cores with f32-grade operands: q and p are pairs of f16 values, 22 bits, so that both products are two
// instructions each; K and V are f16 (a q8_0 element stands for f16(q·d): rounded once, 2^-11 of it, beside the block's own
// step of 2^-8 of its largest); all sums are f32.
//   q        x = q·scale is rounded to f32 once, and a row is held times 2^(10 − e), e the exponent of its largest, so that
//            the pair neither overflows nor loses bits whatever the row's size; a score is s·c, c = log2(e)·2^(e − 10);
//   scores   Sᵀ = K·(qh + ql)ᵀ, keys by rows, so that a lane holds scores of one row (of v_mfma_f32_32x32x16_f16 lane
//            32·hf + c row c's of keys 8(i / 4) + 4hf + i % 4, i < 16);
//   softmax  p = 2^((s − m)·c + 10): the difference first, so p is right for scores of any size. m, the row's reference, is
//            moved to the largest score only when one of its p would pass 2^15 (O and l are rescaled then), whatever the
//            rows beside it do, so that a row's sums are those of the keys it sees. The 10 leaves room below, and drops out
//            with l, which carries it too: the low half's last step is 2^-24, so a weight is held to 2^-22 of itself or 2^-35
//            of the largest (with 3 in its place 2^-28: 2^15 keys at that below one lost 1e-4 of the output together), for
//            an exponent of up to 10 whose own rounding takes the outputs from 2.3 … 3.6e-7 to 2.7 … 4.0e-7 of 64 bits;
//   values   Oᵀ += Vᵀ·(ph + pl)ᵀ, V by transposing LDS reads, p in the lanes that it was made in.
// A key that a row does not see is as if it were not there, whatever the cache holds in it: its score becomes −∞ after the
// product, and values of V that are not finite are taken out of the product of a block that not every row sees, and make
// NaN of the sums of the rows that do see them.
//
// Times below are of calls one after another on an MI355X, 16 q heads on 8 KV heads if nothing else is said.
#include <algorithm>
#include <type_traits>

#include "kv_ops.h"
#include "wave.h"

namespace {

constexpr int D = 128, KB = 32;                // head dim; keys a block
constexpr int K_CHUNKS = 512, TILE = 1024;     // 16-byte chunks of a block's K, of its K and V
constexpr float P_SHIFT = 10.0f, P_ROOM = 5.0f; // log2 of the largest p when m moves; its growth before m must move
constexpr float LOG2E = 1.4426950408889634f;
constexpr float M_NONE = -3.0e38f;             // m before the first key: finite, so that s − m is never ∞ − ∞
constexpr int MAX_SPLIT = 64, TICKET = 32;     // parts of a row group's blocks; words between tickets (128 bytes)

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));
typedef int int2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));
typedef uint16_t ushort2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

struct Args {
    const float *q;
    size_t q_stride;
    float *out;
    HtrKvPlanes kv;
    int n, n_head, group;
    uint32_t per_group;        // ⌈2^32 / group⌉ (group > 1): the quotient of a row below 2^32 / group by one product
    float scale;
    int shift;                 // keys past the first ones' blocks lie this many rows further up in memory
    int n_past;                // tree: the committed keys
    int pos0, window, n_sink;  // window
    int n_rg, n_split;         // row groups, parts of a row group's key blocks
    float *part;               // [n_kv·n_rg·n_split][rows of a part] sums o[128], and each row's (m, l, c)
    float4 *part_ml;
    uint32_t *tickets;         // [n_kv·n_rg], TICKET words apart: zero, self-resetting; NULL: joined by a second launch
    int xl;                    // a row group's workgroups share an XCD, and its L2 shows them each other's stores
};
struct TreeMask {
    uint64_t of[HTR_TREE_MAX];
};

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

// the blocks of U keys that some row of queries ta … tb sees: the blocks 0 … first − 1, then from … to − 1
struct Blocks {
    int first, from, to;
    __device__ __forceinline__ int count() const { return first + max(0, to - from); }
    __device__ __forceinline__ int at(int i) const { return i < first ? i : from + (i - first); }
};
template <bool TREE, int U> __device__ __forceinline__ Blocks blocks_of(const Args &a, int ta, int tb) {
    if constexpr (TREE) {
        return Blocks{0, 0, (a.n_past + a.n + U - 1) / U};
    } else {
        const int pa = a.pos0 + ta, pb = a.pos0 + tb, to = pb / U + 1;
        const int first = min((min(a.n_sink, pb + 1) + U - 1) / U, to), lo = a.window > pa ? 0 : (pa - a.window + 1) / U;
        return Blocks{first, max(first, lo), to};
    }
}

// part `split` of n blocks in n_split even parts
struct Part {
    int i0, i1;
};
__device__ __forceinline__ Part part_of(int n, int split, int n_split) {
    const int per = n / n_split, more = n - per * n_split, i0 = split * per + min(split, more);
    return Part{i0, i0 + per + (split < more ? 1 : 0)};
}
// row r's query
__device__ __forceinline__ int query_of(int group, uint32_t per_group, int r) {
    return group == 1 ? r : (int)__umulhi((uint32_t)r, per_group);
}

// one row: query t, its head, and the keys it sees
template <bool TREE> struct Row {
    int r, t, head, pos;
    uint64_t mask;
    __device__ __forceinline__ Row(const Args &a, const TreeMask &tree, int kvh, int row) {
        const int rc = min(row, a.n * a.group - 1);
        r = row, t = query_of(a.group, a.per_group, rc), head = kvh * a.group + (rc - t * a.group), pos = a.pos0 + t;
        mask = 0;
        if constexpr (TREE) mask = tree.of[t];
    }
};
// the lowest n bits (none for n ≤ 0, all from 32 on)
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? ~0u : (1u << max(n, 0)) - 1; }
// the keys k0 … k0 + 31 that the row sees, a bit each
template <bool TREE> __device__ __forceinline__ uint32_t sees(const Args &a, int pos, uint64_t mask, int k0) {
    const int n = (TREE ? a.n_past : pos + 1) - k0;  // the committed keys among them; those that are not ahead
    if constexpr (TREE) {
        const uint32_t drafted = n < 0 ? (n > -64 ? (uint32_t)(mask >> -n) : 0u) : n < 32 ? (uint32_t)mask << n : 0u;
        return low_bits(n) | drafted;
    } else {
        return low_bits(n) & (~low_bits(n - a.window) | low_bits(a.n_sink - k0));
    }
}
// the blocks of U keys that the queries ta … tb all see the whole of: those before `to` that are among the first keys or in
// the last one's window
template <bool TREE, int U> struct Whole {
    int to, sink, from;
    __device__ __forceinline__ Whole(const Args &a, int ta, int tb) {
        const int out = a.pos0 + tb - a.window;  // the last key that the last query does not see any more
        to = (TREE ? a.n_past : a.pos0 + ta + 1) / U, sink = a.n_sink / U, from = out < 0 ? 0 : out / U + 1;
    }
    __device__ __forceinline__ bool block(int k) const {
        if constexpr (TREE) return k < to;
        else return k < to && (k < sink || k >= from);
    }
};

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

// a row's q·scale as f16 pairs, the B operand of N steps (the lane's 8 dims of step 0 at qrow, of `G` lanes that hold the
// row); the factor of its scores
template <int N, int G> __device__ __forceinline__ float q_pairs(const float *qrow, float scale, half8 (&qh)[N], half8 (&ql)[N]) {
    auto dim = [](int ks) { return N == 4 ? 64 * (ks >> 1) + 8 * (ks & 1) : D / N * ks; };
    float x[N][8], top = 0.0f;
#pragma unroll
    for (int ks = 0; ks < N; ks++) {
        const float4 a0 = *reinterpret_cast<const float4 *>(qrow + dim(ks));
        const float4 a1 = *reinterpret_cast<const float4 *>(qrow + dim(ks) + 4);
        x[ks][0] = a0.x, x[ks][1] = a0.y, x[ks][2] = a0.z, x[ks][3] = a0.w;
        x[ks][4] = a1.x, x[ks][5] = a1.y, x[ks][6] = a1.z, x[ks][7] = a1.w;
    }
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

// ---- up to 16 rows: the keys split over workgroups, shared by the rows --------------------------------------------------------
//
// A workgroup takes 16 rows and a run of units of 16 keys, eight a round, one to each of its eight waves:
//   scores   a wave's own unit against all rows, Sᵀ = K·(qh + ql)ᵀ by v_mfma_f32_16x16x32_f16: lane 16g + c holds row c's
//            scores of keys 4g … 4g + 3; the rows' largest over the waves through LDS (barrier);
//   weights  p = 2^((s − m)·c + 10) as f16 pairs to LDS, in the order of the next products' operands (barrier);
//   values   Oᵀ += Vᵀ·(ph + pl)ᵀ over the round's 128 keys, a wave's own 16 dims. So every K and V value is loaded, and made
//            f16, once for all the rows, no sums of O are merged between waves, and O is 4 registers.
// K and V come straight into LDS, a wave's own unit each: K into one buffer (read by that wave alone, filled again once the
// scores are taken), V into one of two (filled again when all waves are past the values of the round before). q8_0 units as
// they are, int8: an operand's 8 quants become f16 in registers (14 VALU instructions), V's by a transposing read of bytes,
// their scales from LDS in the order of the operand's slots.
//   f16   [16 keys][16 chunks of 16 bytes], K row r's chunk c at 16r + (c ^ r), V's at 16r + (c ^ 2(r % 8));
//   q8_0  [16 keys][8 chunks], row r's chunk c at 8r + (c ^ r / 2), V's of odd units with c ^ 4 too; the scales [16 keys][4]:
// reads of 16 (32) lanes fall on different bank groups.
//
// Bound: latency, of the loads and of a round's two barriers and exchanges. A call takes 5.0 µs up to 128 keys and 0.95 (f16)
// or 1.2 µs (q8_0) a further round; splitting the keys costs 2.4. One token over 8000 q8_0 keys takes 10.2 µs (17.4 MB: 2.5 at
// the 7.0 TB/s of a read). k_attn_decode, for one token, f16 rows and two q heads to a KV head alone, has all its keys' loads in
// flight at once and exchanges between waves only at the end: over 512 / 2048 / 8192 keys 6.4 / 6.4 / 9.2 µs, this kernel
// 7.2 / 7.7 / 9.4 (q8_0 rows 7.4 / 7.7 / 9.7). The waves'
// own blocks of k_kv_attn_split take 9.2 over 1000 keys (here 7.3) and 11.8 over the 8000 (their 32-row products are half or
// more empty, and their sums have to be merged); at 16 rows the two are as fast, above this way is slower (24 rows over 1300
// keys 11.6 and 10.7, over 6000 q8_0 keys 15.1 and 12.5).
constexpr int SW = 8, UK = 16, ST = SW / 2, FR = 16;  // waves; keys of a unit; steps of 32 keys of a round; rows
// Rows × parts that the last workgroup joins itself, in the L2 of its XCD or through the coherence point; more are joined by a
// second launch. In the L2 the two are as fast up to 256 (7 tokens over 1300 keys, 154: 9.4 and 8.8 µs; over 400, 56: 7.6 and
// 8.6), and a launch costs the host 4 µs; with 448 (3000 and more keys) 14.1 and 11.9. Through the coherence point 60 tokens on
// 4 KV heads over 1000 … 4500 keys (128 … 256) take 12.7 … 16.1 and 11.2 … 14.2, one token (16 … 64) 7.6 … 8.7 both ways.
constexpr int JOIN_L2 = 256, JOIN_FAR = 64;

struct JoinArgs {
    const float *part;
    const float4 *part_ml;
    float *out;
    uint32_t per_group;
    int n_split, n_head, group, rows, n_kv, n_rg, tile;  // tile: rows of a row group's part
};

// one row's parts g, g + G, … joined by 32 lanes of 4 dims each; s_w: 64 words of the group's own. LATER: the parts are an
// earlier launch's. Returns Σ l
template <bool LATER>
__device__ __forceinline__ float join_row(const float *part, const float4 *part_ml, size_t first, size_t step, int ns, int g, int G,
                                          float *s_w, int lane, float4 &y) {
    const int j = lane & 31;
    const float *from = part + first * D + 4 * j;
    float4 in[8];
    auto get = [](const float *at) {
        if constexpr (LATER) return *reinterpret_cast<const float4 *>(at);
        const float2 a = get64(at), b = get64(at + 2);
        return make_float4(a.x, a.y, b.x, b.y);
    };
    auto fetch = [&](int p0) {
#pragma unroll
        for (int e = 0; e < 8; e++) in[e] = get(from + (size_t)min(p0 + e * G, ns - 1) * step * D);
    };
    fetch(g);
    float m[2], l[2], top = M_NONE, sum = 0.0f, c = 1.0f;
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const float4 ml = get(reinterpret_cast<const float *>(part_ml + first + (size_t)min(j + 32 * e, ns - 1) * step));
        c = ml.z;
        m[e] = j + 32 * e < ns ? ml.x : M_NONE, l[e] = j + 32 * e < ns ? ml.y : 0.0f;
        top = fmaxf(top, m[e]);
    }
    top = group_max<16>(top, lane);
#pragma unroll
    for (int e = 0; e < 2; e++) {
        const float w = __builtin_amdgcn_exp2f((m[e] - top) * c);
        sum = fmaf(l[e], w, sum);
        s_w[j + 32 * e] = j + 32 * e < ns ? w : 0.0f;
    }
    sum = group_sum<16>(sum, lane);
    __builtin_amdgcn_wave_barrier();
    y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int p = g;;) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float w = p + e * G < ns ? s_w[p + e * G] : 0.0f;
            y.x = fmaf(in[e].x, w, y.x), y.y = fmaf(in[e].y, w, y.y), y.z = fmaf(in[e].z, w, y.z), y.w = fmaf(in[e].w, w, y.w);
        }
        p += 8 * G;
        if (p >= ns) break;
        fetch(p);
    }
    __builtin_amdgcn_wave_barrier();
    return sum;
}
__device__ __forceinline__ void put_row(float *out, int n_head, int group, uint32_t per_group, int kvh, int r, int j, float4 y, float sum) {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // no key seen: zeros
    const int t = query_of(group, per_group, r), head = kvh * group + (r - t * group);
    *reinterpret_cast<float4 *>(out + ((size_t)t * n_head + head) * D + 4 * j) = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
}

// the second launch: two rows a workgroup, four groups of 32 lanes to a row's parts
__global__ __launch_bounds__(256) void k_kv_attn_join(JoinArgs a) {
    __shared__ float s_w[8][MAX_SPLIT];
    __shared__ float4 s_y[8][32];
    const int gr = threadIdx.x >> 5, j = threadIdx.x & 31, g = gr & 3;
    const int id = min((int)blockIdx.x * 2 + (gr >> 2), a.rows * a.n_kv - 1);
    const int kvh = id / a.rows, r = id % a.rows, rg = r / a.tile;
    float4 y;
    const float sum = join_row<true>(a.part, a.part_ml, ((size_t)kvh * a.n_rg + rg) * a.n_split * a.tile + r % a.tile, a.tile, a.n_split, g, 4,
                               s_w[gr], threadIdx.x & 63, y);
    s_y[gr][j] = y;
    __syncthreads();
    if (g != 0 || (int)blockIdx.x * 2 + (gr >> 2) >= a.rows * a.n_kv) return;
#pragma unroll
    for (int e = 1; e < 4; e++) {
        const float4 z = s_y[gr + e][j];
        y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
    }
    put_row(a.out, a.n_head, a.group, a.per_group, kvh, r, j, y, sum);
}

// the last workgroup of a row group to have stored its part joins them all (tile: rows of a part, the group's first at g0);
// s_y: room for a float4 a thread
__device__ __forceinline__ void join_last(const Args &a, int kvh, int rg, int r0, int rows, int tile, size_t g0, int *s_last,
                                          float (&s_w)[2 * SW][MAX_SPLIT], float4 *s_y) {
    const int tid = threadIdx.x, lane = tid & 63;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this thread's stores are performed
    __syncthreads();
    uint32_t *ticket = a.tickets + TICKET * ((size_t)kvh * a.n_rg + rg);
    if (tid == 0)
        *s_last = (a.xl ? __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP)
                        : __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) ==
                  (uint32_t)(a.n_split - 1);
    __syncthreads();
    if (!*s_last) return;
    // 32 lanes a row; where the rows are fewer than the groups of lanes, several groups (of 8 parts at once each) to a row
    const int nr = min(tile, rows - r0), gr = tid >> 5, j = tid & 31;
    const int few = nr > 8 ? 0 : nr > 4 ? 1 : nr > 2 ? 2 : nr > 1 ? 3 : 4;  // log2 of the groups that there are for a row
    const int ns8 = (a.n_split + 7) / 8, lg = 4 - min(few, ns8 > 4 ? 3 : ns8 > 2 ? 2 : ns8 > 1 ? 1 : 0), G = 16 >> lg;
    for (int rb = 0; rb < nr; rb += 1 << lg) {
        const int ri = rb + (gr & ((1 << lg) - 1)), part = gr >> lg;
        float4 y;
        const float sum = join_row<false>(a.part, a.part_ml, g0 + min(ri, nr - 1), tile, a.n_split, part, G, s_w[gr], lane, y);
        if (G > 1) {  // (one pass)
            s_y[tid] = y;
            __syncthreads();
            if (part == 0)
                for (int e = 1; e < G; e++) {
                    const float4 z = s_y[tid + 32 * (e << lg)];
                    y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
                }
        }
        if (part == 0 && ri < nr) put_row(a.out, a.n_head, a.group, a.per_group, kvh, r0 + ri, j, y, sum);
    }
    if (tid == 0) {  // for the next call
        if (a.xl) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
        else __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

template <bool Q8, bool TREE> __global__ __launch_bounds__(64 * SW, 2) void k_kv_attn_few(Args a, TreeMask tree) {
    constexpr int UC = Q8 ? 8 * UK : 16 * UK;                        // 16-byte chunks of a unit's K or V
    constexpr int NL = Q8 ? UK / 8 + 1 : UK / 4;                     // loads of a unit's K or V
    __shared__ __attribute__((aligned(16))) uint4_t s_k[SW][UC], s_v[2][SW][UC];
    __shared__ __attribute__((aligned(16))) uint4_t s_p[2][ST][64];  // weights' high and low halves
    __shared__ __attribute__((aligned(16))) uint32_t s_kd[Q8 ? SW : 1][64], s_vd[2][Q8 ? SW : 1][64];
    __shared__ __attribute__((aligned(16))) uint16_t s_vt[4][ST][4][8];  // V's scales by dims / 32, step, lane group, slot
    __shared__ float s_mx[SW][UK], s_l[SW][UK];
    __shared__ float s_w[SW * 2][MAX_SPLIT];
    __shared__ int s_odd[SW], s_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, c = lane & 15;
    const int kvh = blockIdx.x, rg = blockIdx.y, split = blockIdx.z;
    const int rows = a.n * a.group, r0 = rg * FR;
    const int n_keys = TREE ? a.n_past + a.n : a.pos0 + a.n;
    const int ta = query_of(a.group, a.per_group, r0), tb = query_of(a.group, a.per_group, min(r0 + FR - 1, rows - 1));
    const Blocks blk = blocks_of<TREE, UK>(a, ta, tb);
    const Part part = part_of(blk.count(), split, a.n_split);
    const int i0 = part.i0, i1 = part.i1;
    const int n_round = (i1 - i0 + SW - 1) / SW;
    const size_t head0 = (size_t)kvh * a.kv.n_ctx;

    // the unit i (one past the part's end: the last's, masked) of K, or of V into buffer b; a wave's instruction is 4 (8) whole
    // rows. Rows past the last key are the last key's, and masked
    const uint32_t kx = 16 * ((lane & 15) ^ (lane >> 4)), vx = 16 * ((lane & 15) ^ (2 * (lane >> 4))), r4 = 2 * D * (lane >> 4);
    const uint32_t bx = 16 * ((lane & 7) ^ (lane >> 4)), wx = bx ^ (64 * (wave & 1)), r8 = D * (lane >> 3);
    auto lds_of = [](auto &x) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)(char *)&x; };
    auto load = [&](int i, bool is_v, int b) {
        const int k0 = UK * blk.at(min(i, i1 - 1)), last = min(n_keys - 1 - k0, UK - 1);
        const size_t row = head0 + k0;
        const uint32_t to = is_v ? lds_of(s_v[b][wave]) : lds_of(s_k[wave]);
        const char *base = (const char *)(is_v ? a.kv.v : a.kv.k) + row * (Q8 ? D : 2 * D);
        if constexpr (Q8) {
            lds_load4((is_v ? a.kv.vd : a.kv.kd) + row * 4, 8 * min((lane & 31) >> 1, last) + 4 * (lane & 1),
                      is_v ? lds_of(s_vd[b][wave]) : lds_of(s_kd[wave]));
#pragma unroll
            for (int u = 0; u < 2; u++)
                lds_load16(base, min(r8 + 8 * D * u, (uint32_t)(D * last)) + ((is_v ? wx : bx) ^ (64 * (u & 1))), to + 16 * 64 * u);
        } else {
#pragma unroll
            for (int u = 0; u < 4; u++)
                lds_load16(base, min(r4 + 4 * 2 * D * u, (uint32_t)(2 * D * last)) + (is_v ? vx ^ (128 * (u & 1)) : kx ^ (64 * (u & 3))),
                           to + 16 * 64 * u);
        }
    };
    if (n_round > 0) {
        load(i0 + wave, false, 0);
        load(i0 + wave, true, 0);
    }

    half8 qh[4], ql[4];
    const Row<TREE> row(a, tree, kvh, r0 + c);
    // (the 8 dims of the lane's operand: of two steps 16 in a row, 16 bytes of quants)
    const float sc = q_pairs<4, 4>(a.q + (size_t)row.t * a.q_stride + (size_t)row.head * D + 16 * g, a.scale, qh, ql);
    float m = M_NONE, l = 0.0f;
    // the lane's place in V's units: slots 8g … are keys 4g … 4g + 3 of a step's first unit, then of its second
    const int vrow = Q8 ? 4 * g + ((c >> 1) & 3) : 4 * g + (c >> 2);
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};

    // whether every row sees all keys of the round's units
    const Whole<TREE, UK> full(a, ta, tb);
    auto whole = [&](int rd) {
        const int i = i0 + SW * rd + (lane & 7);
        return __builtin_amdgcn_ballot_w64(!(i < i1 && full.block(blk.at(i)))) == 0;
    };
    for (int rd = 0; rd < n_round; rd++) {
        const bool masked = !whole(rd);  // (what only a masked round does stands behind uniform branches, and is not fetched else)
        const int i = i0 + SW * rd + wave, b = rd & 1;
        const bool more = rd + 1 < n_round;
        wait_loads<NL>();  // K; V is still on its way
        f32x4 s;
        {
            half8 f[4];
            if constexpr (Q8) {
                const uint2_t dk = reinterpret_cast<const uint2_t *>(s_kd[wave])[c];
                half2_t d2[2];
                __builtin_memcpy(d2, &dk, 8);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint4_t w = s_k[wave][8 * c + ((4 * h + g) ^ (c >> 1))];
                    const _Float16 d = g < 2 ? d2[h][0] : d2[h][1];
                    f[2 * h] = dequant8(w[0], w[1], half2_t{d, d});
                    f[2 * h + 1] = dequant8(w[2], w[3], half2_t{d, d});
                }
            } else {
#pragma unroll
                for (int ks = 0; ks < 4; ks++) {
                    const int chunk = 8 * (ks >> 1) + 2 * g + (ks & 1);
                    f[ks] = *reinterpret_cast<const half8 *>(s_k[wave] + 16 * c + (chunk ^ c));
                }
            }
            wait_reads();
            if (more) load(i + SW, false, 0);
#pragma unroll
            for (int ks = 0; ks < 4; ks++) {
                s = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[ks], qh[ks], ks ? s : f32x4{}, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_16x16x32_f16(f[ks], ql[ks], s, 0, 0, 0);
            }
        }
        uint32_t seen = 15u;
        if (masked) {
            const int k0 = UK * blk.at(min(i, i1 - 1)) + here(4 * g);
            seen = i < i1 ? sees<TREE>(a, row.pos, row.mask, k0) : 0u;
#pragma unroll
            for (int x = 0; x < 4; x++) s[x] = seen >> x & 1 ? s[x] : -INFINITY;
        }
        float mx = pair_max<32>(pair_max<16>(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]))));
        if (g == 0) s_mx[wave][c] = mx;
        wait_reads();
        __builtin_amdgcn_s_barrier();  // everyone's largest scores; everyone is past the values of the round before
        asm volatile("" ::: "memory");
        if (more) load(i + SW, true, b ^ 1);
        mx = s_mx[0][c];
#pragma unroll
        for (int w = 1; w < SW; w++) mx = fmaxf(mx, s_mx[w][c]);
        const bool up = (mx - m) * sc > P_ROOM;  // (alike in every wave)
        if (__builtin_amdgcn_ballot_w64(up)) {
            const float to = up ? mx : m, corr = __builtin_amdgcn_exp2f((m - to) * sc);
            m = to;
            l *= corr;
            o *= corr;
        }
        {
            float p[4];
#pragma unroll
            for (int x = 0; x < 4; x++) p[x] = __builtin_amdgcn_exp2f(fmaf(s[x] - m, sc, P_SHIFT));  // not seen: 2^(−∞) = 0
            l += (p[0] + p[1]) + (p[2] + p[3]);
            uint32_t h[2], r[2];
            split2(p[0], p[1], h[0], r[0]);
            split2(p[2], p[3], h[1], r[1]);
            // a weight's sign: not seen
            h[0] |= (~seen & 1u) << 15 | (~seen & 2u) << 30;
            h[1] |= (~seen & 4u) << 13 | (~seen & 8u) << 28;
            reinterpret_cast<uint2_t *>(&s_p[0][wave >> 1][lane])[wave & 1] = uint2_t{h[0], h[1]};
            reinterpret_cast<uint2_t *>(&s_p[1][wave >> 1][lane])[wave & 1] = uint2_t{r[0], r[1]};
        }
        if (more) wait_loads<2 * NL>();  // V
        else wait_loads<0>();
        if constexpr (Q8)
            if (lane < 32) {  // V's scales into the order of the operands' slots
                const uint32_t d2 = s_vd[b][wave][lane];
                const int key = lane >> 1, at = 4 * (wave & 1) + (key & 3);
                s_vt[2 * (lane & 1)][wave >> 1][key >> 2][at] = (uint16_t)d2;
                s_vt[2 * (lane & 1) + 1][wave >> 1][key >> 2][at] = (uint16_t)(d2 >> 16);
            }
        if (masked) {  // does the wave's unit hold a value of V that is not finite (a scale that may make one: 512 and past)?
            uint32_t any = 0;
            if constexpr (Q8) {
                any = scale_past(s_vd[b][wave][here(lane)]);
            } else {
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const uint4_t w = s_v[b][wave][64 * u + here(lane)];
#pragma unroll
                    for (int e = 0; e < 4; e++) any |= ((w[e] & 0x7C007C00u) + 0x04000400u) & 0x80008000u;
                }
            }
            if (lane == 0) s_odd[wave] = 0;
            if (any) s_odd[wave] = 1;
        }
        wait_reads();
        __builtin_amdgcn_s_barrier();  // everyone's weights and V
        asm volatile("" ::: "memory");
        auto vread = [&](int st) {  // Vᵀ of step st, the wave's dims
            half8 v;
            if constexpr (Q8) {
                const uint4_t *unit = s_v[b][2 * st] + UC * ((c >> 3) & 1);
                const int at = 8 * vrow + (wave ^ (vrow >> 1) ^ ((c & 8) >> 1));
                const auto *p = (const __attribute__((address_space(3))) char *)(unit + at) + 8 * (c & 1);
                const int2_t w = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) int2_t *)p);
                v = dequant8((uint32_t)w[0], (uint32_t)w[1], *reinterpret_cast<const half8 *>(s_vt[wave >> 1][st][g]));
            } else {
                const int at = 16 * vrow + ((2 * wave + ((c >> 1) & 1)) ^ (2 * (vrow & 7)));
                const auto *p = (const __attribute__((address_space(3))) char *)(s_v[b][2 * st] + at) + 8 * (c & 1);
                const fp16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)p);
                const fp16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)(p + 16 * UC));
                __builtin_memcpy(&v, &lo, 8);
                __builtin_memcpy((char *)&v + 8, &up, 8);
            }
            return v;
        };
        bool odd = false;
        if (masked) odd = __builtin_amdgcn_ballot_w64(s_odd[here(lane & 7)] != 0) != 0;
        if (!odd) {
#pragma unroll
            for (int st = 0; st < ST; st++) {
                const half8 v = vread(st);
                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, *reinterpret_cast<const half8 *>(&s_p[0][st][lane]), o, 0, 0, 0);
                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, *reinterpret_cast<const half8 *>(&s_p[1][st][lane]), o, 0, 0, 0);
            }
        } else {
            // such values as 0, and NaN into the sums of the rows that see one: a product of ones
            f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
            for (int st = 0; st < ST; st++) {
                const half8 v = vread(st), z = finite(v);
                uint4_t h = s_p[0][st][lane];
                half8 ind;
                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(z, *reinterpret_cast<const half8 *>(&h), o, 0, 0, 0);
                o = __builtin_amdgcn_mfma_f32_16x16x32_f16(z, *reinterpret_cast<const half8 *>(&s_p[1][st][lane]), o, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; e++) h[e] = ((~h[e] >> 15) & 0x00010001u) * 0x3C00u;
                __builtin_memcpy(&ind, &h, 16);
                t = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones_of_not_finite(v), ind, t, 0, 0, 0);
            }
#pragma unroll
            for (int x = 0; x < 4; x++) o[x] = t[x] > 0.0f ? NAN : o[x];
        }
    }
    // Σ l over the lanes and waves (m is the same in every wave)
    l = pair_sum<32>(pair_sum<16>(l));
    if (g == 0) s_l[wave][c] = l;
    __syncthreads();
    const size_t g0 = ((size_t)kvh * a.n_rg + rg) * a.n_split * FR;  // the row group's first row of partial sums
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < SW; w++) l += s_l[w][c];
    if (row.r < rows) {
        if (a.n_split == 1) {
            put_row(a.out, a.n_head, a.group, a.per_group, kvh, row.r, 4 * wave + g, make_float4(o[0], o[1], o[2], o[3]), l);
        } else {
            const size_t pr = g0 + (size_t)split * FR + c;
            float *to = a.part + pr * D + 16 * wave + 4 * g;
            put64(to, o[0], o[1], a.xl);
            put64(to + 2, o[2], o[3], a.xl);
            if (wave == 0 && g == 0) {
                put64(a.part_ml + pr, m, l, a.xl);
                put64(&a.part_ml[pr].z, sc, 0.0f, a.xl);
            }
        }
    }
    if (a.tickets) join_last(a, kvh, rg, r0, rows, FR, g0, &s_last, s_w, reinterpret_cast<float4 *>(&s_k[0][0]));
}

// ---- more rows: the keys split over workgroups, blocks of its own to a wave -----------------------------------------------------
//
// A workgroup takes 32 rows, each of its eight waves every eighth block of 32 keys of its part. A wave loads its own blocks
// straight into LDS of its own, so the waves wait for nobody until their sums are merged; f16 blocks with one buffer for K
// and one for V, each filled again as soon as it is read (K under the softmax and the values, V under the next scores), q8_0
// blocks, half the size, with two, raw: a fragment's 8 quants become f16 in the registers of the one wave that uses them (14
// VALU instructions an operand; V's by a transposing read of bytes).
//   f16   K and V [32 keys][16 chunks of 16 bytes], K row r's chunk c at 16r + (c ^ r % 16), V's at 16r + (c ^ 4(r % 4));
//   q8_0  K and V [32 keys][8 chunks], K row r's chunk c at 8r + (c ^ r / 2 % 8), V's at 8r + (c ^ (r & 2) ^ (r & 8) / 2); their
//         scales [32 keys][4]; V's once more as [dims / 32][key / 16][hf][8], the order of an operand's slots.
// Reads of 16 (32) lanes then fall on different bank groups.
//
// Bound: of few keys latency (8 µs a call up to 300 keys: 2 until the first block is there, 2 for the merge), of many the
// instructions of its two waves a SIMD: a block of f16 is 32 MFMA and some 130 VALU instructions, 16 of them exponentials,
// one of q8_0 224 VALU instructions more (MFMA busy 34 %, VALU 59 % over 40013 keys). 64 tokens over 6001 f16 keys 16.0 µs (27
// MB: 5.5 at a copy's rate), 27 over 40013 q8_0 keys 29.8 (88 MB: 17.8), of real values, whose products lower the clock, 33 …
// 36. With four waves a workgroup the
// kernels alone took 30.9 and 54.9 for 21.2 and 30. Two row tiles to a wave, which halves the conversions, cost 6.7 µs of the
// 27 tokens' call: half as many waves, and each longer.
constexpr int QT = 256 + 256 + 16 + 16;  // 16-byte chunks of a q8_0 buffer: K, V, K scales, V scales

template <bool Q8, bool TREE> __global__ __launch_bounds__(64 * SW, 2) void k_kv_attn_split(Args a, TreeMask tree) {
    constexpr int WAVE = Q8 ? 2 * QT + 16 : TILE;  // chunks of a wave's LDS
    static_assert(WAVE >= 1024, "a wave's sums fit");
    __shared__ __attribute__((aligned(16))) uint4_t s_kv[SW][WAVE];
    __shared__ __attribute__((aligned(16))) uint4_t s_q[2][16 * KB];  // the rows' pairs; then the join's
    __shared__ float s_ml[SW][2][KB], s_c[KB];
    auto &s_w = *reinterpret_cast<float(*)[2 * SW][MAX_SPLIT]>(&s_q[0][0]);
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hf = lane >> 5, c = lane & 31;
    const int kvh = blockIdx.x, rg = blockIdx.y, split = blockIdx.z;
    const int rows = a.n * a.group, r0 = rg * KB;
    const int n_keys = TREE ? a.n_past + a.n : a.pos0 + a.n;
    const int ta = query_of(a.group, a.per_group, r0), tb = query_of(a.group, a.per_group, min(r0 + KB - 1, rows - 1));
    const Blocks blk = blocks_of<TREE, KB>(a, ta, tb);
    const Part part = part_of(blk.count(), split, a.n_split);
    const int i0 = part.i0, i1 = part.i1;
    const size_t head0 = (size_t)kvh * a.kv.n_ctx;

    uint4_t *tile = s_kv[wave];
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4_t *)tile;
    // block i's K or V (f16), or all of it into buffer b (q8_0); a wave's instruction is 4 (8) whole rows. Rows past the last
    // key are the last key's, and are masked
    const uint32_t kx = 16 * ((lane & 15) ^ (lane >> 4)), vx = 16 * ((lane & 15) ^ (4 * (lane >> 4))), r4 = 2 * D * (lane >> 4);
    const uint32_t bx = 16 * ((lane & 7) ^ (lane >> 4)), wx = 16 * ((lane & 7) ^ (2 * ((lane >> 4) & 1))), r8 = D * (lane >> 3);
    auto load = [&](int i, bool is_v) {
        const int k0 = KB * blk.at(i), last = n_keys - 1 - k0;
        const char *base = (const char *)(is_v ? a.kv.v : a.kv.k) + (head0 + k0) * (2 * D);
        const uint32_t to = lds + 16 * (is_v ? K_CHUNKS : 0);
        if (last >= KB - 1) {
#pragma unroll
            for (int u = 0; u < 8; u++)
                lds_load16(base + 2 * D * 4 * u, r4 + (is_v ? vx : kx ^ (64 * (u & 3))), to + 16 * 64 * u);
        } else {
            const int ln = here(lane);
#pragma unroll
            for (int u = 0; u < 8; u++)
                lds_load16(base, 2 * D * min(4 * u + (ln >> 4), last) + (is_v ? vx : kx ^ (64 * (u & 3))), to + 16 * 64 * u);
        }
    };
    auto load_q8 = [&](int i, int b) {
        const int k0 = KB * blk.at(i), last = n_keys - 1 - k0;
        const size_t row = head0 + k0;
        const uint32_t to = lds + 16 * QT * b;
        const char *kb = (const char *)a.kv.k + row * D, *vb = (const char *)a.kv.v + row * D;
        if (last >= KB - 1) {
            lds_load4(a.kv.kd + row * 4, 4 * lane, to + 16 * 512);
            lds_load4(a.kv.vd + row * 4, 4 * lane, to + 16 * 528);
#pragma unroll
            for (int u = 0; u < 8; u++) lds_load16((u < 4 ? kb : vb) + D * 8 * (u & 3), r8 + ((u < 4 ? bx : wx) ^ (64 * (u & 1))), to + 16 * 64 * u);
        } else {
            const int ln = here(lane);
            lds_load4(a.kv.kd + row * 4, 8 * min(ln >> 1, last) + 4 * (ln & 1), to + 16 * 512);
            lds_load4(a.kv.vd + row * 4, 8 * min(ln >> 1, last) + 4 * (ln & 1), to + 16 * 528);
#pragma unroll
            for (int u = 0; u < 8; u++)
                lds_load16(u < 4 ? kb : vb, D * min(8 * (u & 3) + (ln >> 3), last) + ((u < 4 ? bx : wx) ^ (64 * (u & 1))), to + 16 * 64 * u);
        }
    };
    int i = i0 + wave, b = 0;
    if (i < i1) {
        if constexpr (Q8) {
            load_q8(i, 0);
        } else {
            load(i, false);
            load(i, true);
        }
    }

    // the 8 dims of the lane's operand of a step: of two steps 16 in a row, 16 bytes of quants
    auto dims8 = [&](int ks) { return 4 * (ks >> 1) + 2 * hf + (ks & 1); };
    half8 qh[8], ql[8];
    {
        // each thread makes the pairs of 8 dims of a row; the operands come back from LDS (dims 8j … of row c at 32j + (c ^ j):
        // 16 threads' writes and 32 lanes' reads fall on different bank groups)
        const int j = tid & 15, rq = tid >> 4;
        const Row<TREE> mine(a, tree, kvh, r0 + rq);
        half8 h[1], r[1];
        const float f = q_pairs<1, 16>(a.q + (size_t)mine.t * a.q_stride + (size_t)mine.head * D + 8 * j, a.scale, h, r);
        *reinterpret_cast<half8 *>(&s_q[0][KB * j + (rq ^ j)]) = h[0];
        *reinterpret_cast<half8 *>(&s_q[1][KB * j + (rq ^ j)]) = r[0];
        if (j == 0) s_c[rq] = f;
    }
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < 8; ks++) {
        const int j = dims8(ks), at = KB * j + (c ^ j);
        qh[ks] = *reinterpret_cast<const half8 *>(&s_q[0][at]);
        ql[ks] = *reinterpret_cast<const half8 *>(&s_q[1][at]);
    }
    const Row<TREE> row(a, tree, kvh, r0 + c);
    const float sc = s_c[c];
    float m = M_NONE, l = 0.0f;
    f32x16 o[4];
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
        for (int x = 0; x < 16; x++) o[u][x] = 0.0f;

    // the lane's places in a block: K step ks is key c, dims 8·dims8 …; V tile u, step ss, slots 8hf … + 7 are the keys
    // 16ss + 4hf … + 3, then 16ss + 8 + 4hf … + 3 (the lane's scores 8ss …) of dims 32u + 16(lane / 16 % 2) …
    const int vrow = Q8 ? 8 * ((lane >> 3) & 1) + 4 * hf + ((lane >> 1) & 3) : 4 * hf + ((lane & 15) >> 2);
    int va[4];
#pragma unroll
    for (int u = 0; u < 4; u++)
        va[u] = Q8 ? 16 * (256 + 8 * vrow + ((2 * u + ((lane >> 4) & 1)) ^ (vrow & 2) ^ ((vrow & 8) >> 1))) + 8 * (lane & 1)
                   : 16 * (K_CHUNKS + 16 * vrow + ((4 * u + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ (4 * (vrow & 3)))) + 8 * (lane & 1);

    const Whole<TREE, KB> full(a, ta, tb);
    // block i; MASK: not every row sees all of it
    auto step = [&](auto is_masked) {
        constexpr bool MASK = decltype(is_masked)::value;
        const bool more = i + SW < i1;
        uint4_t *buf = tile + (Q8 ? QT * b : 0);
        if constexpr (Q8) {
            if (more) {
                wait_reads();  // of the other buffer, a block ago
                load_q8(i + SW, b ^ 1);
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
            uint4_t w;
#pragma unroll
            for (int ks = 0; ks < 8; ks++) {
                if (ks % 2 == 0) w = buf[8 * c + ((ks + hf) ^ ((c >> 1) & 7))];
                const _Float16 d = d4[ks >> 2][(ks >> 1) & 1];
                const half8 f = dequant8(w[2 * (ks & 1)], w[2 * (ks & 1) + 1], half2_t{d, d});
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, qh[ks], ks ? s : f32x16{}, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, ql[ks], s, 0, 0, 0);
            }
            // the next operand's conversion in the shadow of this one's products, half a conversion to each (as compiled both
            // products went first, and the conversion behind them: 30.4 µs for 29.8 over 40013 keys)
            __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 22, 0);
#pragma unroll
            for (int e = 0; e < 14; e++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x002, 7, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
        } else {
            half8 f[4];
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int ks = 0; ks < 4; ks++) f[ks] = *reinterpret_cast<const half8 *>(buf + 16 * c + (dims8(4 * h + ks) ^ (c & 15)));
                if (h == 1) {
                    wait_reads();
                    if (more) load(i + SW, false);
                }
#pragma unroll
                for (int ks = 0; ks < 4; ks++) {
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[ks], qh[4 * h + ks], h || ks ? s : f32x16{}, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[ks], ql[4 * h + ks], s, 0, 0, 0);
                }
            }
        }
        uint32_t seen = 0;
        if constexpr (MASK) {
            seen = sees<TREE>(a, row.pos, row.mask, KB * blk.at(i) + here(4 * hf));
#pragma unroll
            for (int x = 0; x < 16; x++) s[x] = seen >> (8 * (x >> 2) + (x & 3)) & 1 ? s[x] : -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int x = 1; x < 16; x++) mx = fmaxf(mx, s[x]);
        mx = pair_max<32>(mx);
        const bool up = (mx - m) * sc > P_ROOM;
        if (__builtin_amdgcn_ballot_w64(up)) {
            const float to = up ? mx : m, corr = __builtin_amdgcn_exp2f((m - to) * sc);
            m = to;
            l *= corr;
#pragma unroll
            for (int u = 0; u < 4; u++) o[u] *= corr;
        }
        float ls = 0.0f;
        uint32_t ph[8], pl[8];
#pragma unroll
        for (int x = 0; x < 8; x++) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[2 * x] - m, sc, P_SHIFT));  // not seen: 2^(−∞) = 0
            const float p1 = __builtin_amdgcn_exp2f(fmaf(s[2 * x + 1] - m, sc, P_SHIFT));
            ls += p0;
            ls += p1;
            split2(p0, p1, ph[x], pl[x]);
        }
        l += ls;
        if constexpr (!Q8) {  // V
            if (more) wait_loads<8>();
            else wait_loads<0>();
        }
        auto vread = [&](int u, int ss) {
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
            return v;
        };
        bool odd = false;
        if constexpr (MASK && Q8) {
            odd = __builtin_amdgcn_ballot_w64(scale_past(reinterpret_cast<const uint32_t *>(buf + 528)[here(lane)])) != 0;
        } else if constexpr (MASK) {
            uint32_t top = 0;
#pragma unroll
            for (int u = 0; u < 4; u++) largest(vread(u, 0), top), largest(vread(u, 1), top);
            odd = any_not_finite(top);
        }
#pragma unroll
        for (int ss = 0; ss < 2; ss++) {
            half8 h8, l8;
            __builtin_memcpy(&h8, &ph[4 * ss], 16);
            __builtin_memcpy(&l8, &pl[4 * ss], 16);
#pragma unroll
            for (int u = 0; u < 4; u++) {
                half8 v = vread(u, ss);
                if (odd) v = finite(v);
                o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, h8, o[u], 0, 0, 0);
                o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, l8, o[u], 0, 0, 0);
                if constexpr (MASK) __builtin_amdgcn_sched_barrier(0);  // (few operands in registers at once)
            }
        }
        if constexpr (MASK)
            if (odd) put_nan(o, seen, vread);
        if constexpr (!Q8) {
            wait_reads();
            if (more) load(i + SW, true);
        }
        i += SW;
        b ^= Q8;
    };
    while (i < i1) {
        for (bool all = full.block(blk.at(i)); all; all = i < i1 && full.block(blk.at(i))) step(std::false_type{});
        for (bool some = i < i1; some; some = i < i1 && !full.block(blk.at(i))) step(std::true_type{});
    }

    l = pair_sum<32>(l);

    // the waves' sums through LDS (each its own tile's place): wave w finishes dims 16w … of every row
    wait_reads();
    float4 *so = reinterpret_cast<float4 *>(tile);
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
        for (int x = 0; x < 4; x++)
            so[(4 * u + x) * 64 + lane] = make_float4(o[u][4 * x], o[u][4 * x + 1], o[u][4 * x + 2], o[u][4 * x + 3]);
    if (hf == 0) s_ml[wave][0][c] = m, s_ml[wave][1][c] = l;
    __syncthreads();
    m = M_NONE, l = 0.0f;
#pragma unroll
    for (int p = 0; p < SW; p++) m = fmaxf(m, s_ml[p][0][c]);
    float4 v[2];
#pragma unroll
    for (int x = 0; x < 2; x++) v[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int p = 0; p < SW; p++) {
        const float w = __builtin_amdgcn_exp2f((s_ml[p][0][c] - m) * sc);
        l = fmaf(s_ml[p][1][c], w, l);
        const float4 *from = reinterpret_cast<const float4 *>(s_kv[p]) + 2 * 64 * wave + lane;
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const float4 y = from[64 * x];
            v[x].x = fmaf(y.x, w, v[x].x), v[x].y = fmaf(y.y, w, v[x].y);
            v[x].z = fmaf(y.z, w, v[x].z), v[x].w = fmaf(y.w, w, v[x].w);
        }
    }
    const size_t g0 = ((size_t)kvh * a.n_rg + rg) * a.n_split * KB;  // the row group's first row of partial sums
    if (row.r < rows) {
        if (a.n_split == 1) {
#pragma unroll
            for (int x = 0; x < 2; x++) put_row(a.out, a.n_head, a.group, a.per_group, kvh, row.r, 4 * wave + hf + 2 * x, v[x], l);
        } else {
            const size_t pr = g0 + (size_t)split * KB + c;
            float *to = a.part + pr * D + 16 * wave + 4 * hf;
#pragma unroll
            for (int x = 0; x < 2; x++) {
                put64(to + 8 * x, v[x].x, v[x].y, a.xl);
                put64(to + 8 * x + 2, v[x].z, v[x].w, a.xl);
            }
            if (wave == 0 && hf == 0) {
                put64(a.part_ml + pr, m, l, a.xl);
                put64(&a.part_ml[pr].z, sc, 0.0f, a.xl);
            }
        }
    }
    if (a.tickets) join_last(a, kvh, rg, r0, rows, KB, g0, &s_last, s_w, reinterpret_cast<float4 *>(&s_kv[0][0]));
}

// ---- many rows -----------------------------------------------------------------------------------------------------------------
//
// A workgroup takes 64 rows of a KV head: 4 waves = 2 row tiles × the even / odd key blocks, the two parts merged through
// LDS at the end. A stage is 2 blocks (32 KB), K and V each double-buffered, K a stage ahead of V: the score MFMAs of the
// next stage run under the softmax of this one. The cache is f16 (q8_0 rows are read back first: each is used by many
// workgroups, and 224 VALU instructions a block and wave would be as many as the softmax's).
//
// Bound: the matrix cores' work and the softmax's instructions on the same two waves a SIMD, and the power of the two: 6001
// queries with a window of 1500 of a q8_0 cache, 149 GFLOP as pairs, 178 µs with 13 of reading back (MFMA busy 52 %, VALU
// 44 %; of zeros, at the full clock, 143). 1925 with a window of 512 27.2 µs. 128 rows a workgroup, 8 waves: 198 (their barriers
// hold twice as many).
constexpr int WR = 2, WP = 2;  // row tiles, key parts

template <bool TREE> __global__ __launch_bounds__(64 * WR * WP, 2) void k_kv_attn(Args a, TreeMask tree) {
    __shared__ __attribute__((aligned(16))) uint4_t s_kv[2][WP][TILE];  // [buffer][part][K, V chunks]
    __shared__ float s_ml[WR * WP][2][KB];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hf = lane >> 5, c = lane & 31, rt = wave & 1, kp = wave >> 1;
    const int kvh = blockIdx.x % a.kv.n_kv, rg = a.n_rg - 1 - blockIdx.x / a.kv.n_kv;  // (the longest rows first)
    const int rows = a.n * a.group, r0 = rg * KB * WR;
    const int n_keys = TREE ? a.n_past + a.n : a.pos0 + a.n;
    const Blocks blk = blocks_of<TREE, KB>(a, query_of(a.group, a.per_group, r0),
                                             query_of(a.group, a.per_group, min(r0 + KB * WR - 1, rows - 1)));
    const int nb = blk.count(), n_stage = (nb + WP - 1) / WP;
    const char *kh = (const char *)a.kv.k + (size_t)kvh * a.kv.n_ctx * (2 * D);
    const char *vh = (const char *)a.kv.v + (size_t)kvh * a.kv.n_ctx * (2 * D);

    // a stage's K or V → buffer b: 4 direct loads a wave, each of the 4 waves 4 rows of 16 (keys past the last: the last). A
    // stage's place is worked out once, for its K, and kept for its V a stage later
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4_t *)&s_kv[0][0][64 * wave];
    const int lrow = 4 * wave + (lane >> 4), lc = lane & 15;
    const uint32_t koff = 16 * (lc ^ (lrow & 15)), voff = 16 * (lc ^ (4 * (lrow & 3)));  // the same for row lrow + 16
    struct Place {
        size_t at[WP];  // the blocks' first byte
        int last[WP];   // their last row of a key
    };
    const int skip = blk.from - blk.first, skip_mem = skip - a.shift / KB;
    auto place = [&](int st) {
        Place x;
#pragma unroll
        for (int p = 0; p < WP; p++) {
            const int i = min(WP * st + p, nb - 1), past = i >= blk.first ? 1 : 0;
            x.at[p] = (size_t)(uint32_t)(i + past * skip_mem) * (KB * 2 * D);
            x.last[p] = min(n_keys - 1 - KB * (i + past * skip), KB - 1);
        }
        return x;
    };
    auto issue = [&](const Place &x, int b, bool is_v) {
#pragma unroll
        for (int p = 0; p < WP; p++) {
            const char *base = (is_v ? vh : kh) + x.at[p];
            const uint32_t off = is_v ? voff : koff, last = 2 * D * x.last[p] + off;
#pragma unroll
            for (int h = 0; h < 2; h++)
                lds_load16(base, min(2 * D * (16 * h + lrow) + off, last),
                           lds + 16u * ((b * WP + p) * TILE + (is_v ? K_CHUNKS : 0) + 256 * h));
        }
    };
    Place next = place(0);  // of stage st + 1
    issue(next, 0, false);
    issue(next, 0, true);
    if (n_stage > 1) issue(next = place(1), 1, false);

    const Row<TREE> row(a, tree, kvh, r0 + KB * rt + c);
    const int ta = query_of(a.group, a.per_group, min(r0 + KB * rt, rows - 1));
    const int tb = query_of(a.group, a.per_group, min(r0 + KB * rt + KB - 1, rows - 1));
    half8 qh[8], ql[8];
    const float sc = q_pairs<8, 2>(a.q + (size_t)row.t * a.q_stride + (size_t)row.head * D + 8 * hf, a.scale, qh, ql);
    int ka[8], va[4];
#pragma unroll
    for (int ks = 0; ks < 8; ks++) ka[ks] = 16 * c + ((2 * ks + hf) ^ (c & 15));
    const int vrow = 4 * hf + ((lane & 15) >> 2);
#pragma unroll
    for (int u = 0; u < 4; u++)
        va[u] = 16 * (K_CHUNKS + 16 * vrow + ((4 * u + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ (4 * (vrow & 3)))) + 8 * (lane & 1);

    f32x16 o[4];
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
        for (int x = 0; x < 16; x++) o[u][x] = 0.0f;
    float m = M_NONE, l = 0.0f;

    // stage st in buffer b: its scores are in s; the next stage's are computed into sn under the softmax's VALU work
    auto step = [&](int st, int b, f32x16 &s, f32x16 &sn, auto is_masked) {
        constexpr bool MASK = decltype(is_masked)::value;
        // this wave's loads of K stage st + 1 and V stage st are in, its reads of K stage st and V stage st − 1 have their
        // values; behind the barrier everyone's, and the two buffers are free
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (st + 1 < n_stage) {
            const Place now = next;
            if (st + 2 < n_stage) issue(next = place(st + 2), b, false);
            issue(now, b ^ 1, true);
        }
        uint32_t seen = 0;
        if constexpr (MASK) {
            const int i = WP * st + kp;
            seen = i < nb ? sees<TREE>(a, row.pos, row.mask, KB * blk.at(i) + here(4 * hf)) : 0u;
#pragma unroll
            for (int x = 0; x < 16; x++) s[x] = seen >> (8 * (x >> 2) + (x & 3)) & 1 ? s[x] : -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int x = 1; x < 16; x++) mx = fmaxf(mx, s[x]);
        mx = pair_max<32>(mx);
        const bool up = (mx - m) * sc > P_ROOM;
        if (__builtin_amdgcn_ballot_w64(up)) {
            const float to = up ? mx : m, corr = __builtin_amdgcn_exp2f((m - to) * sc);
            m = to;
            l *= corr;
#pragma unroll
            for (int u = 0; u < 4; u++) o[u] *= corr;
        }
        // the order pinned: behind each score MFMA of the next stage its share of this stage's softmax (left to itself the
        // compiler issues the MFMAs back to back and the softmax behind them)
        // (past the last stage: scores of what the buffer holds, not used)
        const uint4_t *kb = s_kv[b ^ 1][kp];
        const auto *vb = (const __attribute__((address_space(3))) char *)s_kv[b][kp];
        auto vread = [&](int u, int ss) {
            const auto *p = vb + va[u] + 256 * 16 * ss;
            const fp16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)p);
            const fp16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)(p + 256 * 8));
            half8 v;
            __builtin_memcpy(&v, &lo, 8);
            __builtin_memcpy((char *)&v + 8, &up, 8);
            return v;
        };
        uint32_t ph[8], pl[8];
        float ls;
        half8 f[8], v[4];
#pragma unroll
        for (int ks = 0; ks < 3; ks++) f[ks] = *reinterpret_cast<const half8 *>(kb + ka[ks]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < 8; ks++) {
            sn = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[ks], qh[ks], ks ? sn : f32x16{}, 0, 0, 0);
            if (ks + 3 < 8) f[ks + 3] = *reinterpret_cast<const half8 *>(kb + ka[ks + 3]);
            else v[ks - 5] = vread(ks - 5, 0);
            const float2_t p = {__builtin_amdgcn_exp2f(fmaf(s[2 * ks] - m, sc, P_SHIFT)),
                                __builtin_amdgcn_exp2f(fmaf(s[2 * ks + 1] - m, sc, P_SHIFT))};  // not seen: 2^(−∞) = 0
            const half2_t hi = __builtin_convertvector(p, half2_t);
            __builtin_memcpy(&ph[ks], &hi, 4);
            asm volatile("" : "+v"(ph[ks]));  // holds the conversion here
            __builtin_amdgcn_sched_barrier(0);
            sn = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[ks], ql[ks], sn, 0, 0, 0);
            ls = ks ? ls + p[0] : p[0];
            ls += p[1];
            const half2_t lo = __builtin_convertvector((float2_t{minus_half<0>(p[0], ph[ks]), minus_half<1>(p[1], ph[ks])}), half2_t);
            __builtin_memcpy(&pl[ks], &lo, 4);
            asm volatile("" : "+v"(pl[ks]));
            __builtin_amdgcn_sched_barrier(0);
        }
        v[3] = vread(3, 0);
        l += ls;
        bool odd = false;
        if constexpr (MASK) {
            uint32_t top = 0;
#pragma unroll
            for (int u = 0; u < 4; u++) largest(v[u], top), largest(vread(u, 1), top);
            odd = any_not_finite(top);
        }
#pragma unroll
        for (int ss = 0; ss < 2; ss++) {
            half8 h8, l8;
            __builtin_memcpy(&h8, &ph[4 * ss], 16);
            __builtin_memcpy(&l8, &pl[4 * ss], 16);
            half8 vn[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (odd) v[u] = finite(v[u]);
                o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[u], h8, o[u], 0, 0, 0);
                if (ss == 0) vn[u] = vread(u, 1);
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[u], l8, o[u], 0, 0, 0);
                if (ss == 0) v[u] = vn[u];
            }
        }
        if constexpr (MASK)
            if (odd) put_nan(o, seen, vread);
    };
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // K and V stage 0, K stage 1
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    f32x16 s0, s1;
#pragma unroll
    for (int ks = 0; ks < 8; ks++) {
        const half8 f = *reinterpret_cast<const half8 *>(s_kv[0][kp] + ka[ks]);
        s0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, qh[ks], ks ? s0 : f32x16{}, 0, 0, 0);
        s0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, ql[ks], s0, 0, 0, 0);
    }
    // two stages at a time, both kinds of step passing one barrier a stage: a wave's blocks may be masked where another's
    // are not
    const Whole<TREE, KB> full(a, ta, tb);
    auto whole = [&](int st) { return WP * st + kp < nb && full.block(blk.at(WP * st + kp)); };
    for (int st = 0; st < n_stage;) {
        for (; st + 1 < n_stage && whole(st) && whole(st + 1); st += 2) {
            step(st, 0, s0, s1, std::false_type{});
            step(st + 1, 1, s1, s0, std::false_type{});
        }
        for (int e = st + 2; st < min(e, n_stage); st++) {
            step(st, st & 1, s0, s1, std::true_type{});
            s0 = s1;
        }
    }
    l = pair_sum<32>(l);

    // the key parts of each row tile through LDS (the stage buffers, once every wave is done with them): every wave leaves
    // its sums as its lanes hold them, then wave (rt, kp) finishes dims 64kp … of its tile's rows
    __syncthreads();
    float4 *so = reinterpret_cast<float4 *>(&s_kv[0][0][0]);  // [wave][tile][register / 4][lane]
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
        for (int x = 0; x < 4; x++)
            so[((wave * 4 + u) * 4 + x) * 64 + lane] = make_float4(o[u][4 * x], o[u][4 * x + 1], o[u][4 * x + 2], o[u][4 * x + 3]);
    if (hf == 0) s_ml[wave][0][c] = m, s_ml[wave][1][c] = l;
    __syncthreads();
    if (row.r >= rows) return;
    const float m0 = s_ml[rt][0][c], m1 = s_ml[WR + rt][0][c], top = fmaxf(m0, m1);
    float w0 = __builtin_amdgcn_exp2f((m0 - top) * sc), w1 = __builtin_amdgcn_exp2f((m1 - top) * sc);
    const float sum = fmaf(s_ml[rt][1][c], w0, s_ml[WR + rt][1][c] * w1), inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // no key: zeros
    float *orow = a.out + ((size_t)row.t * a.n_head + row.head) * D + 64 * kp + 4 * hf;
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
        for (int x = 0; x < 4; x++) {
            const float4 y0 = so[((rt * 4 + 2 * kp + u) * 4 + x) * 64 + lane], y1 = so[(((WR + rt) * 4 + 2 * kp + u) * 4 + x) * 64 + lane];
            *reinterpret_cast<float4 *>(orow + 32 * u + 8 * x) =
                make_float4(fmaf(y0.x, w0, y1.x * w1) * inv, fmaf(y0.y, w0, y1.y * w1) * inv,
                            fmaf(y0.z, w0, y1.z * w1) * inv, fmaf(y0.w, w0, y1.w * w1) * inv);
        }
}

// the rows that the queries see, read back into room of the device's: from_row on after the first sink_rows, or all of them
// where what lies between is at most a quarter: one launch, 3 µs less than two (2000 queries with a window of 4096 from 4500 on
// 121.5 and 124.9 µs, from 16000 on, three quarters between, 124.3 and 122.2)
int read_back(htr_device *dev, Args &a, int n_keys, int sink_rows, int from_row) {
    if (from_row - sink_rows <= n_keys / 4) sink_rows = from_row = 0;
    const int first = std::min(sink_rows, n_keys), rest = std::max(0, n_keys - from_row);
    const size_t rows = (size_t)sink_rows + rest, bytes = rows * a.kv.n_kv * D * 2;
    void *p;
    HTR_TRY(htr_scratch_kept(dev, SCR_KV_ROWS, 2 * bytes, &p));
    const HtrKvPlanes src = a.kv, dst{p, (char *)p + bytes, nullptr, nullptr, src.n_kv, (int)rows, false};
    if (first) HTR_TRY(htr_kv_read_back(dev, src, 0, dst, 0, first));
    if (rest) HTR_TRY(htr_kv_read_back(dev, src, from_row, dst, sink_rows, rest));
    a.kv = dst, a.shift = from_row - sink_rows;
    return 0;
}

// FEW: 16 rows a workgroup in rounds of 128 keys; else 32 rows in rounds of 256, each of the waves its own blocks of 32
template <bool TREE, bool FEW> int launch_split(htr_device *dev, Args &a, const TreeMask &tree, int max_keys) {
    const int rows = a.n * a.group, tile = FEW ? FR : KB, run = (FEW ? UK : KB) * SW;
    a.n_rg = (rows + tile - 1) / tile;
    const int groups = a.n_rg * a.kv.n_kv, max_run = (max_keys + run - 1) / run;
    // a workgroup a CU, no more parts than rounds; no parts where they would save less than they cost: 64 tokens over 700 keys
    // (3 rounds) 9.0 µs, in parts 11.3; one over 380 keys (3) 6.8 and 7.3, over 500 (4) 7.9 and 7.4
    a.n_split = std::max(1, std::min({dev->n_cu / groups, max_run, MAX_SPLIT}));
    if (max_run <= 3) a.n_split = 1;
    a.xl = groups % 8 == 0 && dev->xcd_round_robin == 1;  // (a launch's workgroups go to the 8 XCDs in turn)
    const bool same = std::min(rows, tile) * a.n_split <= (a.xl ? JOIN_L2 : JOIN_FAR);
    if (a.n_split > 1) {
        void *p;
        HTR_TRY(htr_scratch(dev, SCR_KV_TICKET, (size_t)dev->n_cu * TICKET * 4, &p));
        if (same) a.tickets = (uint32_t *)p;
        const size_t most = (size_t)dev->n_cu * KB;  // rows of partial sums
        HTR_TRY(htr_scratch(dev, SCR_KV_ATTN, most * (D + 4) * 4, &p));
        a.part = (float *)p;
        a.part_ml = (float4 *)(a.part + most * D);
        if (!same) a.xl = 1;  // (the launch's end hands its stores on)
    }
    const dim3 g((unsigned)a.kv.n_kv, (unsigned)a.n_rg, (unsigned)a.n_split), b(64 * SW);
    if constexpr (FEW) {
        if (a.kv.q8) hipLaunchKernelGGL((k_kv_attn_few<true, TREE>), g, b, 0, dev->stream, a, tree);
        else hipLaunchKernelGGL((k_kv_attn_few<false, TREE>), g, b, 0, dev->stream, a, tree);
    } else {
        if (a.kv.q8) hipLaunchKernelGGL((k_kv_attn_split<true, TREE>), g, b, 0, dev->stream, a, tree);
        else hipLaunchKernelGGL((k_kv_attn_split<false, TREE>), g, b, 0, dev->stream, a, tree);
    }
    HTR_TRY(htr_launched(dev, FEW ? "k_kv_attn_few" : "k_kv_attn_split"));
    if (a.n_split == 1 || same) return 0;
    const JoinArgs ja{a.part, a.part_ml, a.out, a.per_group, a.n_split, a.n_head, a.group, rows, a.kv.n_kv, a.n_rg, tile};
    hipLaunchKernelGGL(k_kv_attn_join, dim3((unsigned)((rows * a.kv.n_kv + 1) / 2)), dim3(256), 0, dev->stream, ja);
    return htr_launched(dev, "k_kv_attn_join");
}

// max_keys: the most keys that the queries of a row group see; sink_rows, from_row: the rows 0 … sink_rows − 1 and from_row …
// (both multiples of 32) hold all that is seen
template <bool TREE> int launch(htr_device *dev, Args &a, const TreeMask &tree, int max_keys, int sink_rows, int from_row) {
    const int rows = a.n * a.group;
    // from more than three rounds of 32-row workgroups on the kernel of many rows: with a window of 4096 f16 keys 1000 queries (two
    // rounds) take 61 µs by workgroups of 32 rows and 72 by it, 1500 (three) 88 and 106, 1750 (four) 117 and 107, 4000 233 and 201;
    // of q8_0 80 and 90, 117 and 123, 153 and 122; 1500 from position 0 without a window 35 and 35, 2000 52 and 43
    if (rows > KB && (int64_t)((rows + KB - 1) / KB) * a.kv.n_kv > 3 * dev->n_cu) {
        a.n_rg = (rows + KB * WR - 1) / (KB * WR), a.n_split = 1;
        const unsigned groups = (unsigned)a.n_rg * (unsigned)a.kv.n_kv;  // (check_rows: they fit)
        if (a.kv.q8) HTR_TRY(read_back(dev, a, TREE ? a.n_past + a.n : a.pos0 + a.n, sink_rows, from_row));
        hipLaunchKernelGGL((k_kv_attn<TREE>), dim3(groups), dim3(64 * WR * WP), 0, dev->stream, a, tree);
        return htr_launched(dev, "k_kv_attn");
    }
    if (rows <= FR) return launch_split<TREE, true>(dev, a, tree, max_keys);
    return launch_split<TREE, false>(dev, a, tree, max_keys);
}

int check_rows(const char *me, const float *d_q, size_t q_stride, const htr_kv *kv, const HtrKvPlanes &planes, int n_head,
               float *d_out, int64_t n) {
    if (!d_q || !d_out) return htr_fail("%s: null argument", me);
    if (n_head < 1 || n_head % kv->n_kv) return htr_fail("%s: %d q heads on %d KV heads", me, n_head, kv->n_kv);
    const size_t qd = (size_t)n_head * D;
    if (q_stride < qd || (q_stride & 3))
        return htr_fail("%s: rows %zu floats apart (a multiple of 4, at least %zu)", me, q_stride, qd);
    if (((uintptr_t)d_q | (uintptr_t)d_out) & 15) return htr_fail("%s: pointers must be 16-byte aligned", me);
    const int64_t group = n_head / kv->n_kv;  // (rows · group < 2^32: the kernels' quotients)
    if (n * group > 1 << 30 || n * group * group >= 1ll << 32 ||
        (n * group + KB * WR - 1) / (KB * WR) * kv->n_kv > (int64_t)HTR_MAX_GROUPS)  // (those of the kernel of many rows)
        return htr_fail("%s: %lld queries of %d heads", me, (long long)n, n_head);
    const uintptr_t q0 = (uintptr_t)d_q, q1 = q0 + 4 * (q_stride * (n - 1) + qd), o0 = (uintptr_t)d_out, o1 = o0 + 4 * qd * n;
    if (q0 < o1 && o0 < q1) return htr_fail("%s: the output overlaps the queries", me);
    if (htr_kv_overlaps(planes, d_out, 4 * qd * n)) return htr_fail("%s: the output overlaps the cache", me);
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
    HTR_TRY(check_rows(me, d_q, q_stride, kv, a.kv, n_head, d_out, n));
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
    a.per_group = (uint32_t)(((1ull << 32) + a.group - 1) / a.group);
    a.scale = scale, a.n_past = n_past;
    return launch<true>(dev, a, tree, n_past + n, 0, 0);
}

extern "C" int htr_window_attention(htr_device *dev, const float *d_q, size_t q_stride, int n_q, int pos0, int window,
                                    int n_sink, const htr_kv *kv, int n_head, float scale, float *d_out) {
    const char *me = "htr_window_attention";
    Args a{};
    HTR_TRY(htr_kv_check(me, kv, &a.kv));
    if (n_q < 1 || pos0 < 0 || pos0 > kv->n_ctx - n_q)
        return htr_fail("%s: %d queries from position %d in a %d-row cache", me, n_q, pos0, kv->n_ctx);
    if (window < 1 || n_sink < 0) return htr_fail("%s: a window of %d keys and %d first ones", me, window, n_sink);
    HTR_TRY(check_rows(me, d_q, q_stride, kv, a.kv, n_head, d_out, n_q));
    HTR_TRY(htr_check_alive(dev));
    const HtrOnDevice on(dev);
    a.q = d_q, a.q_stride = q_stride, a.out = d_out, a.n = n_q, a.n_head = n_head, a.group = n_head / kv->n_kv;
    a.per_group = (uint32_t)(((1ull << 32) + a.group - 1) / a.group);
    a.scale = scale, a.pos0 = pos0, a.window = std::min(window, pos0 + n_q), a.n_sink = n_sink;
    const int n_keys = pos0 + n_q, sink = std::min(n_sink, n_keys), sink_rows = (sink + KB - 1) / KB * KB;
    const int from = window > pos0 ? 0 : (pos0 - window + 1) / KB * KB;
    const int64_t span = (int64_t)window + sink + 64;  // of 64 rows' queries
    return launch<false>(dev, a, TreeMask{}, (int)std::min<int64_t>(n_keys, span), sink_rows, std::max(from, sink_rows));
}
