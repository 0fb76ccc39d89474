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
constexpr int MAX_PART_ROWS = 32768;           // rows of partial sums of one call

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float2_t __attribute__((ext_vector_type(2)));
typedef __fp16 fp16x4 __attribute__((ext_vector_type(4)));
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
    float *part;               // [n_kv·n_rg·n_split][32·WR] rows of partial sums: o[128], then (m, l, c) of all
    float *part_ml;
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
    if (a.n_split == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key seen: zeros
        float *orow = a.out + ((size_t)t * a.n_head + head) * D + 4 * hf;
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int x = 0; x < 4; x++)
                *reinterpret_cast<float4 *>(orow + 32 * u + 8 * x) =
                    make_float4(o[u][4 * x] * inv, o[u][4 * x + 1] * inv, o[u][4 * x + 2] * inv, o[u][4 * x + 3] * inv);
        return;
    }
    const size_t pr = (((size_t)kvh * a.n_rg + rg) * a.n_split + split) * (32 * WR) + 32 * rt + c;
    float *prow = a.part + pr * D + 4 * hf;
#pragma unroll
    for (int u = 0; u < 4; u++)
#pragma unroll
        for (int x = 0; x < 4; x++)
            *reinterpret_cast<float4 *>(prow + 32 * u + 8 * x) =
                make_float4(o[u][4 * x], o[u][4 * x + 1], o[u][4 * x + 2], o[u][4 * x + 3]);
    if (hf == 0) *reinterpret_cast<float4 *>(a.part_ml + 4 * pr) = make_float4(m, l, sc, 0.0f);
}

// the parts of a row joined: 32 lanes of 4 dims a row
template <int WR> __global__ __launch_bounds__(256) void k_kv_attn_join(Args a) {
    const int rows = a.n * a.group, lane = threadIdx.x & 31;
    const int id = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (id >= rows * a.kv.n_kv) return;
    const int kvh = id / rows, r = id % rows, rg = r / (32 * WR);
    const size_t pr = ((size_t)kvh * a.n_rg + rg) * a.n_split * (32 * WR) + r % (32 * WR);
    const float4 *ml = reinterpret_cast<const float4 *>(a.part_ml);
    float top = M_NONE;
    for (int p = 0; p < a.n_split; p++) top = fmaxf(top, ml[pr + (size_t)p * 32 * WR].x);
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
    for (int p = 0; p < a.n_split; p++) {
        const size_t at = pr + (size_t)p * 32 * WR;
        const float4 s = ml[at], w4 = *reinterpret_cast<const float4 *>(a.part + at * D + 4 * lane);
        const float w = __builtin_amdgcn_exp2f((s.x - top) * s.z);
        l = fmaf(s.y, w, l);
        v.x = fmaf(w4.x, w, v.x), v.y = fmaf(w4.y, w, v.y), v.z = fmaf(w4.z, w, v.z), v.w = fmaf(w4.w, w, v.w);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int t = r / a.group, head = kvh * a.group + r % a.group;
    *reinterpret_cast<float4 *>(a.out + ((size_t)t * a.n_head + head) * D + 4 * lane) =
        make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
}

template <bool TREE, int WR> int launch(htr_device *dev, Args &a, const TreeMask &tree, int max_blocks) {
    const int rows = a.n * a.group;
    a.n_rg = (rows + 32 * WR - 1) / (32 * WR);
    const int64_t wide = (int64_t)a.n_rg * a.kv.n_kv;
    // enough workgroups for every CU twice, no more parts than stages of blocks, and partial sums that fit their room
    int64_t split = 1;
    if (wide < dev->n_cu) {
        split = std::min<int64_t>((2 * dev->n_cu + wide - 1) / wide, (max_blocks + 4 / WR - 1) / (4 / WR));
        split = std::max<int64_t>(1, std::min<int64_t>(split, MAX_PART_ROWS / (wide * 32 * WR)));
    }
    a.n_split = (int)split;
    if (wide * split > INT32_MAX) return htr_fail("attention: %d rows of %d KV heads", rows, a.kv.n_kv);
    if (split > 1) {
        void *p;
        HTR_TRY(htr_scratch(dev, SCR_KV_ATTN, (size_t)MAX_PART_ROWS * (D + 4) * 4, &p));
        a.part = (float *)p;
        a.part_ml = a.part + (size_t)MAX_PART_ROWS * D;
    }
    const dim3 g((unsigned)(wide * split)), b(256);
    if (a.kv.q8) hipLaunchKernelGGL((k_kv_attn<true, TREE, WR>), g, b, 0, dev->stream, a, tree);
    else hipLaunchKernelGGL((k_kv_attn<false, TREE, WR>), g, b, 0, dev->stream, a, tree);
    HTR_TRY(htr_launched(dev, TREE ? "k_kv_attn<tree>" : "k_kv_attn<window>"));
    if (split == 1) return 0;
    hipLaunchKernelGGL(k_kv_attn_join<WR>, dim3((unsigned)(((int64_t)rows * a.kv.n_kv + 7) / 8)), b, 0, dev->stream, a);
    return htr_launched(dev, "k_kv_attn_join");
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
    return launch<true, 1>(dev, a, tree, (n_past + n + KB - 1) / KB);
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
    return launch<false, 1>(dev, a, TreeMask{}, (int)((span + KB - 1) / KB));
}
