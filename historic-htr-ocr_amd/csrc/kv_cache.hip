// A layer's KV cache in f16 or q8_0 rows: rows normed, turned and stored at positions of their own, rows copied between
// caches of either type (quantised, read back), and rows gathered in place.
//
// q8_0 rows are blocks of 32 values of a head's 128: int8 quants q and one f16 scale d, which stand for f16(q·d), the value
// the read-back gives and the attention works with. For a block of finite values x, saturated to ±65468.5 (127 times the
// largest scale whose 127-fold f16 holds: f16's own largest, 65504, moves by less than a twelfth of its step of 515.5),
//   d = the smallest f16 number with 127·d ≥ max |x|,   q = x / d rounded to the nearest integer, ties to even,
// so |q| ≤ 127 without a clamp and |x − q·d| ≤ d / 2, down to the smallest blocks (a d rounded to nearest would lose up to
// half of a block whose scale is among f16's last subnormals). Both are exact: the quotient's rounding is checked against
// the exact remainder x − q·d, which f32 holds. A block with a NaN or an infinity gets a NaN scale.
//
// Bound: memory; each value passes once. Times below are of calls one after another on an MI355X, where 480008 rows of 8 heads,
// past every cache, pass at 5.7 TB/s (f16 rows copied, 3.9 GB), 5.8 (quantised), 6.0 (read back, 3.0 GB each) and 6.3 (q8_0
// rows copied, 2.1 GB), and a plain copy of 4 GiB at 5.0.
#include <algorithm>

#include "kv_ops.h"
#include "wave.h"

namespace {

constexpr int D = 128, KV_BLOCK = 32;
constexpr float Q8_MAX = 127.0f * 515.5f;  // 515.5: the largest scale whose 127-fold f16 holds
constexpr uint32_t F32_INF = 0x7F800000u;

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

// the f16 scale (as bits) of a block whose largest |x| has the f32 bits `top`
__device__ __forceinline__ uint32_t block_scale(uint32_t top) {
    if (top >= F32_INF) return 0x7E00u;  // a NaN or an infinity
    const float a = fminf(__uint_as_float(top), Q8_MAX);
    const _Float16 h = (_Float16)(a * (1.0f / 127.0f));
    uint16_t b;
    __builtin_memcpy(&b, &h, 2);
    return 127.0f * (float)h < a ? b + 1u : b;  // 127·h is exact: 18 bits
}
// what is read once
template <typename T> __device__ __forceinline__ T load_once(const void *p) {
    return __builtin_nontemporal_load((const __attribute__((address_space(1))) T *)(uintptr_t)p);
}

__device__ __forceinline__ float half_bits(uint32_t b) {
    const uint16_t u = (uint16_t)b;
    _Float16 h;
    __builtin_memcpy(&h, &u, 2);
    return (float)h;
}

// x / d rounded to the nearest integer, ties to even, for |x| ≤ 127·d and d > 0 (inv ≈ 1 / d): the quotient in f32 is within
// 2^-16, so r is the nearest integer or, beside a border, its neighbour; x − r·d is exact in f32
__device__ __forceinline__ int quant(float x, float d, float inv) {
    float r = rintf(x * inv);
    const float e = fmaf(-r, d, x), hd = 0.5f * d;
    const bool odd = ((int)r & 1) != 0;
    if (e > hd || (e == hd && odd)) r += 1.0f;
    else if (e < -hd || (e == -hd && odd)) r -= 1.0f;
    return (int)r;
}
// N of a block's values (|x| ≤ 127·d, or not where the block is not finite), its scale's bits → N quants. x / d + 1.5·2^23 is
// rounded to an integer, two's complement in its low byte; where no remainder reaches half a scale those are the quants
template <int N> __device__ __forceinline__ void quants(const float (&x)[N], uint32_t db, uint32_t *w) {
#pragma unroll
    for (int h = 0; h < N / 4; h++) w[h] = 0u;
    if (db == 0u || db > 0x7C00u) return;
    const float d = half_bits(db), inv = 1.0f / d, big = 12582912.0f;
    uint32_t t[N];
    float far = 0.0f;
#pragma unroll
    for (int e = 0; e < N; e++) {
        const float y = fmaf(x[e], inv, big);
        t[e] = __float_as_uint(y);
        far = fmaxf(far, fabsf(fmaf(big - y, d, x[e])));
    }
    if (far >= 0.5f * d) {  // (4e-5 of the values)
#pragma unroll
        for (int e = 0; e < N; e++) t[e] = (uint32_t)quant(x[e], d, inv);
    }
#pragma unroll
    for (int h = 0; h < N / 4; h++)  // the low bytes of four words
        w[h] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(t[4 * h + 3], t[4 * h + 2], 0x0c0c0400u),
                                     __builtin_amdgcn_perm(t[4 * h + 1], t[4 * h], 0x0c0c0400u), 0x05040100u);
}
typedef uint16_t ushort2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max2_u16(uint32_t a, uint32_t b) {
    ushort2_t x, y;
    __builtin_memcpy(&x, &a, 4);
    __builtin_memcpy(&y, &b, 4);
    x = __builtin_elementwise_max(x, y);
    __builtin_memcpy(&a, &x, 4);
    return a;
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// the largest over the 8 lanes of a block
__device__ __forceinline__ uint32_t block_max(uint32_t v, int lane) {
    v = max(v, lane_swap_u32<4>(v, lane));
    v = max(v, lane_swap_u32<2>(v, lane));
    return max(v, lane_swap_u32<1>(v, lane));
}

__device__ __forceinline__ half2_t scale_pair(uint16_t bits) {
    _Float16 h;
    __builtin_memcpy(&h, &bits, 2);
    return half2_t{h, h};
}

// ---- rows normed, turned and stored ------------------------------------------------------------------------------------

// the value of the lane across lane bit M (as lane_swap)
template <int M> __device__ __forceinline__ double swap_f64(double v, int lane) {
    uint32_t u[2];
    __builtin_memcpy(u, &v, 8);
#pragma unroll
    for (int i = 0; i < 2; i++) u[i] = lane_swap_u32<M>(u[i], lane);
    __builtin_memcpy(&v, u, 8);
    return v;
}
// Σ over the 16 lanes of a row of lanes
__device__ __forceinline__ double row_sum(double v, int lane) {
    v += swap_f64<8>(v, lane);
    v += swap_f64<4>(v, lane);
    v += swap_f64<2>(v, lane);
    return v + swap_f64<1>(v, lane);
}

// 1 / √t: the hardware's estimate (2^-23 or better), squared twice by Newton's step
__device__ __forceinline__ double inv_sqrt(double t) {
    double r = __builtin_amdgcn_rsq(t);
#pragma unroll
    for (int i = 0; i < 2; i++) r = fma(0.5 * r, fma(-t * r, r, 1.0), r);
    return t == INFINITY ? 0.0 : r;
}

struct PostRowsArgs {
    const float *q, *k, *v;
    size_t q_stride, kv_stride;
    const float *qn, *kn, *rope;
    float *q_out;
    HtrKvPlanes kv;
    double eps;
    int n, n_head, pos0, row0;
    const int32_t *pos, *slot;  // PAGES: each row's position and its row of the cache
    int n_pos;
};
enum Place { IN_ORDER, DRAFT, PAGES };  // rows one after another; a draft's positions by depth; both from arrays
struct TreeDepth {
    uint8_t at[HTR_TREE_MAX];
};

// One head of one row to 16 lanes of dims 4j … 4j + 3 and 64 + 4j …, a turn's pairs in one lane. The norm and the turn are in
// f64: what they give is rounded to f32, then to the cache's type, and lies next to a border of that type often enough (4e-4
// of f16 values for f32 sums, an f16 ulp off each, and as many q8_0 quants a step off) that f32 sums would give each order of
// summation a cache of its own. Its 70 operations a lane hide behind the lane's 100 bytes: 1925 rows of 16 + 2·8 heads into
// q8_0 (51 MB) 10.5 µs, 4.9 TB/s, into f16 (55 MB) 10.1; with the library's 1 / sqrt, and V's heads taken through it all too,
// 11.9 and 11.2; with 8 dims in a row to a lane, whose loads skip every other 16 bytes, 13.5 and 13.4. One row: 4 µs, a launch.
template <bool Q8, Place PLACE> __global__ __launch_bounds__(256) void k_post_rows(PostRowsArgs a, TreeDepth depth) {
    const int lane = threadIdx.x & 63, j = lane & 15, heads = a.n_head + 2 * a.kv.n_kv;
    const uint32_t id = blockIdx.x * 16u + (threadIdx.x >> 4), count = (uint32_t)a.n * heads, at = min(id, count - 1);
    const int t = (int)(at / (uint32_t)heads), h = (int)at - t * heads, kvh = h - a.n_head;
    const bool is_q = kvh < 0, is_v = kvh >= a.kv.n_kv;
    int pos = a.pos0 + (PLACE == DRAFT ? depth.at[t] : t), to = a.row0 + t;
    if constexpr (PLACE == PAGES) {  // (the 16 lanes of a head's row go together)
        pos = a.pos[t], to = is_q ? 0 : a.slot[t];
        if ((uint32_t)pos >= (uint32_t)a.n_pos || (uint32_t)to >= (uint32_t)a.kv.n_ctx) return;
    }
    const float *src = is_q   ? a.q + t * a.q_stride + (size_t)h * D
                       : is_v ? a.v + t * a.kv_stride + (size_t)(kvh - a.kv.n_kv) * D
                              : a.k + t * a.kv_stride + (size_t)kvh * D;
    float y[2][4];
#pragma unroll
    for (int u = 0; u < 2; u++) *reinterpret_cast<float4 *>(y[u]) = *reinterpret_cast<const float4 *>(src + 64 * u + 4 * j);
    if (!is_v) {
        const float *w = is_q ? a.qn : a.kn, *turn = a.rope + (size_t)pos * D + 8 * j;
        float wf[2][4], cs[8];
#pragma unroll
        for (int u = 0; u < 2; u++) *reinterpret_cast<float4 *>(wf[u]) = *reinterpret_cast<const float4 *>(w + 64 * u + 4 * j);
#pragma unroll
        for (int u = 0; u < 2; u++) *reinterpret_cast<float4 *>(cs + 4 * u) = *reinterpret_cast<const float4 *>(turn + 4 * u);
        double ss = 0.0;
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) ss = fma((double)y[u][e], (double)y[u][e], ss);
        const double inv = inv_sqrt(fma(row_sum(ss, lane), 1.0 / D, a.eps));
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const double lo = (double)y[0][e] * inv * (double)wf[0][e], up = (double)y[1][e] * inv * (double)wf[1][e];
            const double c = (double)cs[2 * e], s = (double)cs[2 * e + 1];
            y[0][e] = (float)(lo * c - up * s);
            y[1][e] = (float)(lo * s + up * c);
        }
    }
    if (is_q) {
        if (id >= count) return;
        float *o = a.q_out + ((size_t)t * a.n_head + h) * D + 4 * j;
#pragma unroll
        for (int u = 0; u < 2; u++) *reinterpret_cast<float4 *>(o + 64 * u) = make_float4(y[u][0], y[u][1], y[u][2], y[u][3]);
        return;
    }
    const int head = is_v ? kvh - a.kv.n_kv : kvh;
    const size_t row = (size_t)head * a.kv.n_ctx + to;
    if constexpr (Q8) {
        uint32_t db[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < 4; e++) top = max(top, abs_bits(y[u][e]));
            db[u] = block_scale(block_max(top, lane));
        }
        if (id >= count) return;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            uint32_t quad;
#pragma unroll
            for (int e = 0; e < 4; e++) y[u][e] = fminf(fmaxf(y[u][e], -Q8_MAX), Q8_MAX);
            quants(y[u], db[u], &quad);
            *reinterpret_cast<uint32_t *>((char *)(is_v ? a.kv.v : a.kv.k) + row * D + 64 * u + 4 * j) = quad;
            if ((j & 7) == 0) (is_v ? a.kv.vd : a.kv.kd)[row * (D / KV_BLOCK) + 2 * u + (j >> 3)] = (uint16_t)db[u];
        }
    } else {
        if (id >= count) return;
#pragma unroll
        for (int u = 0; u < 2; u++) {
            half4 o;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = (_Float16)y[u][e];
            *reinterpret_cast<half4 *>((_Float16 *)(is_v ? a.kv.v : a.kv.k) + row * D + 64 * u + 4 * j) = o;
        }
    }
}

// ---- rows between caches -------------------------------------------------------------------------------------------------

struct CopyArgs {
    HtrKvPlanes src, dst;
    int src_row, dst_row, n;
};
constexpr int COPY_ROWS = 32, BACK_ROWS = 64;  // rows a workgroup: of a copy or quantised, read back

// blockIdx.y: K and V of each KV head. The f16 rows pass the caches without staying (nontemporal loads, and the read-back's
// stores): 60001 rows of 8 heads quantised and read back, 376 MB each, take 113.7 µs (6.6 TB/s: the quants are still in the last
// cache); 126 with plain stores, 139 with plain loads too (2437 rows: 10.0, 10.0, 9.7).
//
// Quantise: 8 lanes of 16 values to a row, 2 lanes to a block; the workgroup's scales through LDS, so that they leave as whole
// lines too. Alone 66.6 and (2437 rows) 5.2 µs, with 64 rows a workgroup 70.2 and 6.6. Copies: f16 84.3 µs (491 MB), q8_0 44.0
// (261 MB), with 64 rows 88.0 and 44.1, with 16 82.4 and 48.3
__global__ __launch_bounds__(256) void k_kv_quantise(CopyArgs a) {
    __shared__ __attribute__((aligned(8))) uint16_t s_d[COPY_ROWS][4];
    const int tid = threadIdx.x, lane = tid & 63, j = tid & 7, head = blockIdx.y >> 1, is_v = blockIdx.y & 1;
    const _Float16 *src = (const _Float16 *)(is_v ? a.src.v : a.src.k) + ((size_t)head * a.src.n_ctx + a.src_row) * D;
    const size_t to = (size_t)head * a.dst.n_ctx + a.dst_row;
    const int r0 = blockIdx.x * COPY_ROWS, r = tid >> 3;
    uint4_t in[2];
#pragma unroll
    for (int h = 0; h < 2; h++) in[h] = load_once<uint4_t>(src + (size_t)min(r0 + r, a.n - 1) * D + 16 * j + 8 * h);
    // (f16's largest, 65504, is 127.07 of the largest scale: its quant is 127 without being saturated first)
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int e = 0; e < 4; e++) top = max2_u16(top, in[h][e] & 0x7FFF7FFFu);
    top = max(top & 0xFFFFu, top >> 16);  // as f16 bits: those of an infinity and past are the largest too
    top = max(top, lane_swap_u32<1>(top, lane));
    const uint32_t db = block_scale(abs_bits(half_bits(top)));
    uint4_t q;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        half8 v;
        __builtin_memcpy(&v, &in[h], 16);
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (float)v[e];
        uint32_t w[2];
        quants(x, db, w);
        q[2 * h] = w[0], q[2 * h + 1] = w[1];
    }
    if (r0 + r < a.n) *reinterpret_cast<uint4_t *>((char *)(is_v ? a.dst.v : a.dst.k) + (to + r0 + r) * D + 16 * j) = q;
    if ((j & 1) == 0) s_d[r][j >> 1] = (uint16_t)db;
    __syncthreads();
    if (tid < COPY_ROWS && r0 + tid < a.n)
        reinterpret_cast<uint2_t *>((is_v ? a.dst.vd : a.dst.kd) + to * (D / KV_BLOCK))[r0 + tid] = *reinterpret_cast<const uint2_t *>(s_d[tid]);
}

// read back: 16 lanes of 8 values to a row (whole lines leave a wave at once). With plain loads and stores 65.3 µs alone, 2437
// rows 3.9; with 32 rows a workgroup 66.7 and 3.9, with 128 67.3 and 4.2
__global__ __launch_bounds__(256) void k_kv_read_back(CopyArgs a) {
    const int j = threadIdx.x & 15, head = blockIdx.y >> 1, is_v = blockIdx.y & 1;
    const size_t from = (size_t)head * a.src.n_ctx + a.src_row, to = (size_t)head * a.dst.n_ctx + a.dst_row;
    const int r0 = blockIdx.x * BACK_ROWS + (threadIdx.x >> 4);
    uint2_t q[BACK_ROWS / 16];
    uint16_t d[BACK_ROWS / 16];
#pragma unroll
    for (int i = 0; i < BACK_ROWS / 16; i++) {
        const size_t row = from + min(r0 + 16 * i, a.n - 1);
        q[i] = load_once<uint2_t>((const char *)(is_v ? a.src.v : a.src.k) + row * D + 8 * j);
        d[i] = (is_v ? a.src.vd : a.src.kd)[row * (D / KV_BLOCK) + (j >> 2)];
    }
#pragma unroll
    for (int i = 0; i < BACK_ROWS / 16; i++)
        if (r0 + 16 * i < a.n)
            __builtin_nontemporal_store(dequant8(q[i][0], q[i][1], scale_pair(d[i])),
                                        (__attribute__((address_space(1))) half8 *)(uintptr_t)(
                                            (_Float16 *)(is_v ? a.dst.v : a.dst.k) + (to + r0 + 16 * i) * D + 8 * j));
}

// the same type on both sides: a row's bytes (16 or 8 units of 16), its 8 bytes of scales
template <bool Q8> __global__ __launch_bounds__(256) void k_kv_copy(CopyArgs a) {
    constexpr int U = Q8 ? 8 : 16;
    const int head = blockIdx.y >> 1, is_v = blockIdx.y & 1;
    const size_t from = (size_t)head * a.src.n_ctx + a.src_row, to = (size_t)head * a.dst.n_ctx + a.dst_row;
    const uint4_t *src = (const uint4_t *)(is_v ? a.src.v : a.src.k) + from * U;
    uint4_t *dst = (uint4_t *)(is_v ? a.dst.v : a.dst.k) + to * U;
    const int r0 = blockIdx.x * COPY_ROWS, rows = min(COPY_ROWS, a.n - r0);
    for (int i = threadIdx.x; i < rows * U; i += 256) dst[(size_t)r0 * U + i] = src[(size_t)r0 * U + i];
    if (Q8 && (int)threadIdx.x < rows) {
        const uint2_t *sd = (const uint2_t *)(is_v ? a.src.vd : a.src.kd) + from;
        ((uint2_t *)(is_v ? a.dst.vd : a.dst.kd) + to)[r0 + threadIdx.x] = sd[r0 + threadIdx.x];
    }
}

// ---- rows gathered in place ----------------------------------------------------------------------------------------------

struct KeepArgs {
    HtrKvPlanes kv;
    int row0, n;
    int idx[HTR_TREE_MAX];
};
// one plane of one head to a workgroup: every row is held in registers before the first is written
template <bool Q8> __global__ __launch_bounds__(256) void k_kv_keep(KeepArgs a) {
    constexpr int U = Q8 ? 8 : 16, PER = HTR_TREE_MAX * U / 256;
    const int head = blockIdx.x >> 1, is_v = blockIdx.x & 1, tid = threadIdx.x;
    const size_t row0 = (size_t)head * a.kv.n_ctx + a.row0;
    uint4_t *rows = (uint4_t *)(is_v ? a.kv.v : a.kv.k) + row0 * U;
    uint2_t *scales = Q8 ? (uint2_t *)(is_v ? a.kv.vd : a.kv.kd) + row0 : nullptr;
    uint4_t held[PER];
    uint2_t d = {0u, 0u};
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int r = min((tid + 256 * i) / U, a.n - 1);
        held[i] = rows[(size_t)a.idx[r] * U + tid % U];
    }
    if (Q8 && tid < a.n) d = scales[a.idx[tid]];
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int r = (tid + 256 * i) / U;
        if (r < a.n) rows[(size_t)r * U + tid % U] = held[i];
    }
    if (Q8 && tid < a.n) scales[tid] = d;
}

constexpr auto overlap = htr_overlap;

}  // namespace

// ---- ABI -----------------------------------------------------------------------------------------------------------------

HtrOnDevice::HtrOnDevice(htr_device *dev) {
    if (hipGetDevice(&before) != hipSuccess) before = dev->ordinal;
    if (before != dev->ordinal) (void)hipSetDevice(dev->ordinal);
    else before = -1;
}
HtrOnDevice::~HtrOnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
}

int htr_kv_check(const char *what, const htr_kv *kv, HtrKvPlanes *out) {
    if (!kv) return htr_fail("%s: null cache", what);
    if (kv->type != HTR_GGML_F16 && kv->type != HTR_GGML_Q8_0)
        return htr_fail("%s: a cache of type %d (HTR_GGML_F16 %d or HTR_GGML_Q8_0 %d)", what, kv->type, HTR_GGML_F16,
                        HTR_GGML_Q8_0);
    if (kv->n_kv < 1 || kv->n_kv > 4096 || kv->n_ctx < 1)
        return htr_fail("%s: a cache of %d KV heads, %d rows (1 … 4096 heads, at least a row)", what, kv->n_kv, kv->n_ctx);
    if (!kv->d_k || !kv->d_v) return htr_fail("%s: null cache rows", what);
    if (((uintptr_t)kv->d_k | (uintptr_t)kv->d_v) & 15) return htr_fail("%s: the cache rows must be 16-byte aligned", what);
    const bool q8 = kv->type == HTR_GGML_Q8_0;
    if (q8 && (!kv->d_kd || !kv->d_vd)) return htr_fail("%s: a q8_0 cache without scales", what);
    if (q8 && (((uintptr_t)kv->d_kd | (uintptr_t)kv->d_vd) & 7))
        return htr_fail("%s: the cache scales must be 8-byte aligned", what);
    *out = HtrKvPlanes{kv->d_k, kv->d_v, q8 ? kv->d_kd : nullptr, q8 ? kv->d_vd : nullptr, kv->n_kv, kv->n_ctx, q8};
    return 0;
}

namespace {
dim3 copy_grid(const CopyArgs &a, int rows) { return dim3((unsigned)((a.n + rows - 1) / rows), (unsigned)(2 * a.src.n_kv)); }
}  // namespace

int htr_kv_read_back(htr_device *dev, const HtrKvPlanes &src, int src_row, const HtrKvPlanes &dst, int dst_row, int n) {
    const CopyArgs a{src, dst, src_row, dst_row, n};
    hipLaunchKernelGGL(k_kv_read_back, copy_grid(a, BACK_ROWS), dim3(256), 0, dev->stream, a);
    return htr_launched(dev, "k_kv_read_back");
}

namespace {
size_t row_bytes(const HtrKvPlanes &c) { return (size_t)c.n_kv * c.n_ctx * D * (c.q8 ? 1 : 2); }
size_t scale_bytes(const HtrKvPlanes &c) { return c.q8 ? (size_t)c.n_kv * c.n_ctx * 8 : 0; }
struct Plane {
    const void *p;
    size_t n;
};
struct Planes {
    Plane of[4];
    explicit Planes(const HtrKvPlanes &c)
        : of{{c.k, row_bytes(c)}, {c.v, row_bytes(c)}, {c.kd, scale_bytes(c)}, {c.vd, scale_bytes(c)}} {}
};
// a cache that is written to: its planes lie apart
int check_apart(const char *what, const HtrKvPlanes &kv) {
    const Planes c(kv);
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < i; j++)
            if (c.of[i].n && c.of[j].n && overlap(c.of[i].p, c.of[i].n, c.of[j].p, c.of[j].n))
                return htr_fail("%s: the cache's planes overlap", what);
    return 0;
}
}  // namespace

bool htr_kv_overlaps(const HtrKvPlanes &kv, const void *p, size_t n) {
    for (const Plane &c : Planes(kv).of)
        if (c.n && overlap(p, n, c.p, c.n)) return true;
    return false;
}

extern "C" int htr_tree_masks(const int32_t *h_parent, int n, uint64_t *h_mask, int32_t *h_depth) {
    if (!h_parent || !h_mask || !h_depth) return htr_fail("htr_tree_masks: null argument");
    if (n < 1 || n > HTR_TREE_MAX) return htr_fail("htr_tree_masks: %d nodes (1 … %d)", n, HTR_TREE_MAX);
    for (int i = 0; i < n; i++) {
        const int p = h_parent[i];
        if (p < -1 || p >= i) return htr_fail("htr_tree_masks: node %d has parent %d (an earlier node, or -1)", i, p);
        h_mask[i] = (p >= 0 ? h_mask[p] : 0) | 1ull << i;
        h_depth[i] = p >= 0 ? h_depth[p] + 1 : 0;
    }
    return 0;
}

namespace {
// the arguments that the two row writers share, checked; `rows` of the cache or of a table are theirs to check
int post_args(const char *me, const float *d_q, size_t q_stride, const float *d_k, const float *d_v, size_t kv_stride, int n,
              const float *d_q_norm, const float *d_k_norm, const float *d_rope, int n_pos, int n_head, float eps,
              const htr_kv *kv, float *d_q_out, PostRowsArgs *out, size_t *groups) {
    PostRowsArgs &a = *out;
    if (!d_q || !d_k || !d_v || !d_q_norm || !d_k_norm || !d_rope || !d_q_out) return htr_fail("%s: null argument", me);
    if (n_head < 1 || n_head % kv->n_kv) return htr_fail("%s: %d q heads on %d KV heads", me, n_head, kv->n_kv);
    const size_t qd = (size_t)n_head * D, kvd = (size_t)kv->n_kv * D;
    if (q_stride < qd || kv_stride < kvd || ((q_stride | kv_stride) & 3))
        return htr_fail("%s: rows %zu and %zu floats apart (multiples of 4, at least %zu and %zu)", me, q_stride, kv_stride,
                        qd, kvd);
    if (((uintptr_t)d_q | (uintptr_t)d_k | (uintptr_t)d_v | (uintptr_t)d_q_norm | (uintptr_t)d_k_norm | (uintptr_t)d_rope |
         (uintptr_t)d_q_out) & 15)
        return htr_fail("%s: pointers must be 16-byte aligned", me);
    a.q = d_q, a.k = d_k, a.v = d_v, a.q_stride = q_stride, a.kv_stride = kv_stride;
    a.qn = d_q_norm, a.kn = d_k_norm, a.rope = d_rope, a.q_out = d_q_out;
    a.eps = (double)eps, a.n = n, a.n_head = n_head, a.n_pos = n_pos;
    *groups = ((size_t)n * ((size_t)n_head + 2 * kv->n_kv) + 15) / 16;
    return 0;
}
int post_apart(const char *me, const PostRowsArgs &a, size_t groups) {
    // in place (q_out on q's own rows) is the only overlap that the kernel allows
    const size_t n = (size_t)a.n, qd = (size_t)a.n_head * D, kvd = (size_t)a.kv.n_kv * D;
    if (!htr_rows_fit(a.q_stride, n, qd) || !htr_rows_fit(a.kv_stride, n, kvd))
        return htr_fail("%s: %zu rows %zu and %zu floats apart", me, n, a.q_stride, a.kv_stride);
    const size_t q_bytes = 4 * (a.q_stride * (n - 1) + qd), out_bytes = 4 * qd * n;
    const size_t kv_bytes = 4 * (a.kv_stride * (n - 1) + kvd);
    if ((overlap(a.q, q_bytes, a.q_out, out_bytes) && !(a.q == a.q_out && (n == 1 || a.q_stride == qd))) ||
        overlap(a.k, kv_bytes, a.q_out, out_bytes) || overlap(a.v, kv_bytes, a.q_out, out_bytes))
        return htr_fail("%s: the q output overlaps the input rows", me);
    if (htr_kv_overlaps(a.kv, a.q, q_bytes) || htr_kv_overlaps(a.kv, a.k, kv_bytes) || htr_kv_overlaps(a.kv, a.v, kv_bytes) ||
        htr_kv_overlaps(a.kv, a.q_out, out_bytes))
        return htr_fail("%s: the rows or the q output overlap the cache", me);
    const Plane read[5] = {{a.qn, 4 * D}, {a.kn, 4 * D}, {a.rope, (size_t)a.n_pos * D * 4}, {a.pos, a.pos ? 4 * n : 0},
                           {a.slot, a.slot ? 4 * n : 0}};
    for (const auto &w : read)
        if (w.n && (overlap(w.p, w.n, a.q_out, out_bytes) || htr_kv_overlaps(a.kv, w.p, w.n)))
            return htr_fail("%s: the q output or the cache overlaps the norms' weights or the rope table%s", me,
                            a.pos ? ", or the rows' places" : "");
    if (groups > HTR_MAX_GROUPS)
        return htr_fail("%s: %d rows of %d + %d heads in one call (at most %zu heads' rows)", me, a.n, a.n_head, 2 * a.kv.n_kv,
                        16 * HTR_MAX_GROUPS);
    return 0;
}
}  // namespace

extern "C" int htr_qkv_post_rows(htr_device *dev, const float *d_q, size_t q_stride, const float *d_k, const float *d_v,
                                 size_t kv_stride, int n, const float *d_q_norm, const float *d_k_norm,
                                 const float *d_rope, int n_pos, int pos0, const int32_t *h_depth, int n_head, float eps,
                                 const htr_kv *kv, int row0, float *d_q_out) {
    const char *me = "htr_qkv_post_rows";
    PostRowsArgs a{};
    size_t groups;
    HTR_TRY(htr_kv_check(me, kv, &a.kv));
    HTR_TRY(check_apart(me, a.kv));
    HTR_TRY(post_args(me, d_q, q_stride, d_k, d_v, kv_stride, n, d_q_norm, d_k_norm, d_rope, n_pos, n_head, eps, kv, d_q_out, &a,
                      &groups));
    if (n < 1 || row0 < 0 || row0 > kv->n_ctx - n)
        return htr_fail("%s: %d rows from row %d of a %d-row cache", me, n, row0, kv->n_ctx);
    if (h_depth && n > HTR_TREE_MAX) return htr_fail("%s: %d drafted rows (at most %d)", me, n, HTR_TREE_MAX);
    TreeDepth depth{};
    int deepest = n - 1;
    if (h_depth) {
        deepest = 0;
        for (int t = 0; t < n; t++) {
            if (h_depth[t] < 0 || h_depth[t] >= HTR_TREE_MAX)
                return htr_fail("%s: row %d at depth %d (0 … %d)", me, t, h_depth[t], HTR_TREE_MAX - 1);
            depth.at[t] = (uint8_t)h_depth[t];
            deepest = std::max(deepest, h_depth[t]);
        }
    }
    if (pos0 < 0 || n_pos < 1 || deepest >= n_pos || pos0 > n_pos - 1 - deepest)
        return htr_fail("%s: positions %d … %lld of a %d-position rope table", me, pos0, (long long)pos0 + deepest, n_pos);
    HTR_TRY(post_apart(me, a, groups));
    HTR_TRY(htr_check_alive(dev));
    const HtrOnDevice on(dev);
    a.pos0 = pos0, a.row0 = row0;
    const dim3 g((unsigned)groups), b(256);
#define HTR_POST(Q8, PLACE) hipLaunchKernelGGL((k_post_rows<Q8, PLACE>), g, b, 0, dev->stream, a, depth)
    if (a.kv.q8 && h_depth) HTR_POST(true, DRAFT);
    else if (a.kv.q8) HTR_POST(true, IN_ORDER);
    else if (h_depth) HTR_POST(false, DRAFT);
    else HTR_POST(false, IN_ORDER);
    return htr_launched(dev, a.kv.q8 ? "k_post_rows<q8_0>" : "k_post_rows<f16>");
}

extern "C" int htr_qkv_post_pages(htr_device *dev, const float *d_q, size_t q_stride, const float *d_k, const float *d_v,
                                  size_t kv_stride, const htr_pages *pages, const float *d_q_norm, const float *d_k_norm,
                                  const float *d_rope, int n_pos, int n_head, float eps, const htr_kv *kv, float *d_q_out) {
    const char *me = "htr_qkv_post_pages";
    PostRowsArgs a{};
    HtrPages p;
    size_t groups;
    HTR_TRY(htr_kv_check(me, kv, &a.kv));
    HTR_TRY(check_apart(me, a.kv));
    HTR_TRY(htr_pages_check(me, pages, HTR_PAGES_ROWS, &p));
    HTR_TRY(post_args(me, d_q, q_stride, d_k, d_v, kv_stride, p.n_row, d_q_norm, d_k_norm, d_rope, n_pos, n_head, eps, kv,
                      d_q_out, &a, &groups));
    if (n_pos < 1) return htr_fail("%s: a rope table of %d positions", me, n_pos);
    a.pos = p.pos, a.slot = p.slot;
    HTR_TRY(post_apart(me, a, groups));
    HTR_TRY(htr_check_alive(dev));
    const HtrOnDevice on(dev);
    const TreeDepth depth{};
    const dim3 g((unsigned)groups), b(256);
    if (a.kv.q8) HTR_POST(true, PAGES);
    else HTR_POST(false, PAGES);
#undef HTR_POST
    return htr_launched(dev, a.kv.q8 ? "k_post_rows<q8_0, pages>" : "k_post_rows<f16, pages>");
}

extern "C" int htr_kv_copy(htr_device *dev, const htr_kv *src, int src_row, const htr_kv *dst, int dst_row, int n) {
    const char *me = "htr_kv_copy";
    CopyArgs a{};
    HTR_TRY(htr_kv_check(me, src, &a.src));
    HTR_TRY(htr_kv_check(me, dst, &a.dst));
    if (src->n_kv != dst->n_kv) return htr_fail("%s: %d KV heads into %d", me, src->n_kv, dst->n_kv);
    if (n < 0 || src_row < 0 || src_row > src->n_ctx - n || dst_row < 0 || dst_row > dst->n_ctx - n)
        return htr_fail("%s: %d rows from row %d of %d to row %d of %d", me, n, src_row, src->n_ctx, dst_row, dst->n_ctx);
    if ((size_t)n > COPY_ROWS * HTR_MAX_GROUPS)
        return htr_fail("%s: %d rows in one call (at most %zu)", me, n, COPY_ROWS * HTR_MAX_GROUPS);
    // the caches' planes: apart, or the same ones with rows apart
    HTR_TRY(check_apart(me, a.dst));
    const Planes src_planes(a.src), dst_planes(a.dst);
    const Plane *s = src_planes.of, *d = dst_planes.of;
    const bool apart = src_row + n <= dst_row || dst_row + n <= src_row;
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) {
            if (!s[i].n || !d[j].n || !overlap(s[i].p, s[i].n, d[j].p, d[j].n)) continue;
            if (!(i == j && src->type == dst->type && s[i].p == d[j].p && src->n_ctx == dst->n_ctx && apart))
                return htr_fail("%s: rows %d … of the source overlap rows %d … of the destination", me, src_row, dst_row);
        }
    HTR_TRY(htr_check_alive(dev));
    if (n == 0) return 0;
    const HtrOnDevice on(dev);
    a.src_row = src_row, a.dst_row = dst_row, a.n = n;
    const dim3 g = copy_grid(a, COPY_ROWS), b(256);
    if (!a.src.q8 && a.dst.q8) {
        hipLaunchKernelGGL(k_kv_quantise, g, b, 0, dev->stream, a);
        return htr_launched(dev, "k_kv_quantise");
    }
    if (a.src.q8 && !a.dst.q8) return htr_kv_read_back(dev, a.src, src_row, a.dst, dst_row, n);
    if (a.src.q8) hipLaunchKernelGGL(k_kv_copy<true>, g, b, 0, dev->stream, a);
    else hipLaunchKernelGGL(k_kv_copy<false>, g, b, 0, dev->stream, a);
    return htr_launched(dev, a.src.q8 ? "k_kv_copy<q8_0>" : "k_kv_copy<f16>");
}

extern "C" int htr_kv_keep(htr_device *dev, const htr_kv *kv, int row0, const int32_t *h_idx, int n) {
    const char *me = "htr_kv_keep";
    KeepArgs a{};
    HTR_TRY(htr_kv_check(me, kv, &a.kv));
    HTR_TRY(check_apart(me, a.kv));
    if (n < 0 || n > HTR_TREE_MAX) return htr_fail("%s: %d rows (at most %d)", me, n, HTR_TREE_MAX);
    if (n && !h_idx) return htr_fail("%s: null rows", me);
    if (row0 < 0 || row0 > kv->n_ctx - n) return htr_fail("%s: %d rows from row %d of %d", me, n, row0, kv->n_ctx);
    for (int i = 0; i < n; i++) {
        if (h_idx[i] < 0 || h_idx[i] >= kv->n_ctx - row0)
            return htr_fail("%s: row %d + %d of %d", me, row0, h_idx[i], kv->n_ctx);
        a.idx[i] = h_idx[i];
    }
    HTR_TRY(htr_check_alive(dev));
    if (n == 0) return 0;
    const HtrOnDevice on(dev);
    a.row0 = row0, a.n = n;
    const dim3 g((unsigned)(2 * kv->n_kv)), b(256);
    if (a.kv.q8) hipLaunchKernelGGL(k_kv_keep<true>, g, b, 0, dev->stream, a);
    else hipLaunchKernelGGL(k_kv_keep<false>, g, b, 0, dev->stream, a);
    return htr_launched(dev, a.kv.q8 ? "k_kv_keep<q8_0>" : "k_kv_keep<f16>");
}
