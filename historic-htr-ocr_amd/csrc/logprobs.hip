// Log probabilities of given tokens, the entropy of the distribution that each was chosen from, and the likeliest
// alternatives, from rows of logits.
//
// With m the row's largest logit, r = Σ e^(x − m) over all the others and W = Σ e^(x − m)·(m − x),
//
//   log p(i) = (x_i − m) − log(1 + r),   entropy = log(1 + r) + W / (1 + r)   (nats)
//
// The largest logit's own 1 stays out of the sum r, so the log probability and the entropy of a sure choice, both near 0,
// keep their leading digits (log1p); both are sums of terms of one sign, and nothing cancels.
//
// A row is read once, in chunks of 8192 logits (short ones: 2048) that a workgroup holds in registers, 32 (8) a thread; a wave keeps
// m, and r and W in parts by lane. When a chunk raises m, the old one's own 1 joins r, r and W are scaled, and the new one's is left
// out. A row's chunks are shared out among workgroups where the rows are few; the last of them to be done joins the parts, in order.
//
// Alternatives: a wave keeps in LDS every logit past a bound that at least n_top logits reach: the n_top-th largest of its lanes'
// largest so far, found bit by bit from ballots, and anew after 1, 2, 4, … chunks; or the smallest of the waves' (n_top / 4)-th, which
// n_top of theirs together reach. Of the few that are kept (by a wave's own bound 1.3·n_top in a first chunk of random logits, as many
// again over all others) each finds its rank by counting those before it. Where more pass the bound than there is room (equal
// logits), the wave takes the best one by one.
#include <algorithm>

#include "choose_key.h"
#include "kv_ops.h"
#include "wave.h"

namespace {

constexpr int T = 256;                         // threads
constexpr int ROOM = 256;                      // alternatives that a wave has room for
constexpr int MAX_PARTS = 64;                  // workgroups of a row
constexpr int TICKET = 32;                     // words between tickets (128 bytes)
constexpr int SHARED = 9;                      // alternatives from which the waves look for a bound together (with 5 200 rows 30.7 µs for 30.2)
constexpr int FEW = 16;                        // logits a thread of a row that goes by chunks of 8 a thread
constexpr float LOG2E = 1.4426950408889634f;
constexpr float SCALE = 24.0f, ONE = 16777216.0f;  // a wave's sums are held times 2^24: v_exp_f32 gives no subnormal numbers

struct ScoreArgs {
    const float *x;
    size_t stride;
    const int32_t *ids;
    float *logprob, *entropy, *top_lp;
    int32_t *top_ids;
    int n, n_vocab, top, parts;
    // the parts' sums and alternatives [rows·parts][2 + top], and the rows' tickets (zero, self-resetting)
    uint64_t *part;
    uint32_t *tickets;
};

// sums over some logits: the largest, Σ e^(x − m) over the others, Σ e^(x − m)·(m − x); m = −∞: none that counts
struct Sums {
    float m, r, w;
    bool nan;
};
__device__ __forceinline__ Sums join(const Sums &a, const Sums &b) {
    const bool first = a.m >= b.m;
    const float m = first ? a.m : b.m, d = first ? b.m - a.m : a.m - b.m;  // (−∞ − −∞: not used)
    const float r0 = first ? a.r : b.r, w0 = first ? a.w : b.w, r1 = first ? b.r : a.r, w1 = first ? b.w : a.w;
    const bool alone = (first ? b.m : a.m) == -INFINITY;
    const float f = __builtin_amdgcn_exp2f(d * LOG2E), all = 1.0f + r1;
    return Sums{m, alone ? r0 : fmaf(f, all, r0), alone || f == 0.0f ? w0 : fmaf(f, fmaf(all, -d, w1), w0), a.nan || b.nan};
}

// f32 in an unsigned order (−NaN first, NaN last)
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t u) { return __uint_as_float((u & 0x80000000u) ? u & 0x7FFFFFFFu : ~u); }
// a NaN's key comes after −∞'s; no key is 0
__device__ __forceinline__ uint64_t key_of(float v, uint32_t i) { return v == v ? choose_key(v, i) : (uint64_t)(uint32_t)~i; }
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t k) {
#pragma unroll
    for (int d = 32; d; d >>= 1) k = max(k, (uint64_t)__shfl_xor((unsigned long long)k, d));
    return k;
}
__device__ __forceinline__ int count(uint64_t mask) { return (int)__builtin_popcountll(mask); }
__device__ __forceinline__ int before(uint64_t mask) {  // lanes of the mask below this one
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0u));
}

// the ids of the logits of x[from … to) that are −∞ (or NaN) in order, behind the have keys in s_top: one wave
__device__ void fill(const float *x, int from, int to, bool nan, uint64_t *s_top, int &have, int want) {
    const int lane = threadIdx.x & 63;
    for (int i = from; i < to && have < want; i += 64) {
        const float v = i + lane < to ? x[i + lane] : 0.0f;
        const bool is = nan ? v != v : v == -INFINITY;
        const uint64_t mask = __builtin_amdgcn_ballot_w64(is);
        const int at = have + before(mask);
        if (is && at < want) s_top[at] = key_of(v, (uint32_t)(i + lane));
        have = min(want, have + count(mask));
    }
}
// the keys with fewer than `want` larger ones among the n of s_keys, by rank to s_top: all threads, keys apart. s_keys has room for
// 8 more, which are made 0 (behind them a barrier of its own)
__device__ __forceinline__ void rank(uint64_t *s_keys, int n, uint64_t *s_top, int want) {
    if (threadIdx.x < 8) s_keys[n + threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += T) {
        const uint64_t k = s_keys[i];
        int larger = 0;
        for (int j = 0; j < n; j += 8) {
            uint64_t o[8];
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] = s_keys[j + e];
#pragma unroll
            for (int e = 0; e < 8; e++) larger += o[e] > k ? 1 : 0;
        }
        if (larger < want) s_top[larger] = k;
    }
}

// Bound: of many rows HBM: 1925 rows of 151936 with one alternative (1.17 GB) 185 µs, 6.3 TB/s, without 181, with 20 191 (each wave
// by its own bound 215); 200 rows with 5 30 µs. Of few latency: one row 10 µs, 5 for a chunk's loads, sums and alternatives, 4 for
// handing the part over and joining 19; 61 rows with 20 alternatives 21 … 23 (each wave by its own bound 2 more), without 12: what a chunk has
// past its bound is kept and ranked, 400 of 19 parts are ranked again, and 135 of the 1159 workgroups wait for the others. A row's
// parts on one XCD, in whose L2 they are handed over: 61 rows 16.8 … 12.2 µs, for 19.9 and 15.8 through the coherence point.
template <int V, bool TOP, bool XL> __global__ __launch_bounds__(T, 4) void k_logprobs(ScoreArgs a) {
    constexpr int CHUNK = T * V;
    __shared__ __attribute__((aligned(16))) uint64_t s_keys[MAX_PARTS * HTR_TOP_MAX + 8];  // the waves' alternatives, ROOM each; then the parts'
    __shared__ uint64_t s_top[HTR_TOP_MAX];
    __shared__ Sums s_sums[T / 64];
    __shared__ int s_n[T / 64], s_last;
    __shared__ uint32_t s_bound[2][T / 64];
    static_assert(MAX_PARTS * HTR_TOP_MAX >= T / 64 * ROOM, "room");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // XL: the workgroups of a row share an XCD (a launch's go to the 8 XCDs in turn), and its L2 shows them each other's stores
    const int id = XL ? blockIdx.x >> 3 : blockIdx.x, part = id % a.parts, row = XL ? 8 * (id / a.parts) + (blockIdx.x & 7) : id / a.parts;
    if (XL && row >= a.n) return;
    const float *x = a.x + (size_t)row * a.stride;
    // the row from its 16-byte boundary on: logit i at place i + shift
    const int shift = (int)((uintptr_t)x >> 2 & 3), n_place = a.n_vocab + shift;
    const int chunks = (n_place + CHUNK - 1) / CHUNK;
    const int c0 = (int)((int64_t)chunks * part / a.parts), c1 = (int)((int64_t)chunks * (part + 1) / a.parts);
    uint64_t *kept = s_keys + ROOM * wave;

    Sums s{-INFINITY, 0.0f, 0.0f, false};
    float lane_top = -INFINITY, bound = -INFINITY;  // the lane's largest so far; alternatives are larger than the bound
    int n_kept = 0, looked = 0;
    for (int c = c0; c < c1; c++) {
        const int first = c * CHUNK - shift + 4 * tid;  // the thread's first logit; its quads are 4·T apart
        float v[V];
        if (c * CHUNK >= shift && (c + 1) * CHUNK <= n_place) {
#pragma unroll
            for (int q = 0; q < V / 4; q++) {
                typedef float f4 __attribute__((ext_vector_type(4)));
                const f4 y = __builtin_nontemporal_load(reinterpret_cast<const f4 *>(x + first + 4 * T * q));
                v[4 * q] = y[0], v[4 * q + 1] = y[1], v[4 * q + 2] = y[2], v[4 * q + 3] = y[3];
            }
        } else {
#pragma unroll
            for (int q = 0; q < V / 4; q++) {
                const int i = first + 4 * T * q;
                if (i >= 0 && i + 3 < a.n_vocab) {
                    const float4 y = *reinterpret_cast<const float4 *>(x + i);
                    v[4 * q] = y.x, v[4 * q + 1] = y.y, v[4 * q + 2] = y.z, v[4 * q + 3] = y.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) v[4 * q + e] = i + e >= 0 && i + e < a.n_vocab ? x[i + e] : -INFINITY;
                }
            }
        }
        float quad[V / 4], top = -INFINITY;
        bool odd = false;
#pragma unroll
        for (int q = 0; q < V / 4; q++) {
            odd |= __builtin_isunordered(v[4 * q], v[4 * q + 1]) | __builtin_isunordered(v[4 * q + 2], v[4 * q + 3]);
            quad[q] = fmaxf(fmaxf(v[4 * q], v[4 * q + 1]), fmaxf(v[4 * q + 2], v[4 * q + 3]));
            top = fmaxf(top, quad[q]);
        }
        s.nan |= odd;
        const float chunk_top = wave_max(top, lane);
        if (chunk_top > -INFINITY) {
            const bool up = chunk_top > s.m;  // (alike in all lanes)
            int mine = -1;                    // the place of the new largest one, in its lane
            if (__builtin_amdgcn_ballot_w64(up)) {
                if (s.m > -INFINITY) {
                    const float d = s.m - chunk_top, f = __builtin_amdgcn_exp2f(d * LOG2E), all = s.r + (lane == 0 ? ONE : 0.0f);
                    s.w = f == 0.0f ? 0.0f : f * fmaf(all, -d, s.w);
                    s.r = f * all;
                }
                s.m = chunk_top;
                if (lane == (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(top == chunk_top)))
#pragma unroll
                    for (int j = V - 1; j >= 0; j--) mine = v[j] == chunk_top ? j : mine;
            }
            // (a logit 200 and more below the largest adds nothing; the differences stay finite)
            auto add = [&](auto each) {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float d = fmaxf(v[j] - s.m, -200.0f), e = each(j, __builtin_amdgcn_exp2f(fmaf(d, LOG2E, SCALE)));
                    s.r += e;
                    s.w = fmaf(e, -d, s.w);
                }
            };
            if (__builtin_amdgcn_ballot_w64(mine >= 0)) add([&](int j, float e) { return j == mine ? 0.0f : e; });
            else add([](int, float e) { return e; });
        }
        if constexpr (TOP) {
            lane_top = fmaxf(lane_top, top);
            if (((c - c0) & (c - c0 - 1)) == 0) {
                // the largest number of 20 leading bits that a.top lanes reach
                const uint32_t u = ordered(lane_top + 0.0f);  // (−0 as +0)
                auto reached = [&](int lanes) {
                    uint32_t t = 0;
                    for (uint32_t bit = 1u << 31; bit >= 1u << 12; bit >>= 1)
                        if (count(__builtin_amdgcn_ballot_w64(u >= (t | bit))) >= lanes) t |= bit;
                    return t;
                };
                uint32_t t = reached(a.top);
                if (a.top >= SHARED) {  // or that each wave's share of them reaches
                    const uint32_t share = reached((a.top + T / 64 - 1) / (T / 64));
                    uint32_t *all = s_bound[looked++ & 1];
                    if (lane == 0) all[wave] = share;
                    __syncthreads();
                    t = max(t, min(min(all[0], all[1]), min(all[2], all[3])));
                }
                if (t > ordered(-INFINITY)) bound = fmaxf(bound, from_ordered(t == ordered(0.0f) ? t - 2 : t - 1));  // (past −0 too)
            }
            if (__builtin_amdgcn_ballot_w64(top > bound)) {
                const int had = n_kept;
#pragma unroll
                for (int q = 0; q < V / 4; q++) {
                    if (__builtin_amdgcn_ballot_w64(quad[q] > bound) == 0) continue;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const bool is = v[4 * q + e] > bound;
                        const uint64_t mask = __builtin_amdgcn_ballot_w64(is);
                        const int at = n_kept + before(mask);
                        if (is && at < ROOM) kept[at] = choose_key(v[4 * q + e], (uint32_t)(first + 4 * T * q + e));
                        n_kept += count(mask);
                    }
                }
                __builtin_amdgcn_wave_barrier();
                if (n_kept > ROOM) {
                    // the best a.top of those kept before and of this chunk's, one by one
                    uint64_t last = ~0ull, out = 0;
                    int n = 0;
                    for (; n < a.top; n++) {
                        uint64_t k = 0;
                        for (int i = lane; i < had; i += 64)
                            if (kept[i] < last) k = max(k, kept[i]);
#pragma unroll
                        for (int j = 0; j < V; j++) {
                            const uint64_t y = v[j] > bound ? choose_key(v[j], (uint32_t)(first + 4 * T * (j / 4) + j % 4)) : 0;
                            if (y < last) k = max(k, y);
                        }
                        last = wave_max_u64(k);
                        if (lane == n) out = last;
                    }
                    __builtin_amdgcn_wave_barrier();
                    if (lane < n) kept[lane] = out;
                    __builtin_amdgcn_wave_barrier();
                    n_kept = n;
                    bound = from_ordered((uint32_t)(last >> 32));  // (equal ones of later chunks come after)
                }
            }
        }
    }

    // the waves' sums
    s.r = wave_sum(s.r, lane) / ONE, s.w = wave_sum(s.w, lane) / ONE, s.nan = __builtin_amdgcn_ballot_w64(s.nan) != 0;
    if (lane == 0) s_sums[wave] = s, s_n[wave] = n_kept;
    __syncthreads();
    s = join(join(s_sums[0], s_sums[1]), join(s_sums[2], s_sums[3]));
    if constexpr (TOP) {
        // their alternatives next to each other
        int at = 0, n = 0;
        for (int w = 0; w < T / 64; w++) {
            if (w < wave) at += s_n[w];
            n += s_n[w];
        }
        uint64_t mine[ROOM / 64];
#pragma unroll
        for (int i = 0; i < ROOM / 64; i++) mine[i] = lane + 64 * i < n_kept ? kept[lane + 64 * i] : 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ROOM / 64; i++)
            if (lane + 64 * i < n_kept) s_keys[at + lane + 64 * i] = mine[i];
        if (tid < a.top) s_top[tid] = 0;
        rank(s_keys, n, s_top, a.top);
        __syncthreads();
        if (n < a.top && wave == 0) {
            const int from = max(c0 * CHUNK - shift, 0), to = min(c1 * CHUNK - shift, a.n_vocab);
            fill(x, from, to, false, s_top, n, a.top);
            fill(x, from, to, true, s_top, n, a.top);
        }
        __syncthreads();
    }
    if (a.parts > 1) {
        const int words = 2 + a.top;
        uint64_t *out = a.part + ((size_t)row * a.parts + part) * words;
        static constexpr int SCOPE = XL ? __HIP_MEMORY_SCOPE_WORKGROUP : __HIP_MEMORY_SCOPE_AGENT;
        auto put = [](uint64_t *p, uint64_t y) { __hip_atomic_store(p, y, __ATOMIC_RELAXED, XL ? __HIP_MEMORY_SCOPE_WORKGROUP : __HIP_MEMORY_SCOPE_AGENT); };
        auto pair = [](float lo, float hi) { return (uint64_t)__float_as_uint(lo) | (uint64_t)__float_as_uint(hi) << 32; };
        if (tid == 0) put(out, pair(s.m, s.r)), put(out + 1, pair(s.w, s.nan ? 1.0f : 0.0f));
        if (TOP && tid < a.top) put(out + 2 + tid, s_top[tid]);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this thread's stores are performed
        __syncthreads();
        if (tid == 0) {
            const uint32_t got = __hip_atomic_fetch_add(a.tickets + TICKET * row, 1u, __ATOMIC_RELAXED, SCOPE);
            s_last = got == (uint32_t)(a.parts - 1);
            if (s_last) __hip_atomic_store(a.tickets + TICKET * row, 0u, __ATOMIC_RELAXED, SCOPE);  // for the next call
        }
        __syncthreads();
        if (!s_last) return;
        const uint64_t *in = a.part + (size_t)row * a.parts * words;
        auto get = [](const uint64_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
        // a lane a part; each joined with the largest's
        Sums y{-INFINITY, 0.0f, 0.0f, false};
        if (lane < a.parts) {
            const uint64_t p = get(in + (size_t)lane * words), q = get(in + (size_t)lane * words + 1);
            y = Sums{__uint_as_float((uint32_t)p), __uint_as_float((uint32_t)(p >> 32)), __uint_as_float((uint32_t)q), (uint32_t)(q >> 32) != 0};
        }
        const float m = wave_max(y.m, lane);
        const bool is_first = lane == (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(y.m == m));
        const float d = y.m - m, f = __builtin_amdgcn_exp2f(d * LOG2E), all = 1.0f + y.r;
        const bool none = y.m == -INFINITY || f == 0.0f;
        s.r = wave_sum(is_first ? y.r : none ? 0.0f : f * all, lane);
        s.w = wave_sum(is_first ? y.w : none ? 0.0f : f * fmaf(all, -d, y.w), lane);
        s.m = m, s.nan = __builtin_amdgcn_ballot_w64(y.nan) != 0;
        if constexpr (TOP) {
            // a number that a.top keys reach: the smallest of the parts' j-th best, j = ⌈top / parts⌉ (where each has as many)
            const int all_keys = a.parts * a.top, j = (a.top + a.parts - 1) / a.parts;
            uint64_t low = lane < a.parts ? get(in + (size_t)lane * words + 1 + j) : ~0ull;
            low = ~wave_max_u64(~low);
            if (tid == 0) s_n[0] = 0;
            if (tid < a.top) s_top[tid] = 0;
            __syncthreads();
            for (int i = tid; i < all_keys; i += T) {
                const uint64_t k = get(in + (size_t)(i / a.top) * words + 2 + i % a.top);
                if (k && k >= low) s_keys[atomicAdd(&s_n[0], 1)] = k;
            }
            __syncthreads();
            const int n = s_n[0];
            rank(s_keys, n, s_top, a.top);
            __syncthreads();
        }
    }
    // (natural logarithms)
    const bool broken = s.nan || s.m == INFINITY;
    const float ln = log1pf(s.r);
    auto lp = [&](float y) { return broken ? NAN : s.m == -INFINITY ? -INFINITY : (y - s.m) - ln; };
    if (tid == 0) {
        const uint32_t id = (uint32_t)a.ids[row];
        a.logprob[row] = id < (uint32_t)a.n_vocab ? lp(x[id]) : NAN;
        a.entropy[row] = broken ? NAN : s.m == -INFINITY ? 0.0f : ln + s.w / (1.0f + s.r);
    }
    if (TOP && tid < a.top) {
        const uint64_t k = s_top[tid];
        a.top_ids[(size_t)row * a.top + tid] = (int32_t)~(uint32_t)k;
        a.top_lp[(size_t)row * a.top + tid] = lp(from_ordered((uint32_t)(k >> 32)));
    }
}

}  // namespace

// ---- ABI -----------------------------------------------------------------------------------------------------------------

extern "C" int htr_token_logprobs(htr_device *dev, const float *d_logits, size_t stride, int n, int n_vocab, const int32_t *d_ids,
                                  float *d_logprob, float *d_entropy, int n_top, int32_t *d_top_ids, float *d_top_logprob) {
    const char *me = "htr_token_logprobs";
    if (!d_logits || !d_ids || !d_logprob || !d_entropy) return htr_fail("%s: null argument", me);
    if (n < 1 || n > HTR_MAX_ROW || n_vocab < 1 || n_vocab > 1 << 28 || stride < (size_t)n_vocab)
        return htr_fail("%s: %d rows of %d logits, %zu apart (1 … %d rows, 1 … 2^28 logits)", me, n, n_vocab, stride, HTR_MAX_ROW);
    if (n_top < 0 || n_top > HTR_TOP_MAX || n_top > n_vocab)
        return htr_fail("%s: %d alternatives of %d logits (at most %d)", me, n_top, n_vocab, HTR_TOP_MAX);
    if (n_top && (!d_top_ids || !d_top_logprob)) return htr_fail("%s: null alternatives", me);
    const size_t rows = (size_t)n;
    if (!htr_rows_fit(stride, rows, n_vocab)) return htr_fail("%s: %d rows %zu floats apart", me, n, stride);
    const struct {
        const void *p;
        size_t n;
    } of[6] = {{d_logprob, 4 * rows}, {d_entropy, 4 * rows}, {d_top_ids, 4 * rows * n_top}, {d_top_logprob, 4 * rows * n_top},
               {d_logits, 4 * (stride * (rows - 1) + n_vocab)}, {d_ids, 4 * rows}};
    uintptr_t bits = 0;
    for (int i = 0; i < 6; i++) {
        if (!of[i].n) continue;
        bits |= (uintptr_t)of[i].p;
        for (int j = i + 1; i < 4 && j < 6; j++)
            if (of[j].n && htr_overlap(of[i].p, of[i].n, of[j].p, of[j].n)) return htr_fail("%s: an output overlaps another or the inputs", me);
    }
    if (bits & 3) return htr_fail("%s: pointers must be 4-byte aligned", me);
    HTR_TRY(htr_check_alive(dev));
    const HtrOnDevice on(dev);
    ScoreArgs a{d_logits, stride, d_ids, d_logprob, d_entropy, d_top_logprob, d_top_ids, n, n_vocab, n_top, 1, nullptr, nullptr};
    // as many workgroups to a row as the card holds at once, a chunk to each at least (up to a quarter more than it holds)
    const bool few = n_vocab <= FEW * T;
    const int at_once = 4 * dev->n_cu, chunk = T * (few ? 8 : 32), chunks = (n_vocab + chunk - 1) / chunk;
    const int64_t each = std::max<int64_t>(1, ((int64_t)chunks * n + at_once / 4 * 3) / at_once);  // chunks
    a.parts = (int)std::max<int64_t>(1, std::min<int64_t>((chunks + each / 2) / each, MAX_PARTS));  // (of all rows below 2·at_once)
    if (a.parts > 1) {
        void *p;
        HTR_TRY(htr_scratch(dev, SCR_SCORE_TICKET, (size_t)2 * at_once * TICKET * 4, &p));
        a.tickets = (uint32_t *)p;
        HTR_TRY(htr_scratch(dev, SCR_SCORE, (size_t)2 * at_once * (2 + HTR_TOP_MAX) * 8, &p));
        a.part = (uint64_t *)p;
    }
    const bool xl = a.parts > 1 && dev->xcd_round_robin == 1;
    const dim3 g((unsigned)((xl ? (n + 7) / 8 * 8 : n) * a.parts)), b(T);
#define HTR_SCORE(V, TOP)                                                                                                  \
    do {                                                                                                               \
        if (xl) hipLaunchKernelGGL((k_logprobs<V, TOP, true>), g, b, 0, dev->stream, a);                               \
        else hipLaunchKernelGGL((k_logprobs<V, TOP, false>), g, b, 0, dev->stream, a);                                 \
    } while (0)
    if (few && n_top) HTR_SCORE(8, true);
    else if (few) HTR_SCORE(8, false);
    else if (n_top) HTR_SCORE(32, true);
    else HTR_SCORE(32, false);
#undef HTR_SCORE
    return htr_launched(dev, "k_logprobs");
}
