// The tables and row maps of a step of several reads over a cache in pages, made on the device from the reads' lengths.
//
// A cache's rows (htr_kv's n_ctx of them, the same for each KV head) are cut into pages of 2^shift; a read's row i is row
// i % page of page table[read][i / page]. A step takes new rows of many reads, packed in their order. For it
//
//   held = ⌈len / page⌉, need = ⌈(len + new) / page⌉ − held        the pages a read has, and those its new rows ask for
//   upto = Σ need, end = Σ new, both up to and with the read        (a read that ends here, new = −1, asks for none)
//   served: the read's rows fit the table's width and, with end, the step's buffers, and upto ≤ the free pages, or need = 0
//
// Free pages are a ring: page i of those given out in this step is ring[head + i], so where a page goes follows from the sums
// alone, and pages of ended reads go behind the last free one, which no read of this step looks at. So a call writes nothing
// that it reads but the lengths and the pool, each of which its thread has read before the sums: both may be written in place.
#include <algorithm>
#include <type_traits>

#include "kv_ops.h"

namespace {

// A thread a read: one workgroup, of 256 threads for up to 256 reads and 512 rows (24 reads of a token 3.0 µs, by 1024 threads 4.1;
// but 964 rows of 64 reads 6.1 and 5.2), else of 1024. Up to 4096 rows it maps the rows too, more are a second launch's.
constexpr int SMALL = 256, SMALL_ROWS = 512, ROWS_ONE = 4096;
// searches of a thread beside each other, each ten LDS reads behind one another, where there are more than four to a thread (8000
// pages 17.2 µs for 18.7); fewer go one by one (582 reads of a token, 36 of which end, 7.6 µs for 8.9; calls one after another)
constexpr int AT_ONCE = 4;

struct MapArgs {
    HtrPages p;
    const int32_t *len, *add, *pool;
    int32_t *ring, *len_out, *pool_out;
    int n_page;
};

template <typename T> __device__ __forceinline__ T wave_scan(T v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const T o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}
// Σ of v over the threads up to and with this one
template <typename T> __device__ __forceinline__ T block_scan(T v, T *s_wave) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();  // (the waves' sums of the scan before are read)
    if (lane == 63) s_wave[wave] = v;
    __syncthreads();
    for (int w = 0; w < wave; w++) v += s_wave[w];
    return v;
}
// for each of N numbers the first of n ≤ 1024 ascending sums that is past it, n where none is
template <int N> __device__ __forceinline__ void first_past(const uint32_t *sums, int n, const uint32_t (&i)[N], int (&at)[N]) {
#pragma unroll
    for (int k = 0; k < N; k++) at[k] = 0;
    for (int step = 1 << (31 - __builtin_clz((unsigned)n)); step; step >>= 1) {
        uint32_t sum[N];
#pragma unroll
        for (int k = 0; k < N; k++) sum[k] = sums[min(at[k] + step, n) - 1];
#pragma unroll
        for (int k = 0; k < N; k++) at[k] = at[k] + step <= n && sum[k] <= i[k] ? at[k] + step : at[k];
    }
}

// a row's place in the cache: −1 where the table has no page of the cache there
__device__ __forceinline__ int slot_of(int page, int n_page, int pos, int shift) {
    return (uint32_t)page < (uint32_t)n_page ? (page << shift) + (pos & ((1 << shift) - 1)) : -1;
}

template <int THREADS> __global__ __launch_bounds__(THREADS) void k_page_map(MapArgs a, int map_rows) {
    __shared__ uint32_t s_end[THREADS], s_upto[THREADS], s_back[THREADS], s_wave[THREADS / 64], s_taken;
    __shared__ unsigned long long s_two[THREADS / 64];
    __shared__ int s_past[THREADS], s_held[THREADS], s_need[THREADS];
    const int b = threadIdx.x, shift = a.p.shift;
    const bool there = b < a.p.n_seq;
    const int len = there ? a.len[b] : 0, add = there ? a.add[b] : 0;
    // (a ring's state that is none: as near to it as one is)
    const uint32_t n_page = (uint32_t)a.n_page, head = (uint32_t)a.pool[0] % n_page;
    const uint32_t count = (uint32_t)min(max(a.pool[1], 0), a.n_page);
    const bool ends = add < 0;
    const uint32_t mask = (1u << shift) - 1, held = len <= 0 ? 0 : ((uint32_t)len + mask) >> shift;
    if (b == 0) s_taken = 0;
    // (both sums fit 32 bits)
    const unsigned long long two = block_scan(ends ? (unsigned long long)min(held, (uint32_t)a.p.max_pages) << 32 : (unsigned long long)min(add, a.p.n_row + 1), s_two);
    const uint32_t end = (uint32_t)two, back = (uint32_t)(two >> 32);
    const bool fits = there && !ends && len >= 0 && (int64_t)len + add <= (int64_t)a.p.max_pages << shift && end <= (uint32_t)a.p.n_row;
    const uint32_t need = fits ? (((uint32_t)len + (uint32_t)add + mask) >> shift) - held : 0u;
    const uint32_t upto = block_scan(need, s_wave);
    const bool served = fits && (need == 0 || upto <= count);
    s_end[b] = min(end, (uint32_t)a.p.n_row), s_upto[b] = upto, s_back[b] = back;
    s_past[b] = served ? len : -1, s_held[b] = (int)held, s_need[b] = (int)need;
    if (served && need) atomicMax(&s_taken, upto);
    __syncthreads();
    const uint32_t taken = s_taken, returned = min(s_back[THREADS - 1], n_page - count);
    if (there) {
        a.p.start[b + 1] = (int)s_end[b];
        a.p.past[b] = s_past[b];
        a.len_out[b] = ends ? 0 : served ? len + add : len;
    }
    if (b == 0) {
        a.p.start[0] = 0;
        a.pool_out[0] = (int)(head + taken >= n_page ? head + taken - n_page : head + taken);
        a.pool_out[1] = (int)(count - taken + returned);
    }
    auto ring_at = [&](uint32_t i) {  // (i < n_page)
        const uint32_t at = head + i;
        return a.ring + (at >= n_page ? at - n_page : at);
    };
    auto give = [&](auto at_once) {
        constexpr int N = decltype(at_once)::value;
        for (uint32_t i0 = b; i0 < taken; i0 += N * THREADS) {
            uint32_t i[N];
            int at[N], page[N];
#pragma unroll
            for (int k = 0; k < N; k++) i[k] = min(i0 + THREADS * k, taken - 1), page[k] = *ring_at(i[k]);
            first_past(s_upto, a.p.n_seq, i, at);
#pragma unroll
            for (int k = 0; k < N; k++)
                if (i0 + THREADS * k < taken)
                    a.p.table[(size_t)at[k] * a.p.max_pages + s_held[at[k]] + (i[k] - (s_upto[at[k]] - s_need[at[k]]))] = page[k];
        }
    };
    auto take_back = [&](auto at_once) {
        constexpr int N = decltype(at_once)::value;
        for (uint32_t i0 = b; i0 < returned; i0 += N * THREADS) {
            uint32_t i[N];
            int at[N], page[N];
#pragma unroll
            for (int k = 0; k < N; k++) i[k] = min(i0 + THREADS * k, returned - 1);
            first_past(s_back, a.p.n_seq, i, at);
#pragma unroll
            for (int k = 0; k < N; k++) page[k] = a.p.table[(size_t)at[k] * a.p.max_pages + (i[k] - (at[k] ? s_back[at[k] - 1] : 0u))];
#pragma unroll
            for (int k = 0; k < N; k++)
                if (i0 + THREADS * k < returned) *ring_at(count + i[k]) = page[k];
        }
    };
    auto run = [](uint32_t n, auto what) {
        if (n <= AT_ONCE * THREADS) what(std::integral_constant<int, 1>{});
        else what(std::integral_constant<int, AT_ONCE>{});
    };
    run(taken, give);
    run(returned, take_back);
    if (!map_rows) return;
    for (int row = b; row < a.p.n_row; row += THREADS) {
        const uint32_t i[1] = {(uint32_t)row};
        int at[1], pos = -1, page = -1;
        first_past(s_end, a.p.n_seq, i, at);
        const int s = at[0];
        if (s < a.p.n_seq && s_past[s] >= 0) {
            pos = s_past[s] + row - (s ? (int)s_end[s - 1] : 0);
            const int n = pos >> shift;
            // a page that this step gives out is in the ring yet
            page = n < s_held[s] ? a.p.table[(size_t)s * a.p.max_pages + n] : *ring_at(s_upto[s] - s_need[s] + (n - s_held[s]));
        }
        a.p.pos[row] = pos;
        a.p.slot[row] = slot_of(page, a.n_page, pos, shift);
    }
}

// the rows' places of many rows, from the tables
__global__ __launch_bounds__(256) void k_page_rows(MapArgs a) {
    __shared__ uint32_t s_end[HTR_MAX_SEQ];
    for (int b = threadIdx.x; b < a.p.n_seq; b += 256) s_end[b] = (uint32_t)a.p.start[b + 1];
    __syncthreads();
    for (int r = blockIdx.x * 256 + threadIdx.x; r < a.p.n_row; r += gridDim.x * 256) {
        const uint32_t i[1] = {(uint32_t)r};
        int at[1];
        first_past(s_end, a.p.n_seq, i, at);
        const int s = at[0];
        int pos = -1, slot = -1;
        if (s < a.p.n_seq && a.p.past[s] >= 0) {
            pos = a.p.past[s] + r - (s ? (int)s_end[s - 1] : 0);
            slot = slot_of(a.p.table[(size_t)s * a.p.max_pages + (pos >> a.p.shift)], a.n_page, pos, a.p.shift);
        }
        a.p.pos[r] = pos;
        a.p.slot[r] = slot;
    }
}

}  // namespace

int htr_pages_check(const char *what, const htr_pages *p, int uses, HtrPages *out) {
    if (!p) return htr_fail("%s: null pages", what);
    if (p->n_seq < 1 || p->n_seq > HTR_MAX_SEQ || p->n_row < 1 || p->n_row > HTR_MAX_ROW)
        return htr_fail("%s: %d reads of %d rows (1 … %d reads, 1 … %d rows)", what, p->n_seq, p->n_row, HTR_MAX_SEQ, HTR_MAX_ROW);
    if (p->page < 16 || p->page > 1024 || (p->page & (p->page - 1)))
        return htr_fail("%s: pages of %d rows (a power of two, 16 … 1024)", what, p->page);
    if (p->max_pages < 1 || (int64_t)p->max_pages * p->page > INT32_MAX || (int64_t)p->max_pages * p->n_seq > INT32_MAX)
        return htr_fail("%s: a table of %d pages of %d rows for each of %d reads", what, p->max_pages, p->page, p->n_seq);
    if ((uses & HTR_PAGES_TABLE) && (!p->d_start || !p->d_past || !p->d_table)) return htr_fail("%s: null start, past or table", what);
    if ((uses & HTR_PAGES_ROWS) && (!p->d_pos || !p->d_slot)) return htr_fail("%s: null positions or slots", what);
    const uintptr_t t = uses & HTR_PAGES_TABLE ? (uintptr_t)p->d_start | (uintptr_t)p->d_past | (uintptr_t)p->d_table : 0;
    const uintptr_t r = uses & HTR_PAGES_ROWS ? (uintptr_t)p->d_pos | (uintptr_t)p->d_slot : 0;
    if ((t | r) & 3) return htr_fail("%s: the pages' arrays must be 4-byte aligned", what);
    *out = HtrPages{p->n_seq, p->n_row, __builtin_ctz((unsigned)p->page), p->max_pages, p->d_start, p->d_past, p->d_table, p->d_pos,
                    p->d_slot};
    return 0;
}

// ---- ABI -----------------------------------------------------------------------------------------------------------------

extern "C" int htr_page_map(htr_device *dev, const htr_pages *pages, int n_page, const int32_t *d_len, const int32_t *d_new,
                            int32_t *d_ring, const int32_t *d_pool, int32_t *d_len_out, int32_t *d_pool_out) {
    const char *me = "htr_page_map";
    MapArgs a{};
    HTR_TRY(htr_pages_check(me, pages, HTR_PAGES_TABLE | HTR_PAGES_ROWS, &a.p));
    if (!d_len || !d_new || !d_ring || !d_pool || !d_len_out || !d_pool_out) return htr_fail("%s: null argument", me);
    if (n_page < 1 || (int64_t)n_page * pages->page > INT32_MAX)
        return htr_fail("%s: %d pages of %d rows (at most 2^31 - 1 rows)", me, n_page, pages->page);
    if (((uintptr_t)d_len | (uintptr_t)d_new | (uintptr_t)d_ring | (uintptr_t)d_pool | (uintptr_t)d_len_out | (uintptr_t)d_pool_out) & 3)
        return htr_fail("%s: arrays must be 4-byte aligned", me);
    const size_t n = (size_t)a.p.n_seq, rows = (size_t)a.p.n_row;
    const struct {
        const void *p;
        size_t n;
        bool written;
    } of[11] = {{a.p.start, 4 * (n + 1), true}, {a.p.past, 4 * n, true}, {a.p.table, 4 * n * a.p.max_pages, true},
                {a.p.pos, 4 * rows, true}, {a.p.slot, 4 * rows, true}, {d_ring, 4 * (size_t)n_page, true},
                {d_len_out, 4 * n, true}, {d_pool_out, 8, true}, {d_len, 4 * n, false}, {d_new, 4 * n, false}, {d_pool, 8, false}};
    for (int i = 0; i < 8; i++)
        for (int j = i + 1; j < 11; j++) {
            if (!htr_overlap(of[i].p, of[i].n, of[j].p, of[j].n)) continue;
            if (of[i].p == of[j].p && ((i == 6 && j == 8) || (i == 7 && j == 10))) continue;  // in place
            return htr_fail("%s: arrays overlap (the new lengths and the new pool may be the old ones')", me);
        }
    HTR_TRY(htr_check_alive(dev));
    const HtrOnDevice on(dev);
    a.len = d_len, a.add = d_new, a.pool = d_pool, a.ring = d_ring, a.len_out = d_len_out, a.pool_out = d_pool_out, a.n_page = n_page;
    const bool one = a.p.n_row <= ROWS_ONE;
    if (a.p.n_seq <= SMALL && a.p.n_row <= SMALL_ROWS) hipLaunchKernelGGL(k_page_map<SMALL>, dim3(1), dim3(SMALL), 0, dev->stream, a, 1);
    else hipLaunchKernelGGL(k_page_map<HTR_MAX_SEQ>, dim3(1), dim3(HTR_MAX_SEQ), 0, dev->stream, a, one ? 1 : 0);
    HTR_TRY(htr_launched(dev, "k_page_map"));
    if (one) return 0;
    hipLaunchKernelGGL(k_page_rows, dim3((unsigned)std::min((a.p.n_row + 255) / 256, 2048)), dim3(256), 0, dev->stream, a);
    return htr_launched(dev, "k_page_rows");
}
