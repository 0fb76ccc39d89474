// Attention of a step's new tokens of several reads, each over its own rows of a cache in pages. Head dim 128, any number of q
// heads to a KV head, f16 or q8_0 rows.
//
//   out[t][h] = Σ_j p_j·v_j / Σ_j p_j,  p_j = e^(scale·q·k_j − m)  over the rows j ≤ past + i of the read whose i-th row t is
//
// The q heads of a KV head share its keys: a read's rows for a KV head are (i, head of the group), packed, in tiles of 32. The
// operands, the softmax and what is held to how many bits are kv_attention.hip's.
//
// The reads' lengths are on the device, and the launch knows their bounds alone: it is as many workgroups as the card holds at
// once, whatever the reads. Each KV head's tiles in order are a line of work, a tile's length on it its keys and COST more for
// its start and end, and the head's workgroups take equal pieces of the line, wherever that cuts a tile: one read of many keys
// goes to all of them, of many short ones each takes a few, and no list of work is made first. Where a piece begins follows
// from sums over the reads, a lane a read, and within a read from a quadratic equation (a tile's keys grow with its rows'
// positions). The parts of cut tiles go to memory and are joined by a second launch.
#include <algorithm>
#include <type_traits>

#include "kv_attn.h"

namespace {

constexpr int PW = 4;            // waves of a workgroup, two of which a CU holds
constexpr int COST = 64;         // keys that take as long as a tile's start and end
constexpr int LEAST = 128;       // keys of a piece of work, at least: a block for each wave
constexpr int QT = 256 + 256 + 16 + 16;  // 16-byte chunks of a q8_0 buffer: K, V, K scales, V scales

struct Args {
    const float *q;
    size_t q_stride;
    float *out;
    HtrKvPlanes kv;
    HtrPages p;
    int n_head, group;
    uint32_t per_group;  // ⌈2^32 / group⌉ (group > 1): the quotient of a row below 2^32 / group by one product
    int n_page, cap;     // the cache's pages; the rows that the table has room for
    float scale;
    int parts;           // workgroups of a KV head
    float *part;         // [n_kv·parts][2][32] sums o[128], and each row's (m, l, c)
    float4 *part_ml;
};

__device__ __forceinline__ int64_t lane_of(int64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// the line of work: the reads' tiles in order. Uniform but for the 64 reads at hand, a lane each
struct Line {
    const Args &a;
    int first = 0;                // the reads at hand: first …
    int64_t base = 0;             // the line's length before them
    int64_t end;                  // and up to and with each
    int start, n, past;           // its rows and keys; past −1: not served
    __device__ __forceinline__ explicit Line(const Args &args) : a(args) { load(); }

    __device__ __forceinline__ int64_t tile(int held, int rows_to) const { return (int64_t)a.group * (max(held, 0) + COST) + rows_to; }
    __device__ __forceinline__ void load() {
        const int lane = threadIdx.x & 63, b = first + lane;
        const bool there = b < a.p.n_seq;
        const int s0 = there ? a.p.start[b] : 0, s1 = there ? a.p.start[b + 1] : 0, held = there ? a.p.past[b] : -1;
        start = min(max(s0, 0), a.p.n_row);
        n = min(max(s1, start), a.p.n_row) - start;
        past = min(max(held, -1), a.cap);
        const int rows = n * a.group, full = rows / KB;
        end = full * tile(past, 0) + (int64_t)(KB / 2) * full * (full + 1) + (rows % KB ? tile(past, rows) : 0);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t o = __shfl_up((long long)end, d);
            if (lane >= d) end += o;
        }
        end += base;
    }
    __device__ __forceinline__ bool next() {
        if (first + 64 >= a.p.n_seq) return false;
        base = lane_of(end, 63), first += 64;
        load();
        return true;
    }
    __device__ __forceinline__ int64_t total() {
        while (next()) {}
        const int64_t t = lane_of(end, 63);
        if (first) {
            first = 0, base = 0;
            load();
        }
        return t;
    }
};
// how many pieces the line is cut into, and where
__device__ __forceinline__ int pieces(const Args &a, int64_t total) {
    return (int)min((int64_t)a.parts, max((int64_t)1, total / ((int64_t)a.group * (LEAST + COST))));
}
__device__ __forceinline__ int64_t cut(int64_t total, int i, int n) { return i == n ? total : (int64_t)((double)total * i / n); }

// a tile on the line
struct Tile {
    int at;                   // its read: lane `at` of those at hand
    int start, n, past, rows; // the read's
    int tau;                  // its place among the read's tiles
    int64_t begin, len;       // and on the line

    __device__ __forceinline__ void of_read(Line &w, int lane) {
        at = lane;
        start = __builtin_amdgcn_readlane(w.start, at), n = __builtin_amdgcn_readlane(w.n, at), past = __builtin_amdgcn_readlane(w.past, at);
        rows = n * w.a.group;
    }
    __device__ __forceinline__ void measure(const Line &w) { len = w.tile(past, min(KB * (tau + 1), rows)); }
    // the one that holds place x of the line, x before its end
    __device__ __forceinline__ Tile(Line &w, int64_t x) {
        while (lane_of(w.end, 63) <= x && w.next()) {}
        of_read(w, min((int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(w.end > x) | 1ull << 63), 63));
        const int64_t from = at ? lane_of(w.end, at - 1) : w.base;
        const int64_t y = x - from, step = w.tile(past, 0);
        // tau tiles are tau·step + 16·tau·(tau + 1) long
        const double h = 0.5 * ((double)step + KB / 2);
        const int tiles = (rows + KB - 1) / KB;
        tau = min((int)((sqrt(h * h + (double)(KB / 2) * (double)y) - h) / (KB / 2)), tiles - 1);
        auto upto = [&](int t) { return t * step + (int64_t)(KB / 2) * t * (t + 1); };
        while (tau > 0 && upto(tau) > y) tau--;
        while (tau + 1 < tiles && upto(tau + 1) <= y) tau++;
        begin = from + upto(tau);
        measure(w);
    }
    // the next one (there is one)
    __device__ __forceinline__ void next(Line &w) {
        begin += len;
        if (KB * ++tau >= rows) {
            uint64_t more;
            int from = at + 1;
            while ((more = from < 64 ? __builtin_amdgcn_ballot_w64(w.n > 0) >> from << from : 0) == 0) {
                if (!w.next()) break;
                from = 0;
            }
            of_read(w, more ? (int)__builtin_ctzll(more) : 63);
            tau = 0;
        }
        measure(w);
    }
};

// row r's query
__device__ __forceinline__ int query_of(const Args &a, int r) { return a.group == 1 ? r : (int)__umulhi((uint32_t)r, a.per_group); }
__device__ __forceinline__ float *out_row(const Args &a, const Tile &t, int kvh, int r) {
    const int i = query_of(a, r);
    return a.out + ((size_t)(t.start + i) * a.n_head + (size_t)kvh * a.group + (r - i * a.group)) * D;
}

// 4 bytes a lane from p to LDS bytes lds + 4·lane
__device__ __forceinline__ void lds_load4_at(const void *p, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}

// A workgroup's waves take every fourth block of 32 keys of a tile each, into LDS of their own, as k_kv_attn_split's do (the
// layouts there), and wait for nobody until their sums are merged.
template <bool Q8> __global__ __launch_bounds__(64 * PW, 2) void k_page_attn(Args a) {
    constexpr int WAVE = Q8 ? 2 * QT + 16 : TILE;  // chunks of a wave's LDS
    static_assert(WAVE >= 1024, "a wave's sums fit");
    __shared__ __attribute__((aligned(16))) uint4_t s_kv[PW][WAVE];
    __shared__ float s_ml[PW][2][KB];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hf = lane >> 5, c = lane & 31;
    const int kvh = blockIdx.x % a.kv.n_kv, piece = blockIdx.x / a.kv.n_kv;
    Line line(a);
    const int64_t total = line.total();
    const int n_piece = pieces(a, total);
    if (piece >= n_piece) return;
    const int64_t x0 = cut(total, piece, n_piece), x1 = cut(total, piece + 1, n_piece);
    if (x0 >= x1) return;
    const size_t head0 = (size_t)kvh * a.kv.n_ctx;

    uint4_t *tile = s_kv[wave];
    const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4_t *)tile;
    // a wave's instruction is 4 (8) whole rows; half a block lies in one page
    const uint32_t kx = 16 * ((lane & 15) ^ (lane >> 4)), vx = 16 * ((lane & 15) ^ (4 * (lane >> 4))), r4 = 2 * D * (lane >> 4);
    const uint32_t bx = 16 * ((lane & 7) ^ (lane >> 4)), wx = 16 * ((lane & 7) ^ (2 * ((lane >> 4) & 1))), r8 = D * (lane >> 3);
    auto load = [&](int row0, int row1, bool is_v) {
        const char *plane = (const char *)(is_v ? a.kv.v : a.kv.k);
        const char *base[2] = {plane + (head0 + row0) * (2 * D), plane + (head0 + row1) * (2 * D)};
        const uint32_t to = lds + 16 * (is_v ? K_CHUNKS : 0);
#pragma unroll
        for (int u = 0; u < 8; u++)
            lds_load16(base[u >> 2] + 2 * D * 4 * (u & 3), r4 + (is_v ? vx : kx ^ (64 * (u & 3))), to + 16 * 64 * u);
    };
    auto load_q8 = [&](int row0, int row1, int b) {
        const uint32_t to = lds + 16 * QT * b;
        const size_t at[2] = {head0 + row0, head0 + row1};
        const size_t mine = (hf ? at[1] - 16 : at[0]) * 8 + 4 * lane;  // a row's scales are 8 bytes
        lds_load4_at((const char *)a.kv.kd + mine, to + 16 * 512);
        lds_load4_at((const char *)a.kv.vd + mine, to + 16 * 528);
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int h = u & 3;
            lds_load16((const char *)(u < 4 ? a.kv.k : a.kv.v) + at[h >> 1] * D + D * 8 * (h & 1), r8 + ((u < 4 ? bx : wx) ^ (64 * (h & 1))),
                       to + 16 * 64 * u);
        }
    };
    // the 8 dims of the lane's operand of a step; of q8_0 rows two steps are 16 in a row, 16 bytes of quants
    auto dims8 = [&](int ks) { return Q8 ? 4 * (ks >> 1) + 2 * hf + (ks & 1) : 2 * ks + hf; };
    const int vrow = Q8 ? 8 * ((lane >> 3) & 1) + 4 * hf + ((lane >> 1) & 3) : 4 * hf + ((lane & 15) >> 2);
    int va[4];
#pragma unroll
    for (int u = 0; u < 4; u++)
        va[u] = Q8 ? 16 * (256 + 8 * vrow + ((2 * u + ((lane >> 4) & 1)) ^ (vrow & 2) ^ ((vrow & 8) >> 1))) + 8 * (lane & 1)
                   : 16 * (K_CHUNKS + 16 * vrow + ((4 * u + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ (4 * (vrow & 3)))) + 8 * (lane & 1);

    for (Tile t(line, x0);; t.next(line)) {
        const int64_t u0 = max(x0 - t.begin, (int64_t)0), u1 = min(x1 - t.begin, t.len);
        const int r0 = KB * t.tau, r_end = min(r0 + KB, t.rows);
        // the last key that a query sees (past + cap < 2^32)
        auto last_key = [&](int i) { return (int)min((uint32_t)t.past + (uint32_t)i, (uint32_t)a.cap - 1u); };
        const int all_to = t.past < 0 ? 0 : (last_key(query_of(a, r0)) + 1) / KB, last = t.past < 0 ? -1 : last_key(query_of(a, r_end - 1));
        const int nb = (last + KB) / KB;
        const int i0 = u0 == 0 ? 0 : (int)((double)nb * (double)u0 / (double)t.len);
        const int i1 = u1 == t.len ? nb : (int)((double)nb * (double)u1 / (double)t.len);

        // the first rows of the halves of 32 of the wave's blocks: lane 2j + h has block j's half h
        const int32_t *table = a.p.table + (size_t)(line.first + t.at) * a.p.max_pages;
        int rowno = 0, j = 0;  // j: the wave's block
        uint64_t gone = 0;     // of those the ones without a page
        auto pages_from = [&](int jb) {
            const uint32_t key = min(KB * (uint32_t)(i0 + wave + PW * (jb + (lane >> 1))) + 16u * (lane & 1), (uint32_t)last & ~15u);
            const int page = table[key >> a.p.shift];
            const bool bad = (uint32_t)page >= (uint32_t)a.n_page;
            rowno = bad ? 0 : (page << a.p.shift) + (int)(key & ((1u << a.p.shift) - 1));
            gone = __builtin_amdgcn_ballot_w64(bad);
        };
        int i = i0 + wave, b = 0, row0 = 0, row1 = 0;
        uint32_t bad = 0, bad_next = 0;
        auto rows_of = [&](int jn) {
            if (jn && (jn & 31) == 0) pages_from(jn);
            row0 = __builtin_amdgcn_readlane(rowno, 2 * (jn & 31)), row1 = __builtin_amdgcn_readlane(rowno, 2 * (jn & 31) + 1);
            bad_next = (uint32_t)(gone >> (2 * (jn & 31))) & 3u;
        };
        if (i < i1) pages_from(0);
        const int r = r0 + c, rc = min(r, t.rows - 1), qi = query_of(a, rc);
        float qx[8][8];
        q_load<8, Q8>(a.q + (size_t)(t.start + qi) * a.q_stride + ((size_t)kvh * a.group + (rc - qi * a.group)) * D + (Q8 ? 16 : 8) * hf, qx);
        __syncthreads();  // (the sums of the tile before are read)
        if (i < i1) {
            rows_of(0);
            bad = bad_next;
            if constexpr (Q8) {
                load_q8(row0, row1, 0);
            } else {
                load(row0, row1, false);
                load(row0, row1, true);
            }
        }
        half8 qh[8], ql[8];
        const float sc = q_split<8, 2>(qx, a.scale, qh, ql);
        const int keys = t.past < 0 ? 0 : last_key(qi) + 1;  // that the row sees
        float m = M_NONE, l = 0.0f;
        f32x16 o[4];
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int x = 0; x < 16; x++) o[u][x] = 0.0f;

        // block i; MASK: not every row sees all of it, or half of it has no page
        auto step = [&](auto is_masked) {
            constexpr bool MASK = decltype(is_masked)::value;
            const bool more = i + PW < i1;
            uint4_t *buf = tile + (Q8 ? QT * b : 0);
            if constexpr (Q8) {
                if (more) {
                    rows_of(j + 1);
                    wait_reads();  // of the other buffer, a block ago
                    load_q8(row0, row1, b ^ 1);
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
            } else {
                half8 f[4];
#pragma unroll
                for (int h = 0; h < 2; h++) {
#pragma unroll
                    for (int ks = 0; ks < 4; ks++) f[ks] = *reinterpret_cast<const half8 *>(buf + 16 * c + (dims8(4 * h + ks) ^ (c & 15)));
                    if (h == 1) {
                        wait_reads();
                        if (more) {
                            rows_of(j + 1);
                            load(row0, row1, false);
                        }
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
                seen = low_bits(keys - (KB * i + here(4 * hf))) & (bad & 1 ? 0xFFFF0000u : ~0u) & (bad & 2 ? 0x0000FFFFu : ~0u);
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
                    const fp16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)(p + 256 * 8));
                    __builtin_memcpy(&v, &lo, 8);
                    __builtin_memcpy((char *)&v + 8, &hi, 8);
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
                if (more) load(row0, row1, true);
            }
            i += PW, j++;
            b ^= Q8;
            bad = bad_next;
        };
        auto whole = [&] { return i < all_to && bad == 0; };
        while (i < i1) {
            for (bool all = whole(); all; all = i < i1 && whole()) step(std::false_type{});
            for (bool some = i < i1; some; some = i < i1 && !whole()) step(std::true_type{});
        }
        l = pair_sum<32>(l);

        // the waves' sums through LDS (each its own tile's place): wave w finishes dims 32w … of every row
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
        for (int w = 0; w < PW; w++) m = fmaxf(m, s_ml[w][0][c]);
        float4 y[4];
#pragma unroll
        for (int x = 0; x < 4; x++) y[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < PW; w++) {
            const float f = __builtin_amdgcn_exp2f((s_ml[w][0][c] - m) * sc);
            l = fmaf(s_ml[w][1][c], f, l);
            const float4 *from = reinterpret_cast<const float4 *>(s_kv[w]) + 4 * 64 * wave + lane;
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const float4 z = from[64 * x];
                y[x].x = fmaf(z.x, f, y[x].x), y[x].y = fmaf(z.y, f, y[x].y);
                y[x].z = fmaf(z.z, f, y[x].z), y[x].w = fmaf(z.w, f, y[x].w);
            }
        }
        if (r < t.rows) {
            float *to;
            float by = 1.0f;
            if (u0 == 0 && u1 == t.len) {
                by = l == 0.0f ? 0.0f : 1.0f / l;  // no key seen: zeros
                to = out_row(a, t, kvh, r);
            } else {
                const size_t pr = (((size_t)kvh * a.parts + piece) * 2 + (u0 == 0)) * KB + c;
                to = a.part + pr * D;
                if (wave == 0 && hf == 0) a.part_ml[pr] = make_float4(m, l, sc, 0.0f);
            }
#pragma unroll
            for (int x = 0; x < 4; x++)
                *reinterpret_cast<float4 *>(to + 32 * wave + 8 * x + 4 * hf) = make_float4(y[x].x * by, y[x].y * by, y[x].z * by, y[x].w * by);
        }
        if (t.begin + t.len >= x1) break;
    }
}

// the tile that the cut behind a piece goes through, if it is the first cut through it: its parts joined. A piece's two places
// are for the tile that it ends with (1) and the one that it goes on with or begins and ends inside (0). 8 lanes a row
__global__ __launch_bounds__(256) void k_page_attn_join(Args a) {
    const int tid = threadIdx.x, row = tid >> 3, j = tid & 7;
    const int kvh = blockIdx.x % a.kv.n_kv, piece = blockIdx.x / a.kv.n_kv;
    Line line(a);
    const int64_t total = line.total();
    const int n_piece = pieces(a, total);
    if (piece + 1 >= n_piece) return;
    const int64_t x = cut(total, piece + 1, n_piece);
    if (x >= total) return;
    const Tile t(line, x);
    if (t.begin == x || t.begin < cut(total, piece, n_piece)) return;
    int more = 0;  // pieces past this one that have part of it
    while (piece + 1 + more < n_piece && cut(total, piece + 1 + more, n_piece) < t.begin + t.len) more++;
    const int r = KB * t.tau + row;
    if (r >= t.rows) return;
    const size_t first = (((size_t)kvh * a.parts + piece) * 2 + 1) * KB + row;
    auto place = [&](int e) { return e == 0 ? first : first - KB + (size_t)e * (2 * KB); };
    float m = M_NONE;
    for (int e = 0; e <= more; e++) m = fmaxf(m, a.part_ml[place(e)].x);
    float l = 0.0f;
    float4 y[4];
#pragma unroll
    for (int k = 0; k < 4; k++) y[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int e = 0; e <= more; e++) {
        const float4 ml = a.part_ml[place(e)];
        const float f = __builtin_amdgcn_exp2f((ml.x - m) * ml.z);
        l = fmaf(ml.y, f, l);
        const float *from = a.part + place(e) * D + 4 * j;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float4 z = *reinterpret_cast<const float4 *>(from + 32 * k);
            y[k].x = fmaf(z.x, f, y[k].x), y[k].y = fmaf(z.y, f, y[k].y), y[k].z = fmaf(z.z, f, y[k].z), y[k].w = fmaf(z.w, f, y[k].w);
        }
    }
    const float by = l == 0.0f ? 0.0f : 1.0f / l;
    float *to = out_row(a, t, kvh, r) + 4 * j;
#pragma unroll
    for (int k = 0; k < 4; k++) *reinterpret_cast<float4 *>(to + 32 * k) = make_float4(y[k].x * by, y[k].y * by, y[k].z * by, y[k].w * by);
}

}  // namespace

// ---- ABI -----------------------------------------------------------------------------------------------------------------

extern "C" int htr_page_attention(htr_device *dev, const float *d_q, size_t q_stride, const htr_pages *pages, const htr_kv *kv,
                                  int n_head, float scale, float *d_out) {
    const char *me = "htr_page_attention";
    Args a{};
    HTR_TRY(htr_kv_check(me, kv, &a.kv));
    HTR_TRY(htr_pages_check(me, pages, HTR_PAGES_TABLE, &a.p));
    if (!d_q || !d_out) return htr_fail("%s: null argument", me);
    if (n_head < 1 || n_head % kv->n_kv) return htr_fail("%s: %d q heads on %d KV heads", me, n_head, kv->n_kv);
    if (kv->n_ctx < pages->page) return htr_fail("%s: a cache of %d rows in pages of %d", me, kv->n_ctx, pages->page);
    const size_t qd = (size_t)n_head * D, n = (size_t)a.p.n_row;
    if (q_stride < qd || (q_stride & 3)) return htr_fail("%s: rows %zu floats apart (a multiple of 4, at least %zu)", me, q_stride, qd);
    if (((uintptr_t)d_q | (uintptr_t)d_out) & 15) return htr_fail("%s: pointers must be 16-byte aligned", me);
    if (htr_overlap(d_q, 4 * (q_stride * (n - 1) + qd), d_out, 4 * qd * n)) return htr_fail("%s: the output overlaps the queries", me);
    if (htr_kv_overlaps(a.kv, d_out, 4 * qd * n)) return htr_fail("%s: the output overlaps the cache", me);
    const struct {
        const void *p;
        size_t n;
    } read[3] = {{a.p.start, 4 * ((size_t)a.p.n_seq + 1)}, {a.p.past, 4 * (size_t)a.p.n_seq}, {a.p.table, 4 * (size_t)a.p.n_seq * a.p.max_pages}};
    for (const auto &r : read)
        if (htr_overlap(r.p, r.n, d_out, 4 * qd * n)) return htr_fail("%s: the output overlaps the pages' arrays", me);
    const uint64_t group = (uint64_t)(n_head / kv->n_kv);  // (rows · group < 2^32: the kernel's quotients)
    if (n * group * group >= 1ull << 32 || n * group > 1u << 30) return htr_fail("%s: %zu rows of %d heads", me, n, n_head);
    HTR_TRY(htr_check_alive(dev));
    const HtrOnDevice on(dev);
    a.q = d_q, a.q_stride = q_stride, a.out = d_out, a.n_head = n_head, a.group = n_head / kv->n_kv;
    a.n_page = kv->n_ctx / pages->page, a.scale = scale;
    a.per_group = (uint32_t)(((1ull << 32) + a.group - 1) / a.group), a.cap = a.p.max_pages << a.p.shift;
    a.parts = std::max(1, 2 * dev->n_cu / kv->n_kv);
    const unsigned groups = (unsigned)(a.parts * kv->n_kv);
    if (a.parts > 1) {
        const size_t rows = (size_t)4 * dev->n_cu * KB;  // two places for each of 2·n_cu pieces
        void *p;
        HTR_TRY(htr_scratch(dev, SCR_PAGE_ATTN, rows * (D + 4) * 4, &p));
        a.part = (float *)p;
        a.part_ml = (float4 *)(a.part + rows * D);
    }
    if (a.kv.q8) hipLaunchKernelGGL(k_page_attn<true>, dim3(groups), dim3(64 * PW), 0, dev->stream, a);
    else hipLaunchKernelGGL(k_page_attn<false>, dim3(groups), dim3(64 * PW), 0, dev->stream, a);
    HTR_TRY(htr_launched(dev, a.kv.q8 ? "k_page_attn<q8_0>" : "k_page_attn<f16>"));
    if (a.parts == 1) return 0;
    hipLaunchKernelGGL(k_page_attn_join, dim3(groups - (unsigned)kv->n_kv), dim3(256), 0, dev->stream, a);
    return htr_launched(dev, "k_page_attn_join");
}
