// Attention of a step's new tokens of several reads, each over its own rows of a cache in pages. Head dim 128, any number of q
// heads to a KV head, f16 or q8_0 rows.
//
//   out[t][h] = Σ_j p_j·v_j / Σ_j p_j,  p_j = e^(scale·q·k_j − m)  over the rows j ≤ past + i of the read whose i-th row t is
//
// The q heads of a KV head share its keys: a read's rows for a KV head are (i, head of the group), packed, in tiles. The
// operands, the softmax and what is held to how many bits are kv_attention.hip's.
//
// The reads' lengths are on the device, and the launch knows their bounds alone: it is as many workgroups as the card holds at
// once, whatever the reads (twice: once for each height of tile). Each KV head's tiles in order are a line of work, a tile's
// length on it its keys and COST more for its start and end, and the head's workgroups take equal pieces of the line, wherever
// that cuts a tile: one read of many keys goes to all of them, of many short ones each takes a few, and no list of work is made
// first. Where a piece begins follows from sums over the reads, a lane a read. The parts of a cut tile are joined by a second
// launch, of tokens by the last of the tile's workgroups. (So joined, 32 parts of a wide tile went through one workgroup: 65 rows
// over 8000 keys, when they took 47 µs by a second launch, 182, in pairs 75. More and smaller pieces, or smaller ones for the
// workgroups that begin later, were slower: 64 reads' tokens, when they took 105, 110 … 124.)
//
// Tiles come in two heights, each with a line of its own. Of up to 32 rows (a step's token, or what is left of a prompt) the waves
// share out the keys, every fourth block of 32 to each, loaded into LDS of its own, so that nobody waits for anybody until the
// four sums are merged. More are tiles of 128, 32 to a wave, all of which use each block, staged for them together. (Four prompts
// of 1925 in tiles of 32 rows alone 309 µs, with both 158.)
//
// Times here and below are of calls one after another on an MI355X, 16 q heads on 8 KV heads.
#include <algorithm>
#include <type_traits>

#include "kv_attn.h"

namespace {

constexpr int PW = 4;                       // waves of a workgroup, two of which a CU holds
constexpr int NARROW = KB, WIDE = KB * PW;  // rows of a tile
constexpr int COST = 128;                   // keys that take as long as a tile's start and end (with 64 four prompts 182 µs for 166)
constexpr int LEAST = 192;                  // a piece's length, at least: a block for each wave, and a tile's start
constexpr int SLIVER = 4;                   // blocks of a tile's beginning or end that are not cut off for themselves
constexpr int FEW = 128;                    // rows of a step (for a KV head) that go by narrow tiles alone, up to 4 of a read's on average
constexpr float CUT = 2.0f;                 // keys that take as long as joining a row of a part in the launch
constexpr int TICKET = 32;                  // words between tickets (128 bytes)
constexpr int SHARES = 4;                   // workgroups of the join to a wide piece
constexpr int QT = 256 + 256 + 16 + 16;     // 16-byte chunks of a q8_0 buffer: K, V, K scales, V scales

// where the parts of a height's cut tiles wait. A piece has two places: 1 for the tile that it begins and does not end, 0 for
// the one that it goes on with
struct Part {
    int first, n;        // the pieces that have a part of the tile: first … first + n − 1; n = 0: the place is empty
    int start, r0, rows; // its read's first row of the buffers; its first row of the read, its rows
};
struct Parts {
    float *sums;  // [n_kv·pieces][2][rows of a tile][128]
    float4 *ml;   // [n_kv·pieces][2][rows of a tile]: a row's (m, l, c)
    Part *of;     // [n_kv·pieces][2]
};
struct Args {
    const float *q;
    size_t q_stride;
    float *out;
    HtrKvPlanes kv;
    HtrPages p;
    int n_head, group;
    uint32_t per_group;  // ⌈2^31 / group⌉: the quotient of a row below 2^31 / group by one product
    int n_page, cap;     // the cache's pages; the rows that the table has room for
    float scale;
    int pieces;          // workgroups of a KV head and height
    int wide;            // those of the wide tiles: pieces, or none where no read has so many rows
    double per_piece;    // 1 / pieces
    uint32_t *tickets;   // [n_kv·pieces], TICKET words apart
    Parts part[2];
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t lane_of(int64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
    return (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ int64_t uniform(int64_t v) { return lane_of(v, 0); }
__device__ __forceinline__ int lane_id() { return here(threadIdx.x & 63); }  // (here: what is made of it is not kept in registers for later)
// row r's query
__device__ __forceinline__ int query_of(const Args &a, int r) { return (int)__umulhi(2u * (uint32_t)r, a.per_group); }

// 64 reads of the line of work at hand, in LDS
struct Reads {
    int64_t end[64];                 // the line's length up to and with each
    int start[64], n[64], past[64];  // its rows and keys; past −1: not served
};
// read b: its rows of the buffers, the keys before them
struct Read {
    int start, n, past;
    __device__ __forceinline__ Read(const Args &a, int b) {
        const bool there = b < a.p.n_seq;
        const int s0 = there ? a.p.start[b] : 0, s1 = there ? a.p.start[b + 1] : 0, held = there ? a.p.past[b] : -1;
        start = min(max(s0, 0), a.p.n_row), n = min(max(s1, start), a.p.n_row) - start, past = min(max(held, -1), a.cap);
    }
};
// the lines: of wide tiles, of the narrow ones behind them, of narrow ones alone
enum Kind { REST, TALL, ALL };
template <Kind K> __device__ __forceinline__ int64_t line_step(const Args &a, int past) {
    return (int64_t)(K == TALL ? a.group : 1) * (max(past, 0) + (int64_t)COST);
}
// a read's length on a line; n: 0 where it has no tile on it
template <Kind K> __device__ __forceinline__ int64_t line_length(const Args &a, Read &x) {
    const int rows = x.n * a.group, full = rows / WIDE, rest = rows % WIDE;
    const int64_t step = line_step<K>(a, x.past);
    if constexpr (K == ALL) return (rows + NARROW - 1) / NARROW * (step + x.n);
    x.n = (K == TALL ? full == 0 && rest <= NARROW : rest > NARROW || rest == 0) ? 0 : x.n;
    const int64_t len = K == TALL ? full * step + (int64_t)(WIDE / 2) * full * (full + 1) + (rest > NARROW ? step + rows : 0) : step + x.n;
    return x.n ? len : 0;
}
// a line: the reads' tiles in order. A narrow tile's length is its read's keys and COST. A wide one's is group times that, up to
// its last row (of a read's first k tiles k·step + 64·k·(k + 1) in all, step = group·(past + COST))
template <Kind K> struct Line {
    static constexpr bool W = K == TALL;
    const Args &a;
    Reads &r;
    int first = 0;     // the reads at hand: first …
    int64_t base = 0;  // the line's length before them
    int64_t total, piece;
    __device__ __forceinline__ Line(const Args &args, Reads &reads, const Read &x) : a(args), r(reads) {  // x: read `lane`
        float most = 0.0f;  // ALL: a tile's length by its rows
        auto look = [&](const Read &y) {
            if constexpr (K == ALL) most = fmaxf(most, (float)(step(y.past) + y.n) * (float)min(y.n * a.group, NARROW));
            return load(y);
        };
        total = look(x);
        if (a.p.n_seq > 64) {
            while (first + 64 < a.p.n_seq) base = total, first += 64, total = look(Read(a, first + lane_id()));
            first = 0, base = 0;
            load(x);
        }
        piece = uniform(max((int64_t)((double)total * a.per_piece) + 1, (int64_t)LEAST * (W ? a.group : 1)));
        // (a tile of k keys and r rows in p parts takes k / p keys' time and p·r rows' join, the least at pieces of √(CUT·k·r))
        if constexpr (K == ALL) piece = max(piece, (int64_t)uniform((int)__builtin_sqrtf(wave_max(most, lane_id()) * CUT)));
    }
    // where piece i begins
    __device__ __forceinline__ int64_t cut(int i) const { return i >= a.pieces ? total : min(i * piece, total); }
    __device__ __forceinline__ int piece_of(int64_t x) const {
        const float each = (float)(int64_t)((uint64_t)(uint32_t)here((int)(piece >> 32)) << 32 | (uint32_t)here((int)piece));
        int i = min((int)((float)x * __builtin_amdgcn_rcpf(each)), a.pieces - 1);  // (or one beside it)
        i -= i > 0 && cut(i) > x;
        i += i + 1 < a.pieces && cut(i + 1) <= x;
        return uniform(i);
    }
    __device__ __forceinline__ int64_t step(int past) const { return line_step<K>(a, past); }
    // the reads from `first` on; their end on the line
    __device__ __forceinline__ int64_t load() { return load(Read(a, first + lane_id())); }
    __device__ __forceinline__ int64_t load(Read x) {
        const int lane = lane_id();
        int64_t end = line_length<K>(a, x);
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t lo = __builtin_amdgcn_ds_bpermute(4 * (lane - d), (int)(uint32_t)end), hi = __builtin_amdgcn_ds_bpermute(4 * (lane - d), (int)(end >> 32));
            if (lane >= d) end += (int64_t)((uint64_t)hi << 32 | lo);
        }
        end += base;
        r.end[lane] = end, r.start[lane] = x.start, r.n[lane] = x.n, r.past[lane] = x.past;
        return lane_of(end, 63);
    }
};

// a tile on the line
template <Kind K> struct Tile {
    static constexpr bool W = K == TALL;
    int at;                    // its read: of those at hand
    int start, n, past;        // the read's
    int r0, rows;              // narrow: its first row of the read, its rows; wide: the read's rows in wide tiles
    int tau;                   // its place among the read's tiles
    int last, nb;              // the last key that one of its rows sees; its blocks of keys
    int64_t begin, len;        // and on the line

    // the last key that query i sees (past + i < 2^32)
    __device__ __forceinline__ int last_key(const Args &a, int i) const {
        return past < 0 ? -1 : (int)min((uint32_t)past + (uint32_t)i, (uint32_t)a.cap - 1u);
    }
    __device__ __forceinline__ int last_of(const Args &a, int r) const { return last_key(a, query_of(a, min(r, rows - 1))); }
    __device__ __forceinline__ void of_read(const Line<K> &w, int i) {
        at = i, start = uniform(w.r.start[i]), n = uniform(w.r.n[i]), past = uniform(w.r.past[i]);
        rows = n * w.a.group, r0 = rows / WIDE * WIDE;
        if constexpr (!W) rows -= r0;
        else if (rows - r0 <= NARROW) rows = r0;
        tau = 0;
    }
    __device__ __forceinline__ void measure(const Line<K> &w) {
        if constexpr (K == ALL) r0 = NARROW * tau, rows = min(NARROW, n * w.a.group - r0);
        len = w.step(past) + (W ? min(WIDE * (tau + 1), rows) : n);
        last = W ? last_of(w.a, WIDE * (tau + 1) - 1) : last_key(w.a, K == ALL ? query_of(w.a, r0 + rows - 1) : n - 1);
        nb = blocks_to(last);
    }
    // the block that place x of the line (begin < x < begin + len) cuts the tile in front of; 0 and nb: it does not
    __device__ __forceinline__ int block_at(const Line<K> &w, int64_t x) const {
        const int64_t u = x - begin;
        // (wide: to 22 bits, the same for all that ask)
        const int b = W ? uniform((int)((float)u * __builtin_amdgcn_rcpf((float)here(KB * w.a.group)))) : (int)(u / KB);
        return b < SLIVER ? 0 : b > nb - SLIVER ? nb : b;
    }
    // the one that holds place x of the line, x before its end
    __device__ __forceinline__ Tile(Line<K> &w, int64_t x) {
        int64_t mine = w.r.end[lane_id()];
        for (int64_t t; (t = lane_of(mine, 63)) <= x && w.first + 64 < w.a.p.n_seq; mine = w.r.end[lane_id()]) {
            w.base = t, w.first += 64;
            w.load();
        }
        of_read(w, (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(mine > x) | 1ull << 63));
        begin = at ? lane_of(mine, at - 1) : w.base;
        const int64_t y = x - begin, step = w.step(past);
        if constexpr (K == ALL) {
            const int tiles = (n * w.a.group + NARROW - 1) / NARROW;
            tau = uniform(min((int)((float)y * __builtin_amdgcn_rcpf((float)(step + n))), tiles - 1));  // (or one beside it)
            tau -= tau > 0 && tau * (step + n) > y;
            tau += tau + 1 < tiles && (tau + 1) * (step + n) <= y;
            begin += tau * (step + n);
        }
        if constexpr (W) {
            const float half = WIDE / 2, mid = 0.5f * ((float)step + half);
            const int tiles = (rows + WIDE - 1) / WIDE;
            tau = uniform(min((int)((float)y / (__builtin_sqrtf(mid * mid + half * (float)y) + mid)), tiles - 1));  // (or one beside it)
            auto upto = [&](int t) { return t * step + (int64_t)(WIDE / 2) * t * (t + 1); };
            tau -= tau > 0 && upto(tau) > y;
            tau += tau + 1 < tiles && upto(tau + 1) <= y;
            begin += upto(tau);
        }
        measure(w);
    }
    // the next one (there is one)
    __device__ __forceinline__ void next(Line<K> &w) {
        begin += len;
        if (K == REST || (K == ALL ? NARROW * ++tau >= n * w.a.group : WIDE * ++tau >= rows)) {
            uint64_t more;
            for (int from = at + 1;; from = 0) {
                more = from < 64 ? __builtin_amdgcn_ballot_w64(w.r.n[lane_id()] > 0) >> from << from : 0;
                if (more || w.first + 64 >= w.a.p.n_seq) break;
                w.base = begin, w.first += 64;
                w.load();
            }
            of_read(w, more ? (int)__builtin_ctzll(more) : 63);
        }
        measure(w);
    }
};

// the blocks i0 … i1 − 1 of a tile that are a piece's
struct Share {
    int i0, i1;
    bool all;
};
template <Kind K> __device__ __forceinline__ Share share_of(const Line<K> &w, const Tile<K> &t, int64_t x0, int64_t x1) {
    Share s{0, t.nb, true};
    if (x0 > t.begin) s.i0 = t.block_at(w, x0);
    if (x1 < t.begin + t.len) s.i1 = t.block_at(w, x1);
    s.all = s.i0 == 0 && s.i1 == t.nb;
    return s;
}
// a piece's place for its part of a cut tile, and in `to` (of that place, or of LDS) which pieces have the others (the last wave's
// work: of few keys it has the least)
__device__ __forceinline__ size_t place_of(const Args &a, const Share &share, int kvh, int piece) {
    return ((size_t)kvh * a.pieces + piece) * 2 + (share.i0 == 0);
}
template <Kind K> __device__ __forceinline__ void part_of(const Line<K> &w, const Tile<K> &t, Part &to) {
    if (threadIdx.x < 64 * (PW - 1)) return;
    int first = w.piece_of(t.begin), end = first + 1;
    if (w.cut(end) < t.begin + t.len && t.block_at(w, w.cut(end)) == 0) first++, end++;  // (it leaves the beginning to the next one)
    for (end = max(w.piece_of(t.begin + t.len - 1) + 1, end); end - 1 > first && t.block_at(w, w.cut(end - 1)) == t.nb;) end--;
    if (threadIdx.x == 64 * (PW - 1))
        to = K == TALL ? Part{first, end - first, t.start, WIDE * t.tau, min(WIDE, t.rows - WIDE * t.tau)}
                       : Part{first, end - first, t.start, t.r0, t.rows};
}
// the two places of a piece that has no cut tile are empty (the same wave's stores, in order)
template <bool W> __device__ __forceinline__ void no_parts(const Args &a, int kvh, int piece) {
    const int k = (int)threadIdx.x - 64 * (PW - 1);
    if (k >= 0 && k < 2) a.part[W].of[((size_t)kvh * a.pieces + piece) * 2 + k].n = 0;
}
__device__ __forceinline__ float *out_row(const Args &a, int start, int kvh, int r) {
    const int i = query_of(a, r);
    return a.out + ((size_t)(start + i) * a.n_head + (size_t)kvh * a.group + (r - i * a.group)) * D;
}
__device__ __forceinline__ const float *q_row(const Args &a, int start, int kvh, int r) {
    const int i = query_of(a, r);
    return a.q + (size_t)(start + i) * a.q_stride + ((size_t)kvh * a.group + (r - i * a.group)) * D;
}

// the first rows of the halves of a run of blocks b0, b0 + step, …: lane 2j + h has the j-th one's half h, of 32 at a time. Half a
// block lies in one page
struct Rows {
    int at[2];
    uint32_t bad;  // bit h: half h has no page
};
struct Run {
    const int32_t *table;
    int b0, step, last, shift, n_page;
    int row;
    uint64_t gone;  // the halves without a page
    __device__ __forceinline__ void fetch(int j) {
        const int lane = lane_id();
        const uint32_t key = min(KB * (uint32_t)(b0 + step * (j + (lane >> 1))) + 16u * (lane & 1), (uint32_t)last & ~15u);
        const int page = table[key >> shift];
        const bool bad = (uint32_t)page >= (uint32_t)n_page;
        row = bad ? 0 : (page << shift) + (int)(key & ((1u << shift) - 1));
        gone = __builtin_amdgcn_ballot_w64(bad);
    }
    __device__ __forceinline__ Rows of(int j) {
        if (j && (j & 31) == 0) fetch(j);
        return Rows{{__builtin_amdgcn_readlane(row, 2 * (j & 31)), __builtin_amdgcn_readlane(row, 2 * (j & 31) + 1)},
                    (uint32_t)(gone >> (2 * (j & 31))) & 3u};
    }
};
template <Kind K> __device__ __forceinline__ Run run_of(const Args &a, const Line<K> &w, const Tile<K> &t, int b0, int step) {
    return Run{a.p.table + (size_t)(w.first + t.at) * a.p.max_pages, b0, step, t.last, a.p.shift, a.n_page, 0, 0};
}
// the keys of block i that a row of `keys` sees, of the lane's 16 (bits 0 … 3, 8 … 11, 16 …, 24 …)
__device__ __forceinline__ uint32_t sees(int keys, int i, int hf, uint32_t bad) {
    return low_bits(keys - (KB * i + here(4 * hf))) & (bad & 1 ? 0xFFFF0000u : ~0u) & (bad & 2 ? 0x0000FFFFu : ~0u);
}

// 4 bytes a lane from p to LDS bytes lds + 4·lane
__device__ __forceinline__ void lds_load4_at(const void *p, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}

constexpr int WAVE_F16 = TILE, WAVE_Q8 = 2 * QT + 16;  // 16-byte chunks of a wave's LDS: K and V of a block; two raw ones
constexpr int RAW = 1024 + 1024 + 256;                 // bytes of 8 raw rows: K, V, their scales (64 + 64, twice)
struct Shared {
    Reads reads[PW];  // (each wave its own: nobody waits)
    float ml[PW][2][KB];
    Part part;  // of the tile at hand
    int last;   // its last part is this one
};

// The rows ra … rb − 1 of a cut tile: 32 lanes of 4 dims to a row; where the rows are fewer than the groups of 32, several groups to
// a row's parts. HERE: parts that workgroups of this launch stored
struct Join {
    float4 y[8][32];
    float2 ml[8];
};
template <bool HERE> __device__ __forceinline__ void join_rows(const Args &a, int w, int kvh, const Part &t, int ra, int rb, Join &sh) {
    constexpr int U = HERE ? 8 : 4;  // parts of a row at once: here the row's one workgroup waits for each load, there many do
    const int tid = threadIdx.x, gr = tid >> 5, j = tid & 31, nr = rb - ra;
    const Parts &p = a.part[w];
    const int height = w ? WIDE : NARROW;
    auto get = [](const float4 *from) {
        if constexpr (!HERE) return *from;
        const float2 lo = get64(from), hi = get64(&from->z);
        return make_float4(lo.x, lo.y, hi.x, hi.y);
    };
    const int lg = nr > 4 ? 3 : nr > 2 ? 2 : nr > 1 ? 1 : 0, G = 8 >> lg;  // 2^lg rows at once, G groups to each
    for (int r = ra; r < rb; r += 1 << lg) {
        const int row = min(r + (gr & ((1 << lg) - 1)), rb - 1), g = gr >> lg;
        float top = M_NONE, sum = 0.0f;
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float c = 0.0f;
        const uint32_t at0 = ((uint32_t)(kvh * a.pieces + t.first) * 2) * height + row;  // (times 128: below 2^25)
        for (int e0 = g; e0 < t.n; e0 += U * G) {
            float4 ml[U], in[U];
#pragma unroll
            for (int q = 0; q < U; q++) {
                const int e = e0 + q * G;
                ml[q] = make_float4(M_NONE, 0.0f, c, 0.0f), in[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (e < t.n) {
                    const uint32_t at = at0 + (uint32_t)(2 * e + (e == 0)) * height;
                    ml[q] = get(p.ml + at);
                    in[q] = get(reinterpret_cast<const float4 *>(p.sums + (at * D + 4 * j)));
                }
            }
            c = ml[0].z;  // (a row's parts have the same)
            float to = top;
#pragma unroll
            for (int q = 0; q < U; q++) to = fmaxf(to, ml[q].x);
            const float f = __builtin_amdgcn_exp2f((top - to) * c);
            top = to, sum *= f, y.x *= f, y.y *= f, y.z *= f, y.w *= f;
#pragma unroll
            for (int q = 0; q < U; q++) {
                const float h = __builtin_amdgcn_exp2f((ml[q].x - to) * c);
                sum = fmaf(ml[q].y, h, sum);
                y.x = fmaf(in[q].x, h, y.x), y.y = fmaf(in[q].y, h, y.y), y.z = fmaf(in[q].z, h, y.z), y.w = fmaf(in[q].w, h, y.w);
            }
        }
        if (G > 1) {  // (one pass)
            __syncthreads();
            sh.y[gr][j] = y;
            if (j == 0) sh.ml[gr] = make_float2(top, sum);
            __syncthreads();
            if (g == 0) {
                float to = top;
                for (int e = 1; e < G; e++) to = fmaxf(to, sh.ml[gr + (e << lg)].x);
                const float f = __builtin_amdgcn_exp2f((top - to) * c);
                sum *= f, y.x *= f, y.y *= f, y.z *= f, y.w *= f;
                for (int e = 1; e < G; e++) {
                    const float4 z = sh.y[gr + (e << lg)][j];
                    const float2 ml = sh.ml[gr + (e << lg)];
                    const float h = __builtin_amdgcn_exp2f((ml.x - to) * c);
                    sum = fmaf(ml.y, h, sum);
                    y.x = fmaf(z.x, h, y.x), y.y = fmaf(z.y, h, y.y), y.z = fmaf(z.z, h, y.z), y.w = fmaf(z.w, h, y.w);
                }
            }
        }
        if (g == 0 && r + (gr & ((1 << lg) - 1)) < rb) {
            const float by = sum == 0.0f ? 0.0f : 1.0f / sum;  // no key seen: zeros
            *reinterpret_cast<float4 *>(out_row(a, t.start, kvh, t.r0 + row) + 4 * j) = make_float4(y.x * by, y.y * by, y.z * by, y.w * by);
        }
    }
}

// ---- reads of few rows -------------------------------------------------------------------------------------------------------
//
// A wave's block is K and V in its own LDS (layouts and products are k_kv_attn_split's): f16 one buffer each, filled again as soon
// as it is read, q8_0 raw in two.
//
// Bound: of few keys latency (a token over 1300 keys 10.9 µs, of which lengths, pages, keys, each a load that the next one waits
// for, 5 µs, and the join 2); of many HBM: 64 reads' tokens over 300 … 6000 f16 keys (505 MB) 100 µs, over 8000 (2.1 GB) 350, 6.2 TB/s
// of them from one to the other; over q8_0 rows (269 MB) 67, where conversions and softmax take as long as the loads.
// JOIN: who joins the parts of a cut tile: a second launch, or the last of its workgroups, which share an XCD or do not
enum Joins { SECOND, NEAR, FAR };
template <bool Q8, Joins JOIN> __device__ __forceinline__ void narrow(const Args &a, int kvh, int piece, const Read &x, uint4_t *s_kv, Shared &sh) {
    constexpr bool ONE = JOIN != SECOND, XL = JOIN == NEAR;
    constexpr int WAVE = Q8 ? WAVE_Q8 : WAVE_F16;
    static_assert(WAVE >= 1024, "a wave's sums fit");
    const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), hf = lane >> 5, c = lane & 31;
    if (!ONE && a.pieces > 1) no_parts<false>(a, kvh, piece);
    constexpr Kind K = ONE ? ALL : REST;
    Line<K> line(a, sh.reads[wave], x);
    const int64_t x0 = line.cut(piece), x1 = line.cut(piece + 1);
    if (x0 >= x1) return;
    const size_t head0 = (size_t)kvh * a.kv.n_ctx;
    uint4_t *tile = s_kv + WAVE * wave;
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
    for (Tile<K> t(line, x0);; t.next(line)) {
        const Share own = share_of(line, t, x0, x1);
        if (own.i0 < own.i1 || own.all) {
            const int i1 = own.i1, rc = t.r0 + min(c, t.rows - 1);
            const int all_to = (t.last_key(a, query_of(a, t.r0)) + 1) / KB;  // blocks that all rows see the whole of
            const int keys = t.last_key(a, query_of(a, rc)) + 1;             // keys that the lane's row sees
            int i = own.i0 + wave, j = 0, b = 0;
            Run run = run_of(a, line, t, i, PW);
            if (i < i1) run.fetch(0);
            float qx[8][8];
            q_load<8, Q8>(q_row(a, t.start, kvh, rc) + (Q8 ? 16 : 8) * hf, qx);
            __syncthreads();  // (the sums of the tile before are read)
            Rows now{{0, 0}, 0}, then{{0, 0}, 0};
            if (i < i1) {
                now = run.of(0);
                if constexpr (Q8) {
                    load_q8(now.at[0], now.at[1], 0);
                } else {
                    load(now.at[0], now.at[1], false);
                    load(now.at[0], now.at[1], true);
                }
            }
            const size_t place = place_of(a, own, kvh, piece), part = place * NARROW;
            if (!own.all) part_of(line, t, ONE ? sh.part : a.part[0].of[place]);
            half8 qh[8], ql[8];
            const float sc = q_split<8, 2>(qx, a.scale, qh, ql);
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
                        then = run.of(j + 1);
                        wait_reads();  // of the other buffer, a block ago
                        load_q8(then.at[0], then.at[1], b ^ 1);
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
                                then = run.of(j + 1);
                                load(then.at[0], then.at[1], false);
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
                    seen = sees(keys, i, hf, now.bad);
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
                    if (more) load(then.at[0], then.at[1], true);
                }
                i += PW, j++;
                b ^= Q8;
                now = then;
            };
            auto whole = [&] { return i < all_to && now.bad == 0; };
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
            if (hf == 0) sh.ml[wave][0][c] = m, sh.ml[wave][1][c] = l;
            __syncthreads();
            m = M_NONE, l = 0.0f;
#pragma unroll
            for (int w = 0; w < PW; w++) m = fmaxf(m, sh.ml[w][0][c]);
            float4 y[4];
#pragma unroll
            for (int x = 0; x < 4; x++) y[x] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < PW; w++) {
                const float f = __builtin_amdgcn_exp2f((sh.ml[w][0][c] - m) * sc);
                l = fmaf(sh.ml[w][1][c], f, l);
                const float4 *from = reinterpret_cast<const float4 *>(s_kv + WAVE * w) + 4 * 64 * wave + lane;
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const float4 z = from[64 * x];
                    y[x].x = fmaf(z.x, f, y[x].x), y[x].y = fmaf(z.y, f, y[x].y), y[x].z = fmaf(z.z, f, y[x].z), y[x].w = fmaf(z.w, f, y[x].w);
                }
            }
            const float by = !own.all ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;  // no key seen: zeros
            float *to = own.all ? out_row(a, t.start, kvh, rc) : a.part[0].sums + (part + c) * D;
            to += 32 * wave + 4 * hf;
            float4 *ml = a.part[0].ml + part + c;
            if (ONE && !own.all) {
                if (c < t.rows) {
#pragma unroll
                    for (int x = 0; x < 4; x++) put64(to + 8 * x, y[x].x, y[x].y, XL), put64(to + 8 * x + 2, y[x].z, y[x].w, XL);
                    if (wave == 0 && hf == 0) put64(ml, m, l, XL), put64(&ml->z, sc, 0.0f, XL);
                }
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this thread's stores are performed
                __syncthreads();
                const Part whole = sh.part;
                if (threadIdx.x == 0) {
                    uint32_t *ticket = a.tickets + (size_t)TICKET * (kvh * a.pieces + whole.first);
                    constexpr int SCOPE = XL ? __HIP_MEMORY_SCOPE_WORKGROUP : __HIP_MEMORY_SCOPE_AGENT;
                    sh.last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, SCOPE) == (uint32_t)(whole.n - 1);
                    if (sh.last) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, SCOPE);  // for the next call
                }
                __syncthreads();
                if (sh.last) {
                    join_rows<true>(a, 0, kvh, whole, 0, whole.rows, *reinterpret_cast<Join *>(s_kv));
                    __syncthreads();  // (the next tile's loads go there)
                }
                if (t.begin + t.len >= x1) break;
                continue;
            }
            if (!own.all && c < t.rows && wave == 0 && hf == 0) *ml = make_float4(m, l, sc, 0.0f);
            if (c < t.rows)
#pragma unroll
                for (int x = 0; x < 4; x++)
                    *reinterpret_cast<float4 *>(to + 8 * x) = make_float4(y[x].x * by, y[x].y * by, y[x].z * by, y[x].w * by);
        }
        if (t.begin + t.len >= x1) break;
    }
}

// ---- reads of many rows ------------------------------------------------------------------------------------------------------
//
// Bound: the matrix cores and their power: four chunks of 2000 over 8000 keys (590 GFLOP, as pairs twice that) 1.025 ms, 1.15
// PFLOP/s, where a library f16 product of 8192³ reaches 1.14, over q8_0 rows 1.14 ms (with a block's quants in registers until
// they are made f16, 56 registers spilled, 2.06); four prompts of 1925 (121 GFLOP as pairs) 158 µs, of which 9 % of the products
// are of keys past a row's own, 13 µs the second launch, 20 that workgroups wait for the last. Of two waves on a SIMD the one at
// its scores goes first (without 1.046 ms; the one at its values first 1.043). Loads four stages ahead or one, and a barrier a
// stage or every second one, take the same time.
template <bool Q8> __device__ __forceinline__ void wide(const Args &a, int kvh, int piece, const Read &x, uint4_t *s_kv, Shared &sh) {
    const int wave = uniform((int)threadIdx.x >> 6);
    if (a.pieces > 1) no_parts<true>(a, kvh, piece);
    Line<TALL> line(a, sh.reads[wave], x);
    const int64_t x0 = line.cut(piece), x1 = line.cut(piece + 1);
    if (x0 >= x1) return;
    const size_t head0 = (size_t)kvh * a.kv.n_ctx;

    for (Tile<TALL> t(line, x0);; t.next(line)) {
        const Share own = share_of(line, t, x0, x1);
        if (own.i0 < own.i1 || own.all) {
            const int lane = lane_id(), hf = lane >> 5, c = lane & 31;
            // K and V of a block as f16, K a block ahead of V: the next block's scores are computed under this one's softmax (the layouts
            // are k_kv_attn's). f16 rows: four buffers, filled two at a time, behind every second barrier; a wave loads 4 rows of each half
            // straight into LDS. q8_0 rows: two buffers, and four raw ones of each wave's own, which has 8 rows of a block: loaded straight
            // into LDS four blocks ahead, and made f16 by the wave that loaded them, K two blocks and V one before they are used
            char *stage = reinterpret_cast<char *>(s_kv);
            const uint32_t slds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)stage, slds = slds0 + 16u * 64 * wave;
            const int lrow = Q8 ? 8 * wave + (lane >> 3) : 4 * wave + (lane >> 4), lc = Q8 ? lane & 7 : lane & 15;
            const uint32_t koff = 2 * D * lrow + 16 * (lc ^ (lrow & 15)), voff = 2 * D * lrow + 16 * (lc ^ (4 * (lrow & 3)));  // the same for row lrow + 16
            auto issue = [&](const Rows &x, int b, bool is_v) {
#pragma unroll
                for (int h = 0; h < 2; h++)
                    lds_load16((const char *)(is_v ? a.kv.v : a.kv.k) + (head0 + x.at[h]) * (2 * D), is_v ? voff : koff,
                               slds + 16u * (b * TILE + (is_v ? K_CHUNKS : 0) + 256 * h));
            };
            const int raw0 = 16 * 2 * TILE + RAW * 4 * wave;
            auto issue_q8 = [&](const Rows &x, int slot) {
                const size_t row = head0 + x.at[0] + (x.at[1] - x.at[0]) * (wave >> 1) + 8 * (wave & 1);
                const uint32_t to = slds0 + raw0 + RAW * slot;
                lds_load16((const char *)a.kv.k + row * D, 16 * lane, to);
                lds_load16((const char *)a.kv.v + row * D, 16 * lane, to + 1024);
                lds_load4_at((const char *)(lane & 16 ? a.kv.vd : a.kv.kd) + row * 8 + 4 * (lane & 15), to + 2048);  // a row's scales are 8 bytes
            };
            // the lane's bytes: 16 raw quants, their scale, and two f16 chunks of K and of V (the other one at ^ 16)
            const int c_raw = raw0 + 16 * lane, c_d = raw0 + 2048 + 8 * (lane >> 3) + 2 * (lc >> 1);
            const int c_k = 16 * (16 * lrow + ((2 * lc) ^ (lrow & 15))), c_v = 16 * (K_CHUNKS + 16 * lrow + ((2 * lc) ^ (4 * (lrow & 3))));
            auto commit = [&](int slot, int b, bool is_v) {
                const uint4_t q = *reinterpret_cast<const uint4_t *>(stage + here(c_raw) + RAW * slot + (is_v ? 1024 : 0));
                const _Float16 d = *reinterpret_cast<const _Float16 *>(stage + here(c_d) + RAW * slot + (is_v ? 64 : 0));
                const int to = here(is_v ? c_v : c_k);
                *reinterpret_cast<half8 *>(stage + to + 16 * TILE * b) = dequant8(q[0], q[1], half2_t{d, d});
                *reinterpret_cast<half8 *>(stage + (to ^ 16) + 16 * TILE * b) = dequant8(q[2], q[3], half2_t{d, d});
            };
            // the lane's bytes of a block: K's step ks at k_at ^ 32·ks (chunk 2ks + hf of row c), V's tile u at v_at ^ 64·u
            const int vrow = 4 * hf + ((lane & 15) >> 2);
            const int k_at = 16 * (16 * c + (hf ^ (c & 15)));
            const int v_at = 16 * (K_CHUNKS + 16 * vrow + ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ (4 * (vrow & 3)))) + 8 * (lane & 1);
            const int i0 = own.i0, n_st = own.i1 - i0;
            const int r0 = WIDE * t.tau + KB * wave, rc = min(r0 + c, t.rows - 1);
            const WaveBlocks mine = wave_blocks(r0 < t.rows, t.last_of(a, r0), t.last_of(a, r0 + KB - 1));
            Run run = run_of(a, line, t, i0, 1);
            if (n_st > 0) run.fetch(0);
            Rows r_last{{0, 0}, 0};  // f16: of the last stage whose K is on its way
            uint32_t gone = 0;       // and the halves without a page of this stage and those after it, a pair of bits each
            half8 qh[8], ql[8];
            float sc;
            {
                float qx[8][8];
                q_load<8>(q_row(a, t.start, kvh, rc) + 8 * hf, qx);
                __syncthreads();  // (the tile before is done with the buffers)
                if constexpr (Q8) {
                    if (n_st > 0)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const Rows x = run.of(min(e, n_st - 1));
                            gone |= x.bad << (2 * e);
                            issue_q8(x, e);
                        }
                } else {
                    if (n_st > 0) {
                        const Rows one = run.of(0), two = run.of(min(1, n_st - 1));
                        r_last = run.of(min(2, n_st - 1));
                        gone = one.bad | two.bad << 2 | r_last.bad << 4;
                        issue(one, 0, false), issue(two, 1, false), issue(r_last, 2, false);
                        issue(one, 0, true), issue(two, 1, true);
                    }
                }
                sc = q_split<8, 2>(qx, a.scale, qh, ql);
            }
            if constexpr (Q8) {
                wait_loads<0>();
                commit(0, 0, false), commit(0, 0, true), commit(1, 1, false);
            }
            float m = M_NONE, l = 0.0f;
            f32x16 o[4];
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int x = 0; x < 16; x++) o[u][x] = 0.0f;

            // stage st in buffer b: its scores are in s; the next stage's are computed into sn under the softmax's VALU work
            auto step = [&](int st, int b, f32x16 &s, f32x16 &sn, auto is_masked) {
                constexpr bool MASK = decltype(is_masked)::value;
                // this wave's loads of K stage st + 1 and V stage st (f16: of the stages after them too) are in, its reads of K stage
                // st and V stage st − 1 have their values; behind the barrier everyone's, and the buffers are free
                if (Q8 || (st & 1) == 0) {
                    if constexpr (Q8) asm volatile("s_waitcnt vmcnt(3) lgkmcnt(0)" ::: "memory");
                    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                    __builtin_amdgcn_s_barrier();
                    asm volatile("" ::: "memory");
                }
                const uint32_t bad = gone & 3u;
                {  // (past the last stage: its loads once more)
                    if constexpr (Q8) {
                        const Rows four = run.of(min(st + 4, n_st - 1));
                        gone |= four.bad << 8;
                        issue_q8(four, st & 3);
                    } else if ((st & 1) == 0) {
                        const Rows three = run.of(min(st + 3, n_st - 1)), four = run.of(min(st + 4, n_st - 1));
                        gone |= three.bad << 6 | four.bad << 8;
                        issue(three, (st + 3) & 3, false), issue(four, st & 3, false);
                        issue(r_last, (st + 2) & 3, true), issue(three, (st + 3) & 3, true);
                        r_last = four;
                    }
                    gone >>= 2;
                }
                auto convert = [&] {
                    if constexpr (Q8) commit((st + 2) & 3, b, false), commit((st + 1) & 3, b ^ 1, true);
                };
                const int i = i0 + st;
                if constexpr (MASK)
                    if (i >= mine.any) {
                        convert();
                        return;
                    }
                uint32_t seen = 0;
                if constexpr (MASK) {
                    const int keys = t.last_of(a, r0 + (lane_id() & 31)) + 1;  // that the lane's row sees
                    seen = sees(keys, i, hf, bad);
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
                // the order pinned: behind each score MFMA of the next stage its share of this stage's softmax
                // (past the last stage: scores of what the buffer holds, not used)
                const char *kb = stage + (Q8 ? 16 * TILE * (b ^ 1) : 0);
                // (the sums below are not kept from stage to stage)
                const int k0 = here(k_at + (Q8 ? 0 : 16 * TILE * ((st + 1) & 3))), v0 = here(v_at + (Q8 ? 0 : 16 * TILE * (st & 3)));
                const auto *vb = (const __attribute__((address_space(3))) char *)stage + (Q8 ? 16 * TILE * b : 0);
                auto vread = [&](int u, int ss) {
                    const auto *p = vb + (v0 ^ 64 * u) + 256 * 16 * ss;
                    const fp16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)p);
                    const fp16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4 *)(p + 256 * 8));
                    half8 v;
                    __builtin_memcpy(&v, &lo, 8);
                    __builtin_memcpy((char *)&v + 8, &hi, 8);
                    return v;
                };
                uint32_t ph[8], pl[8];
                float ls;
                half8 f[8], v[4];
#pragma unroll
                for (int ks = 0; ks < 3; ks++) f[ks] = *reinterpret_cast<const half8 *>(kb + (k0 ^ 32 * ks));
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int ks = 0; ks < 8; ks++) {
                    sn = __builtin_amdgcn_mfma_f32_32x32x16_f16(f[ks], qh[ks], ks ? sn : f32x16{}, 0, 0, 0);
                    if (ks + 3 < 8) f[ks + 3] = *reinterpret_cast<const half8 *>(kb + (k0 ^ 32 * (ks + 3)));
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
                convert();
                __builtin_amdgcn_s_setprio(0);
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
                __builtin_amdgcn_s_setprio(1);  // (scores before a neighbour's values)
                if constexpr (MASK)
                    if (odd) put_nan(o, seen, vread);
            };
            // K and V of stage 0, K of stage 1
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            f32x16 s0, s1;
#pragma unroll
            for (int ks = 0; ks < 8; ks++) {  // (without a stage: scores of what the buffer holds, not used)
                const half8 f = *reinterpret_cast<const half8 *>(stage + (k_at ^ 32 * ks));
                s0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, qh[ks], ks ? s0 : f32x16{}, 0, 0, 0);
                s0 = __builtin_amdgcn_mfma_f32_32x32x16_f16(f, ql[ks], s0, 0, 0, 0);
            }
            // two stages at a time, both kinds of step passing one barrier a stage: a wave's blocks may be masked where another's
            // are not
            auto whole2 = [&](int st) { return st + 1 < n_st && i0 + st + 1 < mine.whole && (gone & 15u) == 0; };
            for (int st = 0; st < n_st;) {
                for (; whole2(st); st += 2) {
                    step(st, 0, s0, s1, std::false_type{});
                    step(st + 1, 1, s1, s0, std::false_type{});
                }
                for (int e = st + 2; st < min(e, n_st); st++) {
                    step(st, st & 1, s0, s1, std::true_type{});
                    s0 = s1;
                }
            }
            const size_t place = place_of(a, own, kvh, piece), part = place * WIDE;
            if (!own.all) part_of(line, t, a.part[1].of[place]);
            l = pair_sum<32>(l);
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // (the next tile's loads go over these buffers)

            const int ln = lane_id(), row_of = KB * wave + (ln & 31), r = WIDE * t.tau + row_of, half = ln >> 5;
            const float by = !own.all ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;  // no key seen: zeros
            float *to;
            if (own.all) {
                to = out_row(a, t.start, kvh, min(r, t.rows - 1));
            } else {
                const size_t row = part + row_of;
                to = a.part[1].sums + row * D;
                if (r < t.rows && half == 0) a.part[1].ml[row] = make_float4(m, l, sc, 0.0f);
            }
            if (r < t.rows)
#pragma unroll
                for (int u = 0; u < 4; u++)
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        *reinterpret_cast<float4 *>(to + 4 * half + 32 * u + 8 * x) =
                            make_float4(o[u][4 * x] * by, o[u][4 * x + 1] * by, o[u][4 * x + 2] * by, o[u][4 * x + 3] * by);
        }
        if (t.begin + t.len >= x1) break;
    }
}

// The workgroups of wide tiles and those of narrow ones, of the kind first that has more to do: 64 tokens beside 512 rows 134 µs,
// narrow first, for 145; four prompts with their last narrow tiles 155, wide first, for 161. Where neither has much more (f16; over
// q8_0 rows it is no faster), half of each kind in turn, so that a CU has one of each: two chunks of 509 rows beside 61 tokens 146
// µs for 157 (wide first) and 159. To tell costs 1 µs. In turn one by one, a CU got two of one kind and its neighbour none.
// By r, the narrow line's length over the wide one's (chunks of 512 rows beside 20 or 61 tokens; µs in turn, wide first, narrow first):
//   over 5000 keys, the wide line 172000: r 0.03 113 108 112, 0.1 115 116 117, 0.2 124 129 131, 0.5 153 169 169, 1.2 229 260 244
//   over 2000, 76000: r 4.5 295 313 299, 6 375 389 370;   over 900, 41000: r 1.2 75 82 79, 4.5 173 190 177, 6 217 232 218
//   over 400, 25000: r 0.6 48 42 46, 1.2 53 53 56, 2 69 73 76;   over 1500 q8_0 keys: r 1.7 106 104 102, 2.3 117 121 118
// so in turn from r 0.15 to 5, where the wide line is 1.5 of the least pieces to each of its workgroups (36864 here), and else by r 2.
constexpr float TURNS_FROM = 0.15f, TURNS_TO = 5.0f, TURNS_PIECES = 1.5f, NARROW_FIRST = 2.0f;
template <bool Q8> __global__ __launch_bounds__(64 * PW, 2) void k_page_attn(Args a) {
    __shared__ __attribute__((aligned(16))) uint4_t s_kv[PW * (Q8 ? WAVE_Q8 : WAVE_F16)];
    static_assert(!Q8 || 16 * PW * WAVE_Q8 >= 16 * 2 * TILE + 4 * RAW * PW, "the wide tiles' buffers fit");
    __shared__ Shared sh;
    const int kvh = blockIdx.x % a.kv.n_kv, unit = blockIdx.x / a.kv.n_kv;
    const Read mine(a, lane_id());
    bool is_narrow = true;
    int piece = unit;
    if (a.wide) {
        float lw = 0.0f, ln = 0.0f;  // the lines' lengths, about
        Read x = mine;
        for (int first = 64;; x = Read(a, first + lane_id()), first += 64) {
            const int rows = x.n * a.group, rest = rows % WIDE;
            const float tiles = (float)(rows / WIDE + (rest > NARROW)), held = (float)max(x.past, 0) + COST;
            lw = fmaf(tiles, fmaf(held, (float)a.group, WIDE / 2 * tiles), lw);
            ln += rest > 0 && rest <= NARROW ? held + (float)x.n : 0.0f;
            if (first >= a.p.n_seq) break;
        }
        lw = wave_sum(lw, lane_id()), ln = wave_sum(ln, lane_id());
        const bool narrow_first = __builtin_amdgcn_ballot_w64(ln >= NARROW_FIRST * lw) != 0;  // (alike in all lanes)
        const bool halves = !Q8 && __builtin_amdgcn_ballot_w64(ln > TURNS_FROM * lw && ln < TURNS_TO * lw &&
                                                               lw > TURNS_PIECES * LEAST * a.group * a.pieces) != 0;
        // n of the one kind, n of the other, and what is left of each
        const int n = halves ? (a.pieces + 1) / 2 : a.pieces, left = a.pieces - n;
        const bool other = unit >= n && (unit < 2 * n || unit >= 2 * n + left);
        piece = unit < n ? unit : unit < 2 * n + left ? unit - n : unit - n - left;
        is_narrow = other != narrow_first;
    }
    if (uniform((int)is_narrow)) narrow<Q8, SECOND>(a, kvh, piece, mine, s_kv, sh);
    else wide<Q8>(a, kvh, piece, mine, s_kv, sh);
}

// Tokens: narrow tiles alone, the parts of a cut one joined by the last of its workgroups. A token over 1300 keys 10.9 µs, by the
// other kernel and its second launch 12.9; 64 reads' 100 for 104, 16 and 48 rows of another read 33 for 38; on one KV head, whose
// workgroups are on all XCDs, 7 tokens 13.9 for 16.4. But a read of 16 rows over 32000 keys 41 for 34, of 64 rows 62 for 59; and of
// more rows, where a step of 200 tokens would take 212 for 218, one read of 130 102 for 72.
template <bool Q8, Joins JOIN> __global__ __launch_bounds__(64 * PW, 2) void k_page_few(Args a) {
    __shared__ __attribute__((aligned(16))) uint4_t s_kv[PW * (Q8 ? WAVE_Q8 : WAVE_F16)];
    __shared__ Shared sh;
    narrow<Q8, JOIN>(a, blockIdx.x % a.kv.n_kv, blockIdx.x / a.kv.n_kv, Read(a, lane_id()), s_kv, sh);
}

// The second launch: the rows of a cut tile shared out among as many workgroups as it has parts (SHARES times as many), those of
// the pieces
__global__ __launch_bounds__(256) void k_page_attn_join(Args a) {
    __shared__ Join sh;
    const int kvh = blockIdx.x % a.kv.n_kv, unit = blockIdx.x / a.kv.n_kv, share = unit / a.pieces, piece = unit - share * a.pieces;
    const int w = share > 0, shares = w ? SHARES : 1;  // (share 0: the narrow tiles')
    const size_t mine = ((size_t)kvh * a.pieces + piece) * 2;
    const Part both[2] = {a.part[w].of[mine], a.part[w].of[mine + 1]};
    for (int k = 0; k < 2; k++) {
        const Part &t = both[k];
        if (t.n == 0) continue;
        const int mth = (piece - t.first) * shares + (w ? share - 1 : 0), of = t.n * shares;
        join_rows<false>(a, w, kvh, t, t.rows * mth / of, t.rows * (mth + 1) / of, sh);
    }
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
    if (!htr_rows_fit(q_stride, n, qd)) return htr_fail("%s: %zu rows %zu floats apart", me, n, q_stride);
    if (((uintptr_t)d_q | (uintptr_t)d_out) & 15) return htr_fail("%s: pointers must be 16-byte aligned", me);
    if (htr_overlap(d_q, 4 * (q_stride * (n - 1) + qd), d_out, 4 * qd * n)) return htr_fail("%s: the output overlaps the queries", me);
    if (htr_kv_overlaps(a.kv, d_out, 4 * qd * n)) return htr_fail("%s: the output overlaps the cache", me);
    const struct {
        const void *p;
        size_t n;
    } read[3] = {{a.p.start, 4 * ((size_t)a.p.n_seq + 1)}, {a.p.past, 4 * (size_t)a.p.n_seq}, {a.p.table, 4 * (size_t)a.p.n_seq * a.p.max_pages}};
    for (const auto &r : read)
        if (htr_overlap(r.p, r.n, d_out, 4 * qd * n)) return htr_fail("%s: the output overlaps the pages' arrays", me);
    const uint64_t group = (uint64_t)(n_head / kv->n_kv);  // (rows · group < 2^31: the kernel's quotients)
    if (n * group * group >= 1ull << 31 || n * group > 1u << 30) return htr_fail("%s: %zu rows of %d heads", me, n, n_head);
    const double rows = (double)(n * group), held = (double)a.p.max_pages * pages->page;  // (a line's length, whatever the arrays hold)
    if (a.p.n_seq * (rows / WIDE + 2) * group * (held + rows + COST) >= 0x1p62)
        return htr_fail("%s: %d reads of %zu rows of %d heads over up to %.0f rows", me, a.p.n_seq, n, n_head, held);
    HTR_TRY(htr_check_alive(dev));
    const HtrOnDevice on(dev);
    a.q = d_q, a.q_stride = q_stride, a.out = d_out, a.n_head = n_head, a.group = n_head / kv->n_kv;
    a.n_page = kv->n_ctx / pages->page, a.scale = scale;
    a.per_group = (uint32_t)(((1ull << 31) + a.group - 1) / a.group), a.cap = a.p.max_pages << a.p.shift;
    a.pieces = std::max(1, 2 * dev->n_cu / kv->n_kv), a.per_piece = 1.0 / a.pieces;
    a.wide = n * group > NARROW ? a.pieces : 0;
    if (a.pieces > 1) {
        const size_t at_once = (size_t)2 * dev->n_cu;
        void *p;
        HTR_TRY(htr_scratch(dev, SCR_PAGE_TICKET, at_once * TICKET * 4, &p));
        if (n * group <= FEW && n <= 4 * (size_t)a.p.n_seq) a.tickets = (uint32_t *)p, a.wide = 0;  // tokens, by what the sizes say
        HTR_TRY(htr_scratch(dev, SCR_PAGE_ATTN, 2 * at_once * ((NARROW + WIDE) * (D + 4) * 4 + 2 * sizeof(Part)), &p));
        float *at = (float *)p;
        for (int w = 0; w < 2; w++) {
            const size_t rows = 2 * at_once * (w ? WIDE : NARROW);
            a.part[w] = Parts{at, (float4 *)(at + rows * D), (Part *)(at + rows * (D + 4))};
            at += rows * (D + 4) + 2 * at_once * sizeof(Part) / 4;
        }
    }
    const unsigned groups = (unsigned)((a.wide + a.pieces) * kv->n_kv);
    const dim3 g(groups), b(64 * PW);
    if (a.tickets) {
        const bool near = kv->n_kv % 8 == 0 && dev->xcd_round_robin == 1;  // (a launch's workgroups go to the 8 XCDs in turn)
        if (a.kv.q8 && near) hipLaunchKernelGGL((k_page_few<true, NEAR>), g, b, 0, dev->stream, a);
        else if (a.kv.q8) hipLaunchKernelGGL((k_page_few<true, FAR>), g, b, 0, dev->stream, a);
        else if (near) hipLaunchKernelGGL((k_page_few<false, NEAR>), g, b, 0, dev->stream, a);
        else hipLaunchKernelGGL((k_page_few<false, FAR>), g, b, 0, dev->stream, a);
        return htr_launched(dev, a.kv.q8 ? "k_page_few<q8_0>" : "k_page_few<f16>");
    }
    if (a.kv.q8) hipLaunchKernelGGL(k_page_attn<true>, g, b, 0, dev->stream, a);
    else hipLaunchKernelGGL(k_page_attn<false>, g, b, 0, dev->stream, a);
    HTR_TRY(htr_launched(dev, a.kv.q8 ? "k_page_attn<q8_0>" : "k_page_attn<f16>"));
    if (a.pieces == 1) return 0;
    hipLaunchKernelGGL(k_page_attn_join, dim3((unsigned)((SHARES * a.wide + a.pieces) * kv->n_kv)), dim3(256), 0, dev->stream, a);
    return htr_launched(dev, "k_page_attn_join");
}
