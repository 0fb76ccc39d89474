// What the operators on a layer's KV cache share (kv_cache.hip, kv_attention.hip).
#pragma once

#include "htr_internal.h"

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

// int8 quants → f16(q·d): a byte q ^ 0x80 under the high byte 0x64 is the f16 number 1024 + 128 + q, so one packed
// subtraction gives q exactly, and one packed product rounds q·d once
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

// a checked cache's planes, as the kernels take them
struct HtrKvPlanes {
    void *k, *v;          // f16 or int8 [n_kv][n_ctx][128]
    uint16_t *kd, *vd;    // q8_0: f16 scales [n_kv][n_ctx][4]
    int n_kv, n_ctx;
    bool q8;
};
// the most workgroups of 256 threads along a grid's first dimension, which takes less than 2^32 threads (a launch of more
// fails, and leaves the device dead)
constexpr size_t HTR_MAX_GROUPS = (1u << 24) - 1;
// 0 with *out filled, or -1 with the message of what is wrong with the cache
int htr_kv_check(const char *what, const htr_kv *kv, HtrKvPlanes *out);

// whether [p, p + n) touches the cache's memory
bool htr_kv_overlaps(const HtrKvPlanes &kv, const void *p, size_t n);
// rows of a q8_0 cache as f16 into another's (n ≥ 1, in range: not checked)
int htr_kv_read_back(htr_device *dev, const HtrKvPlanes &src, int src_row, const HtrKvPlanes &dst, int dst_row, int n);

// a checked batch of reads over a cache in pages, as the kernels take it
struct HtrPages {
    int n_seq, n_row, shift, max_pages;  // shift: log2 of a page's rows
    int32_t *start, *past, *table, *pos, *slot;
};
constexpr int HTR_MAX_SEQ = 1024, HTR_MAX_ROW = 1 << 21;  // reads and rows of a step: their sums fit 32 bits
// 0 with *out filled, or -1 with the message of what is wrong with the sizes, or with the arrays that the call uses
enum { HTR_PAGES_TABLE = 1, HTR_PAGES_ROWS = 2 };  // start, past and table; pos and slot
int htr_pages_check(const char *what, const htr_pages *p, int uses, HtrPages *out);
inline bool htr_overlap(const void *a, size_t na, const void *b, size_t nb) {
    return (uintptr_t)a < (uintptr_t)b + nb && (uintptr_t)b < (uintptr_t)a + na;
}

// whether n ≥ 1 rows of `row` floats (below 2^40), `stride` apart, end within 2^62 bytes: what htr_overlap is told of such rows has
// not wrapped, and no row lies in front of the first
inline bool htr_rows_fit(size_t stride, size_t n, size_t row) { return n == 1 || stride <= ((1ull << 60) - row) / (n - 1); }

// the device made current for a call's launches, and the caller's own again afterwards
struct HtrOnDevice {
    explicit HtrOnDevice(htr_device *dev);
    ~HtrOnDevice();
    int before = -1;
};
