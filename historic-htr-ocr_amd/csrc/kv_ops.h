// What the operators on a layer's KV cache share (kv_cache.hip, kv_attention.hip).
#pragma once

#include "htr_internal.h"

// a checked cache's planes, as the kernels take them
struct HtrKvPlanes {
    void *k, *v;          // f16 or int8 [n_kv][n_ctx][128]
    uint16_t *kd, *vd;    // q8_0: f16 scales [n_kv][n_ctx][4]
    int n_kv, n_ctx;
    bool q8;
};
// 0 with *out filled, or -1 with the message of what is wrong with the cache
int htr_kv_check(const char *what, const htr_kv *kv, HtrKvPlanes *out);

// whether [p, p + n) touches the cache's memory
bool htr_kv_overlaps(const HtrKvPlanes &kv, const void *p, size_t n);
// rows of a q8_0 cache as f16 into another's (n ≥ 1, in range: not checked)
int htr_kv_read_back(htr_device *dev, const HtrKvPlanes &src, int src_row, const HtrKvPlanes &dst, int dst_row, int n);

// the device made current for a call's launches, and the caller's own again afterwards
struct HtrOnDevice {
    explicit HtrOnDevice(htr_device *dev);
    ~HtrOnDevice();
    int before = -1;
};
