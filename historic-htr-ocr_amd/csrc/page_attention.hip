// Attention of a step's new tokens of several reads, each over its own rows of a cache in pages. Head dim 128, any number of q
// heads to a KV head, f16 or q8_0 rows.
//
//   out[t][h] = Σ_j p_j·v_j / Σ_j p_j,  p_j = e^(scale·q·k_j − m)  over the rows j ≤ past + i of the read whose i-th row t is
//
// The reads' lengths are on the device, so the launch knows their bounds alone.
#include <algorithm>

#include "kv_ops.h"
#include "wave.h"

namespace {

constexpr int D = 128;
constexpr float LOG2E = 1.4426950408889634f;

struct Args {
    const float *q;
    size_t q_stride;
    float *out;
    HtrKvPlanes kv;
    HtrPages p;
    int n_head, group, n_page;
    float scale;
};

// a wave a row and head: two dims a lane, one key after another
template <bool Q8> __global__ __launch_bounds__(256) void k_page_attn(Args a) {
    const int lane = threadIdx.x & 63, id = blockIdx.x * 4 + (threadIdx.x >> 6), t = id / a.n_head, h = id % a.n_head;
    if (t >= a.p.n_row) return;
    int b = 0;
    while (b < a.p.n_seq && a.p.start[b + 1] <= t) b++;
    if (b == a.p.n_seq) return;  // behind the last read
    const int past = a.p.past[b], start = max(a.p.start[b], 0), kvh = h / a.group;
    const int cap = (int)min((int64_t)a.p.max_pages << a.p.shift, (int64_t)INT32_MAX);
    const int keys = past < 0 || t < start ? 0 : (int)min((int64_t)past + (t - start) + 1, (int64_t)cap);
    const float2 qv = *reinterpret_cast<const float2 *>(a.q + t * a.q_stride + (size_t)h * D + 2 * lane);
    float m = -3.0e38f, l = 0.0f, ox = 0.0f, oy = 0.0f;
    for (int j = 0; j < keys; j++) {
        const int page = a.p.table[(size_t)b * a.p.max_pages + (j >> a.p.shift)];
        if ((uint32_t)page >= (uint32_t)a.n_page) continue;
        const size_t row = (size_t)kvh * a.kv.n_ctx + ((size_t)page << a.p.shift) + (j & ((1 << a.p.shift) - 1));
        float k[2], v[2];
        for (int e = 0; e < 2; e++) {
            if constexpr (Q8) {
                const _Float16 *dk = (const _Float16 *)a.kv.kd + row * 4 + lane / 16, *dv = (const _Float16 *)a.kv.vd + row * 4 + lane / 16;
                k[e] = (float)(_Float16)((float)((const int8_t *)a.kv.k)[row * D + 2 * lane + e] * (float)*dk);
                v[e] = (float)(_Float16)((float)((const int8_t *)a.kv.v)[row * D + 2 * lane + e] * (float)*dv);
            } else {
                k[e] = (float)((const _Float16 *)a.kv.k)[row * D + 2 * lane + e];
                v[e] = (float)((const _Float16 *)a.kv.v)[row * D + 2 * lane + e];
            }
        }
        const float s = wave_sum(fmaf(qv.x * a.scale, k[0], qv.y * a.scale * k[1]), lane);
        if (s > m) {
            const float c = __builtin_amdgcn_exp2f((m - s) * LOG2E);
            m = s, l *= c, ox *= c, oy *= c;
        }
        const float p = __builtin_amdgcn_exp2f((s - m) * LOG2E);
        l += p;
        ox = fmaf(p, v[0], ox), oy = fmaf(p, v[1], oy);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // no key: zeros
    *reinterpret_cast<float2 *>(a.out + ((size_t)t * a.n_head + h) * D + 2 * lane) = make_float2(ox * inv, oy * inv);
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
    HTR_TRY(htr_check_alive(dev));
    const HtrOnDevice on(dev);
    a.q = d_q, a.q_stride = q_stride, a.out = d_out, a.n_head = n_head, a.group = n_head / kv->n_kv;
    a.n_page = kv->n_ctx / pages->page, a.scale = scale;
    const dim3 g((unsigned)((n * n_head + 3) / 4)), b(256);
    if (a.kv.q8) hipLaunchKernelGGL(k_page_attn<true>, g, b, 0, dev->stream, a);
    else hipLaunchKernelGGL(k_page_attn<false>, g, b, 0, dev->stream, a);
    return htr_launched(dev, a.kv.q8 ? "k_page_attn<q8_0>" : "k_page_attn<f16>");
}
