// Log probabilities of given tokens, the entropy of the distribution that each was chosen from, and the likeliest
// alternatives, from rows of logits.
//
// With m the row's largest logit, r = Σ e^(x − m) over all the others and W = Σ e^(x − m)·(m − x),
//
//   log p(i) = (x_i − m) − log(1 + r),   entropy = log(1 + r) + W / (1 + r)   (nats)
//
// The largest logit's own 1 stays out of the sum r, so the log probability and the entropy of a sure choice, both near 0,
// keep their leading digits (log1p); both are sums of terms of one sign, and nothing cancels.
#include <algorithm>

#include "choose_key.h"
#include "kv_ops.h"
#include "wave.h"

namespace {

constexpr int T = 256;

struct ScoreArgs {
    const float *x;
    size_t stride;
    const int32_t *ids;
    float *logprob, *entropy, *top_lp;
    int32_t *top_ids;
    int n, n_vocab, top;
};

__device__ __forceinline__ float block_sum(float v, float *s) {
    v = wave_sum(v, threadIdx.x & 63);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    return (s[0] + s[1]) + (s[2] + s[3]);
}

// a workgroup a row: its largest logit by order of choice, the sums, then the alternatives one by one
__global__ __launch_bounds__(T) void k_logprobs(ScoreArgs a) {
    __shared__ float s_f[4];
    __shared__ uint64_t s_k[4];
    const int tid = threadIdx.x, lane = tid & 63, row = blockIdx.x;
    const float *x = a.x + (size_t)row * a.stride;
    auto block_key = [&](uint64_t k) {
#pragma unroll
        for (int d = 32; d; d >>= 1) k = max(k, (uint64_t)__shfl_xor((unsigned long long)k, d));
        __syncthreads();
        if (lane == 0) s_k[tid >> 6] = k;
        __syncthreads();
        return max(max(s_k[0], s_k[1]), max(s_k[2], s_k[3]));
    };
    auto key = [&](int i) { return x[i] == x[i] ? choose_key(x[i], (uint32_t)i) : (uint64_t)(uint32_t)~i; };  // NaN below all
    uint64_t best = 0;
    for (int i = tid; i < a.n_vocab; i += T) best = max(best, key(i));
    best = block_key(best);
    const uint32_t at = ~(uint32_t)best;
    const float m = x[at];
    float r = 0.0f, w = 0.0f, bad = 0.0f;
    for (int i = tid; i < a.n_vocab; i += T) {
        const float d = x[i] - m, e = expf(d);
        if (!(x[i] < INFINITY)) bad = 1.0f;
        if ((uint32_t)i != at) {
            r += e;
            if (!(e == 0.0f)) w = fmaf(e, -d, w);
        }
    }
    r = block_sum(r, s_f);
    w = block_sum(w, s_f);
    bad = block_sum(bad, s_f);
    const float ln = log1pf(r);
    auto lp = [&](float v) { return bad > 0.0f ? NAN : m == -INFINITY ? -INFINITY : (v - m) - ln; };
    if (tid == 0) {
        const uint32_t id = (uint32_t)a.ids[row];
        a.logprob[row] = id < (uint32_t)a.n_vocab ? lp(x[id]) : NAN;
        a.entropy[row] = bad > 0.0f ? NAN : m == -INFINITY ? 0.0f : ln + w / (1.0f + r);
    }
    uint64_t last = best;
    for (int k = 0; k < a.top; k++) {
        if (k) {
            uint64_t next = 0;
            for (int i = tid; i < a.n_vocab; i += T) {
                const uint64_t c = key(i);
                if (c < last) next = max(next, c);
            }
            last = block_key(next);
        }
        if (tid == 0) {
            const uint32_t i = ~(uint32_t)last;
            a.top_ids[(size_t)row * a.top + k] = (int32_t)i;
            a.top_lp[(size_t)row * a.top + k] = lp(x[i]);
        }
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
    const ScoreArgs a{d_logits, stride, d_ids, d_logprob, d_entropy, d_top_logprob, d_top_ids, n, n_vocab, n_top};
    hipLaunchKernelGGL(k_logprobs, dim3((unsigned)n), dim3(T), 0, dev->stream, a);
    return htr_launched(dev, "k_logprobs");
}
