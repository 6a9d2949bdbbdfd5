// Attention over the 8-bit paged cache (strata_kv8_attend).
#include "kv8.cuh"

#include <cmath>

namespace strata {
namespace {

constexpr int kThreads = 128;

// One CTA: one token and query head, block after block: 64 logits, the running maximum and sum of the
// softmax, and the weighted value rows, all in 32 bits.
__global__ void __launch_bounds__(kThreads) k_kv8_attend(const Kv8 c, const float *q, long long stride, int heads, const Kv8Runs runs,
                                                         const int *picks, int top, float scale, float *y) {
    __shared__ float q_s[256], p_s[kKvBlock];
    const int tid = threadIdx.x, token = blockIdx.x, h = blockIdx.y, head = h / (heads / c.kv_heads);
    const RunAt a = run_at(c, runs, token / runs.count);
    const int seen = visible_keys(c, a, token % runs.count);
    const int nb = (seen + kKvBlock - 1) / kKvBlock, n = picks ? top : nb;
    for (int i = tid; i < 256; i += kThreads) q_s[i] = i < c.dim ? q[(long long)token * stride + (size_t)h * c.dim + i] * scale : 0.0f;
    float m = -INFINITY, sum = 0.0f, acc[2] = {0.0f, 0.0f};
    for (int i = 0; i < n; ++i) {
        const int block = picks ? picks[((size_t)token * c.kv_heads + head) * top + i] : i;
        if (block < 0 || block >= nb) continue;
        const int page = page_of(c, a.sequence, block);
        if (page < 0) continue;
        __syncthreads();
        const int8_t *k = page_codes(c, page, head, 0), *v = page_codes(c, page, head, 1);
        const float sk = page_scales(c, page, head)[0], sv = page_scales(c, page, head)[1];
        if (tid < kKvBlock) {
            float dot = 0.0f;
            for (int ch = 0; ch < c.dim; ++ch) dot += q_s[ch] * (float)k[key_byte(tid, ch)];
            p_s[tid] = block * kKvBlock + tid < seen ? dot * sk : -INFINITY;
        }
        __syncthreads();
        float top_now = m;
        for (int t = 0; t < kKvBlock; ++t) top_now = fmaxf(top_now, p_s[t]);
        const float shrink = expf(m - top_now);
        m = top_now;
        sum *= shrink;
        float part[2] = {0.0f, 0.0f};
        for (int t = 0; t < kKvBlock; ++t) {
            const float w = expf(p_s[t] - m);
            sum += w;
            for (int j = 0; j < 2; ++j)
                if (tid + j * kThreads < c.dim) part[j] += w * (float)v[(tid + j * kThreads) * kKvBlock + t];
        }
        for (int j = 0; j < 2; ++j) acc[j] = acc[j] * shrink + part[j] * sv;
    }
    for (int j = 0; j < 2; ++j) {
        const int ch = tid + j * kThreads;
        if (ch < c.dim) y[((size_t)token * heads + h) * c.dim + ch] = sum == 0.0f ? 0.0f : acc[j] / sum;
    }
}

}  // namespace

cudaError_t kv8_attend(const Kv8 &c, const float *q, long long stride, int heads, const Kv8Runs &r, const int *picks, int top, float scale,
                       float *y, cudaStream_t s) {
    k_kv8_attend<<<dim3(r.segments * r.count, heads), kThreads, 0, s>>>(c, q, stride, heads, r, picks, top, scale, y);
    return cudaGetLastError();
}

}  // namespace strata
