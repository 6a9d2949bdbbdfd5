// Norms of queries and keys for each head with the position's rotation in the same pass (strata_qk_rope).
//
// Bound by bytes: a group of LANES lanes has a head row, reads it once from memory (what a channel is paired with comes from
// L1), and writes it once. A block has heads of one token, so that no index is divided. 8191 tokens of 24 + 2 heads of
// 256: 84 us, 5.2 TB/s; partners through shuffles took 94 us.
#include "mixers.cuh"

namespace strata {
namespace {

constexpr int kQkThreads = 256;

// C: groups of VEC channels a lane.
template <int VEC, int C, int LANES>
__global__ void __launch_bounds__(kQkThreads)
    k_qk_rope(const __grid_constant__ QkRope W, const __grid_constant__ QkRopeRows A, const __grid_constant__ MixRuns r) {
    kv8_enter();
    constexpr int N = VEC * C;
    const int sub = threadIdx.x % LANES, run = blockIdx.z, t = blockIdx.x, head = blockIdx.y * (kQkThreads / LANES) + threadIdx.x / LANES;
    if (head >= W.heads + W.kv_heads) return;
    const unsigned mates = LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1) << ((threadIdx.x & 31) / LANES * LANES);
    const MixRun me = mix_run(r, W.sequences, run, W.err);
    const long long row = (long long)run * r.count + t;
    const bool is_q = head < W.heads;
    float *y = is_q ? A.yq + (row * W.heads + head) * W.dim : A.yk + (row * W.kv_heads + head - W.heads) * W.dim;
    const float *x = is_q ? A.q + row * A.q_stride + head * A.q_head_stride : A.k + row * A.k_stride + (long long)(head - W.heads) * W.dim;
    const float *w = is_q ? W.q_weight : W.k_weight;
    if (me.sequence >= 0 && t >= me.tokens) return;
    const int half = W.rotary / 2;
    long long at = 0;
    bool zero = me.sequence < 0;
    if (!zero) {
        at = (long long)A.start[run] + t;
        if (at < 0 || at >= W.cells) {
            raise_error(W.err, kErrIndex);
            zero = true;
        }
    }
    const auto channel = [&](int i) { return (i / VEC * LANES + sub) * VEC + i % VEC; };
    const auto load = [&](const float *p, int c, float *f) {
        if constexpr (VEC == 4) {
            const float4 g = *reinterpret_cast<const float4 *>(p + c);
            f[0] = g.x, f[1] = g.y, f[2] = g.z, f[3] = g.w;
        } else {
            f[0] = p[c];
        }
    };
    float v[N], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i += VEC) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i + e] = 0.0f;
        if (!zero && channel(i) < W.dim) load(x, channel(i), v + i);
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum = fmaf(v[i + e], v[i + e], sum);
    }
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(mates, sum, m);
    const float inv = rsqrtf(__fdividef(sum, (float)W.dim) + A.epsilon);
#pragma unroll
    for (int i = 0; i < N; i += VEC) {
        const int c = channel(i);
        if (c >= W.dim || zero) continue;
        float g[VEC];
        load(w, c, g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i + e] *= inv * g[e];
        if (c < W.rotary) {  // VEC divides half, so a group has partners side by side
            const bool lower = c < half;
            const int other = lower ? c + half : c - half, pair = lower ? c : other;
            float b[VEC], co[VEC], si[VEC];
            load(x, other, b);
            load(w, other, g);
            load(W.cos + at * half, pair, co);
            load(W.sin + at * half, pair, si);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                b[e] *= inv * g[e];
                v[i + e] = v[i + e] * co[e] + (lower ? -b[e] : b[e]) * si[e];
            }
        }
    }
    __syncwarp(mates);  // all of the row has been read: y may be x
#pragma unroll
    for (int i = 0; i < N; i += VEC) {
        const int c = channel(i);
        if (c >= W.dim) continue;
        if constexpr (VEC == 4)
            *reinterpret_cast<float4 *>(y + c) = float4{v[i], v[i + 1], v[i + 2], v[i + 3]};
        else
            y[c] = v[i];
    }
}

template <int VEC, int C, int LANES>
cudaError_t launch_qk(const QkRope &w, const QkRopeRows &a, const MixRuns &r, cudaStream_t s) {
    const int per = kQkThreads / LANES;
    return kv8_launch(k_qk_rope<VEC, C, LANES>, dim3((unsigned)r.count, (unsigned)((w.heads + w.kv_heads + per - 1) / per), (unsigned)r.segments),
                      dim3(kQkThreads), 0, 1, s, w, a, r);
}

}  // namespace

cudaError_t qk_rope(const QkRope &w, const QkRopeRows &a, const MixRuns &r, cudaStream_t s) {
    const bool vec = w.dim % 4 == 0 && w.rotary % 8 == 0 && a.q_stride % 4 == 0 && a.q_head_stride % 4 == 0 && a.k_stride % 4 == 0 &&
                     mix_aligned16(a.q) && mix_aligned16(a.k) && mix_aligned16(a.yq) && mix_aligned16(a.yk) && mix_aligned16(w.q_weight) &&
                     mix_aligned16(w.k_weight) && mix_aligned16(w.cos) && mix_aligned16(w.sin);
    if (!vec) return launch_qk<1, 8, 32>(w, a, r, s);
    if (w.dim <= 32) return launch_qk<4, 1, 8>(w, a, r, s);
    if (w.dim <= 64) return launch_qk<4, 1, 16>(w, a, r, s);
    if (w.dim <= 128) return launch_qk<4, 1, 32>(w, a, r, s);
    return launch_qk<4, 2, 32>(w, a, r, s);
}

}  // namespace strata
