// The delta-rule layer's inputs from its [q | k | v] projection (strata_delta_inputs): a causal convolution of each channel
// that goes on from the sequence's history, SiLU, and the L2 norms of the heads of q and k, in one pass over the rows.
//
// Bound by bytes: each row is read once and written once. LANES lanes have a head's channels, VEC next to each other, and
// walk over kTile tokens with the last taps - 1 rows in registers; the norm's sum stays inside the lanes.
#include "mixers.cuh"

#include <cmath>

namespace strata {
namespace {

constexpr int kRowThreads = 256, kTile = 16, kMaxTaps = 8;

// C: groups of VEC channels a lane.
template <int TAPS, int VEC, int C, int LANES>
__global__ void __launch_bounds__(kRowThreads) k_delta_inputs(DeltaNet n, DeltaInputs A, MixRuns r) {
    kv8_enter();
    constexpr int W = VEC * C, ROOM = TAPS > 0 ? TAPS : kMaxTaps;
    const int taps = TAPS > 0 ? TAPS : n.taps;
    const int sub = threadIdx.x % LANES, heads = 2 * n.key_heads + n.value_heads;
    const int across = (heads + kRowThreads / LANES - 1) / (kRowThreads / LANES);  // blocks that share a tile
    const int head = (int)(blockIdx.x % across) * (kRowThreads / LANES) + threadIdx.x / LANES;
    const int run = blockIdx.y, t0 = (int)(blockIdx.x / across) * kTile;
    const MixRun me = mix_run_alone(r, n.sequences, run, n.err);
    if (head >= heads) return;  // (a whole group of LANES lanes, which is all that meets below)
    const unsigned mates = LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1) << ((threadIdx.x & 31) / LANES * LANES);
    const long long first = (long long)run * r.count, kd = (long long)n.key_heads * n.dim, vd = (long long)n.value_heads * n.dim;
    const bool is_q = head < n.key_heads, normed = head < 2 * n.key_heads;
    float *out = is_q ? A.q + head * n.dim : normed ? A.k + (head - n.key_heads) * n.dim : A.v + (long long)(head - 2 * n.key_heads) * n.dim;
    const long long ow = normed ? kd : vd;
    const auto channel = [&](int i) { return (i / VEC * LANES + sub) * VEC + i % VEC; };  // of the head
    const auto load = [&](const float *p, float (&x)[W]) {
#pragma unroll
        for (int i = 0; i < W; i += VEC) {
            const int c = channel(i);
            if constexpr (VEC == 4) {
                const float4 f = c < n.dim ? *reinterpret_cast<const float4 *>(p + c) : float4{0, 0, 0, 0};
                x[i] = f.x, x[i + 1] = f.y, x[i + 2] = f.z, x[i + 3] = f.w;
            } else {
                x[i] = c < n.dim ? p[c] : 0.0f;
            }
        }
    };
    const auto store = [&](float *p, const float (&x)[W]) {
#pragma unroll
        for (int i = 0; i < W; i += VEC) {
            const int c = channel(i);
            if (c >= n.dim) continue;
            if constexpr (VEC == 4)
                *reinterpret_cast<float4 *>(p + c) = float4{x[i], x[i + 1], x[i + 2], x[i + 3]};
            else
                p[c] = x[i];
        }
    };
    if (me.sequence < 0) {
        const float zero[W] = {};
        for (int t = t0; t < min(r.count, t0 + kTile); ++t) store(out + (first + t) * ow, zero);
        return;
    }
    if (t0 >= me.tokens) return;
    const long long c0 = (long long)head * n.dim;
    const float *x = A.x + first * A.row_stride + c0;
    float w[ROOM][W], past[ROOM][W];  // past[m]: the row m tokens back, [0] the token's own
#pragma unroll
    for (int i = 0; i < W; ++i)
#pragma unroll
        for (int m = 0; m < ROOM; ++m) w[m][i] = m < taps && channel(i) < n.dim ? n.weight[(c0 + channel(i)) * taps + taps - 1 - m] : 0.0f;
    float *history = n.history + ((long long)me.sequence * n.channels() + c0) * (taps - 1);
#pragma unroll
    for (int m = 1; m < ROOM; ++m) {  // rows before the tile: past[m - 1] is t0 - m here
        if (m >= taps) break;
        if (t0 - m >= 0) {
            load(x + (t0 - m) * A.row_stride, past[m - 1]);
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i)
                past[m - 1][i] = channel(i) < n.dim ? history[(long long)channel(i) * (taps - 1) + taps - 1 - m + t0] : 0.0f;
        }
    }
    const int end = min(me.tokens, t0 + kTile);
    for (int t = t0; t < end; ++t) {
#pragma unroll
        for (int m = ROOM - 1; m > 0; --m)
#pragma unroll
            for (int i = 0; i < W; ++i) past[m][i] = past[m - 1][i];
        load(x + t * A.row_stride, past[0]);
        float s[W], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            s[i] = 0.0f;
#pragma unroll
            for (int m = ROOM - 1; m >= 0; --m)
                if (m < taps) s[i] = fmaf(w[m][i], past[m][i], s[i]);
            s[i] = s[i] / (1.0f + expf(-s[i]));
            sum = fmaf(s[i], s[i], sum);
        }
        if (normed) {
#pragma unroll
            for (int m = LANES / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(mates, sum, m);
            const float inv = (is_q ? A.q_scale : 1.0f) / sqrtf(sum + A.epsilon);
#pragma unroll
            for (int i = 0; i < W; ++i) s[i] *= inv;
        }
        store(out + (first + t) * ow, s);
    }
    if (t0 == 0 && taps > 1) {
        // the first tile's lanes alone have read the history: they leave the run's last taps - 1 rows in its place
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int c = channel(i);
            if (c >= n.dim) continue;
            float *mine = history + (long long)c * (taps - 1);
            for (int m = 0; m < taps - 1; ++m) {  // ascending: a short run moves its history down
                const int t = me.tokens - (taps - 1) + m;
                mine[m] = t >= 0 ? x[t * A.row_stride + c] : mine[m + me.tokens];
            }
        }
    }
}

template <int TAPS, int VEC, int C, int LANES>
cudaError_t launch_inputs(const DeltaNet &n, const DeltaInputs &a, const MixRuns &r, cudaStream_t s) {
    const int heads = 2 * n.key_heads + n.value_heads, per = kRowThreads / LANES;
    return kv8_launch(k_delta_inputs<TAPS, VEC, C, LANES>, dim3((unsigned)((heads + per - 1) / per) * ((r.count + kTile - 1) / kTile), r.segments),
                      dim3(kRowThreads), 0, 1, s, n, a, r);
}
template <int TAPS>
cudaError_t pick_inputs(const DeltaNet &n, const DeltaInputs &a, const MixRuns &r, cudaStream_t s) {
    const bool vec = n.dim % 4 == 0 && a.row_stride % 4 == 0 && mix_aligned16(a.x) && mix_aligned16(a.q) && mix_aligned16(a.k) && mix_aligned16(a.v);
    if (!vec) return launch_inputs<TAPS, 1, 8, 32>(n, a, r, s);
    if (n.dim <= 32) return launch_inputs<TAPS, 4, 1, 8>(n, a, r, s);
    if (n.dim <= 64) return launch_inputs<TAPS, 4, 1, 16>(n, a, r, s);
    if (n.dim <= 128) return launch_inputs<TAPS, 4, 1, 32>(n, a, r, s);
    return launch_inputs<TAPS, 4, 2, 32>(n, a, r, s);
}

}  // namespace

cudaError_t delta_inputs(const DeltaNet &n, const DeltaInputs &given, const MixRuns &r, cudaStream_t s) {
    DeltaInputs a = given;
    if (a.q_scale == 0) a.q_scale = (float)(1 / std::sqrt((double)n.dim));
    return n.taps == 4 ? pick_inputs<4>(n, a, r, s) : pick_inputs<0>(n, a, r, s);
}

}  // namespace strata
