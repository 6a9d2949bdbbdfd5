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
__global__ void __launch_bounds__(kRowThreads)
    k_delta_inputs(const __grid_constant__ DeltaNet n, const __grid_constant__ DeltaInputs A, const __grid_constant__ MixRuns r) {
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
    float *history = n.history + ((long long)me.sequence * n.channels() + c0) * (taps - 1);
    constexpr bool kWide = TAPS == 4 && VEC == 4;  // four channels' weights are four vectors, their histories three
    if constexpr (kWide) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float4 f = channel(i) < n.dim ? reinterpret_cast<const float4 *>(n.weight)[c0 + channel(i)] : float4{0, 0, 0, 0};
            w[3][i] = f.x, w[2][i] = f.y, w[1][i] = f.z, w[0][i] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
            for (int m = 0; m < ROOM; ++m) w[m][i] = m < taps && channel(i) < n.dim ? n.weight[(c0 + channel(i)) * taps + taps - 1 - m] : 0.0f;
    }
    float old[kWide ? 3 * W : 1];  // the history of lanes that have the run's first tile: three values a channel
    if constexpr (kWide) {
        if (t0 == 0) {
#pragma unroll
            for (int i = 0; i < W; i += 4)
#pragma unroll
                for (int e = 0; e < 3; ++e) {
                    const float4 f = channel(i) < n.dim ? reinterpret_cast<const float4 *>(history + 3 * channel(i))[e] : float4{0, 0, 0, 0};
                    old[3 * i + 4 * e] = f.x, old[3 * i + 4 * e + 1] = f.y, old[3 * i + 4 * e + 2] = f.z, old[3 * i + 4 * e + 3] = f.w;
                }
        }
    }
#pragma unroll
    for (int m = 1; m < ROOM; ++m) {  // rows before the tile: past[m - 1] is t0 - m here
        if (m >= taps) break;
        if (t0 - m >= 0) {
            load(x + (t0 - m) * A.row_stride, past[m - 1]);
        } else if constexpr (kWide) {
#pragma unroll
            for (int i = 0; i < W; ++i) past[m - 1][i] = old[3 * i + 3 - m];
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i)
                past[m - 1][i] = channel(i) < n.dim ? history[(long long)channel(i) * (taps - 1) + taps - 1 - m + t0] : 0.0f;
        }
    }
    const int end = min(me.tokens, t0 + kTile);
    constexpr int kAhead = W <= 4 ? 4 : 1;  // rows in flight
    for (int t1 = t0; t1 < end; t1 += kAhead) {
        float ahead[kAhead][W];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (t1 + u < end) load(x + (t1 + u) * A.row_stride, ahead[u]);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (t1 + u >= end) break;
#pragma unroll
            for (int m = ROOM - 1; m > 0; --m)
#pragma unroll
                for (int i = 0; i < W; ++i) past[m][i] = past[m - 1][i];
            float s[W], sum = 0.0f;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                past[0][i] = ahead[u][i];
                s[i] = 0.0f;
#pragma unroll
                for (int m = ROOM - 1; m >= 0; --m)
                    if (m < taps) s[i] = fmaf(w[m][i], past[m][i], s[i]);
                s[i] = __fdividef(s[i], 1.0f + expf(-s[i]));
                sum = fmaf(s[i], s[i], sum);
            }
            if (normed) {
#pragma unroll
                for (int m = LANES / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(mates, sum, m);
                const float inv = (is_q ? A.q_scale : 1.0f) / sqrtf(sum + A.epsilon);
#pragma unroll
                for (int i = 0; i < W; ++i) s[i] *= inv;
            }
            store(out + (first + t1 + u) * ow, s);
        }
    }
    if (t0 == 0 && taps > 1) {
        // the first tile's lanes alone have read the history: they leave the run's last taps - 1 rows in its place
        if constexpr (kWide) {
#pragma unroll
            for (int i = 0; i < W; i += 4) {
                if (channel(i) >= n.dim) continue;
                float now[3][4];
#pragma unroll
                for (int m = 0; m < 3; ++m) {
                    const int t = me.tokens - 3 + m;
                    if (t >= 0) {
                        const float4 f = *reinterpret_cast<const float4 *>(x + t * A.row_stride + channel(i));
                        now[m][0] = f.x, now[m][1] = f.y, now[m][2] = f.z, now[m][3] = f.w;
                    } else {  // a short run moves its history down
#pragma unroll
                        for (int e = 0; e < 4; ++e) now[m][e] = t == -3 ? old[3 * (i + e)] : t == -2 ? old[3 * (i + e) + 1] : old[3 * (i + e) + 2];
                    }
                }
                float4 *to = reinterpret_cast<float4 *>(history + 3 * channel(i));
                to[0] = float4{now[0][0], now[1][0], now[2][0], now[0][1]};
                to[1] = float4{now[1][1], now[2][1], now[0][2], now[1][2]};
                to[2] = float4{now[2][2], now[0][3], now[1][3], now[2][3]};
            }
            return;
        }
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
    const bool vec = n.dim % 4 == 0 && a.row_stride % 4 == 0 && mix_aligned16(a.x) && mix_aligned16(a.q) && mix_aligned16(a.k) && mix_aligned16(a.v) &&
                     mix_aligned16(n.weight) && mix_aligned16(n.history);
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
