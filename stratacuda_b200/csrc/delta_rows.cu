// The delta-rule layer's inputs from its [q | k | v] projection (strata_delta_inputs): a causal convolution of each channel
// that goes on from the sequence's history, SiLU, and the L2 norms of the heads of q and k, in one pass over the rows.
//
// Bound by bytes: each row is read once and written once. LANES lanes have a head's channels, VEC next to each other, and
// walk over kTile tokens with the last taps - 1 rows in registers; the norm's sum stays inside the lanes. Tokens go in groups of four,
// so that four rows are in flight and the window does not move through registers: 8191 tokens of 10240 channels 135 us, 5.0 TB/s
// (192 us row by row); a token of each of 64 sessions 6 us.
#include "mixers.cuh"

#include <cmath>

namespace strata {
namespace {

constexpr int kRowThreads = 256, kTile = 16, kMaxTaps = 8;

// C: groups of VEC channels a lane.
template <int TAPS, int VEC, int C, int LANES>
__global__ void __launch_bounds__(kRowThreads, TAPS == 4 && VEC == 4 && C == 1 ? 3 : 1)
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
    float *history = n.history + ((long long)me.sequence * n.channels() + c0) * (taps - 1);
    constexpr bool kWide = TAPS == 4 && VEC == 4;  // four channels' weights are four vectors, their histories three
    constexpr int kAhead = W <= 4 ? 4 : 1;         // rows in flight
    // Of the widths that have registers for it, the next rows while these are worked on: 4096 tokens of 8192 channels, heads of 256, 67 us
    // (72 without), of 4096 channels with three taps 43 (49). Four taps of a vector a lane would have two blocks a multiprocessor in place of three.
    constexpr bool kNext = !(TAPS == 4 && W == 4);
    float w[ROOM][W], row[ROOM - 1 + kAhead][W];   // row[i] is token t + i - (ROOM - 1); fewer taps than ROOM are the last ones
    const int skip = ROOM - taps;
    if constexpr (kWide) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const float4 f = channel(i) < n.dim ? reinterpret_cast<const float4 *>(n.weight)[c0 + channel(i)] : float4{0, 0, 0, 0};
            w[0][i] = f.x, w[1][i] = f.y, w[2][i] = f.z, w[3][i] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
#pragma unroll
            for (int m = 0; m < ROOM; ++m) w[m][i] = m >= skip && channel(i) < n.dim ? n.weight[(c0 + channel(i)) * taps + m - skip] : 0.0f;
    }
    // The rows before the tile. The first tile's lanes alone read the history, and leave the run's last taps - 1 rows in its place.
    if (t0 > 0) {
#pragma unroll
        for (int m = 0; m < ROOM - 1; ++m)
            if (m >= skip) load(x + (t0 + m - (ROOM - 1)) * A.row_stride, row[m]);
    } else if constexpr (kWide) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            if (channel(i) >= n.dim) {
#pragma unroll
                for (int m = 0; m < 3; ++m) row[m][i] = row[m][i + 1] = row[m][i + 2] = row[m][i + 3] = 0.0f;
                continue;
            }
            float4 *at = reinterpret_cast<float4 *>(history + 3 * channel(i));
            const float4 f = at[0], g = at[1], h = at[2];
            row[0][i] = f.x, row[1][i] = f.y, row[2][i] = f.z, row[0][i + 1] = f.w;
            row[1][i + 1] = g.x, row[2][i + 1] = g.y, row[0][i + 2] = g.z, row[1][i + 2] = g.w;
            row[2][i + 2] = h.x, row[0][i + 3] = h.y, row[1][i + 3] = h.z, row[2][i + 3] = h.w;
            float now[3][4];
#pragma unroll
            for (int m = 0; m < 3; ++m) {
                const int t = me.tokens - 3 + m;
                if (t >= 0) {
                    const float4 v = *reinterpret_cast<const float4 *>(x + t * A.row_stride + channel(i));
                    now[m][0] = v.x, now[m][1] = v.y, now[m][2] = v.z, now[m][3] = v.w;
                } else {  // a short run moves its history down
#pragma unroll
                    for (int e = 0; e < 4; ++e) now[m][e] = t == -3 ? row[0][i + e] : t == -2 ? row[1][i + e] : row[2][i + e];
                }
            }
            at[0] = float4{now[0][0], now[1][0], now[2][0], now[0][1]};
            at[1] = float4{now[1][1], now[2][1], now[0][2], now[1][2]};
            at[2] = float4{now[2][2], now[0][3], now[1][3], now[2][3]};
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int c = channel(i);
            float *mine = history + (long long)c * (taps - 1);
#pragma unroll
            for (int m = 0; m < ROOM - 1; ++m)
                row[m][i] = m >= skip && c < n.dim ? mine[m - skip] : 0.0f;
            if (c >= n.dim) continue;
            for (int m = 0; m < taps - 1; ++m) {  // ascending: a short run moves its history down
                const int t = me.tokens - (taps - 1) + m;
                mine[m] = t >= 0 ? x[t * A.row_stride + c] : mine[m + me.tokens];
            }
        }
    }
    const int end = min(me.tokens, t0 + kTile);
    const float scale = is_q ? A.q_scale : 1.0f;
    float next[kAhead][W];
    const auto fetch = [&](int t, float(*to)[W]) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (t + u < end) load(x + (t + u) * A.row_stride, to[u]);
    };
    if (kNext) fetch(t0, next);
#pragma unroll 1
    for (int t = t0; t < end; t += kAhead) {
        if constexpr (kNext) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
#pragma unroll
                for (int i = 0; i < W; ++i) row[ROOM - 1 + u][i] = next[u][i];
            fetch(t + kAhead, next);
        } else {
            fetch(t, row + ROOM - 1);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            float s[W], sum = 0.0f;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                s[i] = 0.0f;
#pragma unroll
                for (int m = 0; m < ROOM; ++m)
                    if (TAPS > 0 || m >= skip) s[i] = fmaf(w[m][i], row[u + m][i], s[i]);
                s[i] = __fdividef(s[i], 1.0f + expf(-s[i]));
                sum = fmaf(s[i], s[i], sum);
            }
            if (normed) {
#pragma unroll
                for (int m = LANES / 2; m > 0; m >>= 1) sum += __shfl_xor_sync(mates, sum, m);
                const float inv = scale * rsqrtf(sum + A.epsilon);
#pragma unroll
                for (int i = 0; i < W; ++i) s[i] *= inv;
            }
            if (t + u < end) store(out + (first + t + u) * ow, s);
        }
#pragma unroll
        for (int m = 0; m < ROOM - 1; ++m)
#pragma unroll
            for (int i = 0; i < W; ++i) row[m][i] = row[m + kAhead][i];
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
