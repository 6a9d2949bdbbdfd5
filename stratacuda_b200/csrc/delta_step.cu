// The gated delta rule token by token (strata_delta_rule): single tokens and short runs of many sequences.
//
// With the state S [key][value] of a value head before the token, and decay a, strength b:
//   d = b (v - a S^T k),  y = a S^T q + (k . q) d,  S <- a S + k d^T
// so that prediction and result come from one pass over the state as it was: one exchange between warps a token.
// A block has 32 value columns of a head (columns do not meet), its 128 threads 4 columns by ROWS keys each, in registers.
#include "delta_chunk.cuh"

namespace strata {
namespace {

constexpr int kStepThreads = 128, kStepCols = 32;

template <bool VEC>
__device__ __forceinline__ float4 load4(const float *p, int left) {
    if (VEC) return left > 0 ? *reinterpret_cast<const float4 *>(p) : float4{0, 0, 0, 0};
    return float4{left > 0 ? p[0] : 0.0f, left > 1 ? p[1] : 0.0f, left > 2 ? p[2] : 0.0f, left > 3 ? p[3] : 0.0f};
}
template <bool VEC>
__device__ __forceinline__ void store4(float *p, int left, float4 x) {
    if (VEC) {
        if (left > 0) *reinterpret_cast<float4 *>(p) = x;
        return;
    }
    if (left > 0) p[0] = x.x;
    if (left > 1) p[1] = x.y;
    if (left > 2) p[2] = x.z;
    if (left > 3) p[3] = x.w;
}
__device__ __forceinline__ float sum_groups(float x) {  // over the warp's four groups of 8 lanes
    x += __shfl_xor_sync(0xffffffffu, x, 8);
    return x + __shfl_xor_sync(0xffffffffu, x, 16);
}
__device__ __forceinline__ void add_to(float4 &a, float b, const float4 &c) {
    a.x = fmaf(b, c.x, a.x);
    a.y = fmaf(b, c.y, a.y);
    a.z = fmaf(b, c.z, a.z);
    a.w = fmaf(b, c.w, a.w);
}

// VEC: rows of the state, of v and of y can be read four columns at a time.
template <int ROWS, bool VEC>
__global__ void __launch_bounds__(kStepThreads, ROWS <= 8 ? 6 : 3)
    k_delta_step(const __grid_constant__ DeltaNet n, const __grid_constant__ DeltaRule A, const __grid_constant__ MixRuns r) {
    kv8_enter();
    constexpr int D = ROWS * 16;  // keys there is room for
    __shared__ float kq[2][2][D];
    __shared__ float4 part[2][4][2][8];
    __shared__ float part_kq[2][4];
    const int slices = (n.dim + kStepCols - 1) / kStepCols, h = blockIdx.x / slices, run = blockIdx.y;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = warp * 4 + (lane >> 3);
    const int col = (int)(blockIdx.x % slices) * kStepCols + 4 * (lane & 7), row0 = group * ROWS, left = n.dim - col;
    const long long first = (long long)run * r.count;  // the run's first row
    const MixRun me = mix_run_alone(r, n.sequences, run, n.err);
    const long long vw = (long long)n.value_heads * n.dim, vat = (long long)h * n.dim + col, kat = (long long)(h % n.key_heads) * n.dim;
    if (me.sequence < 0) {
        for (long long t = group; t < r.count; t += 16) store4<VEC>(A.y + (first + t) * vw + vat, left, float4{0, 0, 0, 0});
        return;
    }
    if (!me.tokens) return;
    // A token's rows are fetched while the token before it is worked on: key and query, a channel or two a thread, through
    // shared memory, decay, strength and this thread's columns of v in registers
    constexpr int E = (D + kStepThreads - 1) / kStepThreads;
    struct Next {
        float k[E], q[E], a, b;
        float4 v;
    };
    const float *kp = A.k + first * A.k_stride + kat, *qp = A.q + first * A.q_stride + kat, *vp = A.v + first * A.v_stride + vat;
    const float *ap = A.decay + first * n.value_heads + h, *bp = A.beta + first * n.value_heads + h;
    const auto fetch = [&](int t, Next &x) {
        if (t >= me.tokens) return;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = tid + e * kStepThreads;
            x.k[e] = i < n.dim ? kp[t * A.k_stride + i] : 0.0f;
            x.q[e] = i < n.dim ? qp[t * A.q_stride + i] : 0.0f;
        }
        x.a = ap[(long long)t * n.value_heads], x.b = bp[(long long)t * n.value_heads];
        x.v = load4<VEC>(vp + t * A.v_stride, left);
    };
    const auto stage = [&](int t, const Next &x) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = tid + e * kStepThreads;
            if (D % kStepThreads == 0 || i < D) kq[t & 1][0][i] = x.k[e], kq[t & 1][1][i] = x.q[e];
        }
    };
    Next x{};
    fetch(0, x);
    float *sp = n.state + ((long long)me.sequence * n.dim + row0) * vw + vat;
    float4 S[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) S[i] = row0 + i < n.dim ? load4<VEC>(sp + i * vw, left) : float4{0, 0, 0, 0};
    float *yp = A.y + first * vw + vat;
    stage(0, x);
    __syncthreads();
    for (int t = 0; t < me.tokens; ++t) {
        const float a = x.a, b = x.b;
        const float4 v = x.v;
        fetch(t + 1, x);
        float k[ROWS], dot = 0.0f;
        float4 p{0, 0, 0, 0}, y{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            k[i] = kq[t & 1][0][row0 + i];
            const float q = kq[t & 1][1][row0 + i];
            dot = fmaf(k[i], q, dot);
            add_to(p, k[i], S[i]);
            add_to(y, q, S[i]);
        }
        p = float4{sum_groups(p.x), sum_groups(p.y), sum_groups(p.z), sum_groups(p.w)};
        y = float4{sum_groups(y.x), sum_groups(y.y), sum_groups(y.z), sum_groups(y.w)};
        dot = sum_groups(dot);
        if (lane < 8) {
            part[t & 1][warp][0][lane] = p;
            part[t & 1][warp][1][lane] = y;
        }
        if (lane == 0) part_kq[t & 1][warp] = dot;
        if (t + 1 < me.tokens) stage(t + 1, x);
        __syncthreads();
        p = y = float4{0, 0, 0, 0};
        dot = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            add_to(p, 1.0f, part[t & 1][w][0][lane & 7]);
            if (warp == 0) add_to(y, 1.0f, part[t & 1][w][1][lane & 7]);
            dot += part_kq[t & 1][w];
        }
        const float4 d{b * (v.x - a * p.x), b * (v.y - a * p.y), b * (v.z - a * p.z), b * (v.w - a * p.w)};
        if (group == 0)
            store4<VEC>(yp + t * vw, left, float4{fmaf(dot, d.x, a * y.x), fmaf(dot, d.y, a * y.y), fmaf(dot, d.z, a * y.z), fmaf(dot, d.w, a * y.w)});
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            S[i] = float4{a * S[i].x, a * S[i].y, a * S[i].z, a * S[i].w};
            add_to(S[i], k[i], d);
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
        if (row0 + i < n.dim) store4<VEC>(sp + i * vw, left, S[i]);
}

template <bool VEC>
cudaError_t launch_step(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, cudaStream_t s) {
    const dim3 grid((unsigned)n.value_heads * ((n.dim + kStepCols - 1) / kStepCols), (unsigned)r.segments);
    const auto kernel = n.dim <= 32 ? k_delta_step<2, VEC> : n.dim <= 64 ? k_delta_step<4, VEC> : n.dim <= 128 ? k_delta_step<8, VEC> : k_delta_step<16, VEC>;
    return kv8_launch(kernel, grid, dim3(kStepThreads), 0, 1, s, n, a, r);
}

}  // namespace

cudaError_t delta_step(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, cudaStream_t s) {
    const bool vec = n.dim % 4 == 0 && a.v_stride % 4 == 0 && mix_aligned16(n.state) && mix_aligned16(a.v) && mix_aligned16(a.y);
    return vec ? launch_step<true>(n, a, r, s) : launch_step<false>(n, a, r, s);
}

}  // namespace strata
