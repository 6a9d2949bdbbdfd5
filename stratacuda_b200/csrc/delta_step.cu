// The gated delta rule token by token (strata_delta_rule): single tokens and short runs of many sequences.
//
// With the state S [key][value] of a value head before the token, and decay a, strength b:
//   d = b (v - a S^T k),  y = a S^T q + (k . q) d,  S <- a S + k d^T
// so that prediction and result come from one pass over the state as it was: one exchange between warps a token.
// A block has 32 value columns of a head (columns do not meet), a thread of its WARPS warps 4 columns by ROWS keys, in registers.
//
// Single tokens of many sequences are bound by the states' bytes (64 sessions of 32 heads of 128: 54 us, 5 TB/s of 268 MB), runs by
// instructions and the way from token to token: rows come through asynchronous copies kAhead tokens ahead, keys and queries twice
// so that products are paired (one session, 0.7 us a token; 0.83 with rows fetched one token ahead).
#include "delta_chunk.cuh"

namespace strata {
namespace {

using delta::both;
using delta::fma2;

constexpr int kStepCols = 32, kAhead = 4, kRing = 8;
// Of heads of more than 64 keys, blocks up to which four warps share one: with few blocks the way from token to token is shorter (one
// session of 32 heads of 128, 32 tokens: 25 us against 32), with many two warps need fewer instructions (16 sessions 106 us against 117).
constexpr int kFewBlocks = 2 * 148;

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
using Pair = unsigned long long;  // of F32, in one register pair
__device__ __forceinline__ float4 sum_groups(Pair x, Pair y) {
    float4 f;
    unpack2(x, f.x, f.y);
    unpack2(y, f.z, f.w);
    return float4{sum_groups(f.x), sum_groups(f.y), sum_groups(f.z), sum_groups(f.w)};
}
__device__ __forceinline__ void copy4(float *to, const float *from, bool in) {  // zero where not `in`
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(static_cast<unsigned>(__cvta_generic_to_shared(to))), "l"(from), "r"(in ? 4 : 0)
                 : "memory");
}

// VEC: rows of the state and of y can be read and written four columns at a time.
template <int ROWS, int WARPS, bool VEC>
__global__ void __launch_bounds__(32 * WARPS, WARPS == 2 ? 8 : ROWS <= 8 ? 6 : 3)
    k_delta_step(const __grid_constant__ DeltaNet n, const __grid_constant__ DeltaRule A, const __grid_constant__ MixRuns r) {
    kv8_enter();
    constexpr int D = ROWS * 4 * WARPS, kStepThreads = 32 * WARPS;  // keys there is room for
    struct Token {
        float2 k[D], q[D];  // each twice, as a pair
        float v[kStepCols], a, b, pad[2];
    };
    __shared__ __align__(16) Token ring[kRing];
    __shared__ float4 part[2][2][WARPS][8];
    __shared__ float part_kq[2][WARPS];
    const int slices = (n.dim + kStepCols - 1) / kStepCols, h = blockIdx.x / slices, run = blockIdx.y, col0 = (int)(blockIdx.x % slices) * kStepCols;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, group = warp * 4 + (lane >> 3), mine = 4 * (lane & 7);
    const int row0 = group * ROWS, left = n.dim - col0 - mine;
    const long long first = (long long)run * r.count;  // the run's first row
    const MixRun me = mix_run_alone(r, n.sequences, run, n.err);
    const long long vw = (long long)n.value_heads * n.dim, vat = (long long)h * n.dim + col0, kat = (long long)(h % n.key_heads) * n.dim;
    float *yp = A.y + first * vw + vat + mine;
    if (me.sequence < 0) {
        for (long long t = group; t < r.count; t += 4 * WARPS) store4<VEC>(yp + t * vw, left, float4{0, 0, 0, 0});
        return;
    }
    if (!me.tokens) return;
    const float *kp = A.k + first * A.k_stride + kat, *qp = A.q + first * A.q_stride + kat, *vp = A.v + first * A.v_stride + vat;
    const float *ap = A.decay + first * n.value_heads + h, *bp = A.beta + first * n.value_heads + h;
    const auto fetch = [&](int t) {
        if (t < me.tokens) {
            Token &x = ring[t % kRing];
#pragma unroll
            for (int i = tid; i < D; i += kStepThreads) {
                const bool in = i < n.dim;
                const float *k = in ? kp + t * A.k_stride + i : kp, *q = in ? qp + t * A.q_stride + i : qp;
                copy4(&x.k[i].x, k, in), copy4(&x.k[i].y, k, in);
                copy4(&x.q[i].x, q, in), copy4(&x.q[i].y, q, in);
            }
            if (tid < kStepCols) copy4(&x.v[tid], col0 + tid < n.dim ? vp + t * A.v_stride + tid : vp, col0 + tid < n.dim);
            if (tid == 32) copy4(&x.a, ap + (long long)t * n.value_heads, true);
            if (tid == 33) copy4(&x.b, bp + (long long)t * n.value_heads, true);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int t = 0; t < kAhead; ++t) fetch(t);
    float *sp = n.state + ((long long)me.sequence * n.dim + row0) * vw + vat + mine;
    Pair S[ROWS][2];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const float4 f = row0 + i < n.dim ? load4<VEC>(sp + i * vw, left) : float4{0, 0, 0, 0};
        S[i][0] = pack2(f.x, f.y), S[i][1] = pack2(f.z, f.w);
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
    __syncthreads();
#pragma unroll 1
    for (int t = 0; t < me.tokens; ++t) {
        const Token &x = ring[t % kRing];
        const int turn = t & 1;
        fetch(t + kAhead);
        Pair p0 = 0, p1 = 0, y0 = 0, y1 = 0;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < ROWS; i += 2) {
            const ulonglong2 k = *reinterpret_cast<const ulonglong2 *>(&x.k[row0 + i]), q = *reinterpret_cast<const ulonglong2 *>(&x.q[row0 + i]);
            p0 = fma2(k.x, S[i][0], p0), p1 = fma2(k.x, S[i][1], p1);
            y0 = fma2(q.x, S[i][0], y0), y1 = fma2(q.x, S[i][1], y1);
            p0 = fma2(k.y, S[i + 1][0], p0), p1 = fma2(k.y, S[i + 1][1], p1);
            y0 = fma2(q.y, S[i + 1][0], y0), y1 = fma2(q.y, S[i + 1][1], y1);
            float a, b, c, d, same;
            unpack2(k.x, a, same), unpack2(q.x, b, same), unpack2(k.y, c, same), unpack2(q.y, d, same);
            dot = fmaf(a, b, fmaf(c, d, dot));
        }
        const float4 p = sum_groups(p0, p1), y = sum_groups(y0, y1);
        dot = sum_groups(dot);
        if (lane < 8) {
            part[turn][0][warp][lane] = p;
            part[turn][1][warp][lane] = y;
        }
        if (lane == 0) part_kq[turn][warp] = dot;
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");  // the next token's rows
        __syncthreads();
        const float a = x.a, b = x.b;
        const float4 v = *reinterpret_cast<const float4 *>(&x.v[mine]);
        const auto total = [&](int which) {
            const float4 *f = &part[turn][which][0][lane & 7];
            float4 s = f[0];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) s.x += f[8 * w].x, s.y += f[8 * w].y, s.z += f[8 * w].z, s.w += f[8 * w].w;
            return s;
        };
        const float4 s = total(0);
        const float4 d{b * (v.x - a * s.x), b * (v.y - a * s.y), b * (v.z - a * s.z), b * (v.w - a * s.w)};
        const Pair d0 = pack2(d.x, d.y), d1 = pack2(d.z, d.w), aa = both(a);
#pragma unroll
        for (int i = 0; i < ROWS; i += 2) {
            const ulonglong2 k = *reinterpret_cast<const ulonglong2 *>(&x.k[row0 + i]);
            S[i][0] = fma2(k.x, d0, mul2_rn(aa, S[i][0])), S[i][1] = fma2(k.x, d1, mul2_rn(aa, S[i][1]));
            S[i + 1][0] = fma2(k.y, d0, mul2_rn(aa, S[i + 1][0])), S[i + 1][1] = fma2(k.y, d1, mul2_rn(aa, S[i + 1][1]));
        }
        if (warp == t % WARPS && lane < 8) {
            const float4 z = total(1);
            float c = part_kq[turn][0];
#pragma unroll
            for (int w = 1; w < WARPS; ++w) c += part_kq[turn][w];
            store4<VEC>(yp + t * vw, left, float4{fmaf(c, d.x, a * z.x), fmaf(c, d.y, a * z.y), fmaf(c, d.z, a * z.z), fmaf(c, d.w, a * z.w)});
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        float4 f;
        unpack2(S[i][0], f.x, f.y);
        unpack2(S[i][1], f.z, f.w);
        if (row0 + i < n.dim) store4<VEC>(sp + i * vw, left, f);
    }
}

template <int ROWS, int WARPS, bool VEC>
cudaError_t launch_step(dim3 grid, const DeltaNet &n, const DeltaRule &a, const MixRuns &r, cudaStream_t s) {
    return kv8_launch(k_delta_step<ROWS, WARPS, VEC>, grid, dim3(32 * WARPS), 0, 1, s, n, a, r);
}
template <bool VEC>
cudaError_t pick_step(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, cudaStream_t s) {
    const dim3 grid((unsigned)n.value_heads * ((n.dim + kStepCols - 1) / kStepCols), (unsigned)r.segments);
    if (n.dim > 128) return launch_step<16, 4, VEC>(grid, n, a, r, s);
    if (n.dim <= 32) return launch_step<4, 2, VEC>(grid, n, a, r, s);
    if (n.dim <= 64) return launch_step<8, 2, VEC>(grid, n, a, r, s);
    if ((long long)grid.x * grid.y > kFewBlocks) return launch_step<16, 2, VEC>(grid, n, a, r, s);
    return launch_step<8, 4, VEC>(grid, n, a, r, s);
}

}  // namespace

cudaError_t delta_step(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, cudaStream_t s) {
    const bool vec = n.dim % 4 == 0 && mix_aligned16(n.state) && mix_aligned16(a.y);
    return vec ? pick_step<true>(n, a, r, s) : pick_step<false>(n, a, r, s);
}

}  // namespace strata
