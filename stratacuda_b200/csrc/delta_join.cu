// The chunked delta rule over parts of runs: the states before the parts (delta_chunk.cuh).
//
// A part takes the state before it to  S' = F S + N,  with F where the part's tokens take the identity without values and N where they
// take zeros (delta_chain.cu). Part after part: a block has COLS columns of a head's state, a thread EACH of a row; the
// transitions come through asynchronous copies one part ahead. F32 throughout.
// Transitions of decays up to one and strengths that keep the state bounded have no element above one. Where one is above
// kLargest, or not finite, differences of large terms could lose what the state keeps: that run and head is taken whole.
#include "delta_chunk.cuh"

namespace strata {
namespace {

using delta::both;
using delta::fma2;
using delta::larger;

constexpr float kLargest = 2.0f;

template <int D, int COLS>
struct JoinSmem {
    float f[2][D][D + 4];
    float s[2][D][COLS];
};

template <int D, int COLS, int EACH>
__global__ void __launch_bounds__(D *COLS / EACH) k_delta_join(const __grid_constant__ DeltaNet n, const __grid_constant__ MixRuns r, const __grid_constant__ DeltaSlab slab) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    constexpr int kThreads = D * COLS / EACH, kVec = EACH / 4;
    JoinSmem<D, COLS> &M = *reinterpret_cast<JoinSmem<D, COLS> *>(smem_raw);
    kv8_enter();
    const int tid = threadIdx.x, row = tid % D, group = tid / D, slice = (int)(blockIdx.x % (D / COLS)), chain = (int)(blockIdx.x / (D / COLS));
    const int m = chain % slab.ratio, h = slab.head0 + chain / slab.ratio % slab.heads + m * n.key_heads, run = slab.run0 + chain / slab.ratio / slab.heads;
    const MixRun me = mix_run_alone(r, n.sequences, run, n.err);
    const int begin = slab.chunk0 * kChunk, col = slice * COLS + group * EACH;
    if (me.sequence < 0 || begin >= me.tokens || slice * COLS >= n.dim) return;
    const int chunks = min(slab.chunks, (me.tokens - begin + kChunk - 1) / kChunk), last = (chunks - 1) / slab.part_chunks;
    float *const own = slab.states + (long long)chain * (slab.parts - 1) * (2 * D * D);
    const auto fetch = [&](int p) {
        const float *from = own + (long long)p * (2 * D * D);
        float(*to)[D + 4] = M.f[p & 1];
#pragma unroll
        for (int i = 0; i < D * D / 4 / kThreads; ++i) {
            const int at = (i * kThreads + tid) * 4;
            const unsigned smem = (unsigned)__cvta_generic_to_shared(&to[at / D][at % D]);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem), "l"(from + at) : "memory");
        }
    };
    if (last > 1) fetch(1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    // the state before the first part moves here: the last part's block writes the real one
    const float *real = n.state + ((long long)me.sequence * n.dim + row) * n.value_heads * n.dim + (long long)h * n.dim + col;
    ulonglong2 end[kVec], next[kVec];  // four columns each
#pragma unroll
    for (int c = 0; c < kVec; ++c) {
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = row < n.dim && col + 4 * c + e < n.dim ? real[4 * c + e] : 0.0f;
        *reinterpret_cast<float4 *>(own + row * D + col + 4 * c) = float4{x[0], x[1], x[2], x[3]};
    }
    const auto ends = [&](int p) { return reinterpret_cast<ulonglong2 *>(own + (2 * p + 1) * (D * D) + row * D + col); };
#pragma unroll
    for (int c = 0; c < kVec; ++c) {
        if (last > 0) end[c] = ends(0)[c];
        if (last > 1) next[c] = ends(1)[c];
    }
    float most = 0.0f;
    for (int p = 1; p < last; ++p) {
        ulonglong2 sum[kVec];
#pragma unroll
        for (int c = 0; c < kVec; ++c) {
            // rows past the head's channels hold nothing
            reinterpret_cast<ulonglong2 *>(&M.s[p & 1][row][group * EACH])[c] = row < n.dim ? end[c] : ulonglong2{0, 0};
            sum[c] = next[c];
            if (p + 1 < last) next[c] = ends(p + 1)[c];
        }
        if (p + 1 < last) fetch(p + 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        __syncthreads();
        const float *f = M.f[p & 1][row];
        const auto four = [&](int j, float4 a) {
            const float w[4] = {a.x, a.y, a.z, a.w};
            most = larger(larger(most, w[0], w[1]), w[2], w[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < kVec; ++c) {
                    const ulonglong2 s = reinterpret_cast<const ulonglong2 *>(&M.s[p & 1][j + e][group * EACH])[c];
                    sum[c].x = fma2(both(w[e]), s.x, sum[c].x), sum[c].y = fma2(both(w[e]), s.y, sum[c].y);
                }
        };
        const int whole = n.dim & ~3;
#pragma unroll 4
        for (int j = 0; j < whole; j += 4) four(j, *reinterpret_cast<const float4 *>(f + j));
        if (whole < n.dim) {
            const float4 a = *reinterpret_cast<const float4 *>(f + whole);
            four(whole, float4{a.x, whole + 1 < n.dim ? a.y : 0.0f, whole + 2 < n.dim ? a.z : 0.0f, 0.0f});
        }
        if (row >= n.dim) most = 0.0f;
#pragma unroll
        for (int c = 0; c < kVec; ++c) ends(p)[c] = end[c] = sum[c];
        __syncthreads();  // the buffers' next turn
    }
    const int large = __syncthreads_or(!(most <= kLargest));
    if (slice == 0 && tid == 0) slab.whole[chain] = large;
}

template <int D, int COLS, int EACH>
cudaError_t launch_join(const DeltaNet &n, const MixRuns &r, const DeltaSlab &slab, cudaStream_t s) {
    const cudaError_t e = mix_shared_memory<k_delta_join<D, COLS, EACH>>(sizeof(JoinSmem<D, COLS>));
    if (e != cudaSuccess) return e;
    return kv8_launch(k_delta_join<D, COLS, EACH>, dim3((unsigned)(slab.runs * slab.heads * slab.ratio * (D / COLS))), dim3(D * COLS / EACH), sizeof(JoinSmem<D, COLS>), 1, s, n, r, slab);
}

}  // namespace

cudaError_t delta_join(const DeltaNet &n, const MixRuns &r, const DeltaSlab &slab, cudaStream_t s) {
    // narrow while that is at most a block a multiprocessor
    if (slab.runs * slab.heads * slab.ratio <= 148 / 16) return n.dim <= 64 ? launch_join<64, 8, 4>(n, r, slab, s) : launch_join<128, 8, 4>(n, r, slab, s);
    return n.dim <= 64 ? launch_join<64, 16, 8>(n, r, slab, s) : launch_join<128, 16, 8>(n, r, slab, s);
}

}  // namespace strata
