// Choosing the blocks that a query attends to (strata_kv8_select).
#include "kv8.cuh"

namespace strata {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float block_max(float x, float *red) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, s));
    __syncthreads();
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = x;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) x = fmaxf(x, red[i]);
    return x;
}
// A float's bits in an order that compares as unsigned words.
__device__ __forceinline__ unsigned ordered(float f) {
    const unsigned u = __float_as_uint(f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One CTA: one token and key/value head. The group's queries become two rows of 8-bit codes
// (positive and negative parts), every block's bound is an integer product with its marks, and the
// top-th largest ordered bound is found bit by bit; blocks above it and the lowest of those equal to
// it are written in ascending order.
template <int P>
__global__ void __launch_bounds__(kThreads) k_kv8_select(const Kv8 c, const float *q, long long stride, int heads, const Kv8Runs runs, int top,
                                                         int first, int last, int *picks) {
    extern __shared__ unsigned key_s[];  // [blocks in sight]
    __shared__ float red[kThreads / 32];
    __shared__ __align__(16) int8_t pos_s[P], neg_s[P];
    __shared__ int count_s, taken_s[kThreads];
    const int tid = threadIdx.x, head = blockIdx.y;
    const int token = blockIdx.x, run = token / runs.count;
    const RunAt a = run_at(c, runs, run);
    const int nb = (visible_keys(c, a, token % runs.count) + kKvBlock - 1) / kKvBlock;
    int *out = picks + ((size_t)token * c.kv_heads + head) * top;
    if (nb <= top) {
        for (int i = tid; i < top; i += kThreads) out[i] = i < nb ? i : -1;
        return;
    }
    const int group = heads / c.kv_heads;
    const float *x = q + (long long)token * stride + (size_t)head * group * c.dim;
    float amax = 0.0f;
    for (int i = tid; i < group * c.dim; i += kThreads) amax = fmaxf(amax, isfinite(x[i]) ? fabsf(x[i]) : 0.0f);
    amax = block_max(amax, red);
    const float unit = amax < 0x1p-100f ? 0.0f : __fdiv_rn(32767.0f, amax);
    int pos = 0, neg = 0;
    if (tid < c.dim)
        for (int h = 0; h < group; ++h) {
            const float f = x[h * c.dim + tid];
            const int r = isfinite(f) ? __float2int_rn(__fmul_rn(f, unit)) : 0;
            pos += max(r, 0);
            neg += min(r, 0);
        }
    const float big = block_max((float)max(pos, -neg), red);
    const float fine = big > 0.0f ? __fdiv_rn(127.0f, big) : 0.0f;
    if (tid < P) {
        pos_s[tid] = (int8_t)__float2int_rn(__fmul_rn((float)pos, fine));
        neg_s[tid] = (int8_t)__float2int_rn(__fmul_rn((float)neg, fine));
    }
    __syncthreads();
    for (int b = tid; b < nb; b += kThreads) {
        unsigned key = 0xffffffffu;
        if (b >= first && b < nb - last) {
            const int page = page_of(c, a.sequence, b);
            int dot = 0;
            float scale = 0.0f;
            if (page >= 0) {
                const uint4 *m = reinterpret_cast<const uint4 *>(page_marks(c, page, head));
                for (int i = 0; i < P / 16; ++i) {
                    const uint4 lo = m[i], hi = m[P / 16 + i];
                    const uint4 n = reinterpret_cast<const uint4 *>(neg_s)[i], p = reinterpret_cast<const uint4 *>(pos_s)[i];
                    dot = __dp4a((int)lo.x, (int)n.x, dot), dot = __dp4a((int)lo.y, (int)n.y, dot);
                    dot = __dp4a((int)lo.z, (int)n.z, dot), dot = __dp4a((int)lo.w, (int)n.w, dot);
                    dot = __dp4a((int)hi.x, (int)p.x, dot), dot = __dp4a((int)hi.y, (int)p.y, dot);
                    dot = __dp4a((int)hi.z, (int)p.z, dot), dot = __dp4a((int)hi.w, (int)p.w, dot);
                }
                scale = page_scales(c, page, head)[0];
            }
            key = min(ordered(__fmul_rn((float)dot, scale)), 0xfffffffeu);
        }
        key_s[b] = key;
    }
    // the largest threshold that at least `top` keys reach, from its highest bit down
    unsigned least = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const unsigned trial = least | 1u << bit;
        __syncthreads();
        if (tid == 0) count_s = 0;
        __syncthreads();
        int n = 0;
        for (int b = tid; b < nb; b += kThreads) n += key_s[b] >= trial;
        atomicAdd(&count_s, n);
        __syncthreads();
        if (count_s >= top) least = trial;
    }
    // each thread writes a run of blocks of its own; keys equal to the threshold fill what is left, lowest first
    const int each = (nb + kThreads - 1) / kThreads, b0 = tid * each, b1 = min(nb, b0 + each);
    int above = 0, equal = 0;
    for (int b = b0; b < b1; ++b) {
        above += key_s[b] > least;
        equal += key_s[b] == least;
    }
    taken_s[tid] = above | equal << 16;
    __syncthreads();
    if (tid == 0) {
        int room = top;
        for (int i = 0; i < kThreads; ++i) room -= taken_s[i] & 65535;
        int at = 0;
        for (int i = 0; i < kThreads; ++i) {
            const int up = taken_s[i] & 65535, eq = min(room, taken_s[i] >> 16);
            taken_s[i] = at | eq << 16;
            at += up + eq;
            room -= eq;
        }
    }
    __syncthreads();
    int at = taken_s[tid] & 65535, eq = taken_s[tid] >> 16;
    for (int b = b0; b < b1; ++b) {
        const bool same = key_s[b] == least;
        if (key_s[b] > least || (same && eq > 0)) {
            out[at++] = b;
            eq -= same;
        }
    }
}

template <int P>
cudaError_t launch(const Kv8 &c, const float *q, long long stride, int heads, const Kv8Runs &r, int top, int first, int last, int *picks,
                   cudaStream_t s) {
    const size_t smem = (size_t)c.blocks * 4;
    cudaError_t e = cudaFuncSetAttribute(k_kv8_select<P>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    k_kv8_select<P><<<dim3(r.segments * r.count, c.kv_heads), kThreads, smem, s>>>(c, q, stride, heads, r, top, first, last, picks);
    return cudaGetLastError();
}

}  // namespace

cudaError_t kv8_select(const Kv8 &c, const float *q, long long stride, int heads, const Kv8Runs &r, int top, int first, int last, int *picks,
                       cudaStream_t s) {
    if (c.padded == 64) return launch<64>(c, q, stride, heads, r, top, first, last, picks, s);
    if (c.padded == 128) return launch<128>(c, q, stride, heads, r, top, first, last, picks, s);
    return launch<256>(c, q, stride, heads, r, top, first, last, picks, s);
}

}  // namespace strata
