// The gated delta rule in chunks of 64 tokens on the 5th-generation tensor cores: what its two kernels share.
//
// With P_i the product of a chunk's decays up to token i, G_ij that of those after j up to i, E_i that of those after i:
//   A_ij = beta_i G_ij (k_i . k_j) for j < i,   T = (I + A)^-1,   U = T diag(beta) V,   W = T diag(beta P) K        delta_prepare.cu
//   D = U - W S,   y_i = P_i q_i S + sum_{j <= i} G_ij (q_i . k_j) D_j,   S <- P_63 S + sum_i E_i k_i D_i^T          delta_chain.cu
// (with keys as they are scaled for the products, by a power of two e_i each: k_i 2^-e_i, beta_i 2^2e_i, and as V and D what they add to the
// state, beta_i 2^e_i v_i and 2^e_i d_i; so that keys and strengths of all sizes meet in factors of one size.)
// The first line needs no state: all chunks of all heads at once. The second goes from chunk to chunk. Products of decays are
// formed by multiplication alone, so that zero decays need no care.
//
// Runs of few states are taken in parts at once: a state goes into a part and out of it as  S' = F S + N, with F and N where the identity
// without values and zeros end; then the parts follow from the states before them.                  delta_chain.cu, delta_join.cu
//
// Products. Each F32 factor is two FP16 halves, times a power of two that brings the largest value of its row (or of its
// TMEM lane, or tile) to 2^13; lo is held 2^11 times as large as it is. That is 22 bits for whatever is within 2^-27 of the largest, and
// 2^-49 of it below. lo hi + hi lo + hi hi are three FP16 products with F32 sums; lo lo would be 2^-22 of the result. The large product
// comes last, its first step takes the sum so far times 2^-11: sums in TMEM are cut, not rounded, and each step at full size costs up to
// 2^-24 of the sum, always towards zero (a prompt's result is 2.5e-7 off in the 2-norm; with hi hi first three times as much).
//
// What a lane holds of a chunk's 64 tokens has one power of two, also of tokens that are to come, or that a decay has taken away. A chunk in
// which that hides a value of V, or a difference, from a token whose state holds nothing larger is walked token by token.
//
// Workspace: a slot for each run, key head and chunk of a slab, in the layout that the second kernel's tensor-core operands
// have in shared memory (rows of 128 bytes, 128-byte swizzle): Q above K [2 x 64 tokens][D], hi and lo; then for each of the key
// head's value heads W^T [D][64], hi and lo, the products G (q . k) [64][64], hi and lo, U [64][D] in F32 and the rows' factors.
#pragma once
#include "mixers.cuh"
#include "pf_gemm.cuh"

namespace strata {

constexpr int kChunk = 64;
constexpr int kSortedRuns = 128;        // at most, where runs are taken by their lengths
constexpr float kDeltaLarge = 0x1p60f;  // past this, or not finite: the chunk is walked token by token

struct DeltaFactors {  // of a chunk's rows, for one value head
    float z[64];       // W's scale taken back
    float q[64];       // P over Q's scale
    float attn[64];    // G (q . k)'s scale taken back
    float k[64];       // E over 2^13
    float end;         // P of the last token
    int walk;          // token by token
    int counted;       // tokens up to the last one with a query or a key: rows that fill up a batch have neither
    int pad[29];
};
struct DeltaSlab {  // runs, key heads and chunks [first, first + n) of a call
    int run0, runs, head0, heads, chunk0, chunks;
    int ratio;   // value heads of a key head
    int sorted;  // the second kernel takes long runs first
    int ahead;  // the first kernel runs while the slab before is on its way through the second
    unsigned char *slots;
    long long slot_bytes;
    // Runs in parts of part_chunks chunks that are on their way at once (parts > 1): of each run and head, for each part p but the
    // last, its transition and its end without it ([dim D][dim D] each), then the end with it; in the first one's transition's place
    // the state before it. And whether a run and head has to be taken whole.
    int parts, part_chunks;
    float *states;
    int *whole;
};
template <int D>
struct DeltaSlot {
    static constexpr int tile = 64 * D * 2 * 2, attn = 64 * 64 * 2 * 2, u = 64 * D * 4;  // bytes; hi and lo
    static constexpr int heads = 2 * tile;  // behind Q and K
    static constexpr int w = 0, g = tile, uu = tile + attn, factors = uu + u, head_bytes = factors + (int)sizeof(DeltaFactors);
    __host__ __device__ static long long bytes(int ratio) { return heads + (long long)ratio * head_bytes; }
};

cudaError_t delta_step(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, cudaStream_t s);
cudaError_t delta_prepare(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, const DeltaSlab &slab, bool vec, cudaStream_t s);
cudaError_t delta_chain(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, const DeltaSlab &slab, cudaStream_t s);
cudaError_t delta_ends(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, const DeltaSlab &slab, cudaStream_t s);  // transitions and ends of parts
cudaError_t delta_join(const DeltaNet &n, const MixRuns &r, const DeltaSlab &slab, cudaStream_t s);                     // states before them

#ifdef __CUDACC__
namespace delta {

using namespace pf;

// 8, 16 or 32 columns of this thread's TMEM lane, and 8 or 16 written.
__device__ __forceinline__ void tmem_read(unsigned taddr, float (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
          "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_read8(unsigned taddr, float (&v)[8]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_read(unsigned taddr, float (&v)[32]) { tmem_ld32(taddr, v); }
__device__ __forceinline__ void tmem_write(unsigned taddr, const unsigned (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_write(unsigned taddr, const unsigned (&r)[16]) { tmem_st16(taddr, r); }
__device__ __forceinline__ void tmem_written() {
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    tc_fence_before();
}
__device__ __forceinline__ void to_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// The power of two that brings a largest magnitude to [2^13, 2^14), and its reciprocal.
__device__ __forceinline__ int exponent_of(float largest) { return min(max((int)(__float_as_uint(largest) >> 23) - 127, -113), 127); }
__device__ __forceinline__ float scale_of(int e) { return __uint_as_float((unsigned)(140 - e) << 23); }
__device__ __forceinline__ float unscale_of(int e) { return __uint_as_float((unsigned)(114 + e) << 23); }
// Largest magnitudes; NaN where one is.
__device__ __forceinline__ float larger(float a, float b, float c) {
    float d;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float smaller(float a, float b, float c) {  // of magnitudes
    float d;
    asm("min.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Below this magnitude a value has less than 22 bits beside a largest one of exponent e. (Where that is as small as it gets, F32 ends first.)
__device__ __forceinline__ float hidden_below(int e) { return e > -113 ? unscale_of(e) * 0x1p-14f : 0.0f; }
template <int N>
__device__ __forceinline__ float largest(float m, const float (&x)[N]) {
#pragma unroll
    for (int i = 0; i + 1 < N; i += 2) m = larger(m, x[i], x[i + 1]);
    return m;
}
__device__ __forceinline__ float warp_largest(float x) {
    float r;
    asm volatile("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ bool past(float largest) { return !(largest <= kDeltaLarge); }
// Pairs of F32 as one 64-bit register pair.
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ unsigned long long both(float x) { return pack2(x, x); }
// A pair times powers of two as FP16 halves, hi first where products with it begin before lo is there. lo is held kLow times as
// large: it keeps 11 bits where hi itself is as small as FP16 gets. (What hi leaves is a sum of an F32 and an FP16 number in one
// instruction: conversions back to F32 share a pipe with paired operations, which bounds a split. With them, and products by kLow one by one,
// 2048 tokens over 32 heads of 128 take 8% longer.)
constexpr float kLow = 0x1p11f;
__device__ __forceinline__ float less_half(float x, unsigned short negative) {
    float d;
    asm("add.rn.f32.f16 %0, %1, %2;" : "=f"(d) : "h"(negative), "f"(x));
    return d;
}
__device__ __forceinline__ unsigned split_hi(unsigned long long x, unsigned long long by) {
    float a, b;
    unpack2(mul2_rn(x, by), a, b);
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned *>(&h);
}
__device__ __forceinline__ unsigned split_lo(unsigned long long x, unsigned long long by, unsigned hi) {
    float a, b;
    unpack2(mul2_rn(x, by), a, b);
    const unsigned h = hi ^ 0x80008000u;
    unpack2(mul2_rn(pack2(less_half(a, (unsigned short)h), less_half(b, (unsigned short)(h >> 16))), both(kLow)), a, b);
    const __half2 l = __floats2half2_rn(a, b);
    return *reinterpret_cast<const unsigned *>(&l);
}
__device__ __forceinline__ void split2(unsigned long long x, unsigned long long by, unsigned &hi, unsigned &lo) { hi = split_hi(x, by), lo = split_lo(x, by, hi); }
template <int N>
__device__ __forceinline__ void split(const float (&x)[N], float scale, unsigned (&hi)[N / 2], unsigned (&lo)[N / 2]) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) split2(pack2(x[2 * i], x[2 * i + 1]), both(scale), hi[i], lo[i]);
}
__device__ __forceinline__ float larger2(float m, unsigned long long x) {
    float a, b;
    unpack2(x, a, b);
    return larger(m, a, b);
}
__device__ __forceinline__ float smaller2(float m, unsigned long long x) {
    float a, b;
    unpack2(x, a, b);
    return smaller(m, a, b);
}
// Byte of 16-byte piece c of row r: rows of 128 bytes, 128-byte swizzle.
__device__ __forceinline__ int piece(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }
// Pieces [first, first + N / 4) of row r of a tile from pairs.
template <int N>
__device__ __forceinline__ void put_pieces(unsigned char *tile, int r, int first, const unsigned (&x)[N]) {
#pragma unroll
    for (int c = 0; c < N / 4; ++c) *reinterpret_cast<uint4 *>(tile + piece(r, first + c)) = uint4{x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]};
}
// Operand with its rows along the sum (a tile [sum][64 channels a panel] read the other way round): 64 channels of 8 rows are
// an atom; panels are `panel` bytes apart, the next 8 rows 1024.
__device__ __forceinline__ unsigned long long turned_desc(unsigned smem_addr, unsigned panel) {
    return (unsigned long long)((smem_addr & 0x3FFFFu) >> 4) | ((unsigned long long)(panel >> 4) << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ unsigned turned_idesc(int M, int N) { return idesc_f16(M, N) | (1u << 16); }  // the narrow operand
constexpr unsigned kTurnedWide = 1u << 15;                                                                // the 128-row one

// Step k of product 0 (lo hi), 1 (hi lo) or 2 (hi hi) of a sum; the last one's first step takes what the others gave times 2^-11, 1 / kLow.
__device__ __forceinline__ void mma_step(unsigned tmem_d, unsigned long long a, unsigned long long b, unsigned idesc, int product, int k) {
    if (product < 2 || k) return mma_f16(tmem_d, a, b, idesc, product || k);
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.eq.b32 p, 0, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p, 11;\n\t}" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc)
        : "memory");
}
__device__ __forceinline__ void mma_step_ts(unsigned tmem_d, unsigned tmem_a, unsigned long long b, unsigned idesc, int product, int k) {
    if (product < 2 || k) return mma_f16_ts(tmem_d, tmem_a, b, idesc, product || k);
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.eq.b32 p, 0, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p, 11;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(b), "r"(idesc)
        : "memory");
}

// A channel's 64 tokens over a warp, two a lane: what each adds to the state of it (size[0] of token `lane`, size[1] of lane + 32), what is left
// of the state at it (decay, up to one), and `held` before them. Whether there is a token among `wanted` (bits as sizes) that sees less than
// limit but something: neither of its own (`seen`) nor of what the state holds.
__device__ __forceinline__ bool see_less(const float (&size)[2], const float (&decay)[2], const float (&seen)[2], const bool (&wanted)[2], float held, float limit, int lane) {
    bool any = false;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        float d = decay[e], b = size[e];  // over tokens so far: held after them is max(d held, b)
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const float d0 = __shfl_up_sync(0xffffffffu, d, s), b0 = __shfl_up_sync(0xffffffffu, b, s);
            if (lane >= s) b = fmaxf(d * b0, b), d *= d0;
        }
        const float after = fmaxf(d * held, b), before = __shfl_up_sync(0xffffffffu, after, 1);
        const float most = fmaxf(seen[e], decay[e] * (lane ? before : held));
        any |= wanted[e] & (most > 0.0f) & (most < limit);
        held = __shfl_sync(0xffffffffu, after, 31);
    }
    return __any_sync(0xffffffffu, any);
}

// Waits of a block's threads, with a limit; past it, all of them let everything through and the block reports.
struct Waits {
    int *abort_flag;
    unsigned *err;
    __device__ __forceinline__ void operator()(unsigned long long *b, unsigned parity) const {
        if (bar_try(b, parity)) return;
        const long long began = clock64();
        while (!bar_try(b, parity)) {
            if (*(volatile int *)abort_flag) return;
            if (clock64() - began > 2000000000LL) {  // about a second
                atomicExch(abort_flag, 1);
                raise_error(err, kErrWaitTimeout);
                return;
            }
        }
    }
    // The same of a whole warp: one lane looks (32 that look at one barrier take 15 clocks each way, 16 warps of them 250).
    __device__ __forceinline__ void warp(unsigned long long *b, unsigned parity, int lane) const {
        if (lane == 0) (*this)(b, parity);
        __syncwarp();
    }
};

// After a wait has run out: time for copies and products in flight, before shared memory and TMEM go.
__device__ __forceinline__ void settle(const int *abort_flag) {
    if (!*(volatile const int *)abort_flag) return;
    const long long began = clock64();
    while (clock64() - began < 4000000) {
    }
}

}  // namespace delta
#endif

}  // namespace strata
