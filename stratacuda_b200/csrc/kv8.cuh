// Device helpers of the 8-bit paged key/value cache kernels.
#pragma once
#include "common.cuh"
#include "kv8.h"

#include <cuda_fp16.h>

namespace strata {

// Programmatic dependent launch, by all of these kernels: a kernel may be placed while the one before it still runs, and
// its first act is to wait until that has finished and its writes are visible; then it lets the next one be placed. Only
// launch latency overlaps: about 2 us a kernel of a token step.
__device__ __forceinline__ void kv8_enter() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
template <typename... KT, typename... AT>
inline cudaError_t kv8_launch(void (*k)(KT...), dim3 grid, dim3 block, size_t smem, unsigned cluster, cudaStream_t s, AT &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, static_cast<AT &&>(args)...);
}

// A run's sequence and first position, or sequence -1 for an idle slot (a sequence outside the
// cache is reported and treated as idle).
struct RunAt {
    int sequence, start;
};
__device__ __forceinline__ RunAt run_at(const Kv8 &c, const Kv8Runs &r, int i) {
    RunAt a{r.sequence[i], r.start[i]};
    if (a.sequence < -1 || a.sequence >= c.sequences) {
        raise_error(c.err, kErrIndex);
        a.sequence = -1;
    }
    return a;
}
// Keys that token j of a run sees: those at or before its own position, none for an idle slot.
// Positions past the table are reported and left out.
__device__ __forceinline__ int visible_keys(const Kv8 &c, const RunAt &a, int j) {
    if (a.sequence < 0) return 0;
    const long long n = (long long)a.start + j + 1, most = (long long)c.blocks * kKvBlock;
    if (n > most) raise_error(c.err, kErrIndex);
    return n <= 0 ? 0 : (int)(n > most ? most : n);
}
// The page of a sequence's block, or -1 (reported) when the table holds none.
__device__ __forceinline__ int page_of(const Kv8 &c, int sequence, int block) {
    const int p = c.table[(size_t)sequence * c.blocks + block];
    if (p >= 0 && p < c.pages) return p;
    raise_error(c.err, kErrIndex);
    return -1;
}
__device__ __forceinline__ int8_t *page_codes(const Kv8 &c, int page, int head, int kind) {
    return c.codes + (((size_t)page * c.kv_heads + head) * 2 + kind) * c.padded * kKvBlock;
}
__device__ __forceinline__ int8_t *page_marks(const Kv8 &c, int page, int head) {
    return c.marks + ((size_t)page * c.kv_heads + head) * 2 * c.padded;
}
__device__ __forceinline__ float *page_scales(const Kv8 &c, int page, int head) { return c.scales + ((size_t)page * c.kv_heads + head) * 2; }
// Byte of key channel ch of token t in a page: panels of 64 channels, token rows of 64 bytes.
__device__ __forceinline__ int key_byte(int t, int ch) { return ((ch >> 6) * kKvBlock + t) * 64 + (ch & 63); }

// Four signed codes as two FP16 pairs: the bits 0x6400 | (c + 128) are 1152 + c, less 1152 is c, exactly.
__device__ __forceinline__ void codes_to_half(unsigned w, unsigned &b0, unsigned &b1) {
    const unsigned u = w ^ 0x80808080u, k1152 = 0x64806480u;
    const unsigned p0 = __byte_perm(u, 0x64646464u, 0x4140), p1 = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 k = *reinterpret_cast<const __half2 *>(&k1152);
    const __half2 h0 = __hsub2(*reinterpret_cast<const __half2 *>(&p0), k), h1 = __hsub2(*reinterpret_cast<const __half2 *>(&p1), k);
    b0 = *reinterpret_cast<const unsigned *>(&h0);
    b1 = *reinterpret_cast<const unsigned *>(&h1);
}
// a pair of floats as FP16 halves: x = hi + lo to 2^-22 of x (2^-25 absolute for small x)
__device__ __forceinline__ void split_pair(float x, float y, unsigned &hi, unsigned &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const unsigned *>(&h);
    lo = *reinterpret_cast<const unsigned *>(&l);
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

}  // namespace strata
