// Cache pages as operands of the tensor cores' integer products (tcgen05 kind::i8): rows of 64 codes as they lie in memory,
// fetched by TMA with a 64-byte swizzle.
#pragma once
#include "kv8.cuh"
#include "pf_gemm.cuh"

#include <cudaTypedefs.h>

#include <mutex>

namespace strata {
namespace {

// Shared-memory matrix descriptor: K-major, 64-byte rows and swizzle, 8-row groups 512 bytes apart.
__device__ __forceinline__ unsigned long long sw64_desc(unsigned smem_addr) {
    return (unsigned long long)((smem_addr & 0x3FFFFu) >> 4) | (1ull << 16) | (32ull << 32) | (1ull << 46) | (4ull << 61);
}
// Byte of a 64-byte row in that layout.
__device__ __forceinline__ int sw64_byte(int row, int at) { return row * 64 + ((((at >> 4) ^ (row >> 1)) & 3) << 4) + (at & 15); }
// Instruction descriptor, kind::i8: S32 sums (bits 4-5 = 2), A signed (bits 7-9 = 1), B signed or not (bits 10-12), both
// K-major, M = 128.
__device__ __forceinline__ unsigned idesc_i8(int N, bool b_signed) {
    return (2u << 4) | (1u << 7) | ((unsigned)b_signed << 10) | ((unsigned)(N >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void mma_i8(unsigned tmem_d, unsigned long long a, unsigned long long b, unsigned idesc, int accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Three signed 8-bit digits of four whole numbers |v| <= 2^22, digit e of v[k] in byte k of d[e]: with 128 added at each
// digit's place the digits are the bytes, less 128 each.
__device__ __forceinline__ void digits_of(const int (&v)[4], unsigned (&d)[3]) {
    unsigned w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = (unsigned)(v[k] + 0x808080) ^ 0x808080u;
    const unsigned a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);
    d[0] = __byte_perm(a, b, 0x5410);
    d[1] = __byte_perm(a, b, 0x7632);
    d[2] = __byte_perm(__byte_perm(w[0], w[1], 0x0062), __byte_perm(w[2], w[3], 0x0062), 0x5410);
}
inline PFN_cuTensorMapEncodeTiled_v12000 encoder() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}
// The cache's codes as {64 bytes, rows of a page, pages}, fetched in boxes of box_rows rows of one page.
inline bool page_map(const Kv8 &c, unsigned box_rows, CUtensorMap *map) {
    const auto encode = encoder();
    const cuuint64_t dims[3] = {64, 2ull * c.kv_heads * c.padded, (cuuint64_t)c.pages}, strides[2] = {64, dims[1] * 64};
    const cuuint32_t box[3] = {64, box_rows, 1}, steps[3] = {1, 1, 1};
    return encode && encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, c.codes, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace
}  // namespace strata
