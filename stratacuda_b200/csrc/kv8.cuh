// Device helpers of the 8-bit paged key/value cache kernels.
#pragma once
#include "common.cuh"
#include "kv8.h"

namespace strata {

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

}  // namespace strata
