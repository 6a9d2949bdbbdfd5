// Internal interface of the 8-bit paged key/value cache (kv8_append.cu, kv8_select.cu,
// kv8_attend.cu, checked and launched by kv8_api.cu and api.cu). The format and the operators'
// definitions are in include/strata_cuda.h.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <cstddef>

namespace strata {

constexpr int kKvBlock = 64;  // tokens of a page

// Device view of one layer's cache.
struct Kv8 {
    int kv_heads, dim, padded;  // padded: stored channels, 64, 128 or 256
    int pages, sequences, blocks;
    int8_t *codes;       // [pages][kv_heads][2][padded * 64]
    int8_t *marks;       // [pages][kv_heads][2][padded]
    float *scales;       // [pages][kv_heads][2]
    float *open;         // [sequences][2][64][kv_heads][dim]
    const int *table;    // [sequences][blocks]
    void *workspace;     // STRATA_KV8_WORKSPACE_BYTES
    unsigned *err;       // error word, or null
};
// `segments` runs of `count` tokens; run i continues sequence[i] at position start[i].
struct Kv8Runs {
    int segments, count;
    const int *sequence, *start;
};

inline int kv8_padded(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Argument checks shared by the handle and the pointer forms; 0 or a status with `msg` filled.
// The aligned device addresses are checked by kv8_check_pointers.
int kv8_check_cache(int kv_heads, int dim, int pages, int sequences, int blocks, char *msg, size_t cap);
int kv8_check_runs(int segments, int count, char *msg, size_t cap);
int kv8_check_heads(int heads, int kv_heads, char *msg, size_t cap);
int kv8_check_select(int blocks, int top, int first, int last, char *msg, size_t cap);
int kv8_check_rows(int count, int heads, int kv_heads, char *msg, size_t cap);
int kv8_check_picks(int top, char *msg, size_t cap);
int kv8_check_stride(long long stride, long long width, char *msg, size_t cap);
int kv8_check_alignment(const Kv8 &c, char *msg, size_t cap);

cudaError_t kv8_append(const Kv8 &c, const float *k, const float *v, long long stride, const Kv8Runs &r, cudaStream_t s);
cudaError_t kv8_select(const Kv8 &c, const float *q, long long stride, int heads, const Kv8Runs &r, int top, int first, int last, int *picks,
                       cudaStream_t s);
// picks null: every block. `scale` multiplies q . k.
cudaError_t kv8_attend(const Kv8 &c, const float *q, long long stride, int heads, const Kv8Runs &r, const int *picks, int top, float scale,
                       float *y, cudaStream_t s);
// The same for many tokens a run, every block: 128-row tiles (kv8_prompt.cu), taken by kv8_attend.
cudaError_t kv8_attend_prompt(const Kv8 &c, const float *q, long long stride, int heads, const Kv8Runs &r, float scale, float *y,
                              cudaStream_t s);

}  // namespace strata
