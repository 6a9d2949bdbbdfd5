// Argument checks of the 8-bit paged cache and its entries on caller-owned device memory
// (include/strata_cuda.h). The handle-based entries are in api.cu and share the checks.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>

#include "../../include/strata_cuda.h"
#include "kernels.h"
#include "kv8.h"

namespace strata {

namespace {
int say(char *msg, size_t cap, int code, const char *text) {
    if (msg && cap) snprintf(msg, cap, "%s", text);
    return code;
}
bool aligned(const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
}  // namespace

int kv8_check_cache(int kv_heads, int dim, int pages, int sequences, int blocks, char *msg, size_t cap) {
    if (kv_heads < 1 || kv_heads > 4096) return say(msg, cap, STRATA_ERR_RANGE, "cache kv_heads must be an integer in [1, 4096]");
    if (dim < 1 || dim > 256) return say(msg, cap, STRATA_ERR_RANGE, "cache dim must be an integer in [1, 256]");
    if (pages < 1) return say(msg, cap, STRATA_ERR_RANGE, "cache pages must be an integer >= 1");
    if (sequences < 1) return say(msg, cap, STRATA_ERR_RANGE, "cache sequences must be an integer >= 1");
    if (blocks < 1 || blocks > 0x7fffffff / kKvBlock)
        return say(msg, cap, STRATA_ERR_RANGE, "cache blocks must be an integer in [1, 33554431]: positions are 32-bit");
    return STRATA_OK;
}
int kv8_check_runs(int segments, int count, char *msg, size_t cap) {
    if (segments < 1 || segments > 65535) return say(msg, cap, STRATA_ERR_RANGE, "segments must be an integer in [1, 65535]");
    if (count < 1 || (long long)segments * count > (1 << 24))
        return say(msg, cap, STRATA_ERR_RANGE, "count must be at least 1 and segments * count at most 2^24 tokens");
    return STRATA_OK;
}
int kv8_check_heads(int heads, int kv_heads, char *msg, size_t cap) {
    if (heads < 1 || heads > 65535) return say(msg, cap, STRATA_ERR_RANGE, "heads must be an integer in [1, 65535]");
    if (heads % kv_heads) return say(msg, cap, STRATA_ERR_RANGE, "Attention heads must be divisible by KV heads");
    return STRATA_OK;
}
int kv8_check_select(int blocks, int top, int first, int last, char *msg, size_t cap) {
    if (blocks > STRATA_KV8_SELECT_BLOCKS) return say(msg, cap, STRATA_ERR_RANGE, "selection serves tables of at most 32768 blocks");
    if (top < 1 || top > STRATA_KV8_SELECT_BLOCKS) return say(msg, cap, STRATA_ERR_RANGE, "top must be an integer in [1, 32768]");
    if (first < 0 || last < 0 || (long long)first + last > top)
        return say(msg, cap, STRATA_ERR_RANGE, "first and last must be integers >= 0 with first + last <= top");
    return STRATA_OK;
}
int kv8_check_rows(int count, int heads, int kv_heads, char *msg, size_t cap) {
    // a prompt's rows, whole tiles of 128, are counted in 32 bits
    return (long long)count * (heads / kv_heads) > 0x80000000LL - 128
               ? say(msg, cap, STRATA_ERR_RANGE, "count * heads / kv_heads must be at most 2^31 - 128 rows where every block is attended to")
               : STRATA_OK;
}
int kv8_check_picks(int top, char *msg, size_t cap) {
    // as many blocks as a table can have: lists are walked with 32-bit indices
    return top < 1 || top > 0x7fffffff / kKvBlock ? say(msg, cap, STRATA_ERR_RANGE, "top must be an integer in [1, 33554431]") : STRATA_OK;
}
int kv8_check_stride(long long stride, long long width, char *msg, size_t cap) {
    if (stride < width || stride > (1LL << 40)) return say(msg, cap, STRATA_ERR_LAYOUT, "row_stride is smaller than a row");
    return STRATA_OK;
}
int kv8_check_alignment(const Kv8 &c, char *msg, size_t cap) {
    if (!aligned(c.codes, 16) || !aligned(c.marks, 16) || !aligned(c.workspace, 16))
        return say(msg, cap, STRATA_ERR_LAYOUT, "codes, marks and workspace must start on 16-byte boundaries");
    if (!aligned(c.scales, 4) || !aligned(c.open, 4) || !aligned(c.table, 4) || !aligned(c.err, 4))
        return say(msg, cap, STRATA_ERR_LAYOUT, "scales, open, table and status must start on 4-byte boundaries");
    return STRATA_OK;
}

}  // namespace strata

using namespace strata;

namespace {

// The view of a caller's cache and runs, or a status.
int view(const strata_kv8_cache_dev *cache, int segments, int count, const int32_t *sequence, const int32_t *start, Kv8 *c, Kv8Runs *r,
         char *msg, size_t cap) {
    if (msg && cap) msg[0] = 0;
    if (!cache) return say(msg, cap, STRATA_ERR_RANGE, "null cache");
    if (int e = kv8_check_cache(cache->kv_heads, cache->dim, cache->pages, cache->sequences, cache->blocks, msg, cap)) return e;
    if (int e = kv8_check_runs(segments, count, msg, cap)) return e;
    if (!cache->codes || !cache->marks || !cache->scales || !cache->open || !cache->table || !cache->workspace || !sequence || !start)
        return say(msg, cap, STRATA_ERR_RANGE, "null device pointer");
    *c = Kv8{cache->kv_heads, cache->dim, kv8_padded(cache->dim), cache->pages, cache->sequences, cache->blocks, cache->codes, cache->marks,
             cache->scales, cache->open, cache->table, cache->workspace, cache->status};
    *r = Kv8Runs{segments, count, sequence, start};
    if (!aligned(sequence, 4) || !aligned(start, 4)) return say(msg, cap, STRATA_ERR_LAYOUT, "sequence and start must start on 4-byte boundaries");
    return kv8_check_alignment(*c, msg, cap);
}
int rows(const void *p, uint64_t *stride, long long width, char *msg, size_t cap) {
    if (!p) return say(msg, cap, STRATA_ERR_RANGE, "null device pointer");
    if (!aligned(p, 4)) return say(msg, cap, STRATA_ERR_LAYOUT, "rows must start on 4-byte boundaries");
    if (!*stride) *stride = (uint64_t)width;
    return *stride > (1ull << 40) ? say(msg, cap, STRATA_ERR_LAYOUT, "row_stride is out of range")
                                  : kv8_check_stride((long long)*stride, width, msg, cap);
}
int done(cudaError_t e, char *msg, size_t cap) { return e == cudaSuccess ? STRATA_OK : say(msg, cap, STRATA_ERR_CUDA, cudaGetErrorString(e)); }

}  // namespace

extern "C" int strata_kv8_append_dev(const strata_kv8_cache_dev *cache, const float *k, const float *v, uint64_t row_stride, int32_t segments,
                                     int32_t count, const int32_t *sequence, const int32_t *start, void *stream, char *msg, size_t msg_cap) {
    Kv8 c;
    Kv8Runs r;
    if (int e = view(cache, segments, count, sequence, start, &c, &r, msg, msg_cap)) return e;
    if (int e = rows(k, &row_stride, (long long)c.kv_heads * c.dim, msg, msg_cap)) return e;
    if (int e = rows(v, &row_stride, (long long)c.kv_heads * c.dim, msg, msg_cap)) return e;
    return done(kv8_append(c, k, v, (long long)row_stride, r, static_cast<cudaStream_t>(stream)), msg, msg_cap);
}

extern "C" int strata_kv8_select_dev(const strata_kv8_cache_dev *cache, const float *q, uint64_t row_stride, int32_t heads, int32_t segments,
                                     int32_t count, const int32_t *sequence, const int32_t *start, int32_t top, int32_t first, int32_t last,
                                     int32_t *picks, void *stream, char *msg, size_t msg_cap) {
    Kv8 c;
    Kv8Runs r;
    if (int e = view(cache, segments, count, sequence, start, &c, &r, msg, msg_cap)) return e;
    if (int e = kv8_check_heads(heads, c.kv_heads, msg, msg_cap)) return e;
    if (int e = kv8_check_select(c.blocks, top, first, last, msg, msg_cap)) return e;
    if (int e = rows(q, &row_stride, (long long)heads * c.dim, msg, msg_cap)) return e;
    if (!picks) return say(msg, msg_cap, STRATA_ERR_RANGE, "null device pointer");
    if (!aligned(picks, 4)) return say(msg, msg_cap, STRATA_ERR_LAYOUT, "picks must start on a 4-byte boundary");
    return done(kv8_select(c, q, (long long)row_stride, heads, r, top, first, last, picks, static_cast<cudaStream_t>(stream)), msg, msg_cap);
}

extern "C" int strata_kv8_attend_dev(const strata_kv8_cache_dev *cache, const float *q, uint64_t row_stride, int32_t heads, int32_t segments,
                                     int32_t count, const int32_t *sequence, const int32_t *start, const int32_t *picks, int32_t top,
                                     float scale, float *y, void *stream, char *msg, size_t msg_cap) {
    Kv8 c;
    Kv8Runs r;
    if (int e = view(cache, segments, count, sequence, start, &c, &r, msg, msg_cap)) return e;
    if (int e = kv8_check_heads(heads, c.kv_heads, msg, msg_cap)) return e;
    if (int e = rows(q, &row_stride, (long long)heads * c.dim, msg, msg_cap)) return e;
    if (!y) return say(msg, msg_cap, STRATA_ERR_RANGE, "null device pointer");
    if (!aligned(y, 4) || !aligned(picks, 4)) return say(msg, msg_cap, STRATA_ERR_LAYOUT, "picks and y must start on 4-byte boundaries");
    if (int e = picks ? kv8_check_picks(top, msg, msg_cap) : kv8_check_rows(count, heads, c.kv_heads, msg, msg_cap)) return e;
    if (!std::isfinite(scale)) return say(msg, msg_cap, STRATA_ERR_RANGE, "scale must be finite");
    return done(kv8_attend(c, q, (long long)row_stride, heads, r, picks, top, scale, y, static_cast<cudaStream_t>(stream)), msg, msg_cap);
}

extern "C" int strata_kv8_call_dev(const strata_kv8_call *a) {
    if (!a) return STRATA_ERR_RANGE;
    switch (a->op) {
    case STRATA_KV8_APPEND:
        return strata_kv8_append_dev(a->cache, a->rows, a->v, a->row_stride, a->segments, a->count, a->sequence, a->start, a->stream, a->msg,
                                     a->msg_cap);
    case STRATA_KV8_SELECT:
        return strata_kv8_select_dev(a->cache, a->rows, a->row_stride, a->heads, a->segments, a->count, a->sequence, a->start, a->top, a->first,
                                     a->last, a->picks, a->stream, a->msg, a->msg_cap);
    case STRATA_KV8_ATTEND:
        return strata_kv8_attend_dev(a->cache, a->rows, a->row_stride, a->heads, a->segments, a->count, a->sequence, a->start, a->picks, a->top,
                                     a->scale, a->y, a->stream, a->msg, a->msg_cap);
    }
    return say(a->msg, a->msg_cap, STRATA_ERR_RANGE, "op must be STRATA_KV8_APPEND, _SELECT or _ATTEND");
}
