// The gated delta rule over runs (strata_delta_rule): which form a call takes, and the slabs of the chunked one.
#include "../../include/strata_cuda.h"
#include "delta_chunk.cuh"

#include <algorithm>

namespace strata {
namespace {

// Rows of a run up to which it is taken token by token. A call in chunks takes 35 us however short its runs are (25 us with heads
// of 64), token by token 0.7 us a row, and with more state than the multiprocessors walk at once as much longer as chunks get:
// 16 sessions of 32 heads of 128 92 us in chunks, 106 us token by token at 32 rows; 64 of 8 heads of 64 57 us, 34 us at 32 rows.
int short_run(const DeltaNet &n, const MixRuns &r) {
    if (n.dim <= 64) return 48;
    return (long long)r.segments * n.value_heads <= 148 / 2 ? 44 : 28;
}

}  // namespace

cudaError_t delta_rule(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, cudaStream_t s) {
    const int ratio = n.value_heads / n.key_heads;
    const long long bytes = n.dim <= 64 ? DeltaSlot<64>::bytes(ratio) : DeltaSlot<128>::bytes(ratio);
    const int room = (int)((long long)STRATA_DELTA_WORKSPACE_BYTES / bytes);  // slots
    if (n.dim > 128 || r.count <= short_run(n, r) || room < 1) return delta_step(n, a, r, s);
    const bool vec = n.dim % 4 == 0 && a.q_stride % 4 == 0 && a.k_stride % 4 == 0 && a.v_stride % 4 == 0 && mix_aligned16(a.q) &&
                     mix_aligned16(a.k) && mix_aligned16(a.v);
    // Whole runs where they fit; else as many runs as give each multiprocessor two value heads, and their chunks in turn.
    const int all = (r.count + kChunk - 1) / kChunk, heads = std::min(n.key_heads, room);
    int runs = std::max(1, std::min({r.segments, room / heads, (2 * 148 + heads * ratio - 1) / (heads * ratio)}));
    const int chunks = std::min(all, room / (runs * heads));
    if (chunks == all) runs = std::min(r.segments, room / (heads * chunks));
    for (int run0 = 0; run0 < r.segments; run0 += runs)
        for (int head0 = 0; head0 < n.key_heads; head0 += heads)
            for (int chunk0 = 0; chunk0 < all; chunk0 += chunks) {
                const DeltaSlab slab{run0, std::min(runs, r.segments - run0), head0, std::min(heads, n.key_heads - head0), chunk0,
                                     std::min(chunks, all - chunk0), ratio, static_cast<unsigned char *>(n.workspace), bytes};
                cudaError_t e = delta_prepare(n, a, r, slab, vec, s);
                if (e == cudaSuccess) e = delta_chain(n, a, r, slab, s);
                if (e != cudaSuccess) return e;
            }
    return cudaSuccess;
}

}  // namespace strata
