// The gated delta rule over runs (strata_delta_rule): which form a call takes, and the slabs of the chunked one.
#include "../../include/strata_cuda.h"
#include "delta_chunk.cuh"

#include <algorithm>

namespace strata {
namespace {

constexpr int kSms = 148;

// Rows of a run up to which it is taken token by token. A call in chunks takes 31 us however short its runs are (24 us with heads
// of 64), token by token 0.75 us a row, and with more state than the multiprocessors walk at once as much longer as chunks get. 32 heads of
// 128, in chunks and token by token: one session of 34 rows 31 and 26 us, of 44 31 and 34; two of 36 31 and 32; four of 21 33 and 27, of 28 33
// and 35; 16 of 21 76 and 71, of 24 76 and 81; 8 heads of 64: one of 40 24 and 22 us, of 48 24 and 25; 64 of 40 50 and 41, of 56 51 and 57.
int short_run(const DeltaNet &n, const MixRuns &r) {
    if (n.dim <= 64) return 44;
    return (long long)r.segments * n.value_heads <= kSms / 2 ? 34 : 21;
}

// States up to which runs are taken in parts: with N of them, (148 / N + 3) / 2 parts fill the multiprocessors (of a part but the last
// its end and, but for the first, its transition; then all parts once more, from the states that these give). As one and in parts: one prompt of
// 8191 tokens over 2 heads of 128 444 and 135 us, over 16 505 and 347, over 24 536 and 518; of 2048 over 8 of 64 114 and 63 us, over 24 of 128 160
// and 148. Over 32 three parts are left: 2048 tokens 164 and 167 us, 8191 562 and 661.
constexpr int kSplitStates = 24;

// Parts of a run's chunks, by tenths of microseconds: 3.7 us a chunk as one, 7.1 us a part's chunk twice, 1.5 us to join a part and 15 us
// of two more kernels. (1000 tokens over 4 heads of 128: 80 us as one, 66 in 8 parts; 640 over 8: 60 and 58 us.)
int parts_of(int chunks, int most) {
    int best = 1, least = chunks * 37;
    for (int k = 3; k <= std::min(most, chunks); ++k) {
        const int time = (chunks + k - 1) / k * 71 + k * 15 + 150;
        if (time < least) best = k, least = time;
    }
    return best;
}

// Each block of a run looks for its sequence among the runs before it: segments^2 / 2 numbers for each block of a run. Where twice that is
// past this, a list without sequences that are outside or there twice is made once, at the workspace's end. Single tokens over 32 heads of
// 128, with a look and with the list: 512 runs 409 and 395 us, 1024 821 and 779 us, 8192 7.2 and 6.2 ms; over 4 of 64: 4096 135 and 123 us, 65535 6.3 and
// 1.9 ms. (delta_inputs has no workspace and fewer blocks a run: there
// 65535 runs of 512 channels take 1.0 ms where the look is half of it, 8192 of 8192 channels 0.70 ms where it does not show.)
constexpr double kScanned = 3e7;
constexpr int kListRuns = 65536, kListThreads = 256;
struct RunList {
    int *list, *key, *first;  // the list; a table of sequences, open addressing: the number, and the first run that has it
    int bits;                 // of the table's size, twice the runs at least
};
constexpr long long kListBytes = (1 + 2 + 2) * kListRuns * (long long)sizeof(int);

__global__ void __launch_bounds__(kListThreads) k_list_clear(RunList l) {
    kv8_enter();
    const int i = blockIdx.x * kListThreads + threadIdx.x;
    if (i < 1 << l.bits) l.key[i] = -1, l.first[i] = kListRuns;
}
// A run's place in the table; the order in which runs come does not matter to `first`.
__global__ void __launch_bounds__(kListThreads) k_list_enter(const __grid_constant__ MixRuns r, RunList l, int sequences, unsigned *err) {
    kv8_enter();
    const int i = blockIdx.x * kListThreads + threadIdx.x;
    if (i >= r.segments) return;
    const int mine = r.sequence[i];
    int at = -1;
    if (mine < -1 || mine >= sequences) {
        raise_error(err, kErrIndex);
    } else if (mine >= 0) {
        at = (int)((unsigned)mine * 2654435761u >> (32 - l.bits));
        for (;;) {  // (half of the places stay free)
            const int other = atomicCAS(&l.key[at], -1, mine);
            if (other == -1 || other == mine) break;
            at = (at + 1) & ((1 << l.bits) - 1);
        }
        atomicMin(&l.first[at], i);
    }
    l.list[i] = at;
}
__global__ void __launch_bounds__(kListThreads) k_list_once(const __grid_constant__ MixRuns r, RunList l, unsigned *err) {
    kv8_enter();
    const int i = blockIdx.x * kListThreads + threadIdx.x;
    if (i >= r.segments) return;
    const int at = l.list[i];
    const bool twice = at >= 0 && l.first[at] < i;
    if (twice) raise_error(err, kErrIndex);
    l.list[i] = at < 0 || twice ? -1 : r.sequence[i];
}
cudaError_t list_runs(const MixRuns &r, const RunList &l, const DeltaNet &n, cudaStream_t s) {
    const auto grid = [](int items) { return dim3((unsigned)((items + kListThreads - 1) / kListThreads)); };
    cudaError_t e = kv8_launch(k_list_clear, grid(1 << l.bits), dim3(kListThreads), 0, 1, s, l);
    if (e == cudaSuccess) e = kv8_launch(k_list_enter, grid(r.segments), dim3(kListThreads), 0, 1, s, r, l, n.sequences, n.err);
    return e == cudaSuccess ? kv8_launch(k_list_once, grid(r.segments), dim3(kListThreads), 0, 1, s, r, l, n.err) : e;
}

}  // namespace

cudaError_t delta_rule(const DeltaNet &n, const DeltaRule &a, const MixRuns &given, cudaStream_t s) {
    const int ratio = n.value_heads / n.key_heads;
    const long long bytes = n.dim <= 64 ? DeltaSlot<64>::bytes(ratio) : DeltaSlot<128>::bytes(ratio);
    MixRuns r = given;
    long long space = STRATA_DELTA_WORKSPACE_BYTES;
    if ((double)r.segments * r.segments * n.value_heads * ((n.dim + 31) / 32) > kScanned) {
        space -= kListBytes;
        int *const at = reinterpret_cast<int *>(static_cast<unsigned char *>(n.workspace) + space);
        RunList l{at, at + kListRuns, at + 3 * kListRuns, 1};
        while (1 << l.bits < 2 * r.segments) ++l.bits;
        const cudaError_t e = list_runs(given, l, n, s);
        if (e != cudaSuccess) return e;
        r.sequence = l.list, r.once = true;
    }
    const int room = (int)(space / bytes);  // slots
    if (n.dim > 128 || r.count <= short_run(n, r) || room < 1) return delta_step(n, a, r, s);
    const bool vec = n.dim % 4 == 0 && a.q_stride % 4 == 0 && a.k_stride % 4 == 0 && a.v_stride % 4 == 0 && mix_aligned16(a.q) &&
                     mix_aligned16(a.k) && mix_aligned16(a.v);
    const int all = (r.count + kChunk - 1) / kChunk;
    DeltaSlab slab{0, 0, 0, 0, 0, 0, ratio, 0, 0, static_cast<unsigned char *>(n.workspace), bytes, 1, 0, nullptr, nullptr};
    const auto one = [&] {
        cudaError_t e = delta_prepare(n, a, r, slab, vec, s);
        if (slab.parts > 1) {
            if (e == cudaSuccess) e = delta_ends(n, a, r, slab, s);
            if (e == cudaSuccess) e = delta_join(n, r, slab, s);
        }
        return e == cudaSuccess ? delta_chain(n, a, r, slab, s) : e;
    };
    const int D = n.dim <= 64 ? 64 : 128;
    if ((long long)r.segments * n.value_heads <= kSplitStates) {
        const int states = r.segments * n.value_heads, per = r.segments * n.key_heads, most = (kSms / states + 3) / 2;
        const long long state = 2ll * D * D * sizeof(float) * states, behind = STRATA_DELTA_WORKSPACE_BYTES - state * (most - 1) - 1024;
        const int chunks = std::min<long long>(all, behind / (bytes * per));
        if (chunks > 0 && parts_of(chunks, most) > 1) {
            slab.runs = r.segments, slab.heads = n.key_heads;
            for (; slab.chunk0 < all; slab.chunk0 += slab.chunks) {
                slab.chunks = std::min(chunks, all - slab.chunk0);
                const int parts = parts_of(slab.chunks, most);
                slab.part_chunks = (slab.chunks + parts - 1) / parts;
                slab.parts = (slab.chunks + slab.part_chunks - 1) / slab.part_chunks;
                slab.states = reinterpret_cast<float *>(slab.slots + slab.chunks * per * bytes);
                slab.whole = reinterpret_cast<int *>(slab.states + state / sizeof(float) * (slab.parts - 1));
                const cudaError_t e = one();
                if (e != cudaSuccess) return e;
            }
            return cudaSuccess;
        }
    }
    // Few states leave most multiprocessors idle in the second kernel: there the next slab's first one runs meanwhile, on the
    // workspace's other half. The first slab gives each multiprocessor two blocks, the next ones those that are left. One after another and
    // side by side: one prompt of 2048 tokens over 32 heads of 128 177 and 164 us, of 8191 over 48 876 and 606, two of 1024 over 32 129 and 121;
    // three 179 and 218: with more states than half of the multiprocessors one slab after another.
    if ((long long)r.segments * n.value_heads <= kSms / 2) {
        const int chains = r.segments * n.value_heads, per = r.segments * n.key_heads, most = room / 2 / per;  // chunks of a half
        const int first = std::min(most, 2 * kSms / per), next = std::min(most, std::max(1, 2 * (kSms - chains) / per));
        if (most > 0 && first < all) {
            slab.runs = r.segments, slab.heads = n.key_heads, slab.chunks = first;
            while (slab.chunk0 < all) {
                const cudaError_t e = one();
                if (e != cudaSuccess) return e;
                slab.chunk0 += slab.chunks, slab.chunks = std::min(next, all - slab.chunk0);
                slab.slots = static_cast<unsigned char *>(n.workspace) + (slab.slots == n.workspace ? room / 2 * bytes : 0);
                slab.ahead = 1;
            }
            return cudaSuccess;
        }
    }
    // Of somewhat more states than multiprocessors those of long runs go first, so that none of them begins when others end (24 runs of
    // up to 531 tokens, 8 heads of 64: 88 us without, 80 with it; with two states or more for each multiprocessor it gains nothing and costs 2%).
    // Whole runs where they fit; else as many runs as give each multiprocessor two value heads, and their chunks in turn.
    const int heads = std::min(n.key_heads, room);
    int runs = std::max(1, std::min({r.segments, room / heads, (2 * kSms + heads * ratio - 1) / (heads * ratio)}));
    const int chunks = std::min(all, room / (runs * heads));
    if (chunks == all) runs = std::min(r.segments, room / (heads * chunks));
    for (int run0 = 0; run0 < r.segments; run0 += runs)
        for (int head0 = 0; head0 < n.key_heads; head0 += heads)
            for (int chunk0 = 0; chunk0 < all; chunk0 += chunks) {
                slab.run0 = run0, slab.runs = std::min(runs, r.segments - run0);
                slab.head0 = head0, slab.heads = std::min(heads, n.key_heads - head0);
                slab.chunk0 = chunk0, slab.chunks = std::min(chunks, all - chunk0);
                const int states = slab.runs * slab.heads * ratio;
                slab.sorted = r.lengths && slab.runs <= kSortedRuns && states > kSms && states < 2 * kSms;
                const cudaError_t e = one();
                if (e != cudaSuccess) return e;
            }
    return cudaSuccess;
}

}  // namespace strata
