// Choosing the blocks that a query attends to (strata_kv8_select).
//
// A block's score for a token and key/value head is an integer product: the group's queries as two rows
// of 8-bit codes (negative and positive parts) with the block's two rows of marks, 2 P terms, times the
// block's key scale: the upper bound that the marks give on the group's summed logits, but for the rounding of the codes
// ("bound" below). Products and sums are whole numbers, so any order gives the same score, and the choice repeats exactly.
//   * 16 tokens of a run (two such tiles a CTA) are the rows of an integer tensor-core tile (mma.sync m16n8k32) against 8 blocks a
//     step, whose marks come from global memory in fragment order: 16 consecutive bytes are a lane's operands
//     of two k-steps. One token alone pays for the tile but not for memory: each block's marks are read once.
//   * the bounds, as words that order like the numbers, stay in shared memory; the words' range is halved
//     until exactly `top` of them lie above, which takes a dozen steps instead of 32 when few are equal.
//   * few tokens: a cluster of up to 8 CTAs shares a token's blocks and sends the bounds to its first CTA.
// Measured at 24 heads over 2 of 256 channels: 32 of 1024 blocks for 2048 tokens 47 us (90 T operations/s), bound by the search
// among a token's bounds and by loading marks in fragment order; for 16 sessions 14 us, bound by latency.
#include "../../include/strata_cuda.h"
#include "kv8.cuh"

#include <atomic>
#include <cooperative_groups.h>

namespace strata {
namespace {

namespace cg = cooperative_groups;

constexpr int kTile = 16;       // tokens of a tensor-core tile
constexpr int kTileRows = 32;   // of a CTA: two tiles, whose warps read the same marks soon after one another (L1)
constexpr int kCandidates = 256;
template <bool WIDE>
struct Shape {
    static constexpr int threads = WIDE ? 256 : 512, warps = threads / 32, rows = WIDE ? kTile : kTileRows;
};
constexpr unsigned kForced = 0xffffffffu;

struct Args {
    Kv8 c;
    const float *q;
    long long stride;
    int heads, group;
    Kv8Runs runs;
    int top, first, last;
    int *picks;
    int rows;     // tokens of a CTA (of a cluster), 1 .. 32
    int tiles;    // CTAs (clusters) a run
    int row_len;  // words between the rows of bounds in shared memory
};

// A float's bits in an order that compares as unsigned words; 0 is below every number.
__device__ __forceinline__ unsigned ordered(float f) {
    const unsigned u = __float_as_uint(f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float finite_or_zero(float f) { return isfinite(f) ? f : 0.0f; }
__device__ __forceinline__ void mma_s8(int (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The largest of x over the warps that share a row: the whole block, or this warp.
template <bool WIDE>
__device__ __forceinline__ float row_max(float x, float *red) {
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, s));
    if (!WIDE) return x;
    __syncthreads();
    if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = x;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < Shape<true>::warps; ++i) x = fmaxf(x, red[i]);
    return x;
}

// WIDE: one token a CTA (cluster), all warps on it. Otherwise up to 32 tokens of a run, a warp to a token.
template <int P, bool WIDE>
__global__ void __launch_bounds__(Shape<WIDE>::threads, WIDE ? 2 : 1) k_kv8_select(const __grid_constant__ Args A) {
    constexpr int kThreads = Shape<WIDE>::threads, kWarps = Shape<WIDE>::warps, kRows = Shape<WIDE>::rows;
    extern __shared__ __align__(16) unsigned key_s[];  // [rows][row_len]
    __shared__ __align__(16) int8_t code_s[kRows][2 * P + 16];  // negative parts, positive parts
    __shared__ float red[kWarps];
    __shared__ int count_s[2][kWarps], equal_s[kWarps], have_s[kRows];
    __shared__ unsigned short block_s[WIDE ? 1 : kWarps][kCandidates];
    kv8_enter();
    const cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    // bounds go to the first CTA's shared memory, which is there once that CTA has begun: every CTA says so here, and
    // waits for the others before its first store, with the queries' rounding between
    if (ranks > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int unit = blockIdx.x / ranks, head = unit % A.c.kv_heads, tile = unit / A.c.kv_heads % A.tiles, run = unit / A.c.kv_heads / A.tiles;
    const RunAt at = run_at(A.c, A.runs, run);
    const int j0 = tile * A.rows, rows = min(A.rows, A.runs.count - j0);
    const long long token0 = (long long)run * A.runs.count + j0;
    if (tid < rows) have_s[tid] = (visible_keys(A.c, at, j0 + tid) + kKvBlock - 1) / kKvBlock;

    // the group's queries of each row as two rows of codes
    constexpr int kEach = WIDE ? (P + kThreads - 1) / kThreads : P / 32;  // neighbouring channels of a thread
    constexpr int kHeads = WIDE ? 16 : 4;                                 // heads whose loads are in flight at a time
    const int me = WIDE ? tid : lane, step = WIDE ? kThreads : 32, ch0 = me * kEach;
    for (int r = WIDE ? 0 : warp; r < (WIDE ? 1 : kRows); r += kWarps) {
        int pos[kEach] = {}, neg[kEach] = {};
        if (r < rows) {
            const float *x = A.q + (token0 + r) * A.stride + (size_t)head * A.group * A.c.dim + ch0;
            const bool wide = kEach % 4 == 0 && ch0 + kEach <= A.c.dim && A.c.dim % 4 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
            auto load = [&](int h0, float(&f)[kHeads][kEach]) {
#pragma unroll
                for (int h = 0; h < kHeads; ++h) {
                    const float *src = x + (size_t)(h0 + h) * A.c.dim;
                    if (wide) {
#pragma unroll
                        for (int i = 0; i < kEach / 4; ++i) {
                            const float4 v = h0 + h < A.group ? reinterpret_cast<const float4 *>(src)[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            f[h][4 * i] = v.x, f[h][4 * i + 1] = v.y, f[h][4 * i + 2] = v.z, f[h][4 * i + 3] = v.w;
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < kEach; ++i) f[h][i] = h0 + h < A.group && ch0 + i < A.c.dim ? src[i] : 0.0f;
                    }
                }
            };
            float amax = 0.0f;
            for (int h0 = 0; h0 < A.group; h0 += kHeads) {
                float f[kHeads][kEach];
                load(h0, f);
#pragma unroll
                for (int h = 0; h < kHeads; ++h)
#pragma unroll
                    for (int i = 0; i < kEach; ++i) amax = fmaxf(amax, fabsf(finite_or_zero(f[h][i])));
            }
            amax = row_max<WIDE>(amax, red);
            const float unit_of = amax < 0x1p-100f ? 0.0f : __fdiv_rn(32767.0f, amax);
            for (int h0 = 0; h0 < A.group; h0 += kHeads) {
                float f[kHeads][kEach];
                load(h0, f);
#pragma unroll
                for (int h = 0; h < kHeads; ++h)
#pragma unroll
                    for (int i = 0; i < kEach; ++i) {
                        const int v = __float2int_rn(__fmul_rn(finite_or_zero(f[h][i]), unit_of));
                        pos[i] += max(v, 0);
                        neg[i] += min(v, 0);
                    }
            }
            float big = 0.0f;
#pragma unroll
            for (int i = 0; i < kEach; ++i) big = fmaxf(big, (float)max(pos[i], -neg[i]));
            big = row_max<WIDE>(big, red);
            const float fine = big > 0.0f ? __fdiv_rn(127.0f, big) : 0.0f;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                pos[i] = __float2int_rn(__fmul_rn((float)pos[i], fine));
                neg[i] = __float2int_rn(__fmul_rn((float)neg[i], fine));
            }
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (ch0 + i < P) {
                code_s[r][ch0 + i] = (int8_t)neg[i];
                code_s[r][P + ch0 + i] = (int8_t)pos[i];
            }
    }
    if (WIDE)  // the tile's other rows
        for (int i = tid; i < (kTile - 1) * (2 * P + 16) / 4; i += kThreads) reinterpret_cast<int *>(code_s[1])[i] = 0;
    __syncthreads();
    const int most = have_s[rows - 1];
    const int r0 = WIDE ? 0 : warp / 8 * kTile;  // this warp's tile of rows
    if (ranks > 1) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    if (most > A.top && r0 < rows) {
        unsigned a[P / 32][2][4];  // 64-byte segments of the code rows, two k-steps each
#pragma unroll
        for (int i = 0; i < P / 32; ++i) {
            const uint4 lo = *reinterpret_cast<const uint4 *>(&code_s[r0 + g][i * 64 + t * 16]);
            const uint4 hi = *reinterpret_cast<const uint4 *>(&code_s[r0 + g + 8][i * 64 + t * 16]);
            a[i][0][0] = lo.x, a[i][0][2] = lo.y, a[i][1][0] = lo.z, a[i][1][2] = lo.w;
            a[i][0][1] = hi.x, a[i][0][3] = hi.y, a[i][1][1] = hi.z, a[i][1][3] = hi.w;
        }
        unsigned *keys = cluster.map_shared_rank(key_s, 0);
        const int *table = A.c.table + (size_t)at.sequence * A.c.blocks;
        const int stride_b = 64 * ranks;
        int b0 = (rank * 8 + warp % 8) * 8;
        int entry = b0 + g < most ? table[b0 + g] : -1;
        for (; b0 < most; b0 += stride_b) {
            const int b = b0 + g;
            int page = entry;
            if (b < most && (page < 0 || page >= A.c.pages)) {
                raise_error(A.c.err, kErrIndex);
                page = -1;
            }
            entry = b + stride_b < most ? table[b + stride_b] : -1;
            uint4 m[P / 32];
            float scale = 0.0f;
            if (page >= 0) {
                const uint4 *src = reinterpret_cast<const uint4 *>(page_marks(A.c, page, head)) + t;
#pragma unroll
                for (int i = 0; i < P / 32; ++i) m[i] = src[i * 4];
                scale = page_scales(A.c, page, head)[0];
            } else {
#pragma unroll
                for (int i = 0; i < P / 32; ++i) m[i] = make_uint4(0, 0, 0, 0);
            }
            int d[4] = {0, 0, 0, 0}, d1[4] = {0, 0, 0, 0};  // two chains, so that one product need not wait for the last
#pragma unroll
            for (int i = 0; i < P / 32; ++i) {
                mma_s8(d, a[i][0][0], a[i][0][1], a[i][0][2], a[i][0][3], m[i].x, m[i].y);
                mma_s8(d1, a[i][1][0], a[i][1][1], a[i][1][2], a[i][1][3], m[i].z, m[i].w);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] += d1[e];
            const float s0 = __shfl_sync(0xffffffffu, scale, 8 * t), s1 = __shfl_sync(0xffffffffu, scale, 8 * t + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = r0 + g + (e >> 1) * 8, block = b0 + 2 * t + (e & 1);
                if (r >= rows || block >= most) continue;
                const int have = have_s[r];
                unsigned key = min(ordered(__fmul_rn((float)d[e], e & 1 ? s1 : s0)), kForced - 1);
                if (block < A.first || block >= have - A.last) key = kForced;
                if (block >= have) key = 0;
                keys[r * A.row_len + block] = key;
            }
        }
    }
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    if (rank) return;

    for (int r = WIDE ? 0 : warp; r < rows; r += kWarps) {
        const int have = have_s[r];
        int *out = A.picks + ((size_t)(token0 + r) * A.c.kv_heads + head) * A.top;
        if (have <= A.top) {
            for (int i = me; i < A.top; i += step) out[i] = i < have ? i : -1;
            continue;
        }
        unsigned *key = key_s + r * A.row_len;
        // this warp's blocks: all, or an eighth in whole groups of 128
        const int share = WIDE ? (have + 128 * kWarps - 1) / (128 * kWarps) * 128 : have;
        const int from = WIDE ? min(have, warp * share) : 0, to = WIDE ? min(have, from + share) : have;
        auto row_sum = [&](int n, int which) {  // over the warps on this row; two places, so one barrier a call is enough
            n = __reduce_add_sync(0xffffffffu, n);
            if (!WIDE) return n;
            if (lane == 0) count_s[which][warp] = n;
            __syncthreads();
            n = 0;
#pragma unroll
            for (int i = 0; i < kWarps; ++i) n += count_s[which][i];
            return n;
        };
        // words in a few registers where they fit
        constexpr int kHold = 8;
        unsigned held[kHold];
        unsigned lo = kForced, hi = 0, first_max = 0, second_max = 0;
        int forced = 0;
        for (int b = from + lane; b < to; b += 32) {
            const unsigned k = key[b];
            forced += k == kForced;
            if (k != kForced) {
                lo = min(lo, k);
                hi = max(hi, k);
            }
            second_max = max(second_max, min(first_max, k));
            first_max = max(first_max, k);
        }
        lo = __reduce_min_sync(0xffffffffu, lo);
        hi = __reduce_max_sync(0xffffffffu, hi);
        int n_words = to - from;
        unsigned *words = key + from;
        bool compact = false;
        if (WIDE) {
            if (lane == 0) {
                count_s[1][warp] = (int)lo;
                equal_s[warp] = (int)hi;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kWarps; ++i) {
                lo = min(lo, (unsigned)count_s[1][i]);
                hi = max(hi, (unsigned)equal_s[i]);
            }
        } else if (A.top <= 64) {
            // 32 (64) words at least reach the least of the lanes' largest (second largest): only those that do are
            // candidates, and are moved to the front in their order, with their blocks
            const unsigned least = __reduce_min_sync(0xffffffffu, A.top <= 32 ? first_max : second_max);
            if (least > lo) {
                int n = 0;
                for (int b = lane; b < have; b += 32) n += key[b] >= least;
                n = __reduce_add_sync(0xffffffffu, n);
                if (n <= kCandidates && n > A.top) {
                    compact = true;
                    lo = least == kForced ? lo : least;
                    int at = 0;
                    for (int b = 0; b < have; b += 128) {
                        unsigned k[4], ballot[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) k[i] = b + 32 * i + lane < have ? key[b + 32 * i + lane] : 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) ballot[i] = __ballot_sync(0xffffffffu, k[i] >= least);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (k[i] >= least) {
                                const int to_at = at + __popc(ballot[i] & ((1u << lane) - 1));
                                key[to_at] = k[i];
                                block_s[warp][to_at] = (unsigned short)(b + 32 * i + lane);
                            }
                            at += __popc(ballot[i]);
                        }
                        __syncwarp();
                    }
                    n_words = n;
                }
            }
        }
        const bool hold = n_words <= 32 * kHold;  // (of every warp on the row: they share alike)
        if (hold) {
#pragma unroll
            for (int i = 0; i < kHold; ++i) held[i] = i * 32 + lane < n_words ? words[i * 32 + lane] : 0;
        }
        // at least `top` words reach lo, `above` <= top reach hi; halve until as many as wanted do, or equal words
        // (lo, all of them) are left to fill up with
        int above = row_sum(forced, 0), turn = 1;
        hi += 1;
        while (above != A.top && hi - lo > 1) {
            const unsigned mid = lo + (hi - lo) / 2;
            int n = 0;
            if (hold) {
#pragma unroll
                for (int i = 0; i < kHold; ++i) n += held[i] >= mid;
            } else {
                for (int b = 4 * lane; b < n_words; b += 128) {
                    const uint4 k = *reinterpret_cast<const uint4 *>(words + b);
                    n += (k.x >= mid) + (b + 1 < n_words && k.y >= mid) + (b + 2 < n_words && k.z >= mid) + (b + 3 < n_words && k.w >= mid);
                }
            }
            n = row_sum(n, turn);
            turn ^= 1;
            if (n >= A.top && n != A.top) {
                lo = mid;
            } else {
                hi = mid;
                above = n;
            }
        }
        int room = A.top - above, at_out = 0;
        if (WIDE) {  // where this warp's picks begin, and how many equal ones earlier warps take
            int up = 0, eq = 0;
            for (int b = from + lane; b < to; b += 32) {
                up += key[b] >= hi;
                eq += key[b] == lo && key[b] < hi;
            }
            up = __reduce_add_sync(0xffffffffu, up);
            eq = __reduce_add_sync(0xffffffffu, eq);
            __syncthreads();
            if (lane == 0) {
                count_s[0][warp] = up;
                equal_s[warp] = eq;
            }
            __syncthreads();
            for (int i = 0; i < warp; ++i) {
                const int take = min(room, equal_s[i]);
                at_out += count_s[0][i] + take;
                room -= take;
            }
        }
        for (int b = 0; b < n_words; b += 32) {
            const unsigned k = b + lane < n_words ? words[b + lane] : 0;
            const bool up = k >= hi, eq = !up && k == lo && b + lane < n_words;
            const unsigned equals = __ballot_sync(0xffffffffu, eq);
            const bool take = up || (eq && __popc(equals & ((1u << lane) - 1)) < room);
            const unsigned all = __ballot_sync(0xffffffffu, take);
            if (take) out[at_out + __popc(all & ((1u << lane) - 1))] = compact ? block_s[WIDE ? 0 : warp][b + lane] : from + b + lane;
            at_out += __popc(all);
            room -= min(room, __popc(equals));
        }
    }
}

constexpr int kKeyBytes = 184 * 1024;  // of a tile's bounds, beside the codes and candidates
constexpr int kWideBytes = STRATA_KV8_SELECT_BLOCKS * 4;  // of a token's

// The limit on a kernel's shared memory is the function's, whichever thread's call it serves: the largest, once a device.
template <int P, bool WIDE>
cudaError_t allow_shared_memory() {
    constexpr int kDevices = 64;
    static std::atomic<bool> done[kDevices];
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess || (device < kDevices && done[device].load(std::memory_order_relaxed))) return e;
    e = cudaFuncSetAttribute(k_kv8_select<P, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, WIDE ? kWideBytes : kKeyBytes);
    if (e == cudaSuccess && device < kDevices) done[device].store(true, std::memory_order_relaxed);
    return e;
}

template <int P, bool WIDE>
cudaError_t launch(const Args &A, int ranks, size_t smem, cudaStream_t s) {
    cudaError_t e = allow_shared_memory<P, WIDE>();
    if (e != cudaSuccess) return e;
    const long long ctas = (long long)A.runs.segments * A.tiles * A.c.kv_heads * ranks;
    if (ctas > 0x7fffffff) return cudaErrorInvalidConfiguration;
    return kv8_launch(k_kv8_select<P, WIDE>, dim3((unsigned)ctas), dim3(Shape<WIDE>::threads), smem, ranks, s, A);
}

}  // namespace

cudaError_t kv8_select(const Kv8 &c, const float *q, long long stride, int heads, const Kv8Runs &r, int top, int first, int last, int *picks,
                       cudaStream_t s) {
    constexpr int kSms = 148;
    Args A{c, q, stride, heads, heads / c.kv_heads, r, top, first, last, picks, 1, r.count, (c.blocks + 3) / 4 * 4};
    const long long tokens = (long long)r.segments * r.count * c.kv_heads;
    // Tiles of up to 32 tokens where half of the multiprocessors get one: marks are then read once for 16 or 32 tokens
    int rows = kKeyBytes / (A.row_len * 4);
    rows = rows > kTileRows ? kTileRows : rows;
    if (rows > r.count) rows = r.count;
    if (rows > 1 && tokens >= (long long)rows * kSms / 2) {
        A.rows = rows;
        A.tiles = (r.count + rows - 1) / rows;
        const size_t smem = (size_t)rows * A.row_len * 4;
        if (c.padded == 64) return launch<64, false>(A, 1, smem, s);
        if (c.padded == 128) return launch<128, false>(A, 1, smem, s);
        return launch<256, false>(A, 1, smem, s);
    }
    // A token a cluster; as many CTAs in it as leave each 64 blocks and the device two rounds of CTAs at most
    int ranks = 1;
    while (ranks < 8 && tokens * ranks * 2 <= 4 * kSms && c.blocks >= 128 * ranks) ranks *= 2;
    const size_t smem = (size_t)A.row_len * 4;
    if (c.padded == 64) return launch<64, true>(A, ranks, smem, s);
    if (c.padded == 128) return launch<128, true>(A, ranks, smem, s);
    return launch<256, true>(A, ranks, smem, s);
}

}  // namespace strata
