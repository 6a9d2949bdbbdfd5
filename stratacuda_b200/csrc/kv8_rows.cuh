// What the two token-by-token attention kernels share: arguments, page lists, and the parts that a split call leaves in
// the workspace with the kernel that joins them.
#pragma once
#include "kv8.cuh"

#include <cmath>

namespace strata {
namespace kv8_rows {

constexpr int kJoinThreads = 256;
constexpr int kRows = 16;         // query heads of a unit, at most
constexpr int kMaxTokens = 1024;  // tokens of a split call (their page counts are summed up in shared memory)
constexpr int kMaxCtas = 640;     // CTAs of a split call: two partial results each in the workspace

// Workspace of a split call: page counts are not kept, only what the joining kernel reads.
struct Parts {
    float *acc;   // [2 * CTAs][16][P]
    float2 *ml;   // [2 * CTAs][16] maximum (log2 units), sum
    int2 *cover;  // [units] first and last CTA, and the first one's slot
};
__host__ __device__ inline Parts parts_of(void *ws, int P) {
    char *p = static_cast<char *>(ws);
    Parts r;
    r.acc = reinterpret_cast<float *>(p);
    p += (size_t)2 * kMaxCtas * kRows * P * 4;
    r.ml = reinterpret_cast<float2 *>(p);
    p += (size_t)2 * kMaxCtas * kRows * 8;
    r.cover = reinterpret_cast<int2 *>(p);
    return r;
}

struct Args {
    Kv8 c;
    const float *q;
    long long stride;
    int heads, group, tiles;  // query heads a key/value head, 16-row tiles a group
    Kv8Runs runs;
    const int *picks;
    int top;
    float scale;  // times log2 e
    float *y;
    int split;
};

// Entries of a token's page list: every block in sight, or its picks.
__device__ __forceinline__ int entries(const Args &A, int token, int *sequence, int *seen) {
    const RunAt at = run_at(A.c, A.runs, token / A.runs.count);
    *sequence = at.sequence;
    *seen = visible_keys(A.c, at, token % A.runs.count);
    const int nb = (*seen + kKvBlock - 1) / kKvBlock;
    return A.picks && nb ? A.top : nb;
}

// Joins the partial results of a unit's rows: out = sum_i 2^(m_i - max) acc_i / sum_i 2^(m_i - max) l_i. DEEP parts
// are read at a time by as many groups of threads, and the other threads of the block take further rows.
template <int P, int DEEP>
__global__ static void __launch_bounds__(kJoinThreads) k_kv8_join(const __grid_constant__ Args A) {
    constexpr int kAcross = P / 4, kRowsHere = kJoinThreads / kAcross / DEEP;
    __shared__ float4 acc_s[kJoinThreads];
    __shared__ float sum_s[kJoinThreads];
    const int tid = threadIdx.x, per_token = A.c.kv_heads * A.tiles, unit = blockIdx.x;
    const int at = tid % kAcross, deep = tid / kAcross % DEEP, row = blockIdx.y * kRowsHere + tid / kAcross / DEEP;
    const int token = unit / per_token, sub = unit % per_token, head = sub / A.tiles, row0 = sub % A.tiles * kRows;
    const bool there = row < min(kRows, A.group - row0);
    int sequence, seen;
    kv8_enter();
    const int n = entries(A, token, &sequence, &seen);
    float *dst = A.y + ((size_t)token * A.heads + head * A.group + row0 + row) * A.c.dim;
    if (n == 0) {  // nothing in sight: no CTA had this unit
        for (int i = at; there && deep == 0 && i < A.c.dim; i += kAcross) dst[i] = 0.0f;
        return;
    }
    const Parts W = parts_of(A.c.workspace, P);
    const int2 cover = W.cover[unit];
    const int count = cover.y - cover.x + 1;
    if (count <= 1) return;
    // the unit begins in its first CTA's second slot and goes on in the first slots of the others
    auto slot = [&](int i) { return (size_t)2 * (cover.x + i) + (i == 0); };
    float m = -INFINITY, sum = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (there) {
#pragma unroll 8
        for (int i = 0; i < count; ++i) m = fmaxf(m, W.ml[slot(i) * kRows + row].x);
        if (m == -INFINITY) m = 0.0f;
#pragma unroll 8
        for (int i = deep; i < count; i += DEEP) {
            const float2 ml = W.ml[slot(i) * kRows + row];
            const float4 f = *reinterpret_cast<const float4 *>(W.acc + (slot(i) * kRows + row) * P + at * 4);
            const float w = exp2_fast(ml.x - m);
            sum += w * ml.y;
            acc.x += w * f.x, acc.y += w * f.y, acc.z += w * f.z, acc.w += w * f.w;
        }
    }
    if (DEEP > 1) {
        acc_s[tid] = acc;
        sum_s[tid] = sum;
        __syncthreads();
        if (deep) return;
#pragma unroll
        for (int i = 1; i < DEEP; ++i) {
            const float4 f = acc_s[tid + i * kAcross];
            acc.x += f.x, acc.y += f.y, acc.z += f.z, acc.w += f.w;
            sum += sum_s[tid + i * kAcross];
        }
    }
    if (!there) return;
    const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum), v[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at * 4 + i < A.c.dim) dst[at * 4 + i] = v[i];
}

// few units have many parts each, which a block's threads share; many units have few
template <int P>
cudaError_t launch_join(const Args &A, long long units, int multiprocessors, cudaStream_t s) {
    static_assert((size_t)2 * kMaxCtas * kRows * (256 * 4 + 8) + 65536 * 8 <= (32u << 20), "the workspace holds every partial result");
    constexpr int kSpread = kJoinThreads / (P / 4);
    const int rows = A.group < kRows ? A.group : kRows;
    const bool deep = units * rows < 2LL * multiprocessors;
    return kv8_launch(deep ? k_kv8_join<P, kSpread> : k_kv8_join<P, 1>, dim3((unsigned)units, deep ? rows : (rows + kSpread - 1) / kSpread),
                      dim3(kJoinThreads), 0, 1, s, A);
}

}  // namespace kv8_rows

// csrc/kv8_short.cu: the form for calls of few pages a CTA; whether this call is one.
bool kv8_short_fits(const kv8_rows::Args &A, int multiprocessors);
cudaError_t kv8_attend_short(kv8_rows::Args A, int multiprocessors, cudaStream_t s);

}  // namespace strata
