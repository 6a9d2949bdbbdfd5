// Attention over the 8-bit paged cache (strata_kv8_attend): the form that works token by token.
//
// A unit is one token and key/value head with up to 16 of its group's query heads. With so few rows the
// products are turned round: the cache is the 128-row operand of the 5th-generation tensor cores' integer
// products (tcgen05 kind::i8), which take its codes as they lie in memory, and the queries and weights, as whole
// numbers of several 8-bit digits, are the narrow one. No code is ever converted; every product is exact.
//   S^T[128 tokens][3 digits x rows] = K . Q^T    a query row, scaled by a power of two, has 23 bits in three
//       signed digits; a step is two pages
//   O^T[P channels][4 digits x rows] += V^T . W^T  a weight has 28 bits in four unsigned digits; 32-bit sums in
//       TMEM over up to 256 pages
// A thread of the softmax warps has one of the step's tokens (its TMEM lane): it puts the rows' logits together
// from their digits, takes the exponentials, and writes the weights' digits as the second product's operand.
// Logits, maxima and sums of weights are F32. A row's weights refer to a maximum that follows the true one only
// when a weight would pass 8; then, and at the unit's end, the sums move from TMEM to F32 registers.
//
// Warps: 0-3 softmax, sums and results; 4 looks pages up and fetches keys and values by TMA (64-byte swizzle) into
// two rings, ahead across units; 5 issues the products, S of the next step before O of this; 6-7 make the
// next unit's query digits. One CTA a multiprocessor; every wait is bounded, and past the limit all leave.
//
// Few units (`split`): the pages of all units form one list that the CTAs share evenly, whatever the
// lengths; a unit cut by a CTA border leaves unnormalised partial sums in the workspace and a
// second kernel joins them in CTA order, so results repeat bit for bit.
#include "kv8.cuh"
#include "pf_gemm.cuh"

#include <cudaTypedefs.h>

#include <atomic>
#include <cmath>
#include <mutex>

namespace strata {
namespace {

using namespace pf;

constexpr int kSoft = 128, kFetchWarp = 4, kIssueWarp = 5, kQueryWarp = 6, kThreads = 256;
constexpr int kJoinThreads = 256;
constexpr int kRows = 16;
constexpr int kMaxTokens = 1024;  // tokens of a split call (their page counts are summed up in shared memory)
constexpr int kMaxCtas = 640;     // CTAs of a split call: two partial results each in the workspace
constexpr int kFlushSteps = 128;  // steps that TMEM's 32-bit sums bear (255 * 127 * 128 tokens a step)
constexpr float kGrow = 8.0f;     // weights stay below this, times
constexpr float kUnit = 268435456.0f;  // 2^28, below 2^32
constexpr long long kWaitClocks = 2000000000;  // about a second

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

// P stored channels; R rows that the operands have room for, 4 .. 16.
template <int P, int R>
struct Shape {
    static constexpr int panels = P / 64;
    static constexpr int blocks = P <= 128 ? 1 : 2;             // of 128 channels
    static constexpr int ns = (3 * R + 15) / 16 * 16, nw = 4 * R;  // columns of S and O
    static constexpr int k_ring = 3, v_ring = P == 256 ? 5 : 6;  // steps (two pages), pages
};
// What a slot of the key ring holds: 1 or 2 pages, the end of a unit (0), or the end of all (-1).
struct Step {
    int pages, block[2];
    float k_scale[2], v_scale[2];
    int pad;
};
struct Unit {  // or the part of it that this CTA works on: entries [entry, stop) of its n
    int token, sub, entry, stop, n, seen, sequence, last_cta;
};
template <int P, int R>
struct __align__(1024) Smem {
    using Z = Shape<P, R>;
    unsigned char k[Z::k_ring][Z::panels][128 * 64];  // tokens of two pages, 64 channels a row
    unsigned char v[Z::v_ring][P * 64];               // channels, 64 tokens a row
    unsigned char v_end[P == 64 ? 4096 : 1024];       // (a 64-channel page is read as 128 rows)
    unsigned char q[2][Z::panels][Z::ns * 64];        // row 3 r + digit: 64 channels
    unsigned char w[2][2][Z::nw * 64];                // by step parity and page: row 4 r + digit: 64 tokens
    union {
        struct {
            long long before[kMaxTokens + 1];  // used before the first page is
            long long warp_sum[kThreads / 32];
        };
        struct {
            float row_scale[2][kRows];
            float row_top[4][kRows];
            Unit unit[2];
            Step step[Z::k_ring];
            int fresh[2];  // by step parity: O starts from zero
        };
    };
    unsigned long long k_full[Z::k_ring], k_empty[Z::k_ring], v_full[Z::v_ring], v_empty[Z::v_ring];
    unsigned long long q_full[2], q_empty[2], s_full[2], s_free[2], w_full[2], o_done[2], drained;
    unsigned tmem;
    int abort_flag;
};

struct RowArgs : Args {
    CUtensorMap codes;  // {64 bytes, rows of a page, pages}, boxes of 64 rows, 64-byte swizzle
};

// Entries of a token's page list: every block in sight, or its picks.
__device__ __forceinline__ int entries(const Args &A, int token, int *sequence, int *seen) {
    const RunAt at = run_at(A.c, A.runs, token / A.runs.count);
    *sequence = at.sequence;
    *seen = visible_keys(A.c, at, token % A.runs.count);
    const int nb = (*seen + kKvBlock - 1) / kKvBlock;
    return A.picks && nb ? A.top : nb;
}

// The units of this CTA, in the order in which each role walks them.
struct Walk {
    long long unit, work, work_end, chunk;
    int token, sub, entry;

    __device__ __forceinline__ bool next(const Args &A, int per_token, int tokens, Unit &u) {
        if (A.split) {
            if (work >= work_end) return false;
            while ((u.n = entries(A, token, &u.sequence, &u.seen)) == 0) ++token;  // there is more work, so a token with pages
            u.token = token;
            u.sub = sub;
            u.entry = entry;
            u.stop = (int)min((long long)u.n, entry + (work_end - work));
            u.last_cta = entry == 0 ? (int)((work + u.n - 1) / chunk) : -1;  // the CTA of its last page, where the unit begins here
            work += u.stop - u.entry;
            entry = 0;
            if (++sub == per_token) {
                sub = 0;
                ++token;
            }
            return true;
        }
        if (unit >= (long long)tokens * per_token) return false;
        u.token = (int)(unit / per_token);
        u.sub = (int)(unit % per_token);
        u.entry = 0;
        u.n = u.stop = entries(A, u.token, &u.sequence, &u.seen);
        u.last_cta = -1;
        unit += gridDim.x;
        return true;
    }
};


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
// 16 consecutive columns of this thread's TMEM lane, without the wait.
__device__ __forceinline__ void tmem_ld16(unsigned taddr, int *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// 2^x for a whole x <= 0 or -infinity, exactly; NaN (-infinity less itself) is 1.
__device__ __forceinline__ float two_to(float x) { return x < -126.0f ? 0.0f : isnan(x) ? 1.0f : __uint_as_float((unsigned)(127 + (int)x) << 23); }
// OR of x over the softmax warps (named barrier 1).
__device__ __forceinline__ bool soft_or(bool x) {
    unsigned r;
    asm volatile(
        "{\n\t.reg .pred pi, po;\n\t"
        "setp.ne.u32 pi, %1, 0;\n\t"
        "bar.red.or.pred po, 1, 128, pi;\n\t"
        "selp.u32 %0, 1, 0, po;\n\t}"
        : "=r"(r)
        : "r"((unsigned)x)
        : "memory");
    return r != 0;
}

template <int P, int R>
__global__ void __launch_bounds__(kThreads, 1) k_kv8_rows(const __grid_constant__ RowArgs A) {
    using Z = Shape<P, R>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    Smem<P, R> &M = *reinterpret_cast<Smem<P, R> *>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tokens = A.runs.segments * A.runs.count, per_token = A.c.kv_heads * A.tiles;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (tid == 0) {
        for (int i = 0; i < Z::k_ring; ++i) bar_init(&M.k_full[i], 1), bar_init(&M.k_empty[i], 1 + kSoft / 32);
        for (int i = 0; i < Z::v_ring; ++i) bar_init(&M.v_full[i], 1), bar_init(&M.v_empty[i], 1);
        for (int i = 0; i < 2; ++i) {
            bar_init(&M.q_full[i], 64), bar_init(&M.q_empty[i], 1 + kSoft / 32);
            bar_init(&M.s_full[i], 1), bar_init(&M.s_free[i], kSoft), bar_init(&M.w_full[i], kSoft), bar_init(&M.o_done[i], 1);
        }
        bar_init(&M.drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        M.abort_flag = 0;
    }
    // this CTA's pages [work, work_end) of the list of all units' pages, or units blockIdx.x, + gridDim.x, ...
    Walk walk{};
    walk.unit = blockIdx.x;
    walk.chunk = 1;
    if (A.split) {
        for (int base = 0; base < tokens; base += kThreads) {  // before[i]: entries of a head's pages before token i
            int sequence, seen;
            long long sum = base + tid < tokens ? entries(A, base + tid, &sequence, &seen) : 0;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const long long o = __shfl_up_sync(0xffffffffu, sum, s);
                if (lane >= s) sum += o;
            }
            if (lane == 31) M.warp_sum[warp] = sum;
            __syncthreads();
            long long carry = base ? M.before[base] : 0;
            for (int w = 0; w < warp; ++w) carry += M.warp_sum[w];
            if (base == 0 && tid == 0) M.before[0] = 0;
            if (base + tid < tokens) M.before[base + tid + 1] = carry + sum;
            __syncthreads();
        }
        const long long total = M.before[tokens] * per_token;
        walk.chunk = (total + gridDim.x - 1) / gridDim.x;
        walk.work = walk.chunk * blockIdx.x;
        walk.work_end = min(total, walk.work + walk.chunk);
        if (walk.work >= total) return;
        int lo = 0, hi = tokens - 1;  // the token whose entries hold `work`
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (M.before[mid + 1] * per_token > walk.work) hi = mid;
            else lo = mid + 1;
        }
        const long long n = M.before[lo + 1] - M.before[lo], in = walk.work - M.before[lo] * per_token;
        walk.token = lo;
        walk.sub = (int)(in / n);
        walk.entry = (int)(in % n);
    }
    if (warp == kIssueWarp) {  // TMEM: two buffers of S, 64 columns each, and O, 64 columns a block of 128 channels
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(su32(&M.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = M.tmem, tmem_o = tmem + 128;
    auto wait = [&](unsigned long long *b, unsigned parity) -> bool {
        if (bar_try(b, parity)) return true;
        for (const long long began = clock64(); clock64() - began < kWaitClocks;) {
            if (bar_try(b, parity)) return true;
            if (*(volatile int *)&M.abort_flag) return false;
        }
        atomicOr(&M.abort_flag, 1);
        return false;
    };
    auto wait_all = [&](unsigned long long *b, unsigned parity) { return (bool)__all_sync(0xffffffffu, wait(b, parity)); };

    if (warp < kSoft / 32) {
        // ---------------------------------------------------------------- softmax, sums and results
        const int page = warp >> 1, token_in = (warp & 1) * 32 + lane;  // this thread's token of a step
        const unsigned mine = (unsigned)(warp * 32) << 16;
        unsigned kc = 0, sc = 0;  // key slots, and of them steps with pages, used
        bool ok = true;
        // Every barrier of these warps is a vote; when it is not unanimous, a second one says whether to leave, so that all
        // leave together, wherever each of them is
        auto leave = [&]() { return soft_or(!ok || *(volatile int *)&M.abort_flag); };
        auto meet = [&]() { return !soft_or(!ok) || !leave(); };
        for (unsigned un = 0;; ++un) {
            const unsigned qb = un & 1;
            ok = wait_all(&M.q_full[qb], un >> 1 & 1);
            if (!meet()) break;
            const Unit u = M.unit[qb];
            if (u.token < 0) break;
            float m[R], sum[R], rs[R], o[Z::blocks][R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                m[r] = -INFINITY, sum[r] = 0.0f, rs[r] = M.row_scale[qb][r];
#pragma unroll
                for (int b = 0; b < Z::blocks; ++b) o[b][r] = 0.0f;
            }
            __syncwarp();
            if (lane == 0) bar_arrive(&M.q_empty[qb]);
            float ref = 0.0f;  // a power of two near the first page's value scale: what a weight's digits refer to
            int held = 0;      // steps whose products are in TMEM's sums
            // TMEM's sums of all steps before step number sc join o
            auto flush = [&]() {
                const unsigned last = sc - 1;
                if (!wait_all(&M.o_done[last & 1], last >> 1 & 1)) return false;
                tc_fence_after();
#pragma unroll
                for (int b = 0; b < Z::blocks; ++b)
#pragma unroll
                    for (int c = 0; c < Z::nw; c += 16) {
                        int x[16];
                        tmem_ld16(tmem_o + mine + 64 * b + c, x);
                        tmem_wait_ld();
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            o[b][c / 4 + r] += fmaf(fmaf(fmaf((float)x[4 * r + 3], 256.0f, (float)x[4 * r + 2]), 256.0f, (float)x[4 * r + 1]), 256.0f,
                                                    (float)x[4 * r]);
                    }
                tc_fence_before();
                held = 0;
                return true;
            };
            bool gone = false;
            for (;;) {
                const unsigned ks = kc % Z::k_ring, buf = sc & 1;
                float a[R], p[R], f = 0.0f;
                bool grows = false, here = false;
                ok = ok && wait_all(&M.k_full[ks], kc / Z::k_ring & 1);
                if (ok) {
                    const int pages = M.step[ks].pages, block = M.step[ks].block[page];
                    const float by_k = M.step[ks].k_scale[page], by_v = M.step[ks].v_scale[page], first_v = M.step[ks].v_scale[0];
                    __syncwarp();
                    if (lane == 0) bar_arrive(&M.k_empty[ks]);
                    ++kc;
                    if (pages == 0) break;
                    if (ref == 0.0f) ref = first_v > 0x1p-120f ? __uint_as_float(__float_as_uint(first_v) & 0x7f800000u) : 1.0f;
                    f = by_v / ref;
                    here = page < pages;
                    const int left = here ? u.seen - block * kKvBlock - token_in : 0;
                    ok = wait_all(&M.s_full[buf], sc >> 1 & 1);
                    tc_fence_after();
                    int s[Z::ns];
#pragma unroll
                    for (int c = 0; c < Z::ns; c += 16) tmem_ld16(tmem + mine + 64 * buf + c, s + c);
                    tmem_wait_ld();
                    tc_fence_before();
                    bar_arrive(&M.s_free[buf]);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        // 256 d1 + d0 stays inside 31 bits for 256 channels of codes
                        a[r] = fmaf((float)s[3 * r + 2], 65536.0f, (float)(s[3 * r + 1] * 256 + s[3 * r])) * (by_k * rs[r]);
                        a[r] = left > 0 ? a[r] : -INFINITY;
                        const float e = a[r] - m[r];
                        p[r] = exp2_fast(e);
                        grows |= p[r] * f > kGrow || e > 60.0f;
                    }
                }
                if (soft_or(grows || !ok)) {
                    if (leave()) {
                        gone = true;
                        break;
                    }
                    // all rows move to their maximum over the step
                    if (held) ok = flush();
                    const float lift = fmaxf(f > 0.0f ? log2f(f) : -40.0f, -40.0f);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        float top = a[r] + lift;
#pragma unroll
                        for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                        if (lane == 0) M.row_top[warp][r] = top;
                    }
                    if (!meet()) {
                        gone = true;
                        break;
                    }
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float now = fmaxf(m[r], ceilf(fmaxf(fmaxf(M.row_top[0][r], M.row_top[1][r]), fmaxf(M.row_top[2][r], M.row_top[3][r]))));
                        const float alpha = two_to(m[r] - now);
                        m[r] = now;
                        sum[r] *= alpha;
#pragma unroll
                        for (int b = 0; b < Z::blocks; ++b) o[b][r] *= alpha;
                        p[r] = exp2_fast(a[r] - (now == -INFINITY ? 0.0f : now));
                    }
                } else if (held == kFlushSteps) {
                    ok = flush();
                }
                // the weights' digits; the buffer's last use is over when that step's products are
                if (sc >= 2) ok = ok && wait_all(&M.o_done[buf], (sc - 2) >> 1 & 1);
                if (here && ok) {
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        sum[r] += p[r];
                        const unsigned w = __float2uint_rn(p[r] * f * kUnit);
#pragma unroll
                        for (int d = 0; d < 4; ++d) M.w[buf][page][sw64_byte(4 * r + d, token_in)] = (unsigned char)(w >> (8 * d));
                    }
                }
                if (tid == 0) M.fresh[buf] = held == 0;
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                bar_arrive(&M.w_full[buf]);
                ++held;
                ++sc;
            }
            if (gone) break;
            if (held) ok = flush();
            // ---- the unit is done: the rows' sums over the tokens, then the result or its part
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int x = 16; x > 0; x >>= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], x);
                if (lane == 0) M.row_top[warp][r] = sum[r];
            }
            if (!meet()) break;
#pragma unroll
            for (int r = 0; r < R; ++r) sum[r] = (M.row_top[0][r] + M.row_top[1][r]) + (M.row_top[2][r] + M.row_top[3][r]);
            const int head = u.sub / A.tiles, row0 = u.sub % A.tiles * kRows, rows = min(kRows, A.group - row0);
            const float scale = ref / kUnit;
            if (u.entry == 0 && u.stop == u.n) {
                float *dst = A.y + ((size_t)u.token * A.heads + head * A.group + row0) * A.c.dim;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float inv = sum[r] == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum[r]);
#pragma unroll
                    for (int b = 0; b < Z::blocks; ++b) {
                        const int ch = 128 * b + tid;
                        if (r < rows && ch < A.c.dim) dst[(size_t)r * A.c.dim + ch] = o[b][r] * inv * scale;
                    }
                }
            } else {
                const Parts W = parts_of(A.c.workspace, P);
                const int slot = 2 * blockIdx.x + (u.entry == 0);  // a CTA's first unit may have begun earlier, its last may go on
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (tid == 0) W.ml[slot * kRows + r] = make_float2(m[r], sum[r]);
#pragma unroll
                    for (int b = 0; b < Z::blocks; ++b)
                        if (128 * b + tid < P) W.acc[((size_t)slot * kRows + r) * P + 128 * b + tid] = o[b][r] * scale;
                }
            }
            if (u.last_cta >= 0 && tid == 0) parts_of(A.c.workspace, P).cover[u.token * per_token + u.sub] = make_int2(blockIdx.x, u.last_cta);
            if (!meet()) break;  // row_top is free
        }
    } else if (warp == kFetchWarp) {
        // ---------------------------------------------------------------- pages
        unsigned kc = 0, vc = 0;  // key and value slots asked for
        bool ok = true;
        Unit u;
        auto keys = [&](int n, const int(&page)[2], const int(&block)[2], const float2(&sc)[2], int head) {
            const unsigned s = kc % Z::k_ring;
            if (!wait_all(&M.k_empty[s], (kc / Z::k_ring & 1) ^ 1)) return false;
            if (lane == 0) {
                M.step[s] = Step{n, {block[0], block[1]}, {sc[0].x, sc[1].x}, {sc[0].y, sc[1].y}, 0};
                if (n > 0) {
                    bar_expect(&M.k_full[s], n * P * kKvBlock);
                    for (int i = 0; i < n; ++i)
                        for (int b = 0; b < Z::panels; ++b) tma3(M.k[s][b] + i * 4096, &A.codes, 0, head * 2 * P + 64 * b, page[i], &M.k_full[s]);
                } else {
                    bar_arrive(&M.k_full[s]);
                }
            }
            ++kc;
            return true;
        };
        auto values = [&](int page, int head) {
            const unsigned s = vc % Z::v_ring;
            if (!wait_all(&M.v_empty[s], (vc / Z::v_ring & 1) ^ 1)) return false;
            if (lane == 0) {
                bar_expect(&M.v_full[s], P * kKvBlock);
                for (int b = 0; b < Z::panels; ++b) tma3(M.v[s] + b * 4096, &A.codes, 0, head * 2 * P + P + 64 * b, page, &M.v_full[s]);
            }
            ++vc;
            return true;
        };
        const int none[2] = {-1, -1};
        const float2 zero[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        while (ok && walk.next(A, per_token, tokens, u)) {
            const int head = u.sub / A.tiles, nb = (u.seen + kKvBlock - 1) / kKvBlock;
            int page2[2] = {-1, -1}, block2[2] = {0, 0}, n = 0, behind[2] = {-1, -1};  // the step at hand; values still to be asked for
            float2 scale2[2] = {zero[0], zero[1]};
            auto step = [&]() {  // this step's keys, then the last step's values, which are wanted a step later
                ok = keys(n, page2, block2, scale2, head);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (ok && behind[i] >= 0) ok = values(behind[i], head);
                    behind[i] = i < n ? page2[i] : -1;
                }
                n = 0;
            };
            for (int base = u.entry; base < u.stop && ok; base += 32) {
                // 32 entries looked up at a time, then those that are there in order
                int page = -1, block = -1;
                float2 sc = zero[0];
                if (base + lane < u.stop) {
                    block = A.picks ? A.picks[((size_t)u.token * A.c.kv_heads + head) * A.top + base + lane] : base + lane;
                    if (block >= 0 && block < nb) page = page_of(A.c, u.sequence, block);
                    if (page >= 0) {
                        const float *f = page_scales(A.c, page, head);
                        sc = make_float2(f[0], f[1]);
                    }
                }
                unsigned there = __ballot_sync(0xffffffffu, page >= 0);
                while (there && ok) {
                    const int l = __ffs(there) - 1;
                    there &= there - 1;
                    const int pg = __shfl_sync(0xffffffffu, page, l), bl = __shfl_sync(0xffffffffu, block, l);
                    const float2 s2 = make_float2(__shfl_sync(0xffffffffu, sc.x, l), __shfl_sync(0xffffffffu, sc.y, l));
                    if (n == 0) page2[0] = pg, block2[0] = bl, scale2[0] = s2;
                    else page2[1] = pg, block2[1] = bl, scale2[1] = s2;
                    if (++n == 2) step();
                }
            }
            if (ok && n) step();
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (ok && behind[i] >= 0) ok = values(behind[i], head);
            if (ok) ok = keys(0, none, none, zero, head);  // the end of the unit
        }
        if (ok) ok = keys(-1, none, none, zero, 0);
        if (!ok && lane == 0) {  // let what is in flight land: the last copy of each slot, within the limit
            auto out = [&](unsigned long long *b, unsigned parity) {
                for (const long long began = clock64(); clock64() - began < kWaitClocks && !bar_try(b, parity);) {
                }
            };
            for (unsigned i = 1; i <= Z::k_ring && i <= kc; ++i) out(&M.k_full[(kc - i) % Z::k_ring], (kc - i) / Z::k_ring & 1);
            for (unsigned i = 1; i <= Z::v_ring && i <= vc; ++i) out(&M.v_full[(vc - i) % Z::v_ring], (vc - i) / Z::v_ring & 1);
        }
    } else if (warp == kIssueWarp) {
        // ---------------------------------------------------------------- products
        const unsigned id_s = idesc_i8(Z::ns, true), id_o = idesc_i8(Z::nw, false);
        unsigned kc = 0, vc = 0, sc = 0, un = 0;
        int behind = 0;  // pages of the step whose O is still to be issued
        bool ok = true, begun = false;
        auto sums = [&]() {  // O of step sc - 1
            const unsigned s = sc - 1, buf = s & 1;
            if (!wait_all(&M.w_full[buf], s >> 1 & 1)) return false;
            for (int i = 0; i < behind; ++i)
                if (!wait_all(&M.v_full[(vc + i) % Z::v_ring], (vc + i) / Z::v_ring & 1)) return false;
            tc_fence_after();
            const int fresh = M.fresh[buf];
            if (elect_one()) {
                for (int i = 0; i < behind; ++i) {
                    const unsigned long long v = sw64_desc(su32(M.v[(vc + i) % Z::v_ring])), w = sw64_desc(su32(M.w[buf][i]));
#pragma unroll
                    for (int b = 0; b < Z::blocks; ++b)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            mma_i8(tmem_o + 64 * b, v + b * (8192 >> 4) + 2 * k, w + 2 * k, id_o, !fresh || i > 0 || k > 0);
                    mma_commit(&M.v_empty[(vc + i) % Z::v_ring]);
                }
                mma_commit(&M.o_done[buf]);
            }
            __syncwarp();
            vc += behind;
            behind = 0;
            return true;
        };
        for (;;) {
            const unsigned ks = kc % Z::k_ring;
            if (!(ok = wait_all(&M.k_full[ks], kc / Z::k_ring & 1))) break;
            const int pages = M.step[ks].pages;
            __syncwarp();
            if (pages > 0) {
                const unsigned qb = un & 1, buf = sc & 1;
                if (!begun) {
                    begun = true;
                    if (!(ok = wait_all(&M.q_full[qb], un >> 1 & 1))) break;
                }
                if (!(ok = sc < 2 || wait_all(&M.s_free[buf], (sc - 2) >> 1 & 1))) break;
                tc_fence_after();
                const unsigned long long k = sw64_desc(su32(M.k[ks][0])), q = sw64_desc(su32(M.q[qb][0]));
                if (elect_one()) {
#pragma unroll
                    for (int b = 0; b < Z::panels; ++b)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            mma_i8(tmem + 64 * buf, k + b * (8192 >> 4) + 2 * h, q + b * (Z::ns * 64 >> 4) + 2 * h, id_s, b > 0 || h > 0);
                    mma_commit(&M.k_empty[ks]);
                    mma_commit(&M.s_full[buf]);
                }
                __syncwarp();
                if (behind && !(ok = sums())) break;
                behind = pages;
                ++sc;
            } else {
                if (pages == 0 && !begun && !(ok = wait_all(&M.q_full[un & 1], un >> 1 & 1))) break;  // a unit without pages
                if (behind && !(ok = sums())) break;
                if (elect_one()) {
                    bar_arrive(&M.k_empty[ks]);
                    mma_commit(&M.q_empty[un & 1]);  // the unit's queries have been used
                }
                __syncwarp();
                begun = false;
                ++un;
                if (pages < 0) break;
            }
            ++kc;
        }
        if (elect_one()) mma_commit(&M.drained);
        __syncwarp();
        for (const long long began = clock64(); !bar_try(&M.drained, 0) && clock64() - began < kWaitClocks;) {
        }
    } else {
        // ---------------------------------------------------------------- query digits, a unit ahead
        // a row is P / 8 lanes of 8 channels; rows dealt over the two warps
        constexpr int kLanes = P / 8, kAtOnce = 32 / kLanes;
        const int l = lane % kLanes;
        Unit u;
        for (unsigned n = 0;; ++n) {
            const unsigned b = n & 1;
            const bool more = walk.next(A, per_token, tokens, u);
            if (!wait_all(&M.q_empty[b], (n >> 1 & 1) ^ 1)) break;
            if (!more) u.token = -1;
            const int head = u.sub / A.tiles, row0 = u.sub % A.tiles * kRows, rows = min(kRows, A.group - row0);
            for (int i = (warp - kQueryWarp) * kAtOnce; more && i < R; i += 2 * kAtOnce) {
                const int r = i + lane / kLanes;
                const bool there = r < rows;
                const float *src = A.q + (long long)u.token * A.stride + (size_t)(head * A.group + row0 + r) * A.c.dim + 8 * l;
                float x[8], big = 0.0f;
                if (there && 8 * l + 8 <= A.c.dim && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
                    const float4 a = reinterpret_cast<const float4 *>(src)[0], c = reinterpret_cast<const float4 *>(src)[1];
                    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = c.x, x[5] = c.y, x[6] = c.z, x[7] = c.w;
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = there && 8 * l + k < A.c.dim ? src[k] : 0.0f;
                }
                bool bad = false;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    bad |= !isfinite(x[k]);
                    big = fmaxf(big, fabsf(x[k]));
                }
#pragma unroll
                for (int s = kLanes / 2; s > 0; s >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, s));
                const unsigned all_bad = __ballot_sync(0xffffffffu, bad);
                const bool spoilt = (all_bad >> (lane / kLanes * kLanes) & (kLanes == 32 ? 0xffffffffu : (1u << (kLanes & 31)) - 1)) != 0;
                // a power of two that brings the row's largest value to 2^21 .. 2^22: three signed digits
                const unsigned field = min(275u - (__float_as_uint(big) >> 23), 253u);
                const float up = __uint_as_float(field << 23);
                if (r < R) {
                    // a row with a value that is not finite has no result
                    if (l == 0) M.row_scale[b][r] = spoilt ? __uint_as_float(0x7fc00000u) : __uint_as_float((254u - field) << 23) * A.scale;
                    uint2 d[3] = {};
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        int v = __float2int_rn(x[k] * up);
#pragma unroll
                        for (int e = 0; e < 3; ++e) {
                            const int digit = e < 2 ? ((v + 128) & 255) - 128 : v;
                            v = (v - digit) >> 8;
                            (k < 4 ? d[e].x : d[e].y) |= (unsigned)(digit & 255) << (8 * (k & 3));
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 3; ++e) *reinterpret_cast<uint2 *>(M.q[b][l >> 3] + sw64_byte(3 * r + e, 8 * (l & 7))) = d[e];
                }
            }
            if (warp == kQueryWarp && lane == 0) M.unit[b] = u;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            bar_arrive(&M.q_full[b]);
            if (!more) break;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && M.abort_flag) raise_error(A.c.err, kErrWaitTimeout);
    if (warp == kIssueWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem) : "memory");
    }
}

// Joins the partial results of a unit's row: out = sum_i 2^(m_i - max) acc_i / sum_i 2^(m_i - max) l_i.
template <int P>
__global__ void __launch_bounds__(kJoinThreads) k_kv8_join(const __grid_constant__ Args A) {
    constexpr int kAcross = P / 4, kDeep = kJoinThreads / kAcross;  // threads a row, parts at a time
    __shared__ float weight_s[kMaxCtas], red[kJoinThreads / 32];
    __shared__ float4 acc_s[kJoinThreads];
    __shared__ float sum_s[kDeep];
    const int tid = threadIdx.x, per_token = A.c.kv_heads * A.tiles, unit = blockIdx.x, row = blockIdx.y;
    const int token = unit / per_token, sub = unit % per_token, head = sub / A.tiles, row0 = sub % A.tiles * kRows;
    if (row >= min(kRows, A.group - row0)) return;
    int sequence, seen;
    const int n = entries(A, token, &sequence, &seen);
    float *dst = A.y + ((size_t)token * A.heads + head * A.group + row0 + row) * A.c.dim;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (n == 0) {  // nothing in sight: no CTA had this unit
        for (int i = tid; i < A.c.dim; i += kJoinThreads) dst[i] = 0.0f;
        return;
    }
    const Parts W = parts_of(A.c.workspace, P);
    const int2 cover = W.cover[unit];
    const int count = cover.y - cover.x + 1;
    if (count <= 1) return;
    // the unit begins in its first CTA's second slot and goes on in the first slots of the others
    auto slot = [&](int i) { return (size_t)2 * (cover.x + i) + (i == 0); };
    float m = -INFINITY;
    for (int i = tid; i < count; i += kJoinThreads) {
        weight_s[i] = W.ml[slot(i) * kRows + row].x;
        m = fmaxf(m, weight_s[i]);
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, s));
    if (tid % 32 == 0) red[tid / 32] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kJoinThreads / 32; ++i) m = fmaxf(m, red[i]);
    if (m == -INFINITY) m = 0.0f;
    const int at = tid % kAcross, deep = tid / kAcross;
    float4 acc = make_float4(0, 0, 0, 0);
    float sum = 0.0f;
#pragma unroll 8
    for (int i = deep; i < count; i += kDeep) {
        const float w = exp2_fast(weight_s[i] - m);
        const float4 f = *reinterpret_cast<const float4 *>(W.acc + (slot(i) * kRows + row) * P + at * 4);
        sum += w * W.ml[slot(i) * kRows + row].y;
        acc.x += w * f.x, acc.y += w * f.y, acc.z += w * f.z, acc.w += w * f.w;
    }
    acc_s[tid] = acc;
    if (at == 0) sum_s[deep] = sum;
    __syncthreads();
    if (deep) return;
#pragma unroll
    for (int i = 1; i < kDeep; ++i) {
        const float4 f = acc_s[i * kAcross + at];
        acc.x += f.x, acc.y += f.y, acc.z += f.z, acc.w += f.w;
        sum += sum_s[i];
    }
    const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum), v[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (at * 4 + i < A.c.dim) dst[at * 4 + i] = v[i];
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
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

// What the current device needs set or asked once.
template <int P, int R>
cudaError_t multiprocessors(size_t smem, int *out) {
    constexpr int kDevices = 64;
    static std::atomic<int> known[kDevices];
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    if (device < kDevices && (*out = known[device].load(std::memory_order_relaxed)) > 0) return cudaSuccess;
    e = cudaFuncSetAttribute(k_kv8_rows<P, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess && device < kDevices) known[device].store(*out, std::memory_order_relaxed);
    return e;
}

template <int P, int R>
cudaError_t launch(const Args &args, cudaStream_t s) {
    static_assert((size_t)2 * kMaxCtas * kRows * (256 * 4 + 8) + 65536 * 8 <= (32u << 20), "the workspace holds every partial result");
    // more than half of a multiprocessor's shared memory: one CTA on each
    constexpr size_t kSmem = sizeof(Smem<P, R>) > 120 * 1024 ? sizeof(Smem<P, R>) : 120 * 1024;
    static_assert(kSmem <= 227 * 1024, "fits a multiprocessor");
    RowArgs A;
    static_cast<Args &>(A) = args;
    int slots = 0;
    cudaError_t e = multiprocessors<P, R>(kSmem, &slots);
    if (e != cudaSuccess) return e;
    if (slots > kMaxCtas) slots = kMaxCtas;
    const auto encode = encoder();
    if (!encode) return cudaErrorNotSupported;
    const unsigned long long rows = 2ull * A.c.kv_heads * P;
    const cuuint64_t dims[3] = {64, rows, (cuuint64_t)A.c.pages}, strides[2] = {64, rows * 64};
    const cuuint32_t box[3] = {64, 64, 1}, steps[3] = {1, 1, 1};
    if (encode(&A.codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, A.c.codes, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return cudaErrorInvalidValue;
    const long long tokens = (long long)A.runs.segments * A.runs.count, units = tokens * A.c.kv_heads * A.tiles;
    A.split = tokens <= kMaxTokens && units < 8LL * slots && units <= 65536;
    const long long most = A.split ? units * (A.picks ? A.top : A.c.blocks) : units;
    k_kv8_rows<P, R><<<(unsigned)(most < slots ? most : slots), kThreads, kSmem, s>>>(A);
    e = cudaGetLastError();
    if (e != cudaSuccess || !A.split) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)units, A.group < kRows ? A.group : kRows);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_kv8_join<P>, static_cast<const Args &>(A));
}
template <int P>
cudaError_t launch_rows(const Args &A, cudaStream_t s) {  // room for as many rows as the group has, to the next four
    if (A.group <= 4) return launch<P, 4>(A, s);
    if (A.group <= 8) return launch<P, 8>(A, s);
    if (A.group <= 12) return launch<P, 12>(A, s);
    return launch<P, 16>(A, s);
}

}  // namespace

cudaError_t kv8_attend(const Kv8 &c, const float *q, long long stride, int heads, const Kv8Runs &r, const int *picks, int top, float scale,
                       float *y, cudaStream_t s) {
    const int group = heads / c.kv_heads;
    if (!picks && r.count > 1 && (long long)r.count * group >= 64) return kv8_attend_prompt(c, q, stride, heads, r, scale, y, s);
    const Args A{c, q, stride, heads, group, (group + kRows - 1) / kRows, r, picks, top, scale * 1.4426950408889634f, y, 0};
    if (c.padded == 64) return launch_rows<64>(A, s);
    if (c.padded == 128) return launch_rows<128>(A, s);
    return launch_rows<256>(A, s);
}

}  // namespace strata
