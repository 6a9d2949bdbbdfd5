// Attention over the 8-bit paged cache (strata_kv8_attend): the form that works token by token.
//
// A unit is one token and key/value head with up to 16 of its group's query heads. With so few rows the
// products are turned round: the cache is the 128-row operand of the 5th-generation tensor cores' integer
// products (tcgen05 kind::i8), which take its codes as they lie in memory, and the queries and weights, as whole
// numbers of several 8-bit digits, are the narrow one. No code is ever converted; every product is exact.
//   S^T[128 tokens][3 digits x rows] = K . Q^T    a query row, scaled by a power of two, has 23 bits in three
//       signed digits; a step is two pages
//   O^T[P channels][4 digits x rows] += V^T . W^T  a weight is 31 bits in four unsigned digits; 32-bit sums in
//       TMEM over up to 256 pages
// A thread of the softmax warps has one of the step's tokens (its TMEM lane): it puts the rows' logits together
// from their digits, takes the exponentials, and writes the weights' digits as the second product's operand.
// Logits, references and sums of weights are F32. A row's weights refer to a power of two some way above its maximum,
// which moves only when a weight would pass 2^3; then, and at the unit's end, the sums move from TMEM to F32 registers.
//
// Warps: 0-3 and 4-7 are two softmax groups that take the steps in turn, each with references and sums of its own
// (joined at the unit's end), so that one's latencies run under the other's work; 8 looks pages up and fetches
// keys and values by TMA (64-byte swizzle), ahead across units; one thread of 9 issues S, up to four steps ahead, one
// of 11 O; 10 makes the next unit's query digits. One CTA a multiprocessor; every wait is bounded, and past the limit all leave.
//
// Measured: 64 sessions of up to 16384 tokens, 24 heads over 2 of 256 channels, 115 us, 4.7 TB/s of what has to be read; one
// session of 200001 tokens, 32 heads over 8 of 128, 85 us, 4.8 TB/s. In the first a CTA has 56 steps of two pages in 212
// thousand clocks, 3800 a step with units' beginnings and ends; copies alone ran at 100 and 75 us.
//
// Few units (`split`): the pages of all units form one list that the CTAs share evenly, whatever the
// lengths; a unit cut by a CTA border leaves unnormalised partial sums in the workspace and a
// second kernel joins them in CTA order, so results repeat bit for bit.
#include "kv8_mma.cuh"
#include "kv8_rows.cuh"

#include <atomic>

namespace strata {
namespace {

using namespace pf;
using namespace kv8_rows;

constexpr int kSoft = 128, kKeyWarp = 8, kIssueWarp = 9, kSumWarp = 11, kThreads = 384;  // kSoft: threads of a softmax group
constexpr int kSteps = 8;         // steps looked up ahead
constexpr int kFlushSteps = 128;  // steps that TMEM's 32-bit sums bear (255 * 127 * 128 tokens a step)
constexpr float kGrow = 3.0f;          // log2 of what weights stay below, times
constexpr float kUnit = 268435456.0f;  // 2^28, below 2^32
// log2 of the room that a new reference leaves above the maximum, so that it seldom moves again. A row's largest weight
// is then 2^-4 at least, and rounding to a whole unit exact to 2^-25 of it. (5, 2^26 and room 4 moved less often, a sparse
// prompt of 1024 tokens 426 instead of 445 us, but doubled the result's error to 2e-6.)
constexpr float kRoom = 3.0f;
// What weights refer to: a power of two near the largest value scale of the first 32 pages (of a unit's pages on this CTA) that
// have one but zero. A page's scale counts as 2^kLeastLift of it at least when a row's reference is chosen, and may be up to kFar
// times as large (past that it is reported): references and maxima so stay close enough for F32's exponents, also where parts are joined.
constexpr float kLeastLift = -40.0f, kFar = 0x1p80f;
constexpr long long kWaitClocks = 2000000000;  // about a second

// P stored channels; R rows that the operands have room for, 4 .. 16.
template <int P, int R>
struct Shape {
    static constexpr int panels = P / 64;
    static constexpr int blocks = P <= 128 ? 1 : 2;             // of 128 channels
    static constexpr int ns = (3 * R + 15) / 16 * 16, nw = 4 * R;  // columns of S and O
    static constexpr int k_ring = P == 256 ? 2 : 3, v_ring = P == 256 ? 3 : 4;  // steps
};
// A step: 1 or 2 pages, the end of a unit (0), or the end of all (-1).
struct Step {
    int pages, unit, block[2];
    float k_scale[2], v_scale[2];  // values' over the unit's `ref`
    float ref;
};
struct Unit {  // or the part of it that this CTA works on: entries [entry, stop) of its n
    int token, sub, entry, stop, n, seen, sequence, last_cta;
};
template <int P, int R>
struct __align__(1024) Smem {
    using Z = Shape<P, R>;
    unsigned char k[Z::k_ring][Z::panels][128 * 64];  // tokens of two pages, 64 channels a row
    unsigned char v[Z::v_ring][2][P * 64];            // two pages: channels, 64 tokens a row
    unsigned char v_end[P == 64 ? 4096 : 1024];       // (a 64-channel page is read as 128 rows)
    unsigned char q[2][Z::panels][Z::ns * 64];        // row 3 r + digit: 64 channels
    unsigned char w[2][2][Z::nw * 64];                // by group and page: row 4 r + digit: 64 tokens
    union {
        struct {
            long long before[kMaxTokens + 1];  // used before the first page is
            long long warp_sum[kThreads / 32];
        };
        struct {
            float row_scale[2][kRows];
            float row_top[2][4][kRows];
            float2 group_row[kRows];  // the second group's reference and sum of weights
            Unit unit[2];
            Step step[kSteps];
            float4 list[32];  // pages looked up: page, block (bits), key scale, value scale over the unit's reference
            float group_ref;
            int what[2];  // by group: pages whose weights are there (-1: no more), plus 4 where O starts from zero
        };
    };
    unsigned long long step_full[kSteps], step_empty[kSteps], k_full[Z::k_ring], k_empty[Z::k_ring], v_full[Z::v_ring], v_empty[Z::v_ring];
    unsigned long long q_full[2], q_empty[2], s_full[4], s_free[4], w_full[2], o_done[2], hand_full, hand_free, drained[2];
    unsigned tmem;
    int abort_flag;
};

struct RowArgs : Args {
    CUtensorMap keys, values;  // {64 bytes, rows of a page, pages}, 64-byte swizzle; boxes of 64 rows, of P rows
};

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
// OR of x over a named barrier's threads: a softmax group's (barriers 1 and 2).
__device__ __forceinline__ bool bar_or(int barrier, int threads, bool x) {
    unsigned r;
    asm volatile(
        "{\n\t.reg .pred pi, po;\n\t"
        "setp.ne.u32 pi, %1, 0;\n\t"
        "bar.red.or.pred po, %2, %3, pi;\n\t"
        "selp.u32 %0, 1, 0, po;\n\t}"
        : "=r"(r)
        : "r"((unsigned)x), "r"(barrier), "r"(threads)
        : "memory");
    return r != 0;
}
// The largest of x over the warp; NaN only where all are.
__device__ __forceinline__ float warp_max(float x) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}

template <int P, int R>
__global__ void __launch_bounds__(kThreads, 1) k_kv8_rows(const __grid_constant__ RowArgs A) {
    using Z = Shape<P, R>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    Smem<P, R> &M = *reinterpret_cast<Smem<P, R> *>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int tokens = A.runs.segments * A.runs.count, per_token = A.c.kv_heads * A.tiles;
    if (tid == 0) {
        for (int i = 0; i < Z::k_ring; ++i) bar_init(&M.k_full[i], 1), bar_init(&M.k_empty[i], 1);
        // read by the softmax warps and the one that issues S
        for (int i = 0; i < kSteps; ++i) bar_init(&M.step_full[i], 1), bar_init(&M.step_empty[i], 2 * kSoft / 32 + 1);
        for (int i = 0; i < Z::v_ring; ++i) bar_init(&M.v_full[i], 1), bar_init(&M.v_empty[i], 1);
        for (int i = 0; i < 2; ++i) {
            bar_init(&M.q_full[i], 32), bar_init(&M.q_empty[i], 1 + 2 * kSoft / 32);
            bar_init(&M.w_full[i], kSoft), bar_init(&M.o_done[i], 1);
        }
        for (int i = 0; i < 4; ++i) bar_init(&M.s_full[i], 1), bar_init(&M.s_free[i], kSoft);
        bar_init(&M.hand_full, kSoft), bar_init(&M.hand_free, kSoft);
        bar_init(&M.drained[0], 1), bar_init(&M.drained[1], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        M.abort_flag = 0;
    }
    kv8_enter();
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
    if (warp == kIssueWarp) {  // TMEM: four buffers of S, 64 columns each, and each group's O, 64 columns a block of 128 channels
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&M.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = M.tmem, tmem_o = tmem + 256;
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
    auto wait_out = [&](unsigned long long *b, unsigned parity) {  // the same where others have failed: only the limit ends it
        for (const long long began = clock64(); clock64() - began < kWaitClocks && !bar_try(b, parity);) {
        }
    };

    if (warp < kKeyWarp) {
        // ---------------------------------------------------------------- softmax, sums and results
        const int group = warp >> 2, quarter = warp & 3, page = quarter >> 1, token_in = (quarter & 1) * 32 + lane;  // this thread's token of a step
        const int thread = tid & (kSoft - 1);
        const unsigned mine = (unsigned)(quarter * 32) << 16, own_o = tmem_o + 128 * group;
        unsigned kc = 0, sc = 0;  // steps, and of them those with pages, so far
        bool ok = true, handed = false;  // handed: the second group's last hand-over may not be taken yet
        // Every barrier of these warps is a vote; when it is not unanimous, a second one says whether to leave, so that all
        // leave together, wherever each of them is. Between the groups there are only bounded waits.
        auto leave = [&]() { return bar_or(1 + group, kSoft, !ok || *(volatile int *)&M.abort_flag); };
        auto meet = [&]() { return !bar_or(1 + group, kSoft, !ok) || !leave(); };
        for (unsigned un = 0;; ++un) {
            const unsigned qb = un & 1;
            ok = wait_all(&M.q_full[qb], un >> 1 & 1);
            if (!meet()) break;
            const Unit u = M.unit[qb];
            if (u.token < 0) {  // the group whose step would be next says so to the warp that issues O
                if ((sc & 1) == group) {
                    if (sc >= 2) ok = wait_all(&M.o_done[group], (sc - 2) >> 1 & 1);
                    if (thread == 0) M.what[group] = -1;
                    bar_arrive(&M.w_full[group]);
                }
                break;
            }
            float m[R], sum[R], rs[R], o[Z::blocks][R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                m[r] = -INFINITY, sum[r] = 0.0f, rs[r] = M.row_scale[qb][r];
#pragma unroll
                for (int b = 0; b < Z::blocks; ++b) o[b][r] = 0.0f;
            }
            __syncwarp();
            if (lane == 0) bar_arrive(&M.q_empty[qb]);
            float ref = 0.0f;  // a power of two near the first pages' value scales: what a weight's digits refer to
            int held = 0;      // steps whose products are in TMEM's sums
            unsigned last = 0;  // the group's last step
            // TMEM's sums join o
            auto flush = [&]() {
                if (!wait_all(&M.o_done[group], last >> 1 & 1)) return false;
                tc_fence_after();
#pragma unroll
                for (int b = 0; b < Z::blocks; ++b) {
                    int x[Z::nw];
#pragma unroll
                    for (int c = 0; c < Z::nw; c += 16) tmem_ld16(own_o + mine + 64 * b + c, x + c);
                    tmem_wait_ld();
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        o[b][r] += fmaf(fmaf(fmaf((float)x[4 * r + 3], 256.0f, (float)x[4 * r + 2]), 256.0f, (float)x[4 * r + 1]), 256.0f,
                                        (float)x[4 * r]);
                }
                tc_fence_before();
                held = 0;
                return true;
            };
            auto taken = [&]() {  // before O's columns of TMEM or the other places are written again
                if (handed) ok = ok && wait_all(&M.hand_free, (un - 1) & 1);
                handed = false;
            };
            bool gone = false;
            for (;;) {
                const unsigned ks = kc % kSteps, buf = sc & 3;
                float a[R], f = 0.0f, lift = 0.0f;
                bool grows = false, here = false;
                int pages_now = 0;
                ok = ok && wait_all(&M.step_full[ks], kc / kSteps & 1);
                if (ok) {
                    const int pages = M.step[ks].pages, block = M.step[ks].block[page];
                    const float by_k = M.step[ks].k_scale[page], by_v = M.step[ks].v_scale[page], of_unit = M.step[ks].ref;
                    __syncwarp();
                    if (lane == 0) bar_arrive(&M.step_empty[ks]);
                    ++kc;
                    if (pages == 0) break;
                    if ((sc & 1) != group) {  // the other group's step
                        ++sc;
                        continue;
                    }
                    ref = of_unit;
                    f = by_v;
                    here = page < pages;
                    pages_now = pages;
                    const int left = here ? u.seen - block * kKvBlock - token_in : 0;
                    ok = wait_all(&M.s_full[buf], sc >> 2 & 1);
                    tc_fence_after();
                    int s[Z::ns];
#pragma unroll
                    for (int c = 0; c < Z::ns; c += 16) tmem_ld16(tmem + mine + 64 * buf + c, s + c);
                    lift = fmaxf(f > 0.0f ? log2f(f) : kLeastLift, kLeastLift);
                    tmem_wait_ld();
                    tc_fence_before();
                    bar_arrive(&M.s_free[buf]);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        // 256 d1 + d0 stays inside 31 bits for 256 channels of codes
                        a[r] = fmaf((float)s[3 * r + 2], 65536.0f, (float)(s[3 * r + 1] * 256 + s[3 * r])) * (by_k * rs[r]);
                        a[r] = left > 0 ? a[r] : -INFINITY;
                        grows |= a[r] + lift > m[r] + kGrow;
                    }
                }
                if (bar_or(1 + group, kSoft, grows || !ok)) {
                    if (leave()) {
                        gone = true;
                        break;
                    }
                    // all rows move to their maximum over the step
                    if (held) ok = flush();
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float top = warp_max(a[r] + lift);
                        if (lane == 0) M.row_top[group][quarter][r] = top;
                    }
                    if (!meet()) {
                        gone = true;
                        break;
                    }
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float(*top)[kRows] = M.row_top[group];
                        const float now = fmaxf(m[r], ceilf(fmaxf(fmaxf(top[0][r], top[1][r]), fmaxf(top[2][r], top[3][r]))) + kRoom);
                        const float alpha = two_to(m[r] - now);
                        m[r] = now;
                        sum[r] *= alpha;
#pragma unroll
                        for (int b = 0; b < Z::blocks; ++b) o[b][r] *= alpha;
                    }
                } else if (held == kFlushSteps) {
                    ok = flush();
                }
                // the weights' digits; the buffer's last use is over when that step's products are
                if (sc >= 2) ok = ok && wait_all(&M.o_done[group], (sc - 2) >> 1 & 1);
                taken();
                if (here && ok) {
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float p = exp2_fast(a[r] - (m[r] == -INFINITY ? 0.0f : m[r]));
                        sum[r] += p;
                        const unsigned w = __float2uint_rn(p * f * kUnit);
#pragma unroll
                        for (int d = 0; d < 4; ++d) M.w[group][page][sw64_byte(4 * r + d, token_in)] = (unsigned char)(w >> (8 * d));
                    }
                }
                if (thread == 0) M.what[group] = pages_now + (held == 0 ? 4 : 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                bar_arrive(&M.w_full[group]);
                last = sc;
                ++held;
                ++sc;
            }
            if (gone) break;
            if (held) ok = flush();
            // ---- the unit is done: the rows' sums over the group's tokens
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int x = 16; x > 0; x >>= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], x);
                if (lane == 0) M.row_top[group][quarter][r] = sum[r];
            }
            if (!meet()) break;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float(*part)[kRows] = M.row_top[group];
                sum[r] = (part[0][r] + part[1][r]) + (part[2][r] + part[3][r]);
            }
            // the second group hands its own over, O through its columns of TMEM, and the first writes the result
            if (group == 1) {
                taken();
#pragma unroll
                for (int b = 0; b < Z::blocks; ++b) {
                    unsigned x[16];
#pragma unroll
                    for (int r = 0; r < 16; ++r) x[r] = r < R ? __float_as_uint(o[b][r < R ? r : 0]) : 0u;
                    tmem_st16(own_o + mine + 64 * b, x);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                tc_fence_before();
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (thread == r) M.group_row[r] = make_float2(m[r], sum[r]);
                if (thread == 0) M.group_ref = ref;
                bar_arrive(&M.hand_full);
                handed = true;
                continue;
            }
            ok = wait_all(&M.hand_full, un & 1);
            if (!meet()) break;
            {
                tc_fence_after();
                const float other_ref = M.group_ref / kUnit, own_ref = ref / kUnit;
                const int head = u.sub / A.tiles, row0 = u.sub % A.tiles * kRows, rows = min(kRows, A.group - row0);
                const bool whole = u.entry == 0 && u.stop == u.n;
                const Parts W = parts_of(A.c.workspace, P);
                const int slot = 2 * blockIdx.x + (u.entry == 0);  // a CTA's first unit may have begun earlier, its last may go on
                float *dst = A.y + ((size_t)u.token * A.heads + head * A.group + row0) * A.c.dim;
                float f0[R], f1[R];
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const float2 x = M.group_row[r];
                    const float now = fmaxf(m[r], x.x), l0 = two_to(m[r] - now), l1 = two_to(x.x - now);
                    sum[r] = sum[r] * l0 + x.y * l1;
                    m[r] = now;
                    const float by = !whole ? 1.0f : sum[r] == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum[r]);
                    f0[r] = l0 * by;
                    f1[r] = l1 * by;
                }
#pragma unroll
                for (int b = 0; b < Z::blocks; ++b) {
                    int x[16];
                    tmem_ld16(tmem_o + 128 + mine + 64 * b, x);
                    tmem_wait_ld();
                    const int ch = 128 * b + thread;
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float out = o[b][r] * f0[r] * own_ref + __int_as_float(x[r]) * f1[r] * other_ref;
                        if (whole) {
                            if (r < rows && ch < A.c.dim) dst[(size_t)r * A.c.dim + ch] = out;
                        } else if (ch < P) {
                            W.acc[((size_t)slot * kRows + r) * P + ch] = out;
                        }
                    }
                }
                if (!whole && thread == 0)
#pragma unroll
                    for (int r = 0; r < R; ++r) W.ml[slot * kRows + r] = make_float2(m[r], sum[r]);
                if (u.last_cta >= 0 && thread == 0) W.cover[u.token * per_token + u.sub] = make_int2(blockIdx.x, u.last_cta);
                tc_fence_before();
                bar_arrive(&M.hand_free);
            }
        }
    } else if (warp == kKeyWarp) {
        // ---------------------------------------------------------------- pages, keys and values
        unsigned kc = 0, sc = 0, vc = 0;  // steps; of them those with pages, and those whose values have been asked for
        bool ok = true;
        // a batch: up to 32 entries of a unit, an entry a lane, looked up while the batch before it is being fetched
        struct {
            int unit, head, page, block;  // unit -1: there is no more
            float k_scale, v_scale;
            bool end;  // of the unit
        } batch;
        Unit u;
        int unit = -1, base = 0;
        u.stop = 0;
        auto look_up = [&]() {
            if (base >= u.stop) {
                if (!walk.next(A, per_token, tokens, u)) {
                    batch.unit = -1;
                    return;
                }
                ++unit;
                base = u.entry;
            }
            batch.unit = unit;
            batch.head = u.sub / A.tiles;
            batch.page = -1;
            if (base + lane < u.stop) {
                // the list is walked from its second entry on: the first is mostly the session's first block, which selection
                // picks for its place, and a reference taken from it would soon have to move
                const int e = base + lane + 1 < u.n ? base + lane + 1 : 0;
                batch.block = A.picks ? A.picks[((size_t)u.token * A.c.kv_heads + batch.head) * A.top + e] : e;
                if (batch.block >= 0 && batch.block < (u.seen + kKvBlock - 1) / kKvBlock) batch.page = page_of(A.c, u.sequence, batch.block);
                if (batch.page >= 0) {
                    const float *f = page_scales(A.c, batch.page, batch.head);
                    batch.k_scale = f[0], batch.v_scale = f[1];
                }
            }
            base += 32;
            batch.end = base >= u.stop;
        };
        float ref = 0.0f, per_ref = 0.0f;  // of the unit whose pages are being fetched
        int ref_unit = -1;
        // a step's copies: a lane a box, of 64 key rows or of a page's values
        auto post = [&](int n, int unit_of, int head, int at) {
            const unsigned s = kc % kSteps, k = sc % Z::k_ring, v = vc % Z::v_ring;
            if (!wait_all(&M.step_empty[s], (kc / kSteps & 1) ^ 1)) return false;
            if (lane == 0) {
                const float4 x = M.list[at & 31], y = M.list[(at + 1) & 31];
                M.step[s] = Step{n, unit_of, {__float_as_int(x.y), __float_as_int(y.y)}, {x.z, y.z}, {x.w, y.w}, ref};
                bar_arrive(&M.step_full[s]);
            }
            ++kc;
            if (n <= 0) return true;
            if (!wait_all(&M.k_empty[k], (sc / Z::k_ring & 1) ^ 1)) return false;
            if (lane == 0) bar_expect(&M.k_full[k], n * P * kKvBlock);
            __syncwarp();
            if (lane < n * Z::panels)
                tma3(M.k[k][lane % Z::panels] + lane / Z::panels * 4096, &A.keys, 0, head * 2 * P + 64 * (lane % Z::panels),
                     __float_as_int(M.list[at + lane / Z::panels].x), &M.k_full[k]);
            ++sc;
            if (!wait_all(&M.v_empty[v], (vc / Z::v_ring & 1) ^ 1)) return false;
            if (lane == 0) bar_expect(&M.v_full[v], n * P * kKvBlock);
            __syncwarp();
            if (lane < n) tma3(M.v[v][lane], &A.values, 0, head * 2 * P + P, __float_as_int(M.list[at + lane].x), &M.v_full[v]);
            ++vc;
            return true;
        };
        look_up();
        while (ok && batch.unit >= 0) {
            const int this_unit = batch.unit, head = batch.head;
            const bool end = batch.end;
            const unsigned there = __ballot_sync(0xffffffffu, batch.page >= 0);
            const int count = __popc(there);
            if (this_unit != ref_unit) {  // while all values are zero, nothing refers to it
                const float most = warp_max(batch.page >= 0 ? batch.v_scale : 0.0f);
                ref = most > 0.0f ? __uint_as_float(__float_as_uint(most) & 0x7f800000u) : 1.0f;
                per_ref = __fdiv_rn(1.0f, ref);
                if (most > 0.0f) ref_unit = this_unit;
            }
            if (batch.page >= 0 && batch.v_scale * per_ref > kFar) raise_error(A.c.err, kErrKvScale);
            if (batch.page >= 0)
                M.list[__popc(there & ((1u << lane) - 1))] =
                    make_float4(__int_as_float(batch.page), __int_as_float(batch.block), batch.k_scale, batch.v_scale * per_ref);
            __syncwarp();
            for (int at = 0; at < count && ok; at += 2) {
                ok = post(min(2, count - at), this_unit, head, at);
                if (at == 2) look_up();  // the rings are full for a while
            }
            if (count <= 2) look_up();
            if (ok && end) ok = post(0, this_unit, head, 0);
        }
        if (ok) ok = post(-1, unit + 1, 0, 0);
        if (!ok && lane == 0) {  // let what is in flight land: the last copy of each slot, within the limit
            for (unsigned i = 1; i <= Z::k_ring && i <= sc; ++i) wait_out(&M.k_full[(sc - i) % Z::k_ring], (sc - i) / Z::k_ring & 1);
            for (unsigned i = 1; i <= Z::v_ring && i <= vc; ++i) wait_out(&M.v_full[(vc - i) % Z::v_ring], (vc - i) / Z::v_ring & 1);
        }
    } else if (warp == kSumWarp) {
        // ---------------------------------------------------------------- O
        if (lane == 0) {
            const unsigned id_o = idesc_i8(Z::nw, false);
            for (unsigned sc = 0;; ++sc) {
                const unsigned group = sc & 1, s = sc % Z::v_ring;
                if (!wait(&M.w_full[group], sc >> 1 & 1)) break;
                const int what = M.what[group], pages = what & 3;
                if (what < 0 || !wait(&M.v_full[s], sc / Z::v_ring & 1)) break;
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (i >= pages) continue;
                    const unsigned long long v = sw64_desc(su32(M.v[s][i])), w = sw64_desc(su32(M.w[group][i]));
#pragma unroll
                    for (int b = 0; b < Z::blocks; ++b)
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            mma_i8(tmem_o + 128 * group + 64 * b, v + b * (8192 >> 4) + 2 * k, w + 2 * k, id_o, !(what & 4) || i > 0 || k > 0);
                }
                mma_commit(&M.v_empty[s]);
                mma_commit(&M.o_done[group]);
            }
            mma_commit(&M.drained[1]);
            wait_out(&M.drained[1], 0);
        }
        __syncwarp();
    } else if (warp == kIssueWarp) {
        // ---------------------------------------------------------------- S
        if (lane == 0) {
            const unsigned id_s = idesc_i8(Z::ns, true);
            unsigned sc = 0;
            int unit = -1;  // whose queries are in use
            for (unsigned kc = 0;; ++kc) {
                const unsigned st = kc % kSteps, ks = sc % Z::k_ring, buf = sc & 3;
                if (!wait(&M.step_full[st], kc / kSteps & 1)) break;
                const int pages = M.step[st].pages, next_unit = M.step[st].unit;
                bar_arrive(&M.step_empty[st]);
                if (pages < 0) break;
                if (unit != next_unit && !wait(&M.q_full[next_unit & 1], next_unit >> 1 & 1)) break;
                unit = next_unit;
                if (pages == 0) {
                    mma_commit(&M.q_empty[unit & 1]);  // the unit's queries have been used
                    continue;
                }
                if (sc >= 4 && !wait(&M.s_free[buf], (sc - 4) >> 2 & 1)) break;
                if (!wait(&M.k_full[ks], sc / Z::k_ring & 1)) break;
                tc_fence_after();
                const unsigned long long k = sw64_desc(su32(M.k[ks][0])), q = sw64_desc(su32(M.q[unit & 1][0]));
#pragma unroll
                for (int b = 0; b < Z::panels; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        mma_i8(tmem + 64 * buf, k + b * (8192 >> 4) + 2 * h, q + b * (Z::ns * 64 >> 4) + 2 * h, id_s, b > 0 || h > 0);
                mma_commit(&M.k_empty[ks]);
                mma_commit(&M.s_full[buf]);
                ++sc;
            }
            mma_commit(&M.drained[0]);
            wait_out(&M.drained[0], 0);
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------------- query digits, a unit ahead
        // a row is P / 8 lanes of 8 channels
        constexpr int kLanes = P / 8, kAtOnce = 32 / kLanes;
        const int l = lane % kLanes;
        Unit u;
        for (unsigned n = 0;; ++n) {
            const unsigned b = n & 1;
            const bool more = walk.next(A, per_token, tokens, u);
            if (!wait_all(&M.q_empty[b], (n >> 1 & 1) ^ 1)) break;
            if (!more) u.token = -1;
            const int head = u.sub / A.tiles, row0 = u.sub % A.tiles * kRows, rows = min(kRows, A.group - row0);
            constexpr int kBatch = 4;  // row groups whose loads are in flight together
            for (int i0 = 0; more && i0 < R; i0 += kBatch * kAtOnce) {
                float x[kBatch][8];
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    const int r = i0 + j * kAtOnce + lane / kLanes;
                    const bool there = r < rows;
                    const float *src = A.q + (long long)u.token * A.stride + (size_t)(head * A.group + row0 + r) * A.c.dim + 8 * l;
                    if (there && 8 * l + 8 <= A.c.dim && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
                        const float4 a = reinterpret_cast<const float4 *>(src)[0], c = reinterpret_cast<const float4 *>(src)[1];
                        x[j][0] = a.x, x[j][1] = a.y, x[j][2] = a.z, x[j][3] = a.w, x[j][4] = c.x, x[j][5] = c.y, x[j][6] = c.z, x[j][7] = c.w;
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; ++k) x[j][k] = there && 8 * l + k < A.c.dim ? src[k] : 0.0f;
                    }
                }
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    const int r = i0 + j * kAtOnce + lane / kLanes;
                    float big = 0.0f;
                    bool bad = false;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        bad |= !isfinite(x[j][k]);
                        big = fmaxf(big, fabsf(x[j][k]));
                    }
#pragma unroll
                    for (int s = kLanes / 2; s > 0; s >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, s));
                    const unsigned all_bad = __ballot_sync(0xffffffffu, bad);
                    const bool spoilt = (all_bad >> (lane / kLanes * kLanes) & (kLanes == 32 ? 0xffffffffu : (1u << (kLanes & 31)) - 1)) != 0;
                    // a power of two that brings the row's largest value to 2^21 .. 2^22: three signed digits
                    const unsigned field = min(275u - (__float_as_uint(big) >> 23), 253u);
                    const float up = __uint_as_float(field << 23);
                    if (r >= R) continue;
                    // a row with a value that is not finite has no result
                    if (l == 0) M.row_scale[b][r] = spoilt ? __uint_as_float(0x7fc00000u) : __uint_as_float((254u - field) << 23) * A.scale;
                    unsigned d[2][3];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const int v[4] = {__float2int_rn(x[j][4 * k] * up), __float2int_rn(x[j][4 * k + 1] * up),
                                          __float2int_rn(x[j][4 * k + 2] * up), __float2int_rn(x[j][4 * k + 3] * up)};
                        digits_of(v, d[k]);
                    }
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        *reinterpret_cast<uint2 *>(M.q[b][l >> 3] + sw64_byte(3 * r + e, 8 * (l & 7))) = make_uint2(d[0][e], d[1][e]);
                }
                __syncwarp();
            }
            if (lane == 0) M.unit[b] = u;
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
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
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
    // more than half of a multiprocessor's shared memory: one CTA on each
    constexpr size_t kSmem = sizeof(Smem<P, R>) > 120 * 1024 ? sizeof(Smem<P, R>) : 120 * 1024;
    static_assert(kSmem <= 227 * 1024, "fits a multiprocessor");
    RowArgs A;
    static_cast<Args &>(A) = args;
    int slots = 0;
    cudaError_t e = multiprocessors<P, R>(kSmem, &slots);
    if (e != cudaSuccess) return e;
    if (slots > kMaxCtas) slots = kMaxCtas;
    const long long tokens = (long long)A.runs.segments * A.runs.count, units = tokens * A.c.kv_heads * A.tiles;
    if (kv8_short_fits(A, slots)) return kv8_attend_short(A, slots, s);
    if (!page_map(A.c, 64, &A.keys) || !page_map(A.c, P, &A.values)) return cudaErrorInvalidValue;
    A.split = tokens <= kMaxTokens && units < 8LL * slots && units <= 65536;
    const long long most = A.split ? units * (A.picks ? A.top : A.c.blocks) : units;
    e = kv8_launch(k_kv8_rows<P, R>, dim3((unsigned)(most < slots ? most : slots)), dim3(kThreads), kSmem, 1, s, A);
    if (e != cudaSuccess || !A.split) return e;
    return launch_join<P>(A, units, slots, s);
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
