// Attention over the 8-bit paged cache for prompt chunks (strata_kv8_attend, many tokens a run): tiles of
// 128 query rows on the 5th-generation tensor cores (tcgen05 + TMEM).
//
// A tile is 128 consecutive (token, query head) pairs of one run and key/value head, so that groups of any
// size fill it. Its keys and values pass by page by page (64 tokens):
//   S[128][64] = Q K^T     on integer products (kind::i8): a query row, scaled by a power of two, is 23 bits in three
//                          signed 8-bit digits in shared memory, and the keys' codes are taken as they lie in memory; a digit's
//                          sums are whole numbers in TMEM, exact, and join in F32
//   O[128][P] += W V       the weights as two FP16 halves in TMEM, the A operand, against codes converted to FP16 (exact)
// which gives F32's accuracy at three integer passes for the first product and two FP16 passes for the second. (The
// second on integers would want as many sums as weights have digits, more than TMEM holds.) Maxima and sums are F32.
//
// Warps:
//   0-7  softmax: a row (TMEM lane) is two threads', 32 of a page's tokens each: logits from S, running maximum (the two
//        exchange theirs) and sum, weights into TMEM. O is rescaled only when a row's maximum has grown by more than
//        2^5 (weights are kept times 2^10, so that both ends stay inside FP16), so seldom after the first pages
//   8-9  converters: values to FP16 in the 128-byte-swizzled layout of the MMA operands
//   10   fetches keys by TMA (64-byte swizzle) and values by bulk copies
//   11   one thread issues the MMAs: S of page j + 1 before O of page j, so that S's columns are read and free
//        again while O is computed
// A value scale cannot be applied after the product, since pages add up in one accumulator: weights are
// multiplied by scale / (largest scale of the tile's pages), in their exponents, and a row's running reference is that of
// the products. So FP16's steps are 2^-31 of the row's largest product at most, also for rows that see only small scales.
//
// Measured: 2048 tokens over 16384 keys, 24 heads over 2 of 256 channels, 1365 us, 567 TFLOP/s of the two products as they
// are defined, at a page every 3900 clocks a CTA (2.2 us), the tensor pipe busy for 47%. S alone takes 1250 clocks (24
// instructions of 128 x 64 x 32, bound by reading their operands from shared memory) and O 1000; the rest are the hand-overs
// between products and softmax, for which TMEM has no second set of S's columns at 256 channels. The form with queries in FP16 halves and keys converted as well took
// 1546 us, since its converters and operands take twice the shared-memory traffic.
//
// Every wait is bounded; past the limit all roles leave and the error word is set.
#include "kv8_mma.cuh"

#include <atomic>
#include <cmath>

namespace strata {
namespace {

using namespace pf;

constexpr int kSoftWarps = 8, kConvWarps = 2, kKeyWarp = kSoftWarps + kConvWarps, kMmaWarp = kKeyWarp + 1;
constexpr int kPromptThreads = 32 * (kMmaWarp + 1);
constexpr int kConvThreads = 32 * kConvWarps;
constexpr int kTileRows = 128;
constexpr int kDigits = 3;           // of a query
constexpr float kLiftP = 10.0f;      // weights are stored times 2^10
constexpr float kRoomP = 4.0f;       // log2 of a new reference over its maximum: weights begin at 2^6, far above FP16's subnormals
constexpr float kGrow = 5.0f;        // growth of a maximum (log2) that O's scale bears
constexpr long long kLimit = 2000000000;  // clocks, about a second

constexpr int kFlush = 16;           // pages that add up in TMEM before the sum moves to 32-bit adds
constexpr int kScales = 8;           // pages whose scales are kept: more than are fetched ahead of the softmax
// A unit counts as this many pages more when pages are shared: beginning one takes longer than a page. (Without it
// the CTAs of a prompt's first tiles, which have a page or two each, came last: 1497 tokens from the start, 36 heads over 3
// of 64 channels, took 221 us instead of 84; 98 with 3.)
constexpr int kBegin = 6;
constexpr int kMaxGrid = 160;        // CTAs, each with a slot in the workspace
constexpr int kMaxPairs = 1024;      // (run, tile) pairs of a split call
constexpr int kMaxUnits = 65536;

// Pages [first, stop) of the n that a unit (run, tile, key/value head) attends to; n < 0: no piece is left.
struct Piece {
    int run, tile, head;
    int first, stop, n;
};

template <int P>
struct PromptSmem {  // 1024-byte aligned
    static constexpr int k_ring = P == 256 ? 2 : 3, v_ring = k_ring;
    unsigned char q[kDigits][P / 64][kTileRows * 64];  // panels of 64 channels, a row 64 bytes, swizzled
    unsigned char k[k_ring][P * 64];                   // keys [P / 64][64 tokens][64 bytes], swizzled
    unsigned char v[v_ring][P * 128];                  // values as FP16 [P channels][128 bytes], swizzled
    unsigned char raw[v_ring][P * 64];                 // values as they lie in memory
    float row_scale[kTileRows];
    float2 page_scale[kScales];       // of keys (-1: no page) and values, by page
    float half_row[2][2][kTileRows];  // by page's parity and half: what a row's two threads exchange
    float red[kPromptThreads / 32];
    struct Walk {
        long long unit, work, work_end, chunk;
        int pair, head, page, has_tail;
        Piece tail;
    } walk;  // thread 0's
    Piece piece;
    unsigned long long k_full[k_ring], k_empty[k_ring], raw_full[v_ring], raw_empty[v_ring], v_full[v_ring], v_empty[v_ring];
    unsigned long long s_full, s_free, w_full, o_done, o_free, drained;
    unsigned tmem;
    int abort_flag;
};

struct PromptArgs {
    Kv8 c;
    const float *q;
    long long stride;
    int heads, group, tiles;  // tiles of 128 rows a run and key/value head
    Kv8Runs runs;
    float scale;  // times log2 e
    float *y;
    int split;
    CUtensorMap keys;  // boxes of P rows
};
// Workspace: a CTA's sum of more than kFlush pages, or of the part of a unit that an earlier CTA began,
// as [P / 4][128 rows] float4; per row maximum, sum and value scale of such a part and of a begun one (whose sum is
// in y); the CTAs that share a unit.
struct PromptParts {
    float4 *sum;      // [kMaxGrid][P / 4][128]
    float4 *tail_ml;  // [kMaxGrid][128]
    float4 *head_ml;  // [kMaxGrid][128]
    int2 *cover;      // [units]
};
__host__ __device__ inline PromptParts prompt_parts(void *ws, int P) {
    char *p = static_cast<char *>(ws);
    PromptParts r;
    r.sum = reinterpret_cast<float4 *>(p);
    p += (size_t)kMaxGrid * P * kTileRows * 4;
    r.tail_ml = reinterpret_cast<float4 *>(p);
    p += (size_t)kMaxGrid * kTileRows * 16;
    r.head_ml = reinterpret_cast<float4 *>(p);
    p += (size_t)kMaxGrid * kTileRows * 16;
    r.cover = reinterpret_cast<int2 *>(p);
    return r;
}
static_assert((size_t)kMaxGrid * (256 * kTileRows * 4 + 2 * kTileRows * 16) + (size_t)kMaxUnits * 8 <= (32u << 20), "fits the workspace");

// Pages that a tile of a run attends to: those of its last row.
__device__ __forceinline__ int pair_pages(const PromptArgs &A, int run, int tile) {
    const int last = min(A.runs.count * A.group, (tile + 1) * kTileRows) - 1;
    return (visible_keys(A.c, run_at(A.c, A.runs, run), last / A.group) + kKvBlock - 1) / kKvBlock;
}
__device__ __forceinline__ float *prompt_row(const PromptArgs &A, int run, int head, int r) {
    return A.y + (((size_t)run * A.runs.count + r / A.group) * A.heads + head * A.group + r % A.group) * A.c.dim;
}

// 32 TMEM columns of this thread's lane, without the wait.
__device__ __forceinline__ void tmem_ld32_async(unsigned taddr, unsigned (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
        "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
// 16 of them.
__device__ __forceinline__ void tmem_ld16_async(unsigned taddr, unsigned (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// OR of x over a named barrier's two warps.
__device__ __forceinline__ bool pair_or(int barrier, bool x) {
    unsigned r;
    asm volatile(
        "{\n\t.reg .pred pi, po;\n\t"
        "setp.ne.u32 pi, %1, 0;\n\t"
        "bar.red.or.pred po, %2, 64, pi;\n\t"
        "selp.u32 %0, 1, 0, po;\n\t}"
        : "=r"(r)
        : "r"((unsigned)x), "r"(barrier)
        : "memory");
    return r != 0;
}
// A whole number of |x| < 2^22 in two additions: 1.5 * 2^23 + x is the float whose bits are 0x4b400000 + x.
__device__ __forceinline__ float whole_float(unsigned x) { return __uint_as_float(0x4b400000u + x) - 12582912.0f; }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <int P>
__global__ void __launch_bounds__(kPromptThreads, 1) k_kv8_prompt(const __grid_constant__ PromptArgs A) {
    using Sm = PromptSmem<P>;
    extern __shared__ __align__(1024) unsigned char raw[];  // the swizzled operands repeat every 1024 bytes
    Sm &M = *reinterpret_cast<Sm *>(raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int pairs = A.runs.segments * A.tiles;
    const PromptParts W = prompt_parts(A.c.workspace, P);
    kv8_enter();

    // ---- this CTA's work: units (pair, head) blockIdx.x, + gridDim.x, ... or pages [work, work_end) of all units' list
    if (A.split) {
        long long *before = reinterpret_cast<long long *>(M.v[0]);  // used before the ring is
        long long *part = before + kMaxPairs + 1;
        static_assert(sizeof(M.v) >= (kMaxPairs + 1 + kPromptThreads / 32) * 8, "the page counts fit");
        for (int base = 0; base < pairs; base += kPromptThreads) {  // before[i]: a head's pages, and kBegin a unit, before pair i
            long long sum = base + tid < pairs ? pair_pages(A, (base + tid) / A.tiles, (base + tid) % A.tiles) : 0;
            if (sum) sum += kBegin;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const long long o = __shfl_up_sync(0xffffffffu, sum, s);
                if (lane >= s) sum += o;
            }
            if (lane == 31) part[warp] = sum;
            __syncthreads();
            long long carry = base ? before[base] : 0;
            for (int w = 0; w < warp; ++w) carry += part[w];
            if (base == 0 && tid == 0) before[0] = 0;
            if (base + tid < pairs) before[base + tid + 1] = carry + sum;
            __syncthreads();
        }
        const long long total = before[pairs] * A.c.kv_heads, chunk = (total + gridDim.x - 1) / gridDim.x, work = chunk * blockIdx.x;
        if (work >= total) return;
        if (tid == 0) {
            int lo = 0, hi = pairs - 1;
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (before[mid + 1] * A.c.kv_heads > work) hi = mid;
                else lo = mid + 1;
            }
            const long long n = before[lo + 1] - before[lo], in = work - before[lo] * A.c.kv_heads;
            M.walk.work = work;
            M.walk.work_end = min(total, work + chunk);
            M.walk.chunk = chunk;
            M.walk.pair = lo;
            M.walk.head = (int)(in / n);
            M.walk.page = (int)(in % n);
        }
    }
    if (tid == 0) {
        for (int i = 0; i < Sm::k_ring; ++i) bar_init(&M.k_full[i], 1), bar_init(&M.k_empty[i], 1);
        for (int i = 0; i < Sm::v_ring; ++i) bar_init(&M.v_full[i], kConvThreads), bar_init(&M.v_empty[i], 1);
        for (int i = 0; i < Sm::v_ring; ++i) bar_init(&M.raw_full[i], 1), bar_init(&M.raw_empty[i], kConvWarps);
        bar_init(&M.s_full, 1), bar_init(&M.s_free, 32 * kSoftWarps);
        bar_init(&M.w_full, 32 * kSoftWarps), bar_init(&M.o_done, 1);
        bar_init(&M.o_free, 32 * kSoftWarps);
        bar_init(&M.drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        M.abort_flag = 0;
        M.walk.unit = blockIdx.x;
        M.walk.has_tail = 0;
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&M.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = M.tmem;
    auto wait = [&](unsigned long long *b, unsigned parity) -> bool {
        for (const long long began = clock64();;) {
            if (bar_try(b, parity)) return true;
            if (*(volatile int *)&M.abort_flag) return false;
            if (clock64() - began > kLimit) {
                atomicOr(&M.abort_flag, 1);
                return false;
            }
        }
    };

    // The next piece of the CTA's work (thread 0). The part of a unit that an earlier CTA began comes last: its
    // sum stays in the CTA's workspace slot, which the other pieces use in passing.
    auto next = [&]() {
        auto &w = M.walk;
        Piece p{0, 0, 0, 0, 0, -1};
        if (!A.split) {
            if (w.unit < (long long)pairs * A.c.kv_heads) {
                const int a_tile = A.runs.segments * A.c.kv_heads, rest = (int)(w.unit % a_tile);  // the tiles with the most keys first
                p.tile = A.tiles - 1 - (int)(w.unit / a_tile);
                p.run = rest / A.c.kv_heads;
                p.head = rest % A.c.kv_heads;
                p.n = p.stop = pair_pages(A, p.run, p.tile);
                w.unit += gridDim.x;
            }
            M.piece = p;
            return;
        }
        while (w.work < w.work_end) {
            p.run = w.pair / A.tiles;
            p.tile = w.pair % A.tiles;
            p.head = w.head;
            p.n = pair_pages(A, p.run, p.tile);
            if (p.n == 0) {  // nothing in sight: the joining kernel writes the zeros
                ++w.pair;
                continue;
            }
            if (w.page < kBegin) {  // the CTA that has the first page begins the unit
                w.work += kBegin - w.page;
                w.page = kBegin;
                continue;
            }
            p.first = w.page - kBegin;
            p.stop = (int)min((long long)p.n, p.first + (w.work_end - w.work));
            if (p.first == 0) W.cover[w.pair * A.c.kv_heads + w.head] = make_int2(blockIdx.x, (int)((w.work + p.n - 1) / w.chunk));
            w.work += p.stop - p.first;
            w.page = 0;
            if (++w.head == A.c.kv_heads) {
                w.head = 0;
                ++w.pair;
            }
            if (p.first == 0) {
                M.piece = p;
                return;
            }
            w.tail = p;
            w.has_tail = 1;
        }
        if (w.has_tail) M.piece = w.tail;
        else M.piece.n = -1;
        w.has_tail = 0;
    };

    // counters that go on from piece to piece
    int pages = 0, flushes = 0;
    for (;;) {
        if (tid == 0) next();
        __syncthreads();
        const Piece p = M.piece;
        if (p.n < 0) break;
        const RunAt at = run_at(A.c, A.runs, p.run);
        const int row0 = p.tile * kTileRows, rows = min(kTileRows, A.runs.count * A.group - row0), n = p.stop - p.first, head = p.head;
        if (n == 0) {  // no row of the tile sees a key
            for (int i = tid; i < rows * A.c.dim; i += kPromptThreads) prompt_row(A, p.run, head, row0 + i / A.c.dim)[i % A.c.dim] = 0.0f;
            __syncthreads();
            continue;
        }
        // the table's entry of local page j, to be looked at an iteration later
        const int *table = A.c.table + (size_t)at.sequence * A.c.blocks + p.first;
        auto entry_at = [&](int j) { return j < n ? table[j] : -1; };
        auto checked = [&](int j, int page) {  // an entry of a page that is needed
            if (page >= 0 && page < A.c.pages) return page;
            if (j < n) raise_error(A.c.err, kErrIndex);
            return -1;
        };
        auto scales_of = [&](int page) {
            const float *s = page >= 0 ? page_scales(A.c, page, head) : nullptr;
            return s ? make_float2(s[0], s[1]) : make_float2(-1.0f, 0.0f);
        };
        const int first_page = tid < p.n ? page_of(A.c, at.sequence, tid) : -1;
        const float first_most = first_page >= 0 ? page_scales(A.c, first_page, head)[1] : 0.0f;
        // queries: a row is P / 8 lanes of 8 channels; scaled by a power of two to 2^21 .. 2^22 at most
        {
            constexpr int kLanes = P / 8, kAtOnce = 32 / kLanes;
            const int l = lane % kLanes, ch0 = 8 * l;
            for (int i = warp * kAtOnce + lane / kLanes; i < kTileRows; i += kPromptThreads / 32 * kAtOnce) {
                float x[8], big = 0.0f;
                const int r = row0 + i;
                const float *src = A.q + (p.run * (long long)A.runs.count + r / A.group) * A.stride + (size_t)(head * A.group + r % A.group) * A.c.dim + ch0;
                if (i < rows && ch0 + 8 <= A.c.dim && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
                    const float4 a = reinterpret_cast<const float4 *>(src)[0], b = reinterpret_cast<const float4 *>(src)[1];
                    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k) x[k] = i < rows && ch0 + k < A.c.dim ? src[k] : 0.0f;
                }
                bool bad = false;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    bad |= !isfinite(x[k]);
                    big = fmaxf(big, fabsf(x[k]));
                }
#pragma unroll
                for (int s = kLanes / 2; s > 0; s >>= 1) {
                    big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, s));
                    bad |= __shfl_xor_sync(0xffffffffu, (int)bad, s) != 0;
                }
                const unsigned field = min(275u - (__float_as_uint(big) >> 23), 253u);
                const float up = copysignf(__uint_as_float(field << 23), A.scale);
                // a row with a value that is not finite has no result
                if (l == 0) M.row_scale[i] = bad ? __uint_as_float(0x7fc00000u) : __uint_as_float((254u - field) << 23) * fabsf(A.scale);
                unsigned d[2][kDigits];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int v[4] = {__float2int_rn(x[4 * k] * up), __float2int_rn(x[4 * k + 1] * up), __float2int_rn(x[4 * k + 2] * up),
                                      __float2int_rn(x[4 * k + 3] * up)};
                    digits_of(v, d[k]);
                }
#pragma unroll
                for (int e = 0; e < kDigits; ++e)
                    *reinterpret_cast<uint2 *>(M.q[e][l >> 3] + sw64_byte(i, 8 * (l & 7))) = make_uint2(d[0][e], d[1][e]);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        // the largest value scale of the unit's pages
        float most = first_most;
        for (int j = tid + kPromptThreads; j < p.n; j += kPromptThreads) {
            const int page = page_of(A.c, at.sequence, j);
            if (page >= 0) most = fmaxf(most, page_scales(A.c, page, head)[1]);
        }
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, s));
        if (lane == 0) M.red[warp] = most;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPromptThreads / 32; ++i) most = fmaxf(most, M.red[i]);

        if (warp < kSoftWarps) {
            // ---------------------------------------------------------------- softmax
            const int half = warp >> 2, i = (warp & 3) * 32 + lane;
            const int in_sight = i < rows ? visible_keys(A.c, at, (row0 + i) / A.group) : 0;
            const int seen = in_sight - p.first * kKvBlock - 32 * half;  // from this half of the first page on
            const unsigned mine = tmem + ((unsigned)((warp & 3) * 32) << 16), cols = mine + P + 64 * kDigits + 16 * half;  // O, and the weights
            const float row_scale = in_sight ? M.row_scale[i] : 0.0f, over = most > 0.0f ? __fdiv_rn(1.0f, most) : 0.0f;
            float4 *kept = W.sum + (size_t)blockIdx.x * (P / 4) * kTileRows + i;  // this row's sum of flushed pages, every 128th
            float m = -INFINITY, sum = 0.0f, kept_m = -INFINITY;
            bool ok = true;
            // The two warps of 32 rows meet at a vote; they leave at the same one, which a warp whose wait has failed still comes to.
            auto vote = [&](bool x) -> bool { return pair_or(1 + (warp & 3), x); };
            auto leave = [&]() -> bool { return vote(!ok || *(volatile int *)&M.abort_flag); };
            bool gone = false;
            // O of local page j's group, complete, joins the kept sum
            auto flush = [&](int j) -> bool {
                if (!__all_sync(0xffffffffu, wait(&M.o_done, (pages + j) & 1))) return false;
                tc_fence_after();
                const bool fresh = j < kFlush;
                const float alpha = fresh || kept_m >= m ? 1.0f : exp2_fast(kept_m - m);
                kept_m = m;
                const bool scaled = __any_sync(0xffffffffu, alpha != 1.0f);  // seldom: else the sum is added where it lies
#pragma unroll 1
                for (int k = half * (P / 2); k < (half + 1) * (P / 2); k += 16) {
                    unsigned x[16];
                    float4 f[4];
                    tmem_ld16_async(mine + k, x);
                    if (scaled) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) f[e] = __ldcg(kept + (k / 4 + e) * kTileRows);
                    }
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float4 o = make_float4(__uint_as_float(x[4 * e]), __uint_as_float(x[4 * e + 1]), __uint_as_float(x[4 * e + 2]),
                                               __uint_as_float(x[4 * e + 3]));
                        if (scaled) o = make_float4(f[e].x * alpha + o.x, f[e].y * alpha + o.y, f[e].z * alpha + o.z, f[e].w * alpha + o.w);
                        if (fresh || scaled) kept[(k / 4 + e) * kTileRows] = o;
                        else atomicAdd(kept + (k / 4 + e) * kTileRows, o);  // (this thread alone adds to it)
                    }
                }
                tc_fence_before();
                bar_arrive(&M.o_free);
                return true;
            };
            for (int j = 0; j < n; ++j) {
                const int g = pages + j;
                ok = ok && __all_sync(0xffffffffu, wait(&M.s_full, g & 1));
                tc_fence_after();
                const float2 sc = M.page_scale[g % kScales];
                const int left = sc.x >= 0.0f ? seen - j * kKvBlock : 0;
                float a[32];  // digits' sums joined: logits but for the positive factor c
                {
                    unsigned x[kDigits][32];
#pragma unroll
                    for (int e = 0; e < kDigits; ++e) tmem_ld32_async(mine + P + 64 * e + 32 * half, x[e]);
                    tmem_wait_ld();
                    tc_fence_before();
                    bar_arrive(&M.s_free);
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        a[e] = __fmaf_rn(whole_float(x[2][e]), 65536.0f, (float)((int)x[1][e] * 256 + (int)x[0][e]));
                }
                // a positive factor, so that -infinity stays that; what would be below this makes logits of 0
                const float c = isnan(row_scale) ? row_scale : fmaxf(sc.x * row_scale, 1e-30f);
                // weights take the page's value scale over the tile's largest in the exponent, and a row's reference is that of
                // its largest weight so taken: its weights begin at 2^6 whatever scales other rows' pages have. Values of
                // a scale below 2^-90 of the largest, none among them, count as none
                const float by_v = sc.y * over, fv = fmaxf(by_v, 0x1p-90f), lift = log2f(fv);
                if (__any_sync(0xffffffffu, left < 32)) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) a[k] = k < left ? a[k] : -INFINITY;
                }
                float big[4] = {a[0], a[1], a[2], a[3]};
#pragma unroll
                for (int k = 4; k < 32; ++k) big[k & 3] = fmaxf(big[k & 3], a[k]);
                float top = fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3]));
                top = top * c + lift;
                bool due = j > 0 && j % kFlush == 0;  // the group of pages before this one is to be kept
                if (vote(!ok || top > m + kGrow)) {  // seldom
                    M.half_row[j & 1][half][i] = top;
                    if ((gone = leave())) break;
                    top = fmaxf(top, M.half_row[j & 1][half ^ 1][i]);
                    if (due) {
                        if (!(ok = flush(j - 1))) continue;
                        due = false;
                    }
                    const float now = top > m ? top + kRoomP : m, alpha = now > m ? exp2_fast(m - now) : 1.0f;
                    m = now;
                    sum *= alpha;
                    if (j % kFlush) {
                        if (!(ok = __all_sync(0xffffffffu, wait(&M.o_done, (g - 1) & 1)))) continue;
                        tc_fence_after();
#pragma unroll 1
                        for (int k = half * (P / 2); k < (half + 1) * (P / 2); k += 16) {
                            unsigned x[16];
                            tmem_ld16_async(mine + k, x);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * alpha);
                            tmem_st16(mine + k, x);
                        }
                    }
                }
                const float from = kLiftP - ((m == -INFINITY ? 0.0f : m) - lift);
                float add[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                unsigned hi[16], lo[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float p0 = exp2_fast(__fmaf_rn(a[2 * e], c, from)), p1 = exp2_fast(__fmaf_rn(a[2 * e + 1], c, from));
                    add[(2 * e) & 3] += p0;
                    add[(2 * e + 1) & 3] += p1;
                    split_pair(p0, p1, hi[e], lo[e]);
                }
                if (by_v < 0x1p-90f) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) hi[e] = lo[e] = 0;
                }
                if (g > 0 && !(ok = __all_sync(0xffffffffu, wait(&M.o_done, (g - 1) & 1)))) continue;  // the weights before are used
                tc_fence_after();
                tmem_st16(cols, hi);
                tmem_st16(cols + 32, lo);
                sum += __fdividef((add[0] + add[1]) + (add[2] + add[3]), fv);
                tmem_wait_st();
                tc_fence_before();
                bar_arrive(&M.w_full);
                if (due) ok = flush(j - 1);
            }
            if (!gone) {
                M.half_row[n & 1][half][i] = sum;
                gone = leave();
            }
            if (!gone && (ok = __all_sync(0xffffffffu, wait(&M.o_done, (pages + n - 1) & 1)))) {
                sum += M.half_row[n & 1][half ^ 1][i];
                tc_fence_after();
                const bool whole = n == p.n, flushed = n > kFlush;
                const float inv = !whole ? 1.0f : sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum), by = whole ? most : 1.0f;
                const float alpha = !flushed || kept_m >= m ? 1.0f : exp2_fast(kept_m - m);
                float *dst = i < rows ? prompt_row(A, p.run, head, row0 + i) : nullptr;
                const bool wide = (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
                if (!whole && half == 0) (p.first ? W.tail_ml : W.head_ml)[blockIdx.x * kTileRows + i] = make_float4(m, sum, most, 0.0f);
#pragma unroll 1
                for (int k = half * (P / 2); k < (half + 1) * (P / 2); k += 32) {
                    unsigned x[32];
                    float4 f[8];
                    __syncwarp();
                    tmem_ld32_async(mine + k, x);
                    if (flushed) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[e] = __ldcg(kept + (k / 4 + e) * kTileRows);
                    }
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float4 o = make_float4(__uint_as_float(x[4 * e]), __uint_as_float(x[4 * e + 1]), __uint_as_float(x[4 * e + 2]),
                                               __uint_as_float(x[4 * e + 3]));
                        if (flushed) o = make_float4(f[e].x * alpha + o.x, f[e].y * alpha + o.y, f[e].z * alpha + o.z, f[e].w * alpha + o.w);
                        if (p.first) {
                            kept[(k / 4 + e) * kTileRows] = o;
                        } else if (dst) {
                            const int ch = k + 4 * e;
                            o = make_float4(o.x * inv * by, o.y * inv * by, o.z * inv * by, o.w * inv * by);
                            if (wide && ch + 4 <= A.c.dim) {
                                *reinterpret_cast<float4 *>(dst + ch) = o;
                            } else {
                                if (ch < A.c.dim) dst[ch] = o.x;
                                if (ch + 1 < A.c.dim) dst[ch + 1] = o.y;
                                if (ch + 2 < A.c.dim) dst[ch + 2] = o.z;
                                if (ch + 3 < A.c.dim) dst[ch + 3] = o.w;
                            }
                        }
                    }
                }
            }
        } else if (warp < kKeyWarp) {
            // ---------------------------------------------------------------- converters
            // piece w of a page's values is codes 16 (w % 4) .. of row w / 4, two swizzled 16-byte chunks of FP16
            const int ct = tid - 32 * kSoftWarps;
            for (int j = 0; j < n; ++j) {
                const int g = pages + j, s = g % Sm::v_ring;
                const unsigned turn = g / Sm::v_ring & 1;
                if (!__all_sync(0xffffffffu, wait(&M.raw_full[s], turn) && wait(&M.v_empty[s], turn ^ 1))) break;
#pragma unroll 8
                for (int piece = ct; piece < P * 4; piece += kConvThreads) {
                    const int row = piece >> 2, ch = (piece & 3) * 2;
                    const uint4 w = reinterpret_cast<const uint4 *>(M.raw[s])[piece];
                    uint4 x, z;
                    codes_to_half(w.x, x.x, x.y);
                    codes_to_half(w.y, x.z, x.w);
                    codes_to_half(w.z, z.x, z.y);
                    codes_to_half(w.w, z.z, z.w);
                    unsigned char *dst = M.v[s] + row * 128;
                    *reinterpret_cast<uint4 *>(dst + ((ch ^ (row & 7)) << 4)) = x;
                    *reinterpret_cast<uint4 *>(dst + (((ch + 1) ^ (row & 7)) << 4)) = z;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                bar_arrive(&M.v_full[s]);
                __syncwarp();
                if (lane == 0) bar_arrive(&M.raw_empty[s]);
            }
        } else if (warp == kKeyWarp) {
            // ---------------------------------------------------------------- keys and values
            // 32 pages at a time, a page a lane, the next ones looked up on the way
            int next_page = checked(lane, entry_at(lane));
            float2 next_scale = scales_of(next_page);
            bool ok = true;
            int asked[2] = {0, 0};
            for (int base = 0; base < n && ok; base += 32) {
                const int page = next_page;
                const float2 scale = next_scale;
                next_page = checked(base + 32 + lane, entry_at(base + 32 + lane));
                next_scale = scales_of(next_page);
                for (int e = 0; e < min(32, n - base); ++e) {
                    const int g = pages + base + e, k = g % Sm::k_ring, v = g % Sm::v_ring, at_page = __shfl_sync(0xffffffffu, page, e);
                    if (!(ok = __all_sync(0xffffffffu, wait(&M.k_empty[k], (g / Sm::k_ring & 1) ^ 1)))) break;
                    if (lane == 0 && at_page >= 0) {  // (no key of a page that is not there is in sight: what lies in the rings has no weight)
                        asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(su32(&M.k_full[k])), "r"(P * kKvBlock) : "memory");
                        tma3(M.k[k], &A.keys, 0, head * 2 * P, at_page, &M.k_full[k]);
                    }
                    __syncwarp();
                    if (lane == e) {
                        M.page_scale[g % kScales] = scale;
                        bar_arrive(&M.k_full[k]);
                    }
                    ++asked[0];
                    if (!(ok = __all_sync(0xffffffffu, wait(&M.raw_empty[v], (g / Sm::v_ring & 1) ^ 1)))) break;
                    if (lane == 0) {
                        if (at_page >= 0) {
                            bar_expect(&M.raw_full[v], P * kKvBlock);
                            bulk(M.raw[v], page_codes(A.c, at_page, head, 1), P * kKvBlock, &M.raw_full[v]);
                        } else {
                            bar_arrive(&M.raw_full[v]);
                        }
                    }
                    ++asked[1];
                }
            }
            if (*(volatile int *)&M.abort_flag) {  // what was asked for lands before the CTA leaves
                auto land = [&](unsigned long long *bars, int ring, int count) {
                    for (int a = max(0, count - ring); a < count; ++a)
                        for (const long long began = clock64(); !bar_try(&bars[(pages + a) % ring], (pages + a) / ring & 1) && clock64() - began < kLimit;) {
                        }
                };
                land(M.k_full, Sm::k_ring, asked[0]);
                land(M.raw_full, Sm::v_ring, asked[1]);
            }
        } else {
            // ---------------------------------------------------------------- MMA issuer
            const unsigned id_s = idesc_i8(kKvBlock, true), id_o = idesc_f16(kTileRows, P);
            int freed = flushes;
            bool ok = true;
            auto scores = [&](int j) {
                const int g = pages + j, s = g % Sm::k_ring;
                ok = ok && __all_sync(0xffffffffu, wait(&M.k_full[s], g / Sm::k_ring & 1));
                if (ok && g > 0) ok = __all_sync(0xffffffffu, wait(&M.s_free, (g - 1) & 1));
                if (!ok) return;
                tc_fence_after();
                if (elect_one()) {
#pragma unroll
                    for (int e = 0; e < kDigits; ++e)
#pragma unroll
                        for (int b = 0; b < P / 64; ++b) {
                            const unsigned long long qd = sw64_desc(su32(M.q[e][b])), kd = sw64_desc(su32(M.k[s] + b * 4096));
#pragma unroll
                            for (int k = 0; k < 2; ++k) mma_i8(tmem + P + 64 * e, qd + 2 * k, kd + 2 * k, id_s, b > 0 || k > 0);
                        }
                    mma_commit(&M.k_empty[s]);
                    mma_commit(&M.s_full);
                }
                __syncwarp();
            };
            scores(0);
            for (int j = 0; j < n && ok; ++j) {
                if (j + 1 < n) scores(j + 1);
                const int g = pages + j, s = g % Sm::v_ring;
                ok = ok && __all_sync(0xffffffffu, wait(&M.v_full[s], g / Sm::v_ring & 1) && wait(&M.w_full, g & 1));
                if (ok && j > 0 && j % kFlush == 0) ok = __all_sync(0xffffffffu, wait(&M.o_free, freed++ & 1));
                if (!ok) break;
                tc_fence_after();
                const unsigned w = tmem + P + 64 * kDigits;
                const unsigned long long vd = sw128_desc(su32(M.v[s]));
                if (elect_one()) {
                    // the low halves first: the accumulator is then small, and what an addition drops as well
#pragma unroll
                    for (int h = 1; h >= 0; --h)
#pragma unroll
                        for (int k = 0; k < 4; ++k) mma_f16_ts(tmem, w + 32 * h + 8 * k, vd + 2 * k, id_o, j % kFlush > 0 || k > 0 || h == 0);
                    mma_commit(&M.v_empty[s]);
                    mma_commit(&M.o_done);
                }
                __syncwarp();
            }
        }
        pages += n;
        flushes += (n - 1) / kFlush;
        tc_fence_before();
        __syncthreads();  // the piece is done: its queries, its S and O are free
        tc_fence_after();
        if (*(volatile int *)&M.abort_flag) break;
    }
    __syncthreads();
    if (tid == 0 && M.abort_flag) raise_error(A.c.err, kErrWaitTimeout);
    // every MMA issued must complete before TMEM is released, whether or not the others have given up
    if (warp == kMmaWarp && lane == 0) {
        mma_commit(&M.drained);
        for (const long long began = clock64(); !bar_try(&M.drained, 0) && clock64() - began < kLimit;) {
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Joins the parts of a unit that several CTAs worked on: the begun one in y and the tails in the workspace, all of
// them sums of 2^(logit - m_i) v / most; 32 rows of a tile a block. A warp's lanes are 32 rows in the tails, as they lie
// there, and 32 channels of a row in y; the tails' sum turns in shared memory.
template <int P>
__global__ void __launch_bounds__(256) k_kv8_prompt_join(const __grid_constant__ PromptArgs A) {
    __shared__ float4 tails[P / 4][33];
    __shared__ float2 by[32];  // of a row: what its part in y and what the tails' sum is taken by
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, unit = blockIdx.x, pair = unit / A.c.kv_heads, head = unit % A.c.kv_heads;
    const int run = pair / A.tiles, tile = pair % A.tiles, first = blockIdx.y * 32, i = first + lane;
    const int rows = min(32, A.runs.count * A.group - tile * kTileRows - first);  // of this block, none or fewer at the end
    kv8_enter();
    if (rows <= 0) return;
    const int n = pair_pages(A, run, tile);
    if (n == 0) {
        for (int r = warp; r < rows; r += 8) {
            float *dst = prompt_row(A, run, head, tile * kTileRows + first + r);
            for (int ch = lane; ch < A.c.dim; ch += 32) dst[ch] = 0.0f;
        }
        return;
    }
    const PromptParts W = prompt_parts(A.c.workspace, P);
    const int2 cover = W.cover[unit];
    if (cover.x == cover.y) return;
    float m = -INFINITY;
    if (lane < rows) {
        const float4 begun = W.head_ml[cover.x * kTileRows + i];
        m = begun.x;
        for (int c = cover.x + 1; c <= cover.y; ++c) m = fmaxf(m, W.tail_ml[c * kTileRows + i].x);
        if (m == -INFINITY) m = 0.0f;
        if (warp == 0) {
            const float w0 = exp2_fast(begun.x - m);
            float sum = begun.y * w0;
            for (int c = cover.x + 1; c <= cover.y; ++c) {
                const float4 t = W.tail_ml[c * kTileRows + i];
                sum += t.y * exp2_fast(t.x - m);
            }
            const float inv = (sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum)) * begun.z;
            by[lane] = make_float2(w0 * inv, inv);
        }
        float4 o[P / 32] = {};
        for (int c = cover.x + 1; c <= cover.y; ++c) {
            const float w = exp2_fast(W.tail_ml[c * kTileRows + i].x - m);
#pragma unroll
            for (int j = 0; j < P / 32; ++j) {
                const float4 f = W.sum[((size_t)c * (P / 4) + 8 * j + warp) * kTileRows + i];
                o[j].x += f.x * w, o[j].y += f.y * w, o[j].z += f.z * w, o[j].w += f.w * w;
            }
        }
#pragma unroll
        for (int j = 0; j < P / 32; ++j) tails[8 * j + warp][lane] = o[j];
    }
    __syncthreads();
    for (int r = warp; r < rows; r += 8) {
        float *dst = prompt_row(A, run, head, tile * kTileRows + first + r);
        const float2 w = by[r];
#pragma unroll
        for (int j = 0; j < P / 32; ++j) {
            const int ch = 32 * j + lane;
            if (ch < A.c.dim) dst[ch] = dst[ch] * w.x + reinterpret_cast<const float *>(&tails[ch / 4][r])[ch % 4] * w.y;
        }
    }
}

template <int P>
cudaError_t launch(PromptArgs A, cudaStream_t s) {
    // at least half of an SM's shared memory: two CTAs on one SM would wait for each other's TMEM
    constexpr size_t kSmem = sizeof(PromptSmem<P>) > 120 * 1024 ? sizeof(PromptSmem<P>) : 120 * 1024;
    static_assert(kSmem <= 227 * 1024, "fits an SM");
    int device = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k_kv8_prompt<P>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
    if (e != cudaSuccess) return e;
    if (!page_map(A.c, P, &A.keys)) return cudaErrorInvalidValue;
    const long long pairs = (long long)A.tiles * A.runs.segments, units = pairs * A.c.kv_heads;
    const int most = sms < kMaxGrid ? sms : kMaxGrid;
    // Units shared page by page where whole ones would leave the last round of CTAs uneven
    A.split = pairs <= kMaxPairs && units <= kMaxUnits && units < 8LL * most;
    const long long work = A.split ? units * A.c.blocks : units;
    e = kv8_launch(k_kv8_prompt<P>, dim3((unsigned)(work < most ? work : most)), dim3(kPromptThreads), kSmem, 1, s, A);
    if (e != cudaSuccess || !A.split) return e;
    return kv8_launch(k_kv8_prompt_join<P>, dim3((unsigned)units, kTileRows / 32), dim3(256), 0, 1, s, A);
}

}  // namespace

cudaError_t kv8_attend_prompt(const Kv8 &c, const float *q, long long stride, int heads, const Kv8Runs &r, float scale, float *y, cudaStream_t s) {
    const int group = heads / c.kv_heads;
    const long long rows = (long long)r.count * group;
    const PromptArgs A{c, q, stride, heads, group, (int)((rows + kTileRows - 1) / kTileRows), r, scale * 1.4426950408889634f, y, 0, {}};
    if (c.padded == 64) return launch<64>(A, s);
    if (c.padded == 128) return launch<128>(A, s);
    return launch<256>(A, s);
}

}  // namespace strata
