// Attention over the 8-bit paged cache, token by token, where units have few pages on a CTA or little to read a query row.
//
// The same sums as the form on tcgen05, on 16-row tiles of mma.sync (m16n8k16), whose products answer at once: no tensor
// maps, no TMEM, no digits to prepare, two CTAs a multiprocessor. A unit is one token and key/value head with up to 16
// of its group's query heads.
//   * a page's keys and values of one head are 2 * P * 64 contiguous bytes, fetched by bulk copies
//     into a ring of stages;
//   * S = Q K^T: warp w takes channel panel w % (P / 64) and a slice of the tokens. Q is held in
//     registers as two FP16 halves (query = hi + lo after a power-of-two scaling of its row), the codes
//     are exact in FP16, so two products give S to F32's accuracy. The panels' partial sums go through
//     shared memory;
//   * softmax: 16 lanes a row; running maximum and sum in F32; the weights, times 2^14 to keep small ones
//     out of FP16's subnormals, are split into halves like the queries;
//   * O = alpha O + scale_v (P V): warp w takes P / 8 channels over all 64 tokens.
// The page layouts are the fragment orders: 16 consecutive bytes of a key row (channels) or of a
// value row (tokens) are one lane's operands of four k-steps, the k order being the same on both sides.
// The pages of all units form one list that the CTAs share evenly, as in the other form.
//
// Bound by latency, not by bytes: a page is a copy, a product, a softmax and a product one after the other, with two
// block barriers (about 1.5 us a page and CTA), before that the look-ups and after it the joining kernel. Measured for
// 24 query heads over 2 key/value heads of 256 channels: one session of 2048 tokens 14.2 us (18.6 by the other form),
// 16 sessions with 32 picked blocks each 24.8 us (34.0), 1.3 TB/s.
#include "kv8_rows.cuh"

#include <atomic>

namespace strata {
namespace {

using namespace kv8_rows;

constexpr int kThreads = 256;
constexpr int kList = 256;        // pages looked up at a time
constexpr int kSRow = 72, kPRow = 72;
constexpr float kLift = 14.0f;    // weights are stored times 2^14
constexpr long long kWaitClocks = 2000000000;  // about a second

template <int P>
struct Shape {
    static constexpr int panels = P / 64;
    static constexpr int slices = 8 / panels;        // token slices in S
    static constexpr int s_tiles = 64 / slices / 8;  // 8-token tiles of a warp in S
    static constexpr int o_tiles = P / 64;           // 8-channel tiles of a warp in O
    static constexpr int stages = P == 256 ? 2 : P == 128 ? 4 : 6;
};
template <int P>
struct __align__(128) Smem {
    int8_t page[Shape<P>::stages][2][P * kKvBlock];
    float s[Shape<P>::panels][kRows][kSRow];
    __half p[2][kRows][kPRow];
    float alpha[kRows], row_scale[kRows], row_max[Shape<P>::panels][kRows];
    int list_page[kList], list_block[kList];
    float2 list_scale[kList];
    long long before[kMaxTokens + 1];
    long long warp_sum[kThreads / 32];
    unsigned long long k_full[Shape<P>::stages], v_full[Shape<P>::stages];
};

__device__ __forceinline__ unsigned saddr(const void *p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void fetch(void *dst, const void *src, unsigned bytes, unsigned long long *bar) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(saddr(bar)), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(saddr(dst)), "l"(src),
                 "r"(bytes), "r"(saddr(bar))
                 : "memory");
}
// Waits for a stage, within a limit.
__device__ __forceinline__ bool landed(unsigned long long *bar, unsigned parity) {
    for (const long long began = clock64(); clock64() - began < kWaitClocks;) {
        unsigned ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(saddr(bar)), "r"(parity)
            : "memory");
        if (ok) return true;
    }
    return false;
}
__device__ __forceinline__ void mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int P>
__global__ void __launch_bounds__(kThreads, 2) k_kv8_short(const __grid_constant__ Args A) {
    using Z = Shape<P>;
    extern __shared__ unsigned char smem_raw[];
    Smem<P> &M = *reinterpret_cast<Smem<P> *>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int tokens = A.runs.segments * A.runs.count, per_token = A.c.kv_heads * A.tiles;
    if (tid == 0) {
        for (int i = 0; i < Z::stages; ++i) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(saddr(&M.k_full[i])) : "memory");
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(saddr(&M.v_full[i])) : "memory");
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    kv8_enter();

    // this CTA's pages [work, work_end) of the list of all units' pages
    long long work = 0, work_end = 0, chunk = 1;
    int token = 0, sub = 0, entry = 0;
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
    chunk = (total + gridDim.x - 1) / gridDim.x;
    work = chunk * blockIdx.x;
    work_end = min(total, work + chunk);
    if (work >= work_end) return;
    int lo = 0, hi = tokens - 1;  // the token whose entries hold `work`
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (M.before[mid + 1] * per_token > work) hi = mid;
        else lo = mid + 1;
    }
    token = lo;
    const long long n = M.before[token + 1] - M.before[token], in = work - M.before[token] * per_token;
    sub = (int)(in / n);
    entry = (int)(in % n);

    unsigned fetched = 0;            // pages walked so far: the stage and parity of the next
    unsigned asked[2] = {0, 0};      // thread 0: key and value copies asked for
    bool ok = true;
    for (;;) {
        int sequence, seen;
        const int n = entries(A, token, &sequence, &seen), nb = (seen + kKvBlock - 1) / kKvBlock;
        const int head = sub / A.tiles, row0 = sub % A.tiles * kRows, rows = min(kRows, A.group - row0);
        const int stop = (int)min((long long)n, entry + (work_end - work));

        // queries of rows g and g + 8, channels 16 t .. of this warp's panel
        const int panel = warp % Z::panels, slice = warp / Z::panels;
        unsigned qh[4][4], ql[4][4];
        {
            float x[2][16], big[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = g + 8 * r, ch0 = panel * 64 + 16 * t;
                const float *src = A.q + (long long)token * A.stride + (size_t)(head * A.group + row0 + row) * A.c.dim + ch0;
                big[r] = 0.0f;
                if (row < rows && ch0 + 16 <= A.c.dim && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float4 f = reinterpret_cast<const float4 *>(src)[i];
                        x[r][4 * i] = f.x, x[r][4 * i + 1] = f.y, x[r][4 * i + 2] = f.z, x[r][4 * i + 3] = f.w;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[r][i] = row < rows && ch0 + i < A.c.dim ? src[i] : 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) big[r] = fmaxf(big[r], fabsf(x[r][i]));
                big[r] = fmaxf(big[r], __shfl_xor_sync(0xffffffffu, big[r], 1));
                big[r] = fmaxf(big[r], __shfl_xor_sync(0xffffffffu, big[r], 2));
                if (t == 0 && slice == 0) M.row_max[panel][row] = big[r];
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float b = 0.0f;
#pragma unroll
                for (int i = 0; i < Z::panels; ++i) b = fmaxf(b, M.row_max[i][g + 8 * r]);
                // a power of two that brings the row's largest value to 2^9 .. 2^10
                const unsigned field = min(263u - (__float_as_uint(b) >> 23), 253u);
                const float up = __uint_as_float(field << 23);
                if (warp == 0 && t == 0) M.row_scale[g + 8 * r] = __uint_as_float((254u - field) << 23) * A.scale;
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    split_pair(x[r][4 * s] * up, x[r][4 * s + 1] * up, qh[s][r], ql[s][r]);
                    split_pair(x[r][4 * s + 2] * up, x[r][4 * s + 3] * up, qh[s][2 + r], ql[s][2 + r]);
                }
            }
        }

        float m = -INFINITY, sum = 0.0f;  // of row 2 warp + lane / 16; the sum over this lane's four tokens of each page
        const int srow = warp * 2 + (lane >> 4), stok = (lane & 15) * 4;
        float o[Z::o_tiles][4] = {};
        for (int base = entry; base < stop; base += kList) {
            // look up to 256 pages up, those that are there in order. (A thread's last wait may have failed where others' did
            // not, and all must meet at the same barriers: so they leave together)
            if (!__syncthreads_and(ok)) break;
            int page = -1, block = -1;
            if (base + tid < stop) {
                block = A.picks ? A.picks[((size_t)token * A.c.kv_heads + head) * A.top + base + tid] : base + tid;
                if (block >= 0 && block < nb) page = page_of(A.c, sequence, block);
            }
            const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
            if (lane == 0) M.warp_sum[warp] = __popc(there);
            __syncthreads();
            int at = __popc(there & ((1u << lane) - 1)), count = 0;
#pragma unroll
            for (int w = 0; w < kThreads / 32; ++w) {
                at += w < warp ? (int)M.warp_sum[w] : 0;
                count += (int)M.warp_sum[w];
            }
            if (page >= 0) {
                M.list_page[at] = page;
                M.list_block[at] = block;
                const float *sc = page_scales(A.c, page, head);
                M.list_scale[at] = make_float2(sc[0], sc[1]);
            }
            __syncthreads();
            const unsigned first = fetched;
            auto get = [&](int i, int kind) {
                const unsigned stage = (first + i) % Z::stages;
                ++asked[kind];
                fetch(M.page[stage][kind], page_codes(A.c, M.list_page[i], head, kind), P * kKvBlock, kind ? &M.v_full[stage] : &M.k_full[stage]);
            };
            if (tid == 0)
                for (int i = 0; i < min(count, Z::stages); ++i) get(i, 0), get(i, 1);
            for (int i = 0; i < count; ++i) {
                const unsigned stage = (first + i) % Z::stages, parity = (first + i) / Z::stages & 1;
                const float2 sc = M.list_scale[i];
                ok = ok && landed(&M.k_full[stage], parity);
                float acc[Z::s_tiles][4] = {};
                {
                    uint4 w[Z::s_tiles];
#pragma unroll
                    for (int j = 0; j < Z::s_tiles; ++j)
                        w[j] = *reinterpret_cast<const uint4 *>(M.page[stage][0] + (panel * 64 + (slice * Z::s_tiles + j) * 8 + g) * 64 + t * 16);
#pragma unroll
                    for (int s = 0; s < 4; ++s)
#pragma unroll
                        for (int j = 0; j < Z::s_tiles; ++j) {
                            unsigned b0, b1;
                            codes_to_half(s == 0 ? w[j].x : s == 1 ? w[j].y : s == 2 ? w[j].z : w[j].w, b0, b1);
                            mma(acc[j], qh[s], b0, b1);
                            mma(acc[j], ql[s], b0, b1);
                        }
                }
#pragma unroll
                for (int j = 0; j < Z::s_tiles; ++j) {
                    const int tok = (slice * Z::s_tiles + j) * 8 + 2 * t;
                    *reinterpret_cast<float2 *>(&M.s[panel][g][tok]) = make_float2(acc[j][0], acc[j][1]);
                    *reinterpret_cast<float2 *>(&M.s[panel][g + 8][tok]) = make_float2(acc[j][2], acc[j][3]);
                }
                // every warp has read this page's keys and the last page's values
                if (!__syncthreads_and(ok)) break;
                if (tid == 0) {
                    if (i + Z::stages < count) get(i + Z::stages, 0);
                    if (i > 0 && i - 1 + Z::stages < count) get(i - 1 + Z::stages, 1);
                }
                float4 s4 = *reinterpret_cast<const float4 *>(&M.s[0][srow][stok]);
#pragma unroll
                for (int j = 1; j < Z::panels; ++j) {
                    const float4 f = *reinterpret_cast<const float4 *>(&M.s[j][srow][stok]);
                    s4.x += f.x, s4.y += f.y, s4.z += f.z, s4.w += f.w;
                }
                const float rs = M.row_scale[srow];
                const int left = seen - M.list_block[i] * kKvBlock - stok;  // keys in sight from this lane's first on
                const float a0 = left > 0 ? s4.x * sc.x * rs : -INFINITY, a1 = left > 1 ? s4.y * sc.x * rs : -INFINITY;
                const float a2 = left > 2 ? s4.z * sc.x * rs : -INFINITY, a3 = left > 3 ? s4.w * sc.x * rs : -INFINITY;
                float top_now = fmaxf(fmaxf(a0, a1), fmaxf(a2, a3));
#pragma unroll
                for (int s = 8; s > 0; s >>= 1) top_now = fmaxf(top_now, __shfl_xor_sync(0xffffffffu, top_now, s));
                top_now = fmaxf(top_now, m);
                const float alpha = exp2_fast(m - top_now), from = top_now - kLift;
                m = top_now;
                const float p0 = exp2_fast(a0 - from), p1 = exp2_fast(a1 - from), p2 = exp2_fast(a2 - from), p3 = exp2_fast(a3 - from);
                sum = sum * alpha + ((p0 + p1) + (p2 + p3));
                uint2 hi, lo;
                split_pair(p0, p1, hi.x, lo.x);
                split_pair(p2, p3, hi.y, lo.y);
                *reinterpret_cast<uint2 *>(&M.p[0][srow][stok]) = hi;
                *reinterpret_cast<uint2 *>(&M.p[1][srow][stok]) = lo;
                if ((lane & 15) == 0) M.alpha[srow] = alpha;
                __syncthreads();
                ok = landed(&M.v_full[stage], parity);
                unsigned ph[4][4], pl[4][4];
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint4 a = *reinterpret_cast<const uint4 *>(&M.p[0][g + 8 * r][16 * t + 8 * h]);
                        const uint4 b = *reinterpret_cast<const uint4 *>(&M.p[1][g + 8 * r][16 * t + 8 * h]);
                        ph[2 * h][r] = a.x, ph[2 * h][2 + r] = a.y, ph[2 * h + 1][r] = a.z, ph[2 * h + 1][2 + r] = a.w;
                        pl[2 * h][r] = b.x, pl[2 * h][2 + r] = b.y, pl[2 * h + 1][r] = b.z, pl[2 * h + 1][2 + r] = b.w;
                    }
                float part[Z::o_tiles][4] = {};
                {
                    uint4 w[Z::o_tiles];
#pragma unroll
                    for (int j = 0; j < Z::o_tiles; ++j)
                        w[j] = *reinterpret_cast<const uint4 *>(M.page[stage][1] + ((warp * Z::o_tiles + j) * 8 + g) * 64 + t * 16);
#pragma unroll
                    for (int s = 0; s < 4; ++s)
#pragma unroll
                        for (int j = 0; j < Z::o_tiles; ++j) {
                            unsigned b0, b1;
                            codes_to_half(s == 0 ? w[j].x : s == 1 ? w[j].y : s == 2 ? w[j].z : w[j].w, b0, b1);
                            mma(part[j], ph[s], b0, b1);
                            mma(part[j], pl[s], b0, b1);
                        }
                }
                const float al0 = M.alpha[g], al1 = M.alpha[g + 8];
#pragma unroll
                for (int j = 0; j < Z::o_tiles; ++j) {
                    o[j][0] = o[j][0] * al0 + part[j][0] * sc.y;
                    o[j][1] = o[j][1] * al0 + part[j][1] * sc.y;
                    o[j][2] = o[j][2] * al1 + part[j][2] * sc.y;
                    o[j][3] = o[j][3] * al1 + part[j][3] * sc.y;
                }
            }
            if (ok) fetched = first + count;
        }
        if (!__syncthreads_and(ok)) {  // a copy did not land in time: report, let what is in flight land, leave
            if (tid == 0) {
                raise_error(A.c.err, kErrWaitTimeout);
                for (unsigned i = 0; i < Z::stages; ++i) {  // the last copy of each stage
                    if (asked[0] > i) landed(&M.k_full[i], (asked[0] - 1 - i) / Z::stages & 1);
                    if (asked[1] > i) landed(&M.v_full[i], (asked[1] - 1 - i) / Z::stages & 1);
                }
            }
            return;
        }
#pragma unroll
        for (int s = 8; s > 0; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
        const bool whole = entry == 0 && stop == n;
        if (whole) {
            if ((lane & 15) == 0) M.alpha[srow] = sum;
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int row = g + 8 * r;
                if (row >= rows) continue;
                const float l = M.alpha[row], inv = l == 0.0f ? 0.0f : __fdiv_rn(1.0f, l);
                float *dst = A.y + ((size_t)token * A.heads + head * A.group + row0 + row) * A.c.dim;
#pragma unroll
                for (int j = 0; j < Z::o_tiles; ++j) {
                    const int ch = (warp * Z::o_tiles + j) * 8 + 2 * t;
                    if (ch < A.c.dim) dst[ch] = o[j][2 * r] * inv;
                    if (ch + 1 < A.c.dim) dst[ch + 1] = o[j][2 * r + 1] * inv;
                }
            }
        } else {
            const Parts W = parts_of(A.c.workspace, P);
            const int slot = 2 * blockIdx.x + (entry == 0);  // a CTA's first unit may have begun earlier, its last may go on
            if ((lane & 15) == 0) W.ml[slot * kRows + srow] = make_float2(m, sum);
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int j = 0; j < Z::o_tiles; ++j)
                    *reinterpret_cast<float2 *>(W.acc + ((size_t)slot * kRows + g + 8 * r) * P + (warp * Z::o_tiles + j) * 8 + 2 * t) =
                        make_float2(o[j][2 * r], o[j][2 * r + 1]);
        }
        if (entry == 0 && tid == 0)
            parts_of(A.c.workspace, P).cover[token * per_token + sub] =
                make_int2(blockIdx.x, (int)((work + n - 1) / chunk));  // the CTAs of this unit's first and last page
        work += stop - entry;
        if (work >= work_end) return;
        entry = 0;
        if (++sub == per_token) {
            sub = 0;
            do ++token;
            while (M.before[token + 1] == M.before[token]);
        }
        __syncthreads();
    }
}

// CTAs of k_kv8_short that the current device holds at once; asked of the runtime once per device.
template <int P>
cudaError_t resident_ctas(size_t smem, int *out) {
    constexpr int kDevices = 64;
    static std::atomic<int> known[kDevices];
    int device = 0, sms = 0, fit = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    if (device < kDevices && (*out = known[device].load(std::memory_order_relaxed)) > 0) return cudaSuccess;
    e = cudaFuncSetAttribute(k_kv8_short<P>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, k_kv8_short<P>, kThreads, smem);
    if (e != cudaSuccess) return e;
    if (fit < 1) return cudaErrorInvalidConfiguration;
    *out = fit * sms < kMaxCtas ? fit * sms : kMaxCtas;
    if (device < kDevices) known[device].store(*out, std::memory_order_relaxed);
    return cudaSuccess;
}

template <int P>
cudaError_t launch(Args A, int multiprocessors, cudaStream_t s) {
    constexpr size_t kSmem = sizeof(Smem<P>);
    int slots = 0;
    cudaError_t e = resident_ctas<P>(kSmem, &slots);
    if (e != cudaSuccess) return e;
    const long long units = (long long)A.runs.segments * A.runs.count * A.c.kv_heads * A.tiles, most = units * (A.picks ? A.top : A.c.blocks);
    A.split = 1;
    e = kv8_launch(k_kv8_short<P>, dim3((unsigned)(most < slots ? most : slots)), dim3(kThreads), kSmem, 1, s, A);
    return e != cudaSuccess ? e : launch_join<P>(A, units, multiprocessors, s);
}

}  // namespace

// Chosen for up to kShortPages pages a multiprocessor, and for up to kShortPart pages a part, a unit's pages on one CTA. All
// counts take every block of the table where there are no picks (lengths are known on the device alone).
// A multiprocessor's time in microseconds, fitted to 1000 tokens over 2 heads with 8 and 32 picked blocks: this form takes
// 3 a part and 0.58, 0.74, 1.29 a page at 64, 128, 256 channels whatever the group. The other takes by the group's rows
//            64 channels           128 channels          256 channels
//   4 rows   3.9 and 0.32 a page   4.1 and 0.33          4.8 and 0.42
//   8        5.5 and 0.41          5.8 and 0.39         10.5 and 0.45
//   12       9.2 and 0.48         12.0 and 0.41         16.0 and 0.55
//   16      13.4 and 0.61         14.8 and 0.65         19.2 and 0.81
// so that both are even at kShortPart pages. Where calls are small the other form's fixed costs (its operands' set-up) decide: one
// session over 8 heads of 128 channels takes 23.6 and 27.7 us at 6.9 pages a multiprocessor, 33.8 and 29.7 at 13.8.
constexpr long long kShortPages = 10;
constexpr long long kShortPart[3][4] = {{4, 16, 64, 1LL << 40}, {3, 8, 27, 127}, {2, 8, 17, 33}};

bool kv8_short_fits(const Args &A, int multiprocessors) {
    const long long tokens = (long long)A.runs.segments * A.runs.count, units = tokens * A.c.kv_heads * A.tiles;
    if (tokens > kMaxTokens || units > 65536) return false;
    const long long pages = units * (A.picks ? A.top : A.c.blocks);
    const int rows = A.group < kRows ? (A.group + 3) / 4 - 1 : 3;
    return pages <= kShortPages * multiprocessors || pages <= kShortPart[A.c.padded == 64 ? 0 : A.c.padded == 128 ? 1 : 2][rows] * (units + multiprocessors);
}

cudaError_t kv8_attend_short(Args A, int multiprocessors, cudaStream_t s) {
    if (A.c.padded == 64) return launch<64>(A, multiprocessors, s);
    if (A.c.padded == 128) return launch<128>(A, multiprocessors, s);
    return launch<256>(A, multiprocessors, s);
}

}  // namespace strata
