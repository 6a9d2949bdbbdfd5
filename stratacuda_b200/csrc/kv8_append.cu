// Appending rows to the 8-bit paged cache (strata_kv8_append).
#include "kv8.cuh"

namespace strata {
namespace {

constexpr int kThreads = 256;

constexpr int kFew = 4;  // rows of a run, up to which it is worth trying to add them without forming the block again (FEW)

// One CTA: one kind (keys or values) of one head's block of one run. The block's rows, those that
// the sequence already holds (from `open`) and the new ones, are read into registers, the largest
// magnitude fixes the scale, the codes are laid out in shared memory as the page holds them and
// copied out whole. Bound by memory: 4 bytes read and 1 written a value.
// A few rows added to an open block (decode) mostly leave its scale as it is; then all other codes stand and only the
// new rows' and the marks are written, with the same result. Bound by the latency of the look-ups and of the open rows.
// Measured at 2 heads of 256 channels: a prompt of 8191 tokens 15.7 us (2.7 TB/s; 516 CTAs, a block, kind and head each, are
// 1.2 waves, and loads and stores of a CTA do not overlap), 64 sessions' tokens 7.6 us (9 with the call, which the host bounds).
template <int P, bool WIDE, bool FEW>
__global__ void __launch_bounds__(kThreads) k_kv8_append(const Kv8 c, const float *k, const float *v, long long stride, const Kv8Runs runs) {
    constexpr int kTiles = P / 64;  // 4 tokens x 4 channels a tile, 16 * P / 4 tiles
    __shared__ __align__(16) int8_t page_s[P * kKvBlock];
    __shared__ float red[kThreads / 32];
    __shared__ int lo_s[4][P / 4], hi_s[4][P / 4];
    const int tid = threadIdx.x, head = blockIdx.y >> 1, kind = blockIdx.y & 1;
    kv8_enter();
    const RunAt a = run_at(c, runs, blockIdx.z);
    if (a.sequence < 0) return;
    if (a.start < 0) {
        if (tid == 0) raise_error(c.err, kErrIndex);
        return;
    }
    const long long cells = (long long)c.blocks * kKvBlock;
    long long end = (long long)a.start + runs.count;
    if (end > cells) {
        if (tid == 0) raise_error(c.err, kErrIndex);
        end = cells;
    }
    const int block = a.start / kKvBlock + blockIdx.x;
    if ((long long)block * kKvBlock >= end) return;
    const int r0 = blockIdx.x == 0 ? a.start % kKvBlock : 0;
    const int r1 = (int)min((long long)kKvBlock, end - (long long)block * kKvBlock);
    const int page = page_of(c, a.sequence, block);
    const float *x = kind ? v : k;
    const size_t open_row = (size_t)c.kv_heads * c.dim;
    float *open = c.open + ((size_t)a.sequence * 2 + kind) * kKvBlock * open_row + (size_t)head * c.dim;
    const long long first = (long long)blockIdx.z * runs.count + (long long)block * kKvBlock - a.start;  // input row of the block's row 0
    const float *in = x + first * stride + (size_t)head * c.dim;

    // the run's last block keeps its new rows in 32 bits while it is unfilled. The first block's
    // CTA writes them, after its own reads: it is the only one that reads this head's open rows.
    auto keep = [&]() {
        if (blockIdx.x != 0 || end % kKvBlock == 0) return;
        const int last = (int)(end / kKvBlock), rows = (int)(end % kKvBlock), from = last == block ? r0 : 0;
        const float *src = x + ((long long)blockIdx.z * runs.count + (long long)last * kKvBlock - a.start) * stride + (size_t)head * c.dim;
        for (int i = tid; i < (rows - from) * c.dim; i += kThreads) {
            const int row = from + i / c.dim, ch = i % c.dim;
            const float f = src[(long long)row * stride + ch];
            open[row * open_row + ch] = isfinite(f) ? f : 0.0f;
        }
    };
    // (a run that goes on past this block leaves another's rows in `open`, with which it could not be repeated)
    if (FEW && r0 > 0 && end - (long long)block * kKvBlock <= kKvBlock) {
        // The block's values by channel: the largest magnitude fixes the scale, and the lowest and highest the marks, since
        // rounding keeps order. A page whose scale is that one holds the other rows' codes already.
        constexpr int kAcross = P / 4, kDeep = kThreads / kAcross, kRowsEach = kKvBlock / kDeep;  // a thread: 4 channels, every kDeep-th row
        static_assert(kDeep * kAcross == kThreads && kRowsEach * kDeep == kKvBlock, "whole channels and rows");
        __shared__ __align__(16) float lowest_s[kDeep][P], highest_s[kDeep][P];
        const int ch4 = tid % kAcross * 4, deep = tid / kAcross, ch = tid;
        const float scale = page >= 0 ? page_scales(c, page, head)[kind] : 0.0f;
        float amax = 0.0f;
        bool bad = false;
        {
            float f[kRowsEach][4], lowest[4], highest[4];
#pragma unroll
            for (int i = 0; i < kRowsEach; ++i) {
                const int row = i * kDeep + deep;
                const float *src = row < r0 ? open + row * open_row + ch4 : in + (long long)row * stride + ch4;
                if (WIDE) {
                    const float4 x = row < r1 && ch4 < c.dim ? *reinterpret_cast<const float4 *>(src) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    f[i][0] = x.x, f[i][1] = x.y, f[i][2] = x.z, f[i][3] = x.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) f[i][e] = row < r1 && ch4 + e < c.dim ? src[e] : 0.0f;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                lowest[e] = INFINITY, highest[e] = -INFINITY;
#pragma unroll
                for (int i = 0; i < kRowsEach; ++i) {
                    const bool finite = isfinite(f[i][e]);
                    const float x = finite ? f[i][e] : 0.0f;
                    bad |= !finite;
                    amax = fmaxf(amax, fabsf(x));
                    if (i * kDeep + deep < r1) lowest[e] = fminf(lowest[e], x), highest[e] = fmaxf(highest[e], x);
                }
            }
            *reinterpret_cast<float4 *>(&lowest_s[deep][ch4]) = make_float4(lowest[0], lowest[1], lowest[2], lowest[3]);
            *reinterpret_cast<float4 *>(&highest_s[deep][ch4]) = make_float4(highest[0], highest[1], highest[2], highest[3]);
        }
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, s));
        if (tid % 32 == 0) red[tid / 32] = amax;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kThreads / 32; ++i) amax = fmaxf(amax, red[i]);
        if (page >= 0 && (amax < 0x1p-100f ? 0.0f : __fdiv_rn(amax, 127.0f)) == scale) {
            if (bad) raise_error(c.err, kErrKvValue);
            if (ch < c.dim) {
                const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
                auto code = [&](float x) { return (int8_t)max(-127, min(127, __float2int_rn(__fmul_rn(x, inv)))); };
                int8_t *codes = page_codes(c, page, head, kind), *m = page_marks(c, page, head);
                for (int row = r0; row < r1; ++row) {
                    const float x = in[(long long)row * stride + ch];
                    codes[kind ? ch * kKvBlock + row : key_byte(row, ch)] = code(isfinite(x) ? x : 0.0f);
                }
                if (!kind) {
                    float lowest = INFINITY, highest = -INFINITY;
#pragma unroll
                    for (int d = 0; d < kDeep; ++d) {
                        lowest = fminf(lowest, lowest_s[d][ch]);
                        highest = fmaxf(highest, highest_s[d][ch]);
                    }
                    m[ch] = code(lowest);
                    m[P + ch] = code(highest);
                }
            }
            keep();
            return;
        }
        __syncthreads();  // red is written again below
    }

    // this thread's tiles: neighbouring lanes take neighbouring channels of a key row, and
    // neighbouring token groups of a value channel, so that each kind's packed words lie side by side
    float xs[kTiles][4][4];
    float amax = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
        const int w = i * kThreads + tid;
        const int t4 = kind ? w & 15 : w / (P / 4), c4 = kind ? w >> 4 : w % (P / 4);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int row = t4 * 4 + t, ch = c4 * 4;
            const float *src = row < r0 ? open + row * open_row + ch : in + (long long)row * stride + ch;
            if (WIDE) {
                const float4 f = row < r1 && ch < c.dim ? *reinterpret_cast<const float4 *>(src) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                xs[i][t][0] = f.x, xs[i][t][1] = f.y, xs[i][t][2] = f.z, xs[i][t][3] = f.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) xs[i][t][e] = row < r1 && ch + e < c.dim ? src[e] : 0.0f;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < kTiles; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (!isfinite(xs[i][t][e])) {
                    bad = true;
                    xs[i][t][e] = 0.0f;
                }
                amax = fmaxf(amax, fabsf(xs[i][t][e]));
            }
    if (bad) raise_error(c.err, kErrKvValue);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, s));
    if (tid % 32 == 0) red[tid / 32] = amax;
    __syncthreads();  // also: every read of `open` above is done
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) amax = fmaxf(amax, red[i]);
    const float scale = amax < 0x1p-100f ? 0.0f : __fdiv_rn(amax, 127.0f);
    const float inv = scale > 0.0f ? __fdiv_rn(1.0f, scale) : 0.0f;
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
        const int w = i * kThreads + tid;
        const int t4 = kind ? w & 15 : w / (P / 4), c4 = kind ? w >> 4 : w % (P / 4);
        int q[4][4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) q[t][e] = max(-127, min(127, __float2int_rn(__fmul_rn(xs[i][t][e], inv)))) & 255;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (kind)
                *reinterpret_cast<int *>(page_s + (c4 * 4 + j) * kKvBlock + t4 * 4) = q[0][j] | q[1][j] << 8 | q[2][j] << 16 | q[3][j] << 24;
            else
                *reinterpret_cast<int *>(page_s + key_byte(t4 * 4 + j, c4 * 4)) = q[j][0] | q[j][1] << 8 | q[j][2] << 16 | q[j][3] << 24;
        }
    }
    __syncthreads();
    if (page >= 0) {
        uint4 *dst = reinterpret_cast<uint4 *>(page_codes(c, page, head, kind));
        for (int i = tid; i < P * kKvBlock / 16; i += kThreads) dst[i] = reinterpret_cast<const uint4 *>(page_s)[i];
        if (tid == 0) page_scales(c, page, head)[kind] = scale;
    }
    if (!kind) {  // lowest and highest code of each channel over the rows there are
        for (int w = tid; w < P; w += kThreads) {
            const int quarter = w / (P / 4), c4 = w % (P / 4);
            int lo = 0x7f7f7f7f, hi = (int)0x81818181u;
            for (int t = quarter * 16; t < min(r1, quarter * 16 + 16); ++t) {
                const int codes = *reinterpret_cast<const int *>(page_s + key_byte(t, c4 * 4));
                lo = __vmins4(lo, codes);
                hi = __vmaxs4(hi, codes);
            }
            lo_s[quarter][c4] = lo;
            hi_s[quarter][c4] = hi;
        }
        __syncthreads();
        if (page >= 0 && tid < P / 4) {
            int lo = lo_s[0][tid], hi = hi_s[0][tid];
            for (int i = 1; i < 4; ++i) {
                lo = __vmins4(lo, lo_s[i][tid]);
                hi = __vmaxs4(hi, hi_s[i][tid]);
            }
            int8_t *m = page_marks(c, page, head);
            reinterpret_cast<int *>(m)[tid] = lo;
            reinterpret_cast<int *>(m + P)[tid] = hi;
        }
    }
    keep();
}

}  // namespace

cudaError_t kv8_append(const Kv8 &c, const float *k, const float *v, long long stride, const Kv8Runs &r, cudaStream_t s) {
    const dim3 grid((r.count + kKvBlock - 2) / kKvBlock + 1, c.kv_heads * 2, r.segments);
    // 16-byte loads where every row of a head starts on such a boundary
    const uintptr_t starts = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(c.open);
    const bool wide = starts % 16 == 0 && stride % 4 == 0 && c.dim % 4 == 0;
    const bool few = r.count <= kFew;
    auto launch = [&](auto... kernels) {
        decltype(&k_kv8_append<64, false, false>) all[] = {kernels...};
        return kv8_launch(all[2 * few + wide], grid, dim3(kThreads), 0, 1, s, c, k, v, stride, r);
    };
    if (c.padded == 64)
        return launch(k_kv8_append<64, false, false>, k_kv8_append<64, true, false>, k_kv8_append<64, false, true>, k_kv8_append<64, true, true>);
    if (c.padded == 128)
        return launch(k_kv8_append<128, false, false>, k_kv8_append<128, true, false>, k_kv8_append<128, false, true>,
                      k_kv8_append<128, true, true>);
    return launch(k_kv8_append<256, false, false>, k_kv8_append<256, true, false>, k_kv8_append<256, false, true>, k_kv8_append<256, true, true>);
}

}  // namespace strata
