// The chunked delta rule's first kernel: what a chunk needs that does not depend on the state (delta_chunk.cuh).
//
// A block has a run's chunk and key head, and takes the head's value heads two at a time, one by each warpgroup:
//   [Q; K] K^T      128 rows by 64, once for all of them
//   A, G (q . k)    a thread a row, from its TMEM lane
//   T = (I + A)^-1  of blocks of 16 by substitution, a column a lane, then of blocks twice as large twice, F32 throughout
//   U^T = V^T (T diag(beta))^T   a lane a value channel
//   W = (T diag(beta P)) K       both heads' 64 rows as one operand; K's tile as it lies, read the other way round
// Bound by instructions, most of them the splits into halves: what a row needs twice (its largest value first) waits in TMEM,
// and columns go by 16 in loops that are not unrolled, since code that a block runs once comes slower than it executes (with all
// 64 columns unrolled a prompt of 2048 tokens over 32 heads of 128 took 210 us, most of them without an instruction to issue).
#include "delta_chunk.cuh"

#include <atomic>

namespace strata {
namespace {

using namespace delta;

constexpr int kPrepareThreads = 256, kPitch = 68;

template <int D>
struct __align__(1024) PrepareSmem {
    unsigned char qk[2][D / 64][128 * 128];  // hi, lo: panels of 64 channels; rows 0-63 Q, 64-127 K
    union {                                  // V's rows until they are in TMEM, then T's
        float v[2][64 * D];                  // by head
        struct {
            unsigned char tw[2][128 * 128];    // T diag(beta P) over K's scales: hi, lo; two heads' 64 rows
            unsigned char tu[2][2][64 * 128];  // by head: T diag(beta), hi, lo
        };
    };
    float a[2][64 * kPitch];  // A, then T
    float inv[128];           // Q's and K's scales taken back
    // by head: decays; products of decays up to a token in its half; strengths, and times decays up to the token over K's scale;
    // K's scales taken back, the lower half's times the decays after a token in it
    float decay[2][64], upto[2][64], beta[2][64], beta_w[2][64], inv_k[2][64];
    float inv_tw[2][64], inv_tu[2][64];
    float w_max[2][128];
    int bad_key, bad[2], abort_flag;
    unsigned tmem;
    unsigned long long done;
};

__device__ __forceinline__ void group_sync(int g) { asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory"); }
__device__ __forceinline__ void add2(unsigned long long &d, unsigned long long a, unsigned long long b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(d) : "l"(a), "l"(b));
}
__device__ __forceinline__ ulonglong2 load22(const float *p) { return *reinterpret_cast<const ulonglong2 *>(p); }

// x of (I + L) x = e_c, L the strictly lower part of 16 rows at l
__device__ __forceinline__ void substitute(const float *l, int c, float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float s[4] = {i == c ? 1.0f : 0.0f, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < i; j += 4) {
            const float4 r = *reinterpret_cast<const float4 *>(l + i * kPitch + j);
            s[0] = fmaf(-r.x, x[j], s[0]);
            if (j + 1 < i) s[1] = fmaf(-r.y, x[j + 1], s[1]);
            if (j + 2 < i) s[2] = fmaf(-r.z, x[j + 2], s[2]);
            if (j + 3 < i) s[3] = fmaf(-r.w, x[j + 3], s[3]);
        }
        x[i] = (s[0] + s[1]) + (s[2] + s[3]);
    }
}
// W columns (4 or 8) from c of row r of sign X Y: rows of X at x, Y at y; `terms` (a multiple of 4) of X's row count
template <int W>
__device__ __forceinline__ void times(const float *x, const float *y, int r, int c, int terms, float sign, float *to) {
    unsigned long long s[W / 2] = {};
#pragma unroll 2
    for (int j = 0; j < terms; j += 4) {
        const float4 f = *reinterpret_cast<const float4 *>(x + r * kPitch + j);
        const float g[4] = {f.x * sign, f.y * sign, f.z * sign, f.w * sign};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float *row = y + (j + e) * kPitch + c;
#pragma unroll
            for (int w = 0; w < W; w += 4) {
                const ulonglong2 b = load22(row + w);
                add2(s[w / 2], pack2(g[e], g[e]), b.x);
                add2(s[w / 2 + 1], pack2(g[e], g[e]), b.y);
            }
        }
    }
#pragma unroll
    for (int w = 0; w < W; w += 4) *reinterpret_cast<ulonglong2 *>(to + r * kPitch + c + w) = ulonglong2{s[w / 2], s[w / 2 + 1]};
}
// Products over lanes: of this one's and those before, and of those after.
__device__ __forceinline__ float product_upto(float x, int lane) {
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const float o = __shfl_up_sync(0xffffffffu, x, s);
        if (lane >= s) x *= o;
    }
    return x;
}
__device__ __forceinline__ float product_after(float x, int lane) {
    x = __shfl_down_sync(0xffffffffu, x, 1);
    if (lane == 31) x = 1.0f;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
        const float o = __shfl_down_sync(0xffffffffu, x, s);
        if (lane + s < 32) x *= o;
    }
    return x;
}

// VEC: rows of q, k and v can be read four channels at a time.
template <int D, bool VEC>
__global__ void __launch_bounds__(kPrepareThreads, 1) k_delta_prepare(DeltaNet n, DeltaRule A, MixRuns r, DeltaSlab slab) {
    using Slot = DeltaSlot<D>;
    constexpr int kPanels = D / 64, kW = D / 2;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    PrepareSmem<D> &M = *reinterpret_cast<PrepareSmem<D> *>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = tid >> 7, gt = tid & 127, w4 = warp & 3;
    kv8_enter();
    const int chunk = slab.chunk0 + (int)(blockIdx.x % slab.chunks), head = slab.head0 + (int)(blockIdx.x / slab.chunks % slab.heads);
    const int run = slab.run0 + (int)(blockIdx.x / slab.chunks / slab.heads), t0 = chunk * kChunk;
    const MixRun me = mix_run_alone(r, n.sequences, run, n.err);
    if (me.sequence < 0 || t0 >= me.tokens) return;
    const int tokens = min(kChunk, me.tokens - t0);
    const long long row0 = (long long)run * r.count + t0;
    unsigned char *slot = slab.slots + blockIdx.x * slab.slot_bytes;

    // V's rows of a value head to shared memory, by its warpgroup; zeros behind the run's end and past dim
    const auto fetch_v = [&](int h) {
        const float *from = A.v + row0 * A.v_stride + (long long)h * n.dim;
        constexpr int kPiece = VEC ? 4 : 1;
#pragma unroll 4
        for (int at = gt * kPiece; at < 64 * D; at += 128 * kPiece) {
            const int j = at / D, c = at % D;
            const bool in = j < tokens && c < n.dim;
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(su32(&M.v[g][at])), "l"(in ? from + j * A.v_stride + c : A.v),
                         "n"(kPiece * 4), "r"(in ? kPiece * 4 : 0)
                         : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (g < slab.ratio) fetch_v(head + g * n.key_heads);
    if (tid == 0) {
        bar_init(&M.done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        M.abort_flag = M.bad_key = 0;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&M.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = M.tmem, mine = tmem + ((unsigned)(w4 * 32) << 16);
    // columns: [Q; K] K^T; by head V's halves; W; by head U^T, whose place and W's keep rows until they are split
    const unsigned kRaw = 0, kV = 64 + 64 * g, kWAt = 192, kU = 320 + 64 * g;
    const Waits wait{&M.abort_flag, n.err};
    unsigned phase = 0;

    // Q's and K's rows, a power of two each
    constexpr int kLanes = D / 4, kRows = 32 / kLanes;
#pragma unroll 1
    for (int at = 0; at < 16; at += 8 * kRows) {
        float f[8][4];
        const int ch = 4 * (lane % kLanes);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int row = warp * 16 + at + u * kRows + lane / kLanes, t = row & 63;
            f[u][0] = f[u][1] = f[u][2] = f[u][3] = 0.0f;
            if (t >= tokens || ch >= n.dim) continue;
            const float *p = (row < 64 ? A.q + (row0 + t) * A.q_stride : A.k + (row0 + t) * A.k_stride) + (long long)head * n.dim + ch;
            if (VEC) {
                const float4 x = *reinterpret_cast<const float4 *>(p);
                f[u][0] = x.x, f[u][1] = x.y, f[u][2] = x.z, f[u][3] = x.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) f[u][e] = ch + e < n.dim ? p[e] : 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int row = warp * 16 + at + u * kRows + lane / kLanes;
            float m = largest(0.0f, f[u]);
            if (kLanes == 32) {
                m = warp_largest(m);
            } else {
#pragma unroll
                for (int s = kLanes / 2; s > 0; s >>= 1) m = larger(m, __shfl_xor_sync(0xffffffffu, m, s), 0.0f);
            }
            const int e = exponent_of(m);
            if (lane % kLanes == 0) M.inv[row] = unscale_of(e);
            if (past(m)) M.bad_key = 1;
            unsigned hi[2], lo[2];
            split(f[u], scale_of(e), hi, lo);
            const int to = piece(row, ch % 64 / 8) + ch % 8 * 2;
            *reinterpret_cast<uint2 *>(&M.qk[0][ch / 64][to]) = uint2{hi[0], hi[1]};
            *reinterpret_cast<uint2 *>(&M.qk[1][ch / 64][to]) = uint2{lo[0], lo[1]};
        }
    }
    to_async();
    __syncthreads();
    if (warp == 0) {
        if (elect_one()) {
            const unsigned long long q = sw128_desc(su32(M.qk[0][0]));
#pragma unroll 1
            for (int product = 0; product < 3; ++product) {  // lo hi, hi lo, hi hi
                const unsigned long long x = q + (product == 0) * (kPanels * 1024), y = q + 512 + (product == 1) * (kPanels * 1024);
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    mma_f16(tmem + kRaw, x + k / 4 * 1024 + k % 4 * 2, y + k / 4 * 1024 + k % 4 * 2, idesc_f16(128, 64), product || k);
            }
            mma_commit(&M.done);
        }
        if (lane == 0) {
            for (int i = 0; i < 4 * kPanels; ++i) {  // Q: hi, lo; K: hi, lo
                const int part = i % (2 * kPanels);
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], 8192;" ::"l"(slot + i * 8192),
                             "r"(su32(M.qk[part / kPanels][part % kPanels]) + (i / (2 * kPanels)) * 8192)
                             : "memory");
            }
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
        }
        __syncwarp();
    }

#pragma unroll 1
    for (int pair = 0; pair < slab.ratio; pair += 2) {
        const int m = pair + g, h = head + m * n.key_heads;
        const bool there = m < slab.ratio;
        unsigned char *mine_out = slot + Slot::heads + (long long)m * Slot::head_bytes;
        DeltaFactors *factors = reinterpret_cast<DeltaFactors *>(mine_out + Slot::factors);
        if (gt == 0) M.bad[g] = 0;
        float inv_v = 0.0f;
        if (there) {
            asm volatile("cp.async.wait_all;" ::: "memory");
            group_sync(g);  // V is there, and bad[g] has been cleared
            if (w4 == 0) {
                // decays and strengths, two tokens a lane; rows behind the run's end change nothing
                float a[2], b[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const bool in = lane + 32 * e < tokens;
                    const long long at = (row0 + lane + 32 * e) * n.value_heads + h;
                    a[e] = in ? A.decay[at] : 1.0f;
                    b[e] = in ? A.beta[at] : 0.0f;
                }
                if (past(larger(larger(a[0], a[1], b[0]), b[1], 0.0f))) M.bad[g] = 1;
                const float upto[2] = {product_upto(a[0], lane), product_upto(a[1], lane)};
                const float after[2] = {product_after(a[0], lane), product_after(a[1], lane)};
                const float low = __shfl_sync(0xffffffffu, upto[0], 31), high = __shfl_sync(0xffffffffu, upto[1], 31);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int t = lane + 32 * e;
                    const float p = e ? upto[1] * low : upto[0], inv_k = M.inv[64 + t];
                    M.decay[g][t] = a[e];
                    M.upto[g][t] = upto[e];
                    M.beta[g][t] = b[e];
                    M.beta_w[g][t] = b[e] * p * inv_k;
                    M.inv_k[g][t] = e ? inv_k : inv_k * after[0];
                    factors->q[t] = p * M.inv[t];
                    factors->k[t] = (e ? after[1] : after[0] * high) * inv_k;
                    if (t == 63) factors->end = p;
                }
            }
            // V's column of this lane to TMEM
            const float *column = M.v[g] + (gt < D ? gt : 0);
            float most = 0.0f;
#pragma unroll 1
            for (int j = 0; j < 64; j += 16) {
                float v[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = column[(j + e) * D];
                most = largest(most, v);
            }
            const int e = exponent_of(most);
            inv_v = unscale_of(e);
            if (past(most)) M.bad[g] = 1;
#pragma unroll 1
            for (int j = 0; j < 64; j += 16) {
                float v[16];
                unsigned hi[8], lo[8];
#pragma unroll
                for (int u = 0; u < 16; ++u) v[u] = column[(j + u) * D];
                split(v, scale_of(e), hi, lo);
                tmem_write(mine + kV + j / 2, hi);
                tmem_write(mine + kV + 32 + j / 2, lo);
            }
            tmem_written();
        }
        if (pair == 0) wait(&M.done, phase & 1), ++phase;
        tc_fence_after();
        if (there) {
            group_sync(g);  // the decays are there
            // rows 0-63: products of queries, 64-127: of keys, each times G over the column's scale. Row i of the upper half: the
            // decays up to it in that half times those after column j in the lower one; else their product grows from j = i down.
            const int i = gt & 63;
            const bool key = gt >= 64, upper = w4 & 1;
            const float row_factor = key ? M.inv[gt] * M.beta[g][i] : 1.0f, far = M.upto[g][i];
            float *a_row = &M.a[g][i * kPitch];
            float p = 1.0f, most = 0.0f;
            const int last = upper ? 48 : 16;  // the last columns that count
#pragma unroll 1
            for (int j = last; j >= 0; j -= 16) {
                float x[16];
                tmem_read(mine + kRaw + j, x);
                if (upper && j < 32) {
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const float4 c = *reinterpret_cast<const float4 *>(&M.inv_k[g][j + e]);
                        x[e] *= c.x * far, x[e + 1] *= c.y * far, x[e + 2] *= c.z * far, x[e + 3] *= c.w * far;
                    }
                } else {
                    const int limit = key ? i - 1 : i;
#pragma unroll
                    for (int e = 15; e >= 0; --e) {
                        if (j + e < i) p *= M.decay[g][j + e + 1];
                        x[e] = j + e <= limit ? x[e] * M.inv[64 + j + e] * p : 0.0f;
                    }
                }
                if (key) {
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *reinterpret_cast<float4 *>(a_row + j + e) =
                            float4{x[e] * row_factor, x[e + 1] * row_factor, x[e + 2] * row_factor, x[e + 3] * row_factor};
                } else {
                    most = largest(most, x);
                    tmem_write(mine + kU + j, x);
                }
            }
            if (!key) {
                const int e = exponent_of(most);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
#pragma unroll 1
                for (int j = 0; j < 64; j += 16) {
                    unsigned hi[8] = {}, lo[8] = {};
                    if (j <= last) {
                        float x[16];
                        tmem_read(mine + kU + j, x);
                        split(x, scale_of(e), hi, lo);
                    }
                    put_pieces(mine_out + Slot::g, i, j / 8, hi);
                    put_pieces(mine_out + Slot::g + 8192, i, j / 8, lo);
                }
                factors->attn[i] = unscale_of(e) * M.inv[i];
            }
            group_sync(g);
            // T: inverses of the four blocks of 16 on the diagonal, by two warps; then of pairs of them: the lower left of
            // [B 0; A C]^-1 is -C^-1 (A B^-1), whose second factor waits in the upper right
            float *a = M.a[g];
            const auto at = [&](int row, int col) { return a + row * kPitch + col; };
            if (w4 >= 2) {
                const int block = 32 * (w4 - 2) + (lane & 16);
                float c[16];
                substitute(at(block, block), lane & 15, c);
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 16; ++j) *at(block + j, block + (lane & 15)) = c[j];
            }
            group_sync(g);
            {
                const int two = gt >> 6, row = (gt & 63) >> 2, col = (gt & 3) * 4;  // 64 threads each of two pairs
                float *b = at(32 * two, 32 * two);
                times<4>(b + 16 * kPitch, b, row, col, 16, 1.0f, b + 16);
                group_sync(g);
                times<4>(b + 16 * kPitch + 16, b + 16, row, col, 16, -1.0f, b + 16 * kPitch);
                group_sync(g);
                *reinterpret_cast<float4 *>(b + 16 + row * kPitch + col) = float4{0, 0, 0, 0};
            }
            {
                const int row = gt >> 2, col = (gt & 3) * 8;
                group_sync(g);
                times<8>(at(32, 0), at(0, 0), row, col, 32, 1.0f, at(0, 32));
                group_sync(g);
                times<8>(at(32, 32), at(0, 32), row, col, 8 * w4 + 8, -1.0f, at(32, 0));
                group_sync(g);
            }
        }
        __syncthreads();  // T's rows take V's place
        if (there) {
            // as operands: threads 0-63 for U, 64-127 for W. They wait in W's place.
            const int i = gt & 63, last = w4 & 1 ? 48 : 16;
            const bool key = gt >= 64;
            const float *a_row = &M.a[g][i * kPitch], *by = key ? M.beta_w[g] : M.beta[g];
            const unsigned waiting = mine + kWAt + 64 * g;
            float most = 0.0f;
#pragma unroll 1
            for (int j = 0; j <= last; j += 16) {
                float x[16];
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const float4 t = *reinterpret_cast<const float4 *>(a_row + j + e), b = *reinterpret_cast<const float4 *>(by + j + e);
                    x[e] = t.x * b.x, x[e + 1] = t.y * b.y, x[e + 2] = t.z * b.z, x[e + 3] = t.w * b.w;
                }
                most = largest(most, x);
                tmem_write(waiting + j, x);
            }
            if (past(most)) M.bad[g] = 1;
            const int e = exponent_of(most);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            unsigned char *t_hi = key ? M.tw[0] : M.tu[g][0], *t_lo = key ? M.tw[1] : M.tu[g][1];
            const int t_row = key ? g * 64 + i : i;
#pragma unroll 1
            for (int j = 0; j < 64; j += 16) {
                unsigned hi[8] = {}, lo[8] = {};
                if (j <= last) {
                    float x[16];
                    tmem_read(waiting + j, x);
                    split(x, scale_of(e), hi, lo);
                }
                put_pieces(t_hi, t_row, j / 8, hi);
                put_pieces(t_lo, t_row, j / 8, lo);
            }
            (key ? M.inv_tw[g] : M.inv_tu[g])[i] = unscale_of(e);
        } else if (gt >= 64) {  // rows that no head has
            const unsigned zero[32] = {};
            put_pieces(M.tw[0], 64 + (gt & 63), 0, zero);
            put_pieces(M.tw[1], 64 + (gt & 63), 0, zero);
            M.inv_tw[g][gt & 63] = 0.0f;
        }
        to_async();
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        if (warp == 0) {
            if (elect_one()) {
                const unsigned long long tu = sw128_desc(su32(M.tu[0][0])), tw = sw128_desc(su32(M.tw[0]));
                const unsigned long long keys = turned_desc(su32(M.qk[0][0]) + 8192, 16384);
#pragma unroll 1
                for (int product = 0; product < 3; ++product) {
#pragma unroll
                    for (int w = 0; w < 2; ++w)  // U^T: lanes are value channels (of no head: nobody looks)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            mma_f16_ts(tmem + 320 + 64 * w, tmem + 64 + 64 * w + (product == 0) * 32 + k * 8, tu + w * 1024 + (product == 1) * 512 + k * 2,
                                       idesc_f16(128, 64), product || k);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_f16(tmem + kWAt, tw + (product == 0) * 1024 + k * 2, keys + (product == 1) * (kPanels * 1024) + k * 128, turned_idesc(128, D),
                                product || k);
                }
                mma_commit(&M.done);
            }
            __syncwarp();
        }
        wait(&M.done, phase & 1), ++phase;
        tc_fence_after();
        if (pair + 2 + g < slab.ratio) fetch_v(h + 2 * n.key_heads);  // T's rows have been read
        if (there && w4 < D / 32) {
            float *to = reinterpret_cast<float *>(mine_out + Slot::uu) + gt;
#pragma unroll 1
            for (int i = 0; i < 64; i += 16) {
                float u[16];
                tmem_read(mine + kU + i, u);
#pragma unroll
                for (int e = 0; e < 16; ++e) to[(i + e) * D] = u[e] * inv_v * M.inv_tu[g][i + e];
            }
        }
        // W's rows: lane w4 * 32 + lane is row i of the pair's head `of`; this warpgroup has half of its channels
        const int of = w4 >> 1, i = gt & 63;
        float most = 0.0f;
#pragma unroll 1
        for (int c = 0; c < kW; c += 16) {
            float w[16];
            tmem_read(mine + kWAt + g * kW + c, w);
            most = largest(most, w);
        }
        M.w_max[g][gt] = most;
        __syncthreads();
        most = larger(M.w_max[0][gt], M.w_max[1][gt], 0.0f);
        const float inv_t = M.inv_tw[of][i];
        if (past(most * inv_t)) M.bad[of] = 1;
        if (pair + of < slab.ratio) {
            unsigned char *out = slot + Slot::heads + (long long)(pair + of) * Slot::head_bytes;
            const int e = exponent_of(most);
            const int panel = D == 128 ? g : 0, first = D == 128 ? 0 : g * 4;
#pragma unroll 1
            for (int c = 0; c < kW; c += 16) {
                float w[16];
                unsigned hi[8], lo[8];
                tmem_read(mine + kWAt + g * kW + c, w);
                split(w, scale_of(e), hi, lo);
                put_pieces(out + Slot::w + panel * 8192, i, first + c / 8, hi);
                put_pieces(out + Slot::w + (kPanels + panel) * 8192, i, first + c / 8, lo);
            }
            if (g == 0) reinterpret_cast<DeltaFactors *>(out + Slot::factors)->z[i] = unscale_of(e) * inv_t;
        }
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        if (there && gt == 0) factors->walk = M.bad[g] | M.bad_key;
    }
    if (tid == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    settle(&M.abort_flag);
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <int D, bool VEC>
cudaError_t launch_prepare(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, const DeltaSlab &slab, cudaStream_t s) {
    constexpr int kDevices = 64;
    static std::atomic<bool> done[kDevices];
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess && (device >= kDevices || !done[device].load(std::memory_order_relaxed))) {
        e = cudaFuncSetAttribute(k_delta_prepare<D, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(PrepareSmem<D>));
        if (e == cudaSuccess && device < kDevices) done[device].store(true, std::memory_order_relaxed);
    }
    if (e != cudaSuccess) return e;
    return kv8_launch(k_delta_prepare<D, VEC>, dim3((unsigned)(slab.runs * slab.heads * slab.chunks)), dim3(kPrepareThreads), sizeof(PrepareSmem<D>), 1, s,
                      n, a, r, slab);
}

}  // namespace

cudaError_t delta_prepare(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, const DeltaSlab &slab, bool vec, cudaStream_t s) {
    if (n.dim <= 64) return vec ? launch_prepare<64, true>(n, a, r, slab, s) : launch_prepare<64, false>(n, a, r, slab, s);
    return vec ? launch_prepare<128, true>(n, a, r, slab, s) : launch_prepare<128, false>(n, a, r, slab, s);
}

}  // namespace strata
