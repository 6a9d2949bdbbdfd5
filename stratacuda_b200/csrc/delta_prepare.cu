// The chunked delta rule's first kernel: what a chunk needs that does not depend on the state (delta_chunk.cuh).
//
// A block has a run's chunk and key head, and takes the head's value heads one after another:
//   [Q; K] K^T      128 rows by 64, once for all of them
//   A, G (q . k)    a row's two threads have half of its columns each, from their TMEM lane
//   T = (I + A)^-1  of blocks of 32 by substitution, a column a lane, then -T22 (A21 T11), F32 throughout
//   U^T = (diag(beta) V)^T T^T      a lane a value channel
//   W^T = K^T (T diag(beta P))^T    a lane a key channel; K's tile as it lies, read the other way round
// Bound by instructions (19 k of a warp a chunk and value head), most of them the splits into halves, and by the way from one step to
// the next: two blocks of eight warps a multiprocessor, 100 KB and half of TMEM each, so that one's steps run in the other's waits (288
// chunks of a prompt over 32 heads of 128: 34 us; blocks of sixteen warps take 1.3 times as long). What becomes operands goes through shared
// memory and bulk copies, few and large ones. Code that a block runs once comes slower than it executes, so it is kept short.
// Of a slab ahead the kernel runs beside the second one of the slab before it.
#include "delta_chunk.cuh"

namespace strata {
namespace {

using namespace delta;

constexpr int kPrepareThreads = 256, kPitch = 68;
constexpr float kKey = 0x1p-13f;     // keys are scaled to 2^13, and of size one to all but the products
constexpr float kWScale = 0x1p-19f;  // of W's sums, which are 2^34 at most: 64 terms of two factors below 2^14
// Of G (q . k), with q at up to 2^14: past it F32 ends, though what it weighs may be small. (G (k . k) shows in T.)
constexpr float kLargestWeight = 0x1p110f;

template <int D>
struct __align__(1024) PrepareSmem {
    unsigned char qk[2][D / 64][128 * 128];  // hi, lo: panels of 64 channels; rows 0-63 Q, 64-127 K
    unsigned char more[D == 64 ? 4 : 1][D == 64 ? 64 * 128 : 16];
    union {
        float a[64 * kPitch];  // A, then T
        unsigned char w[2][D * 128];
    };
    float inv[128];  // Q's and K's scales taken back
    // decays; their products up to a token in its half; what a value is added to the state times; strengths, and times decays up to the
    // token (of keys by their power of two); decays after a token in its half, for the lower one, over keys' 2^13
    float decay[64], upto[64], gain[64], beta[64], beta_w[64], behind[64];
    float inv_tu[64];
    float most[2][2][128];  // a row's largest values, by warpgroup; two that are used in turn
    int bad_key, bad[2], abort_flag;  // by turn
    int counted;  // tokens up to the last one with a key and a strength
    unsigned tmem;
    unsigned long long done;

    // Tiles [64][64] of halves, in Q's place once it is not needed any more: G (q . k), hi and lo, and when that has been copied
    // out T diag(beta P) over K's scales; T diag(beta)
    __device__ __forceinline__ unsigned char *tile(int i) { return D == 128 ? qk[i >> 1][i & 1] : more[i]; }
};

__device__ __forceinline__ void bulk_out(void *to, const void *from, unsigned bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(su32(from)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_out_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_out_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

// x of (I + L) x = e_c, L the strictly lower part of 32 rows; at l its negative, by columns. Once x_j is known all later rows have
// their term, so that no row waits for a sum of its own.
__device__ __forceinline__ void substitute(const float *l, int c, float (&x)[32]) {
    unsigned long long s[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = pack2(2 * i == c ? 1.0f : 0.0f, 2 * i + 1 == c ? 1.0f : 0.0f);
#pragma unroll
    for (int j = 0; j < 32; ++j) {
        unpack2(s[j / 2], x[j & ~1], x[j | 1]);
        const unsigned long long by = both(x[j]);
#pragma unroll
        for (int i = (j + 1) / 4; i < 8 && j < 31; ++i) {  // (the pair of x_j itself: its term is zero)
            const ulonglong2 r = *reinterpret_cast<const ulonglong2 *>(l + j * kPitch + 4 * i);
            if (4 * i + 1 > j) s[2 * i] = fma2(r.x, by, s[2 * i]);
            s[2 * i + 1] = fma2(r.y, by, s[2 * i + 1]);
        }
    }
}
// Rows r, r + 1 and four columns from c of X Y, 32 by 32, rows of X at x, Y at y; `terms` (a multiple of 4) of X's rows count.
__device__ __forceinline__ void times(const float *x, const float *y, int r, int c, int terms, float4 (&out)[2]) {
    out[0] = out[1] = float4{0, 0, 0, 0};
#pragma unroll 2
    for (int j = 0; j < terms; j += 4) {
        const float4 f0 = *reinterpret_cast<const float4 *>(x + r * kPitch + j), f1 = *reinterpret_cast<const float4 *>(x + (r + 1) * kPitch + j);
        const float a[4] = {f0.x, f0.y, f0.z, f0.w}, b[4] = {f1.x, f1.y, f1.z, f1.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float4 g = *reinterpret_cast<const float4 *>(y + (j + e) * kPitch + c);
            out[0].x = fmaf(a[e], g.x, out[0].x), out[0].y = fmaf(a[e], g.y, out[0].y), out[0].z = fmaf(a[e], g.z, out[0].z), out[0].w = fmaf(a[e], g.w, out[0].w);
            out[1].x = fmaf(b[e], g.x, out[1].x), out[1].y = fmaf(b[e], g.y, out[1].y), out[1].z = fmaf(b[e], g.z, out[1].z), out[1].w = fmaf(b[e], g.w, out[1].w);
        }
    }
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

// Whether a channel has a token that sees nothing of `limit` or more: not what itself adds to the state, nor what that still has of earlier
// ones (one before the chunk counts, too); by a whole warp. One in 2^25 of normally distributed values makes a thread ask, and then only a
// run's first tokens see nothing larger; tokens of zeros and of strong decays. A token without a key or a strength leaves the state alone.
__device__ __noinline__ bool value_hidden(const DeltaNet &n, const DeltaRule &A, long long row0, int before, int tokens, int h, int channel, const float *key_scales,
                                          float limit) {
    const int lane = threadIdx.x & 31;
    const float *v = A.v + (long long)h * n.dim + channel, *decays = A.decay + h, *strengths = A.beta + h;
    float x[2], decay[2], held = 0.0f;
    bool wanted[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int t = lane + 32 * e;
        const long long row = row0 + t;
        const bool in = t < tokens;
        const float gain = in ? fabsf(strengths[row * n.value_heads] * (key_scales[t] * 0x1p13f)) : 0.0f;
        x[e] = in ? fabsf(v[row * A.v_stride]) * gain : 0.0f;
        decay[e] = in ? fminf(fabsf(decays[row * n.value_heads]), 1.0f) : 1.0f;
        wanted[e] = in & (gain > 0x1p-100f);
    }
    if (before) {
        float key = 0.0f;
        for (int i = lane; i < n.dim; i += 32) key = larger(key, A.k[(row0 - 1) * A.k_stride + (long long)(h % n.key_heads) * n.dim + i], 0.0f);
        held = fabsf(v[(row0 - 1) * A.v_stride] * (strengths[(row0 - 1) * n.value_heads] * (warp_largest(key) * 0.5f)));
    }
    return see_less(x, decay, x, wanted, held, limit, lane);
}

// VEC: rows of q and k can be read four channels at a time.
template <int D, bool VEC>
__global__ void __launch_bounds__(kPrepareThreads, 2) k_delta_prepare(const __grid_constant__ DeltaNet n, const __grid_constant__ DeltaRule A,
                                                                      const __grid_constant__ MixRuns r, const __grid_constant__ DeltaSlab slab) {
    using Slot = DeltaSlot<D>;
    constexpr int kPanels = D / 64, kBulk = 32;  // the thread that copies out
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    PrepareSmem<D> &M = *reinterpret_cast<PrepareSmem<D> *>(smem_raw);
    // half of the columns, row; the warp's number comes from one lane, so that what follows from it is the whole warp's (5% of the kernel)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, half = warp >> 2, gt = tid & 127, w4 = warp & 3;
    if (slab.ahead) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    else kv8_enter();
    // Of a slab ahead, this block makes the kernel end after the second one of the slab before.
    const auto leave = [&] {
        if (slab.ahead && blockIdx.x == gridDim.x - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
    };
    const int chunk = slab.chunk0 + (int)(blockIdx.x % slab.chunks), head = slab.head0 + (int)(blockIdx.x / slab.chunks % slab.heads);
    const int run = slab.run0 + (int)(blockIdx.x / slab.chunks / slab.heads), t0 = chunk * kChunk;
    const MixRun me = mix_run_alone(r, n.sequences, run, n.err);
    if (me.sequence < 0 || t0 >= me.tokens) return leave();
    const int tokens = min(kChunk, me.tokens - t0);
    const long long row0 = (long long)run * r.count + t0;
    unsigned char *slot = slab.slots + blockIdx.x * slab.slot_bytes;

    // Q's and K's rows: sixteen a warp
    constexpr int kLanes = D / 4, kRows = 32 / kLanes, kPasses = 16 / kRows;
    const int ch = 4 * (lane % kLanes);
    float f[kPasses][4];
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        const int row = warp * 16 + u * kRows + lane / kLanes, t = row & 63;
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
    if (tid == 0) {
        bar_init(&M.done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        M.abort_flag = M.bad_key = 0;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 256;" ::"r"(su32(&M.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = M.tmem, mine = tmem + ((unsigned)(w4 * 32) << 16);
    constexpr unsigned kRaw = 0, kV = 64, kU = 128, kW = 192;  // columns: [Q; K] K^T; V's halves; U^T; W^T
    const Waits wait{&M.abort_flag, n.err};
    unsigned phase = 0;
    // a power of two a row
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        const int row = warp * 16 + u * kRows + lane / kLanes;
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
    // V's column of this lane, 32 tokens
    float v[32];
    const auto load_v = [&](int h) {
        const float *p = A.v + (row0 + half * 32) * A.v_stride + (long long)h * n.dim + gt;
#pragma unroll
        for (int j = 0; j < 32; ++j, p += A.v_stride) v[j] = gt < n.dim && half * 32 + j < tokens ? *p : 0.0f;
    };
    load_v(head);
    to_async();
    __syncthreads();
    if (warp == 0) {
        if (elect_one()) {
            const unsigned long long q = sw128_desc(su32(M.qk[0][0]));
#pragma unroll
            for (int product = 0; product < 3; ++product) {  // lo hi, hi lo, hi hi
                const unsigned long long x = q + (product == 0) * (kPanels * 1024), y = q + 512 + (product == 1) * (kPanels * 1024);
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    mma_step(tmem + kRaw, x + k / 4 * 1024 + k % 4 * 2, y + k / 4 * 1024 + k % 4 * 2, idesc_f16(128, 64), product, k);
            }
            mma_commit(&M.done);
        }
        __syncwarp();
    }
    if (tid == kBulk) {
        bulk_out(slot, M.qk, 2 * Slot::tile);
        bulk_out_commit();
    }

#pragma unroll 1
    for (int m = 0; m < slab.ratio; ++m) {
        const int h = head + m * n.key_heads;
        unsigned char *out = slot + Slot::heads + (long long)m * Slot::head_bytes;
        DeltaFactors *factors = reinterpret_cast<DeltaFactors *>(out + Slot::factors);
        if (warp == 4) {
            if (lane == 0) M.bad[m & 1] = 0;
            __syncwarp();
            // decays and strengths, two tokens a lane; rows behind the run's end change nothing
            float a[2], b[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const bool in = lane + 32 * e < tokens;
                const long long at = (row0 + lane + 32 * e) * n.value_heads + h;
                a[e] = in ? A.decay[at] : 1.0f;
                b[e] = in ? A.beta[at] : 0.0f;
            }
            if (past(larger(larger(a[0], a[1], b[0]), b[1], 0.0f))) M.bad[m & 1] = 1;
            const float upto[2] = {product_upto(a[0], lane), product_upto(a[1], lane)};
            const float after[2] = {product_after(a[0], lane), product_after(a[1], lane)};
            const float low = __shfl_sync(0xffffffffu, upto[0], 31), high = __shfl_sync(0xffffffffu, upto[1], 31);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int t = lane + 32 * e;
                const float p = e ? upto[1] * low : upto[0], key = M.inv[64 + t] * 0x1p13f;
                M.decay[t] = a[e];
                M.upto[t] = upto[e];
                M.gain[t] = b[e] * key;
                M.beta[t] = b[e] * key * key;
                M.beta_w[t] = M.beta[t] * p * kKey;
                M.behind[t] = e ? kKey : kKey * after[0];
                factors->q[t] = p * M.inv[t];
                factors->k[t] = (e ? after[1] : after[0] * high) * kKey;
                if (t == 63) factors->end = p;
            }
            const unsigned low_rows = __ballot_sync(0xffffffffu, larger(M.inv[lane], M.inv[64 + lane], 0.0f) > unscale_of(-113));
            const unsigned high_rows = __ballot_sync(0xffffffffu, larger(M.inv[32 + lane], M.inv[96 + lane], 0.0f) > unscale_of(-113));
            const unsigned low_gains = __ballot_sync(0xffffffffu, fabsf(M.gain[lane]) > 0x1p-100f), high_gains = __ballot_sync(0xffffffffu, fabsf(M.gain[32 + lane]) > 0x1p-100f);
            if (lane == 0) M.counted = high_gains ? 64 - __clz(high_gains) : 32 - __clz(low_gains);
            if (lane == 0) factors->counted = high_rows ? 64 - __clz(high_rows) : 32 - __clz(low_rows);
        }
        if (tid == kBulk) bulk_out_read();  // Q's tile, or the last head's W
        __syncthreads();
        // values as what they add to the state
#pragma unroll
        for (int j = 0; j < 32; j += 4) {
            const ulonglong2 g = *reinterpret_cast<const ulonglong2 *>(&M.gain[half * 32 + j]);
            unpack2(mul2_rn(pack2(v[j], v[j + 1]), g.x), v[j], v[j + 1]);
            unpack2(mul2_rn(pack2(v[j + 2], v[j + 3]), g.y), v[j + 2], v[j + 3]);
        }
        M.most[0][half][gt] = largest(0.0f, v);
        __syncthreads();
        const float most_v = larger(M.most[0][0][gt], M.most[0][1][gt], 0.0f);
        const float inv_v = unscale_of(exponent_of(most_v));
        {
            if (past(most_v)) M.bad[m & 1] = 1;
            float least = most_v;
            if (M.counted == kChunk) {
#pragma unroll
                for (int j = 0; j < 32; j += 2) least = smaller(least, v[j], v[j + 1]);
            } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) least = half * 32 + j < M.counted ? smaller(least, v[j], least) : least;
            }
            const float limit = hidden_below(exponent_of(most_v));  // (zero where a lane has zeros)
            for (unsigned ask = __ballot_sync(0xffffffffu, least < limit); ask; ask &= ask - 1) {
                const int who = __ffs(ask) - 1;
                if (value_hidden(n, A, row0, t0, tokens, h, w4 * 32 + who, M.inv + 64, __shfl_sync(0xffffffffu, limit, who))) {
                    M.bad[m & 1] = 1;
                    break;
                }
            }
            unsigned hi[16], lo[16];
            split(v, scale_of(exponent_of(most_v)), hi, lo);
            tmem_write(mine + kV + half * 16, hi);
            tmem_write(mine + kV + 32 + half * 16, lo);
            tmem_written();
        }
        if (m == 0) wait.warp(&M.done, phase & 1, lane), ++phase;
        tc_fence_after();
        // Rows 0-63: products of queries, 64-127: of keys, each times G over the column's scale. Where row and column are of the
        // same half of the tokens, the product of decays grows from the diagonal; else it is that up to the row in its half times
        // that after the column in its own. Columns of the upper half mean nothing to rows of the lower one.
        const int i = gt & 63;
        const bool key = gt >= 64, upper = w4 & 1, empty = !upper && half;
        float *a_row = &M.a[i * kPitch + 32 * half];
        float x[32], most = 0.0f;
        if (!empty) {
            tmem_read(mine + kRaw + 32 * half, x);
            if (upper && !half) {
                const float far = M.upto[i];
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    const float4 c = *reinterpret_cast<const float4 *>(&M.behind[j]);
                    x[j] *= c.x * far, x[j + 1] *= c.y * far, x[j + 2] *= c.z * far, x[j + 3] *= c.w * far;
                }
            } else {
                const int row = i & 31, limit = key ? row - 1 : row;
                const float *decay = &M.decay[32 * half];
                float p = kKey;
#pragma unroll
                for (int j = 31; j >= 0; --j) {
                    if (j < row) p *= decay[j + 1 < 32 ? j + 1 : 31];
                    x[j] = j <= limit ? x[j] * p : 0.0f;
                }
            }
            if (key) {
                const float f = kKey * M.beta[i];
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    const float4 a{x[j] * f, x[j + 1] * f, x[j + 2] * f, x[j + 3] * f};
                    if (upper && !half) {
                        *reinterpret_cast<float4 *>(a_row + j) = a;
                    } else {  // what is substituted: by columns, its negative
                        float *to = &M.a[(32 * half + j) * kPitch + i];
                        to[0] = -a.x, to[kPitch] = -a.y, to[2 * kPitch] = -a.z, to[3 * kPitch] = -a.w;
                    }
                }
            } else {
                most = largest(0.0f, x);
            }
        }
        M.most[1][half][gt] = most;
        __syncthreads();
        if (!key) {
            const float weight = larger(M.most[1][0][gt], M.most[1][1][gt], 0.0f);
            if (!(weight <= kLargestWeight)) M.bad[m & 1] = 1;
            const int e = exponent_of(weight);
            unsigned hi[16] = {}, lo[16] = {};
            if (!empty) split(x, scale_of(e), hi, lo);
            put_pieces(M.tile(0), i, half * 4, hi);
            put_pieces(M.tile(1), i, half * 4, lo);
            if (!half) factors->attn[i] = unscale_of(e) * M.inv[i];
            to_async();
        } else if (!half) {
            // T: the inverses of the two blocks of 32 on the diagonal, a warp each
            float *block = M.a + (w4 == 2 ? 0 : 32 * kPitch + 32), c[32];
            substitute(block, lane, c);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 32; ++j) block[j * kPitch + lane] = c[j];
        }
        __syncthreads();
        if (tid == 128 + kBulk) {
            bulk_out(out + Slot::g, M.tile(0), 8192);
            bulk_out(out + Slot::g + 8192, M.tile(1), 8192);
            bulk_out_commit();
            bulk_out_read();
        }
        if (!half) {
            // the lower left is -T22 (A21 T11); the second factor waits in the upper right
            const int row = (gt >> 3) * 2, col = (gt & 7) * 4;
            float *a12 = M.a + 32, *a21 = M.a + 32 * kPitch, *a22 = a21 + 32;
            float4 o[2];
            times(a21, M.a, row, col, 32, o);
            *reinterpret_cast<float4 *>(a12 + row * kPitch + col) = o[0];
            *reinterpret_cast<float4 *>(a12 + (row + 1) * kPitch + col) = o[1];
            asm volatile("bar.sync 1, 128;" ::: "memory");
            times(a22, a12, row, col, 8 * w4 + 8, o);
            *reinterpret_cast<float4 *>(a21 + row * kPitch + col) = float4{-o[0].x, -o[0].y, -o[0].z, -o[0].w};
            *reinterpret_cast<float4 *>(a21 + (row + 1) * kPitch + col) = float4{-o[1].x, -o[1].y, -o[1].z, -o[1].w};
        }
        __syncthreads();
        // T's rows as operands: threads 0-63 for U, 64-127 for W
        most = 0.0f;
        if (!empty) {  // (the upper right holds what is no part of T)
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
                const float4 t = *reinterpret_cast<const float4 *>(a_row + j);
                x[j] = t.x, x[j + 1] = t.y, x[j + 2] = t.z, x[j + 3] = t.w;
            }
            if (key) {
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    const float4 b = *reinterpret_cast<const float4 *>(&M.beta_w[32 * half + j]);
                    x[j] *= b.x, x[j + 1] *= b.y, x[j + 2] *= b.z, x[j + 3] *= b.w;
                }
            }
            most = largest(0.0f, x);
        }
        M.most[0][half][gt] = most;
        __syncthreads();
        most = larger(M.most[0][0][gt], M.most[0][1][gt], 0.0f);
        if (past(most)) M.bad[m & 1] = 1;
        {
            const int e = exponent_of(most);
            unsigned hi[16] = {}, lo[16] = {};
            if (!empty) split(x, scale_of(e), hi, lo);
            put_pieces(M.tile(key ? 0 : 2), i, half * 4, hi);
            put_pieces(M.tile(key ? 1 : 3), i, half * 4, lo);
            if (!half) {
                if (key) factors->z[i] = unscale_of(e) * (1.0f / kWScale);
                else M.inv_tu[i] = unscale_of(e);
            }
        }
        to_async();
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        if (warp == 0) {
            if (elect_one()) {
                // (of 64 channels the wide operand's second 64 rows are the first ones again, and nobody looks)
                const unsigned long long keys = turned_desc(su32(M.qk[0][0]) + 8192, D == 128 ? 16384 : 0);
                const unsigned long long tw[2] = {sw128_desc(su32(M.tile(0))), sw128_desc(su32(M.tile(1)))};
                const unsigned long long tu[2] = {sw128_desc(su32(M.tile(2))), sw128_desc(su32(M.tile(3)))};
#pragma unroll
                for (int product = 0; product < 3; ++product)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_step_ts(tmem + kU, tmem + kV + (product == 0) * 32 + k * 8, tu[product == 1] + k * 2, idesc_f16(128, 64), product, k);
#pragma unroll
                for (int product = 0; product < 3; ++product)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_step(tmem + kW, keys + (product == 0) * (kPanels * 1024) + k * 128, tw[product == 1] + k * 2, idesc_f16(128, 64) | kTurnedWide,
                                 product, k);
                mma_commit(&M.done);
            }
            __syncwarp();
        }
        if (m + 1 < slab.ratio) load_v(h + n.key_heads);
        wait.warp(&M.done, phase & 1, lane), ++phase;
        tc_fence_after();
        if (w4 < D / 32) {
            tmem_read(mine + kU + half * 32, x);
            float *to = reinterpret_cast<float *>(out + Slot::uu) + half * 32 * D + gt;
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
                const float4 f = *reinterpret_cast<const float4 *>(&M.inv_tu[half * 32 + j]);
                to[j * D] = x[j] * inv_v * f.x, to[j * D + D] = x[j + 1] * inv_v * f.y;
                to[j * D + 2 * D] = x[j + 2] * inv_v * f.z, to[j * D + 3 * D] = x[j + 3] * inv_v * f.w;
            }
            unsigned hi[16], lo[16];
            tmem_read(mine + kW + half * 32, x);
            split(x, kWScale, hi, lo);
            put_pieces(M.w[0], gt, half * 4, hi);
            put_pieces(M.w[1], gt, half * 4, lo);
        }
        to_async();
        tc_fence_before();
        __syncthreads();
        tc_fence_after();
        if (tid == kBulk) {
            factors->walk = M.bad[m & 1] | M.bad_key;
            bulk_out(out + Slot::w, M.w, Slot::tile);
            bulk_out_commit();
        }
        __syncwarp();
    }
    if (tid == kBulk || tid == 128 + kBulk) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    tc_fence_before();
    __syncthreads();
    settle(&M.abort_flag);
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 256;" ::"r"(tmem) : "memory");
    leave();
}

template <int D, bool VEC>
cudaError_t launch_prepare(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, const DeltaSlab &slab, cudaStream_t s) {
    const cudaError_t e = mix_shared_memory<k_delta_prepare<D, VEC>>(sizeof(PrepareSmem<D>));
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
