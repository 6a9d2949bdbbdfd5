// The chunked delta rule's first kernel: what a chunk needs that does not depend on the state (delta_chunk.cuh).
//
// A block has a run's chunk and key head, and takes the head's value heads two at a time, one by each warpgroup:
//   [Q; K] K^T      128 rows by 64, once for all of them
//   A, G (q . k)    a thread a row, from its TMEM lane
//   T = (I + A)^-1  halves' inverses by substitution, a column a lane, then -T22 (A21 T11); F32 throughout
//   U^T = V^T (T diag(beta))^T   a lane a value channel, V straight from memory to TMEM
//   W = (T diag(beta P)) K       both heads' 64 rows as one operand; K's tile as it lies, read the other way round
#include "delta_chunk.cuh"

#include <atomic>

namespace strata {
namespace {

using namespace delta;

constexpr int kPrepareThreads = 256, kPitch = 68;

template <int D>
struct __align__(1024) PrepareSmem {
    unsigned char qk[2][D / 64][128 * 128];  // hi, lo: panels of 64 channels; rows 0-63 Q, 64-127 K
    unsigned char tw[2][128 * 128];          // T diag(beta P) over K's scales: two heads' 64 rows
    unsigned char tu[2][2][64 * 128];        // by head: T diag(beta)
    float a[2][64 * kPitch];                 // A, then T; the upper right quarter has A21 T11
    float inv[128];                          // Q's and K's scales taken back
    float decay[2][64], beta[2][64], upto[2][64];
    float inv_tw[2][64], inv_tu[2][64];
    float w_max[2][128];
    int bad_key, bad[2], abort_flag;
    unsigned tmem;
    unsigned long long done;
};

__device__ __forceinline__ void group_sync(int g) { asm volatile("bar.sync %0, 128;" ::"r"(1 + g) : "memory"); }

// x[j] of the unit triangular system (I + L) x = e_c, L the strictly lower part of 32 rows at l
__device__ __forceinline__ void substitute(const float *l, int c, float (&x)[32]) {
#pragma unroll
    for (int i = 0; i < 32; ++i) {
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
// eight columns of row r of sign * X Y, 32 by 32 at x and y; X's row has `terms` values that count
__device__ __forceinline__ void times(const float *x, const float *y, int r, int c, int terms, float (&out)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) out[e] = 0.0f;
#pragma unroll 8
    for (int j = 0; j < 32; ++j) {
        const float f = j < terms ? x[r * kPitch + j] : 0.0f;
        const float4 a = *reinterpret_cast<const float4 *>(y + j * kPitch + c), b = *reinterpret_cast<const float4 *>(y + j * kPitch + c + 4);
        out[0] = fmaf(f, a.x, out[0]), out[1] = fmaf(f, a.y, out[1]), out[2] = fmaf(f, a.z, out[2]), out[3] = fmaf(f, a.w, out[3]);
        out[4] = fmaf(f, b.x, out[4]), out[5] = fmaf(f, b.y, out[5]), out[6] = fmaf(f, b.z, out[6]), out[7] = fmaf(f, b.w, out[7]);
    }
}

// VEC: rows of q and k can be read four channels at a time.
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
    const unsigned kRaw = 0, kV = 64 + 64 * g, kWAt = 192, kU = 320 + 64 * g;  // columns
    const Waits wait{&M.abort_flag, n.err};
    unsigned phase = 0;

    // Q's and K's rows, a power of two each
    constexpr int kLanes = D / 4, kRows = 32 / kLanes;
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
            unsigned m = __float_as_uint(largest(f[u]));
#pragma unroll
            for (int s = kLanes / 2; s > 0; s >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, s));
            const int e = exponent_of(__uint_as_float(m));
            if (lane % kLanes == 0) M.inv[row] = unscale_of(e);
            if (past(__uint_as_float(m))) M.bad_key = 1;
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
            for (int product = 0; product < 3; ++product) {  // lo hi, hi lo, hi hi
                const int x = product == 0, y = product == 1;
                for (int k = 0; k < D / 16; ++k)
                    mma_f16(tmem + kRaw, sw128_desc(su32(M.qk[x][k / 4])) + k % 4 * 2, sw128_desc(su32(M.qk[y][k / 4]) + 8192) + k % 4 * 2,
                            idesc_f16(128, 64), product || k);
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

    for (int pair = 0; pair < slab.ratio; pair += 2) {
        const int m = pair + g, h = head + m * n.key_heads;
        const bool there = m < slab.ratio;
        unsigned char *mine_out = slot + Slot::heads + (long long)m * Slot::head_bytes;
        DeltaFactors *factors = reinterpret_cast<DeltaFactors *>(mine_out + Slot::factors);
        if (gt == 0) M.bad[g] = 0;
        float inv_v = 0.0f;
        if (there) {
            // decays and strengths; rows behind the run's end change nothing
            const int t = gt & 63;
            const bool in = t < tokens;
            const long long at = (row0 + t) * n.value_heads + h;
            const float x = gt < 64 ? (in ? A.decay[at] : 1.0f) : (in ? A.beta[at] : 0.0f);
            (gt < 64 ? M.decay[g] : M.beta[g])[t] = x;
            // V's column of this lane to TMEM
            float v[64];
            const float *p = A.v + row0 * A.v_stride + (long long)h * n.dim + gt;
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = gt < n.dim && j < tokens ? p[j * A.v_stride] : 0.0f;
            group_sync(g);  // bad[g] has been cleared
            const float most = largest(v);
            const int e = exponent_of(most);
            inv_v = unscale_of(e);
            if (past(most) || past(fabsf(x))) M.bad[g] = 1;
            unsigned hi[32], lo[32];
            split(v, scale_of(e), hi, lo);
            tmem_write(mine + kV, hi);
            tmem_write(mine + kV + 32, lo);
            tmem_written();
        }
        if (pair == 0) wait(&M.done, phase & 1), ++phase;
        tc_fence_after();
        if (there) {
            float x[64];
            tmem_read(mine + kRaw, x);
            const int i = gt & 63;
            const bool key = gt >= 64;
            // x_j G_ij over the scales; the product of decays grows from j = i down
            const float inv_i = M.inv[gt];
            float p = 1.0f;
#pragma unroll
            for (int j = 63; j >= 0; --j) {
                if (j < i) p *= M.decay[g][(j + 1) & 63];
                if (key && i == 63) factors->k[j] = p * M.inv[64 + j];
                x[j] = j < i || (j == i && !key) ? x[j] * M.inv[64 + j] * p * inv_i : 0.0f;
            }
            const float upto = p * M.decay[g][0];
            if (key) {
                const float b = M.beta[g][i];
#pragma unroll
                for (int j = 0; j < 64; j += 4)
                    *reinterpret_cast<float4 *>(&M.a[g][i * kPitch + j]) = float4{x[j] * b, x[j + 1] * b, x[j + 2] * b, x[j + 3] * b};
                M.upto[g][i] = upto;
                if (i == 63) factors->end = upto;
            } else {
                const int e = exponent_of(largest(x));
                unsigned hi[32], lo[32];
                split(x, scale_of(e), hi, lo);
                put_pieces(mine_out + Slot::g, i, 0, hi);
                put_pieces(mine_out + Slot::g + 8192, i, 0, lo);
                factors->attn[i] = unscale_of(e);
                factors->q[i] = upto * inv_i;
            }
            group_sync(g);
            float *a = M.a[g], *a21 = a + 32 * kPitch, *a12 = a + 32, *a22 = a21 + 32;
            if (w4 >= 2) {  // a warp each: the inverses of the two quarters on the diagonal
                float *block = w4 == 2 ? a : a22;
                float c[32];
                substitute(block, lane, c);
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 32; ++j) block[j * kPitch + lane] = c[j];
            }
            group_sync(g);
            float out[8];
            const int row = gt >> 2, col = gt % 4 * 8;
            times(a21, a, row, col, 32, out);
            *reinterpret_cast<float4 *>(a12 + row * kPitch + col) = float4{out[0], out[1], out[2], out[3]};
            *reinterpret_cast<float4 *>(a12 + row * kPitch + col + 4) = float4{out[4], out[5], out[6], out[7]};
            group_sync(g);
            times(a22, a12, row, col, row + 1, out);
            *reinterpret_cast<float4 *>(a21 + row * kPitch + col) = float4{-out[0], -out[1], -out[2], -out[3]};
            *reinterpret_cast<float4 *>(a21 + row * kPitch + col + 4) = float4{-out[4], -out[5], -out[6], -out[7]};
            group_sync(g);
            // T's rows as operands: threads 0-63 for U, 64-127 for W
#pragma unroll
            for (int j = 0; j < 64; j += 4) {
                const float4 f = *reinterpret_cast<const float4 *>(a + i * kPitch + j);
                x[j] = f.x, x[j + 1] = f.y, x[j + 2] = f.z, x[j + 3] = f.w;
            }
#pragma unroll
            for (int j = 0; j < 64; ++j) {
                const float by = key ? M.beta[g][j] * M.upto[g][j] * M.inv[64 + j] : M.beta[g][j];
                x[j] = j <= i ? x[j] * by : 0.0f;
            }
            const float most = largest(x);
            if (past(most)) M.bad[g] = 1;
            const int e = exponent_of(most);
            unsigned hi[32], lo[32];
            split(x, scale_of(e), hi, lo);
            put_pieces(key ? M.tw[0] : M.tu[g][0], key ? g * 64 + i : i, 0, hi);
            put_pieces(key ? M.tw[1] : M.tu[g][1], key ? g * 64 + i : i, 0, lo);
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
                for (int w = 0; w < 2 && pair + w < slab.ratio; ++w)  // U^T: lanes are value channels
                    for (int product = 0; product < 3; ++product)
                        for (int k = 0; k < 4; ++k)
                            mma_f16_ts(tmem + 320 + 64 * w, tmem + 64 + 64 * w + (product == 0) * 32 + k * 8,
                                       sw128_desc(su32(M.tu[w][product == 1])) + k * 2, idesc_f16(128, 64), product || k);
                for (int product = 0; product < 3; ++product)
                    for (int k = 0; k < 4; ++k)
                        mma_f16(tmem + kWAt, sw128_desc(su32(M.tw[product == 0])) + k * 2,
                                turned_desc(su32(M.qk[product == 1][0]) + 8192 + k * 2048, 16384), turned_idesc(128, D), product || k);
                mma_commit(&M.done);
            }
            __syncwarp();
        }
        wait(&M.done, phase & 1), ++phase;
        tc_fence_after();
        if (there) {
            float u[64];
            tmem_read(mine + kU, u);
            float *to = reinterpret_cast<float *>(mine_out + Slot::uu) + gt;
            if (gt < D) {
#pragma unroll
                for (int i = 0; i < 64; ++i) to[i * D] = u[i] * inv_v * M.inv_tu[g][i];
            }
        }
        // W's rows: lane w4 * 32 + lane is row i of the pair's head `of`; this warpgroup has half of its channels
        float w[kW];
        tmem_read(mine + kWAt + g * kW, w);
        const int of = w4 >> 1, i = gt & 63;
        const float inv = M.inv_tw[of][i];
#pragma unroll
        for (int c = 0; c < kW; ++c) w[c] *= inv;
        M.w_max[g][gt] = largest(w);
        __syncthreads();
        const float most = fmaxf(M.w_max[0][gt], M.w_max[1][gt]);
        if (past(M.w_max[0][gt]) || past(M.w_max[1][gt])) M.bad[of] = 1;
        if (pair + of < slab.ratio) {
            unsigned char *out = slot + Slot::heads + (long long)(pair + of) * Slot::head_bytes;
            const int e = exponent_of(most);
            unsigned hi[kW / 2], lo[kW / 2];
            split(w, scale_of(e), hi, lo);
            const int panel = D == 128 ? g : 0, first = D == 128 ? 0 : g * 4;
            put_pieces(out + Slot::w + panel * 8192, i, first, hi);
            put_pieces(out + Slot::w + (kPanels + panel) * 8192, i, first, lo);
            if (g == 0) reinterpret_cast<DeltaFactors *>(out + Slot::factors)->z[i] = unscale_of(e);
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
