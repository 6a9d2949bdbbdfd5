// The chunked delta rule's second kernel: a run's state of one value head, from chunk to chunk (delta_chunk.cuh).
//
// A block has a run's value head. A thread of its sixteen working warps has a value channel (its TMEM lane) with a quarter of
// the state's keys, in F32 registers; the state and the differences go to TMEM as the products' 128-row operand straight from
// there, and what kernel one left comes through bulk copies as the narrow one:
//   Z^T = S^T W^T,  R^T = S^T Q^T        128 value channels by 64 tokens, sums over keys
//   D = U - Z;  new state's part = (E D)^T K        128 by D keys, sums over tokens; K's tile read the other way round
//   Y^T = D^T G^T;  y = P R + Y          128 by 64 tokens
// One warp fetches, one issues; results of a chunk are written while the next one's first product runs.
#include "delta_chunk.cuh"

#include <atomic>

namespace strata {
namespace {

using namespace delta;

constexpr int kWork = 512, kChainThreads = kWork + 64, kFetchWarp = 16, kIssueWarp = 17;

template <int D>
struct __align__(1024) ChainSmem {
    unsigned char w[2][2][D * 128];            // by stage: hi, lo; rows are key channels
    unsigned char q[2][2 * D / 64][64 * 128];  // by stage: hi panels, lo panels
    unsigned char k[2 * D / 64][64 * 128];
    unsigned char g[2][64 * 128];  // hi, lo
    float u[64 * D];
    DeltaFactors factors[2];
    float s_max[4][128];
    float2 d_max[4][128];  // also the sums of chunks that are walked
    unsigned long long w_full[2], w_empty[2], q_full[2], q_empty[2], f_full[2], f_empty[2], k_full, k_empty, g_full, g_empty, u_full, u_empty;
    unsigned long long s_ready, r_free, d_ready, y_ready, z_done, r_done, d_done, y_done;
    unsigned tmem;
    int abort_flag;
};

__device__ __forceinline__ void lane_sync(int w4) { asm volatile("bar.sync %0, 128;" ::"r"(1 + w4) : "memory"); }  // of the same lanes
__device__ __forceinline__ void work_sync() { asm volatile("bar.sync 5, 512;" ::: "memory"); }

template <int D>
__global__ void __launch_bounds__(kChainThreads, 1) k_delta_chain(DeltaNet n, DeltaRule A, MixRuns r, DeltaSlab slab) {
    using Slot = DeltaSlot<D>;
    constexpr int kPart = D / 4;  // keys of a thread; and 16 tokens
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    ChainSmem<D> &M = *reinterpret_cast<ChainSmem<D> *>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    kv8_enter();
    const int m = (int)(blockIdx.x % slab.ratio), head_l = (int)(blockIdx.x / slab.ratio % slab.heads), run_l = (int)(blockIdx.x / slab.ratio / slab.heads);
    const int h = slab.head0 + head_l + m * n.key_heads, run = slab.run0 + run_l;
    const MixRun me = mix_run_alone(r, n.sequences, run, n.err);
    const long long first = (long long)run * r.count, vw = (long long)n.value_heads * n.dim;
    const int begin = slab.chunk0 * kChunk;
    if (me.sequence < 0) {
        const long long end = min((long long)r.count, (long long)begin + (long long)slab.chunks * kChunk), rows = end - begin;
        for (long long i = tid; i < rows * n.dim; i += kChainThreads) A.y[(first + begin + i / n.dim) * vw + (long long)h * n.dim + i % n.dim] = 0.0f;
        return;
    }
    if (begin >= me.tokens) return;
    const int chunks = min(slab.chunks, (me.tokens - begin + kChunk - 1) / kChunk);
    const unsigned char *slots = slab.slots + ((long long)run_l * slab.heads + head_l) * slab.chunks * slab.slot_bytes;
    const long long mine = Slot::heads + (long long)m * Slot::head_bytes;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            bar_init(&M.w_full[i], 1), bar_init(&M.w_empty[i], 1), bar_init(&M.q_full[i], 1), bar_init(&M.q_empty[i], 1);
            bar_init(&M.f_full[i], 1), bar_init(&M.f_empty[i], kWork / 32 + 1);
        }
        bar_init(&M.k_full, 1), bar_init(&M.k_empty, 1), bar_init(&M.g_full, 1), bar_init(&M.g_empty, 1);
        bar_init(&M.u_full, 1), bar_init(&M.u_empty, kWork / 32);
        bar_init(&M.s_ready, kWork / 32), bar_init(&M.r_free, kWork / 32), bar_init(&M.d_ready, kWork / 32), bar_init(&M.y_ready, kWork / 32);
        bar_init(&M.z_done, 1), bar_init(&M.r_done, 1), bar_init(&M.d_done, 1), bar_init(&M.y_done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        M.abort_flag = 0;
    }
    if (warp == kIssueWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&M.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = M.tmem;
    // columns: the state's halves, under whose place Y's operand goes once R has been formed; E D's; Z, R, Y, the new state's part
    constexpr unsigned kS = 0, kSLo = D / 2, kD = 128, kZ = 192, kR = 256, kY = 320, kNew = 384;
    const Waits wait{&M.abort_flag, n.err};

    if (warp == kFetchWarp) {
        if (lane == 0) {
            const auto fetch = [&](void *to, const unsigned char *from, unsigned bytes, unsigned long long *full) {
                bar_expect(full, bytes);
                bulk(to, from, bytes, full);
            };
            for (int c = 0; c < chunks; ++c) {
                const int st = c & 1;
                const unsigned again = (c >> 1 & 1) ^ 1;
                const unsigned char *slot = slots + c * slab.slot_bytes;
                wait(&M.f_empty[st], again);
                fetch(&M.factors[st], slot + mine + Slot::factors, sizeof(DeltaFactors), &M.f_full[st]);
                wait(&M.w_empty[st], again);
                fetch(M.w[st], slot + mine + Slot::w, Slot::tile, &M.w_full[st]);
                wait(&M.q_empty[st], again);
                fetch(M.q[st], slot + Slot::q, Slot::tile, &M.q_full[st]);
                wait(&M.u_empty, (c & 1) ^ 1);
                fetch(M.u, slot + mine + Slot::uu, Slot::u, &M.u_full);
                wait(&M.k_empty, (c & 1) ^ 1);
                fetch(M.k, slot + Slot::k, Slot::tile, &M.k_full);
                wait(&M.g_empty, (c & 1) ^ 1);
                fetch(M.g, slot + mine + Slot::g, Slot::attn, &M.g_full);
            }
        }
        __syncwarp();
    } else if (warp == kIssueWarp) {
        if (elect_one()) {
            unsigned live = 0;  // chunks on the tensor cores so far
            for (int c = 0; c < chunks; ++c) {
                const int st = c & 1;
                const unsigned ph = c >> 1 & 1;
                wait(&M.f_full[st], ph);
                const bool walk = M.factors[st].walk != 0;
                bar_arrive(&M.f_empty[st]);
                if (walk) {  // nothing of it is used
                    wait(&M.w_full[st], ph), wait(&M.q_full[st], ph), wait(&M.k_full, c & 1), wait(&M.g_full, c & 1);
                    bar_arrive(&M.w_empty[st]), bar_arrive(&M.q_empty[st]), bar_arrive(&M.k_empty), bar_arrive(&M.g_empty);
                    continue;
                }
                const unsigned now = live & 1;
                ++live;
                constexpr unsigned kLoTile = D / 64 * 512;  // from a tile's hi panels to its lo ones, in 16-byte units
                wait(&M.w_full[st], ph);
                wait(&M.s_ready, now);
                tc_fence_after();
                const unsigned long long w = turned_desc(su32(M.w[st]), 0), q = sw128_desc(su32(M.q[st]));
#pragma unroll
                for (int product = 0; product < 3; ++product)  // lo hi, hi lo, hi hi
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        mma_f16_ts(tmem + kZ, tmem + (product == 0 ? kSLo : kS) + k * 8, w + (product == 1) * kLoTile + k * 128, turned_idesc(128, 64),
                                   product || k);
                mma_commit(&M.w_empty[st]);
                mma_commit(&M.z_done);
                wait(&M.q_full[st], ph);
                wait(&M.r_free, now);
                tc_fence_after();
#pragma unroll
                for (int product = 0; product < 3; ++product)
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        mma_f16_ts(tmem + kR, tmem + (product == 0 ? kSLo : kS) + k * 8, q + (product == 1) * kLoTile + k / 4 * 512 + k % 4 * 2,
                                   idesc_f16(128, 64), product || k);
                mma_commit(&M.q_empty[st]);
                mma_commit(&M.r_done);
                wait(&M.k_full, c & 1);
                wait(&M.d_ready, now);
                tc_fence_after();
                const unsigned long long keys = turned_desc(su32(M.k[0]), 8192), g = sw128_desc(su32(M.g[0]));
#pragma unroll
                for (int product = 0; product < 3; ++product)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_f16_ts(tmem + kNew, tmem + kD + (product == 0) * 32 + k * 8, keys + (product == 1) * kLoTile + k * 128, turned_idesc(128, D),
                                   product || k);
                mma_commit(&M.k_empty);
                mma_commit(&M.d_done);
                wait(&M.g_full, c & 1);
                wait(&M.y_ready, now);
                tc_fence_after();
#pragma unroll
                for (int product = 0; product < 3; ++product)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_f16_ts(tmem + kY, tmem + kS + (product == 0) * 32 + k * 8, g + (product == 1) * 512 + k * 2, idesc_f16(128, 64), product || k);
                mma_commit(&M.g_empty);
                mma_commit(&M.y_done);
            }
        }
        __syncwarp();
    } else if (warp < kFetchWarp) {
        const int w4 = warp & 3, part = warp >> 2, v = w4 * 32 + lane;
        const unsigned lanes = tmem + ((unsigned)(w4 * 32) << 16);
        const bool in = v < n.dim;
        const auto arrive = [&](unsigned long long *b) {
            __syncwarp();
            if (lane == 0) bar_arrive(b);
        };
        float *state = n.state + ((long long)me.sequence * n.dim + part * kPart) * vw + (long long)h * n.dim + v;
        float S[kPart];
#pragma unroll
        for (int i = 0; i < kPart; ++i) S[i] = in && part * kPart + i < n.dim ? state[i * vw] : 0.0f;
        unsigned live = 0;
        bool owed = false;            // the chunk before has results in TMEM
        float inv_r = 0, inv_y = 0;   // their scales taken back
        // results of chunk c: its tokens part * 16 ..
        const auto write_y = [&](int c) {
            const float4 *fq = reinterpret_cast<const float4 *>(M.factors[c & 1].q + part * 16);
            const float4 *fa = reinterpret_cast<const float4 *>(M.factors[c & 1].attn + part * 16);
            const int t0 = begin + c * kChunk + part * 16, left = in ? me.tokens - t0 : 0;
            float *y = A.y + (first + t0) * vw + (long long)h * n.dim + v;
            float R[16], Y[16];
            tmem_read(lanes + kR + part * 16, R);
            tmem_read(lanes + kY + part * 16, Y);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 q = fq[i], a = fa[i];
                R[4 * i] = fmaf(R[4 * i] * inv_r, q.x, Y[4 * i] * inv_y * a.x);
                R[4 * i + 1] = fmaf(R[4 * i + 1] * inv_r, q.y, Y[4 * i + 1] * inv_y * a.y);
                R[4 * i + 2] = fmaf(R[4 * i + 2] * inv_r, q.z, Y[4 * i + 2] * inv_y * a.z);
                R[4 * i + 3] = fmaf(R[4 * i + 3] * inv_r, q.w, Y[4 * i + 3] * inv_y * a.w);
            }
            if (left >= 16) {
#pragma unroll
                for (int i = 0; i < 16; ++i, y += vw) *y = R[i];
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i, y += vw)
                    if (i < left) *y = R[i];
            }
            arrive(&M.f_empty[c & 1]);
        };
        for (int c = 0; c < chunks; ++c) {
            const int st = c & 1;
            wait(&M.f_full[st], c >> 1 & 1);
            const DeltaFactors &f = M.factors[st];
            if (owed) wait(&M.y_done, (live - 1) & 1), tc_fence_after();
            if (f.walk) {
                if (owed) write_y(c - 1);
                owed = false;
                // token by token: a channel's four threads add up their parts of the keys
                const int t0 = begin + c * kChunk, tokens = min(kChunk, me.tokens - t0);
                for (int t = 0; t < tokens; ++t) {
                    const long long row = first + t0 + t;
                    // (volatile: one after another, not 128 registers of them)
                    const volatile float *kp = A.k + row * A.k_stride + (long long)(slab.head0 + head_l) * n.dim + part * kPart;
                    const volatile float *qp = A.q + row * A.q_stride + (long long)(slab.head0 + head_l) * n.dim + part * kPart;
                    const float a = A.decay[row * n.value_heads + h], b = A.beta[row * n.value_heads + h];
                    const float value = in ? A.v[row * A.v_stride + (long long)h * n.dim + v] : 0.0f;
                    float p = 0.0f, y = 0.0f;
#pragma unroll
                    for (int i = 0; i < kPart; ++i) {
                        S[i] *= a;
                        p = fmaf(S[i], part * kPart + i < n.dim ? kp[i] : 0.0f, p);
                    }
                    M.d_max[part][v].x = p;
                    lane_sync(w4);
                    const float d = b * (value - ((M.d_max[0][v].x + M.d_max[1][v].x) + (M.d_max[2][v].x + M.d_max[3][v].x)));
#pragma unroll
                    for (int i = 0; i < kPart; ++i) {
                        if (part * kPart + i < n.dim) {
                            S[i] = fmaf(kp[i], d, S[i]);
                            y = fmaf(S[i], qp[i], y);
                        }
                    }
                    M.d_max[part][v].y = y;
                    lane_sync(w4);
                    if (part == 0 && in)
                        A.y[row * vw + (long long)h * n.dim + v] = (M.d_max[0][v].y + M.d_max[1][v].y) + (M.d_max[2][v].y + M.d_max[3][v].y);
                }
                arrive(&M.f_empty[st]);
                wait(&M.u_full, c & 1);
                arrive(&M.u_empty);
                continue;
            }
            const unsigned now = live & 1;
            ++live;
            // the state as an operand
            M.s_max[part][v] = largest(0.0f, S);
            lane_sync(w4);
            const int es = exponent_of(larger(larger(M.s_max[0][v], M.s_max[1][v], M.s_max[2][v]), M.s_max[3][v], 0.0f));
            const float inv_s = unscale_of(es);
#pragma unroll
            for (int i = 0; i < kPart; i += 16) {
                float x[16];
                unsigned hi[8], lo[8];
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = S[i + e];
                split(x, scale_of(es), hi, lo);
                tmem_write(lanes + kS + (part * kPart + i) / 2, hi);
                tmem_write(lanes + kSLo + (part * kPart + i) / 2, lo);
            }
            tmem_written();
            arrive(&M.s_ready);
            if (owed) {
                write_y(c - 1);
                tc_fence_before();
            }
            arrive(&M.r_free);
            inv_r = inv_s;
            // differences, and as the decays to the chunk's end leave them
            wait(&M.u_full, c & 1);
            wait(&M.z_done, now);
            tc_fence_after();
            float d[16], e[16];
            const float *u = M.u + part * 16 * D + (v < D ? v : 0);
            const float4 *fz = reinterpret_cast<const float4 *>(f.z + part * 16), *fk = reinterpret_cast<const float4 *>(f.k + part * 16);
            const float by = v < D ? -inv_s : 0.0f, keep = v < D ? 1.0f : 0.0f;
            tmem_read(lanes + kZ + part * 16, d);
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const float4 z = fz[i / 4], k = fk[i / 4];
                d[i] = fmaf(d[i] * by, z.x, u[i * D] * keep), d[i + 1] = fmaf(d[i + 1] * by, z.y, u[i * D + D] * keep);
                d[i + 2] = fmaf(d[i + 2] * by, z.z, u[i * D + 2 * D] * keep), d[i + 3] = fmaf(d[i + 3] * by, z.w, u[i * D + 3 * D] * keep);
                e[i] = d[i] * k.x, e[i + 1] = d[i + 1] * k.y, e[i + 2] = d[i + 2] * k.z, e[i + 3] = d[i + 3] * k.w;
            }
            arrive(&M.u_empty);
            M.d_max[part][v] = float2{largest(0.0f, d), largest(0.0f, e)};
            lane_sync(w4);
            const float2 m0 = M.d_max[0][v], m1 = M.d_max[1][v], m2 = M.d_max[2][v], m3 = M.d_max[3][v];
            const int ed = exponent_of(larger(larger(m0.x, m1.x, m2.x), m3.x, 0.0f)), ee = exponent_of(larger(larger(m0.y, m1.y, m2.y), m3.y, 0.0f));
            unsigned hi[8], lo[8];
            split(e, scale_of(ee), hi, lo);
            tmem_write(lanes + kD + part * 8, hi);
            tmem_write(lanes + kD + 32 + part * 8, lo);
            tmem_written();
            arrive(&M.d_ready);
            split(d, scale_of(ed), hi, lo);
            wait(&M.r_done, now);  // the state's halves have been read
            tc_fence_after();
            tmem_write(lanes + kS + part * 8, hi);
            tmem_write(lanes + kS + 32 + part * 8, lo);
            tmem_written();
            arrive(&M.y_ready);
            inv_y = unscale_of(ed);
            // the new state
            wait(&M.d_done, now);
            tc_fence_after();
            const float inv_e = unscale_of(ee), end = f.end;
#pragma unroll
            for (int i = 0; i < kPart; i += 16) {
                float x[16];
                tmem_read(lanes + kNew + part * kPart + i, x);
#pragma unroll
                for (int e = 0; e < 16; ++e) S[i + e] = fmaf(x[e], inv_e, S[i + e] * end);
            }
            tc_fence_before();
            owed = true;
        }
        if (owed) {
            wait(&M.y_done, (live - 1) & 1);
            tc_fence_after();
            write_y(chunks - 1);
        }
        work_sync();
        if (!*(volatile int *)&M.abort_flag) {
#pragma unroll
            for (int i = 0; i < kPart; ++i)
                if (in && part * kPart + i < n.dim) state[i * vw] = S[i];
        }
    }
    tc_fence_before();
    __syncthreads();
    settle(&M.abort_flag);
    if (warp == kIssueWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <int D>
cudaError_t launch_chain(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, const DeltaSlab &slab, cudaStream_t s) {
    constexpr int kDevices = 64;
    static std::atomic<bool> done[kDevices];
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess && (device >= kDevices || !done[device].load(std::memory_order_relaxed))) {
        e = cudaFuncSetAttribute(k_delta_chain<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(ChainSmem<D>));
        if (e == cudaSuccess && device < kDevices) done[device].store(true, std::memory_order_relaxed);
    }
    if (e != cudaSuccess) return e;
    return kv8_launch(k_delta_chain<D>, dim3((unsigned)(slab.runs * slab.heads * slab.ratio)), dim3(kChainThreads), sizeof(ChainSmem<D>), 1, s, n, a, r,
                      slab);
}

}  // namespace

cudaError_t delta_chain(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, const DeltaSlab &slab, cudaStream_t s) {
    return n.dim <= 64 ? launch_chain<64>(n, a, r, slab, s) : launch_chain<128>(n, a, r, slab, s);
}

}  // namespace strata
