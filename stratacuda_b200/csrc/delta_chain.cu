// The chunked delta rule's second kernel: a run's state of one value head, from chunk to chunk (delta_chunk.cuh).
//
// A block has a run's value head. A thread of its sixteen working warps has a value channel (its TMEM lane) with a quarter of
// the state's keys, in F32 registers; the state and the differences go to TMEM as the products' 128-row operand straight from
// there, and what kernel one left comes through bulk copies as the narrow one:
//   Z^T = S^T W^T,  R^T = S^T Q^T        128 value channels by 64 tokens, sums over keys
//   D = U - Z;  new state's part = (E D)^T K        128 by D keys, sums over tokens; K's tile read the other way round
//   Y^T = D^T G^T;  y = P R + Y          128 by 64 tokens
// One warp fetches, one issues; results of a chunk are written while the next one's first product runs.
//
// Bound by the way round: a product, its differences, the next product and the new state cannot overlap one another. A chunk of 128
// channels takes 6100 clocks (3.1 us): the four products 2700 of the tensor cores, half of them on that way, the rest splits, scales and
// hand-overs. Products begin with the upper half of their 128-row operand while the lower one is made (5% of the time). 18 warps leave 96
// registers a thread, which the loop over chunks needs all: what it needs seldom is in shared memory (8%).
#include "delta_chunk.cuh"

namespace strata {
namespace {

using namespace delta;

constexpr int kWork = 512, kChainThreads = kWork + 64, kFetchWarp = 16, kIssueWarp = 17;

template <int D>
struct __align__(1024) ChainSmem {
    unsigned char w[2][2][D * 128];         // by stage: hi, lo; rows are key channels
    unsigned char qk[2][D / 64][128 * 128];  // hi, lo: panels of 64 channels; rows 0-63 Q, 64-127 K
    unsigned char g[2][64 * 128];  // hi, lo
    struct {
        float u[64 * D];
        DeltaFactors f;
    } row[2];  // by stage, as they follow one another in a slot
    float s_max[4][128];
    float2 d_max[4][128];  // also the sums of chunks that are walked
    unsigned long long w_full[2], w_empty[2], row_full[2], row_empty[2], qk_full, qk_empty, g_full, g_empty;
    unsigned long long s_hi, s_ready, r_free, d_hi, d_ready, y_ready, z_done, d_done, y_done;
    // What a chunk needs seldom: its loop has no registers to spare. Where the state goes and is walked, rows to_next floats apart;
    // the part's first row, its tokens, the value head.
    float *to;
    long long to_next, row0;
    int tokens, head;
    unsigned tmem;
    int abort_flag, picked;
};

__device__ __forceinline__ void lane_sync(int w4) { asm volatile("bar.sync %0, 128;" ::"r"(1 + w4) : "memory"); }  // of the same lanes
__device__ __forceinline__ void work_sync() { asm volatile("bar.sync 5, 512;" ::: "memory"); }
__device__ __forceinline__ bool any_work(bool mine) {  // of all working threads
    int any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.s32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, 5, 512, p;\n\t"
        "selp.s32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"((int)mine)
        : "memory");
    return any != 0;
}

// A chunk token by token, on the state in memory: a channel's four threads add up their parts of the keys, four rows in flight. With few
// registers of its own, so that the loop over chunks keeps them: 420 us a chunk of 128 channels, 49 us of 64 (with the state in registers
// or eight rows in flight 84 and 390 us, but then prompts that walk nothing take 6 to 12% longer).
template <int D, bool ENDS>
__device__ __noinline__ void walk_chunk(const DeltaNet &n, const DeltaRule &A, ChainSmem<D> &M, long long row, int tokens, int h, int part, int v, bool values) {
    constexpr int kPart = D / 4, kRows = 4;
    const long long vw = (long long)n.value_heads * n.dim, key = (long long)(h % n.key_heads) * n.dim + part * kPart, next = M.to_next;
    const bool in = v < n.dim;
    const int keys = in ? min(kPart, n.dim - part * kPart) : 0;
    float *const state = M.to + part * kPart * next + v;
    for (int t = 0; t < tokens; ++t, ++row) {
        const float *kp = A.k + row * A.k_stride + key, *qp = A.q + row * A.q_stride + key;
        const float a = A.decay[row * n.value_heads + h], b = A.beta[row * n.value_heads + h];
        const float value = in && values ? A.v[row * A.v_stride + (long long)h * n.dim + v] : 0.0f;
        float p = 0.0f, y = 0.0f;
#pragma unroll 1
        for (int i = 0; i < keys; i += kRows) {
            float s[kRows], k[kRows];
#pragma unroll
            for (int j = 0; j < kRows; ++j) s[j] = i + j < keys ? state[(i + j) * next] : 0.0f, k[j] = i + j < keys ? kp[i + j] : 0.0f;
#pragma unroll
            for (int j = 0; j < kRows; ++j) p = fmaf(s[j] * a, k[j], p);
        }
        M.d_max[part][v].x = p;
        lane_sync(v >> 5);
        const float d = b * (value - ((M.d_max[0][v].x + M.d_max[1][v].x) + (M.d_max[2][v].x + M.d_max[3][v].x)));
#pragma unroll 1
        for (int i = 0; i < keys; i += kRows) {
            float s[kRows], k[kRows], q[kRows];
#pragma unroll
            for (int j = 0; j < kRows; ++j) {
                s[j] = i + j < keys ? state[(i + j) * next] : 0.0f, k[j] = i + j < keys ? kp[i + j] : 0.0f;
                q[j] = !ENDS && i + j < keys ? qp[i + j] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < kRows; ++j) {
                s[j] = fmaf(k[j], d, s[j] * a);
                y = fmaf(s[j], q[j], y);
                if (i + j < keys) state[(i + j) * next] = s[j];
            }
        }
        M.d_max[part][v].y = y;
        lane_sync(v >> 5);
        if (!ENDS && part == 0 && in) A.y[row * vw + (long long)h * n.dim + v] = (M.d_max[0][v].y + M.d_max[1][v].y) + (M.d_max[2][v].y + M.d_max[3][v].y);
    }
}

// Whether a channel has a token, of a quarter's, that sees nothing of `limit` or more: not its own difference without the state, nor what the
// state, `held` before the chunk, still has of earlier ones; by a whole warp. Seldom called, as the first kernel's value_hidden. A token whose
// query weighs nothing has a result of zeros exactly.
template <int D>
__device__ __forceinline__ bool difference_hidden(const DeltaRule &A, int heads, long long row, int h, const float *u, const DeltaFactors &f, float held, int quarter,
                                                  float limit) {
    const int lane = threadIdx.x & 31;
    float x[2], decay[2];
    bool wanted[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int t = lane + 32 * e;
        const bool in = t < f.counted;
        x[e] = in ? fabsf(u[t * D]) : 0.0f;
        decay[e] = in ? fminf(fabsf(A.decay[(row + t) * heads + h]), 1.0f) : 1.0f;
        wanted[e] = in & (t >> 4 == quarter) & (f.attn[t] > 0x1p-120f);
    }
    return see_less(x, decay, x, wanted, held, limit, lane);
}

// ENDS: nothing but where parts of runs end, from zeros and (their transition) without values from the identity. SORTED: a kernel of its own,
// since a run's number from memory takes registers that the other form has not to spare (2% of its time).
template <int D, bool ENDS, bool SORTED>
__global__ void __launch_bounds__(kChainThreads, 1) k_delta_chain(const __grid_constant__ DeltaNet n, const __grid_constant__ DeltaRule A,
                                                                  const __grid_constant__ MixRuns r, const __grid_constant__ DeltaSlab slab) {
    using Slot = DeltaSlot<D>;
    constexpr bool kEarlyU = D == 64 || ENDS;
    constexpr int kPart = D / 4;  // keys of a thread; and 16 tokens
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    ChainSmem<D> &M = *reinterpret_cast<ChainSmem<D> *>(smem_raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    kv8_enter();
    int block = (int)blockIdx.x;
    bool transition = false;
    int part = 0;
    if (ENDS) transition = block & 1, block >>= 1;
    if (slab.parts > 1) part = block % (slab.parts - ENDS), block /= slab.parts - ENDS;
    const int chain = block, m = block % slab.ratio, head_l = block / slab.ratio % slab.heads;
    int run_l = block / slab.ratio / slab.heads;
    if (SORTED) {  // the run with the run_l-th most tokens
        int *tokens = reinterpret_cast<int *>(M.s_max);
        const int i = slab.run0 + tid;
        if (tid < slab.runs) tokens[tid] = r.sequence[i] < 0 ? 0 : r.lengths[i];
        __syncthreads();
        if (tid < slab.runs) {
            int rank = 0;
            for (int j = 0; j < slab.runs; ++j) rank += tokens[j] > tokens[tid] || (tokens[j] == tokens[tid] && j < tid);
            if (rank == run_l) M.picked = tid;
        }
        __syncthreads();
        run_l = M.picked;
    }
    const int h = slab.head0 + head_l + m * n.key_heads, run = slab.run0 + run_l;
    const MixRun me = mix_run_alone(r, n.sequences, run, n.err);
    const long long first = (long long)run * r.count, vw = (long long)n.value_heads * n.dim;
    int begin = slab.chunk0 * kChunk;
    if (me.sequence < 0) {
        if (ENDS || part > 0) return;
        const long long end = min((long long)r.count, (long long)begin + (long long)slab.chunks * kChunk), rows = end - begin;
        for (long long i = tid; i < rows * n.dim; i += kChainThreads) A.y[(first + begin + i / n.dim) * vw + (long long)h * n.dim + i % n.dim] = 0.0f;
        return;
    }
    if (begin >= me.tokens) return;
    int chunks = min(slab.chunks, (me.tokens - begin + kChunk - 1) / kChunk), chunk = 0;
    // where the state comes from (null: zeros or the identity), and where it goes
    float *const real = n.state + (long long)me.sequence * n.dim * vw + (long long)h * n.dim;
    float *from = real, *to = real;
    long long from_next = vw, to_next = vw;
    if (slab.parts > 1) {
        const int last = (chunks - 1) / slab.part_chunks;
        float *const own = slab.states + (long long)chain * (slab.parts - 1) * (2 * D * D);
        if (ENDS) {
            if (part >= last || (transition && part == 0)) return;
            if (part > 0) from = nullptr;
            to = own + (2 * part + !transition) * (D * D), to_next = D;
        } else {
            const bool whole = slab.whole[chain] != 0;
            if (part > (whole ? 0 : last)) return;
            from = own + (part ? 2 * part - 1 : 0) * (D * D), from_next = D;
            if (!whole && part < last) to = from, to_next = D;
            if (whole) part = -1;
        }
        if (part >= 0) chunk = part * slab.part_chunks, chunks = min(slab.part_chunks, chunks - chunk), begin += chunk * kChunk;
    }

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            bar_init(&M.w_full[i], 1), bar_init(&M.w_empty[i], 1);
            bar_init(&M.row_full[i], 1), bar_init(&M.row_empty[i], kWork / 32 + 1);
        }
        bar_init(&M.qk_full, 1), bar_init(&M.qk_empty, 1), bar_init(&M.g_full, 1), bar_init(&M.g_empty, 1);
        bar_init(&M.s_hi, kWork / 32), bar_init(&M.d_hi, kWork / 32), bar_init(&M.s_ready, kWork / 32), bar_init(&M.r_free, kWork / 32), bar_init(&M.d_ready, kWork / 32), bar_init(&M.y_ready, kWork / 32);
        bar_init(&M.z_done, 1), bar_init(&M.d_done, 1), bar_init(&M.y_done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        M.abort_flag = 0;
        M.to = to, M.to_next = to_next;
        M.row0 = first + begin, M.tokens = me.tokens - begin, M.head = h;
    }
    if (warp == kIssueWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&M.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const unsigned tmem = M.tmem;
    // columns: the state's halves; E D's; Z, and when it has been read D's halves; R, Y, the new state's part
    constexpr unsigned kS = 0, kSLo = D / 2, kE = 128, kZ = 192, kR = 256, kY = 320, kNew = 384;
    const Waits wait{&M.abort_flag, n.err};

    if (warp == kFetchWarp) {
        if (lane == 0) {
            const unsigned char *slot = slab.slots + (((long long)run_l * slab.heads + head_l) * slab.chunks + chunk) * slab.slot_bytes;
            const long long mine = Slot::heads + (long long)m * Slot::head_bytes;
            const auto fetch = [&](void *to, const unsigned char *from, unsigned bytes, unsigned long long *full) {
                bar_expect(full, bytes);
                bulk(to, from, bytes, full);
            };
            for (int c = 0; c < chunks; ++c, slot += slab.slot_bytes) {
                const int st = c & 1;
                const unsigned again = (c >> 1 & 1) ^ 1, again1 = (c & 1) ^ 1;
                wait(&M.w_empty[st], again);
                fetch(M.w[st], slot + mine + Slot::w, Slot::tile, &M.w_full[st]);
                wait(&M.row_empty[st], again);
                fetch(&M.row[st], slot + mine + Slot::uu, sizeof M.row[st], &M.row_full[st]);
                wait(&M.qk_empty, again1);
                fetch(M.qk, slot, 2 * Slot::tile, &M.qk_full);
                if (ENDS) continue;
                wait(&M.g_empty, again1);
                fetch(M.g, slot + mine + Slot::g, Slot::attn, &M.g_full);
            }
        }
        __syncwarp();
    } else if (warp == kIssueWarp) {
        if (elect_one()) {
            constexpr unsigned kLoW = D * 8, kLoQk = D / 64 * 1024;  // from hi to lo, in 16-byte units
            const unsigned long long q = sw128_desc(su32(M.qk)), keys = turned_desc(su32(M.qk) + 8192, 16384), g = sw128_desc(su32(M.g));
            unsigned live = 0;  // chunks on the tensor cores so far
            for (int c = 0; c < chunks; ++c) {
                const int st = c & 1;
                const unsigned ph = c >> 1 & 1, ph1 = c & 1;
                wait(&M.row_full[st], ph);
                const bool walk = M.row[st].f.walk != 0;
                bar_arrive(&M.row_empty[st]);
                if (walk) {  // nothing of it is used
                    wait(&M.w_full[st], ph), wait(&M.qk_full, ph1);
                    bar_arrive(&M.w_empty[st]), bar_arrive(&M.qk_empty);
                    if (ENDS) continue;
                    wait(&M.g_full, ph1);
                    bar_arrive(&M.g_empty);
                    continue;
                }
                const unsigned now = live & 1;
                ++live;
                const unsigned long long w = turned_desc(su32(M.w[st]), 0);
                wait(&M.w_full[st], ph);
                wait(&M.s_hi, now);
                tc_fence_after();
#pragma unroll
                for (int product = 0; product < 3; ++product) {  // hi lo, lo hi, hi hi
                    if (product == 1) {
                        wait(&M.s_ready, now);
                        tc_fence_after();
                    }
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        mma_step_ts(tmem + kZ, tmem + (product == 1 ? kSLo : kS) + k * 8, w + (product == 0) * kLoW + k * 128, turned_idesc(128, 64),
                                    product, k);
                }
                mma_commit(&M.z_done);
                mma_commit(&M.w_empty[st]);
                wait(&M.qk_full, ph1);
                if (!ENDS) {
                    wait(&M.r_free, now);
                    tc_fence_after();
#pragma unroll
                    for (int product = 0; product < 3; ++product)
#pragma unroll
                        for (int k = 0; k < D / 16; ++k)
                            mma_step_ts(tmem + kR, tmem + (product == 0 ? kSLo : kS) + k * 8, q + (product == 1) * kLoQk + k / 4 * 1024 + k % 4 * 2,
                                        idesc_f16(128, 64), product, k);
                }
                wait(&M.d_hi, now);
                tc_fence_after();
#pragma unroll
                for (int product = 0; product < 3; ++product) {  // hi lo, lo hi, hi hi
                    if (product == 1) {
                        wait(&M.d_ready, now);
                        tc_fence_after();
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_step_ts(tmem + kNew, tmem + kE + (product == 1) * 32 + k * 8, keys + (product == 0) * kLoQk + k * 128, turned_idesc(128, D),
                                    product, k);
                }
                mma_commit(&M.d_done);
                mma_commit(&M.qk_empty);
                if (ENDS) continue;
                wait(&M.g_full, ph1);
                wait(&M.y_ready, now);
                tc_fence_after();
#pragma unroll
                for (int product = 0; product < 3; ++product)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_step_ts(tmem + kY, tmem + kZ + (product == 0) * 32 + k * 8, g + (product == 1) * 512 + k * 2, idesc_f16(128, 64), product, k);
                mma_commit(&M.y_done);
                mma_commit(&M.g_empty);
            }
        }
        __syncwarp();
    } else {
        const int w4 = warp & 3, quarter = warp >> 2, v = w4 * 32 + lane;
        const unsigned lanes = tmem + ((unsigned)(w4 * 32) << 16);
        const bool in = v < n.dim;
        const int keys = in ? n.dim - quarter * kPart : 0;  // how many of the thread's there are, or more
        const auto arrive = [&](unsigned long long *b) {
            __syncwarp();
            if (lane == 0) bar_arrive(b);
        };
        unsigned long long S[kPart / 2];
        const auto load_state = [&](const float *p, long long next) {
#pragma unroll
            for (int i = 0; i < kPart / 2; ++i, p += 2 * next) S[i] = pack2(2 * i < keys ? p[0] : 0.0f, 2 * i + 1 < keys ? p[next] : 0.0f);
        };
        const auto store_state = [&] {
            const long long next = M.to_next;
            float *p = M.to + quarter * kPart * next + v;
#pragma unroll
            for (int i = 0; i < kPart / 2; ++i, p += 2 * next) {
                float a, b;
                unpack2(S[i], a, b);
                if (2 * i < keys) p[0] = a;
                if (2 * i + 1 < keys) p[next] = b;
            }
        };
        if (!ENDS || from) {
            load_state(from + quarter * kPart * from_next + v, from_next);
        } else {
#pragma unroll
            for (int i = 0; i < kPart / 2; ++i)
                S[i] = pack2(transition && quarter * kPart + 2 * i == v ? 1.0f : 0.0f, transition && quarter * kPart + 2 * i + 1 == v ? 1.0f : 0.0f);
        }
        unsigned live = 0;
        bool owed = false;           // the chunk before has results in TMEM
        float inv_r = 0, inv_y = 0;  // their scales taken back
        // results of chunk c: its tokens quarter * 16 ..
        const auto write_y = [&](int c) {
            const DeltaFactors &f = M.row[c & 1].f;
            const int t0 = begin + c * kChunk + quarter * 16, left = in ? M.tokens - c * kChunk - quarter * 16 : 0;
            // (uniform row addresses and a lane's offset)
            const char *row = reinterpret_cast<const char *>(A.y + (first + t0) * vw + (long long)h * n.dim);
            const long long next = vw * 4;
            const unsigned at = v * 4;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float R[8], Y[8];
                tmem_read8(lanes + kR + quarter * 16 + half * 8, R);
                tmem_read8(lanes + kY + quarter * 16 + half * 8, Y);
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const ulonglong2 q = *reinterpret_cast<const ulonglong2 *>(f.q + quarter * 16 + half * 8 + i);
                    const ulonglong2 a = *reinterpret_cast<const ulonglong2 *>(f.attn + quarter * 16 + half * 8 + i);
                    const auto sum = [&](int j, unsigned long long q, unsigned long long a) {
                        const unsigned long long r = mul2_rn(pack2(R[j], R[j + 1]), both(inv_r)), y = mul2_rn(pack2(Y[j], Y[j + 1]), both(inv_y));
                        unpack2(fma2(r, q, mul2_rn(y, a)), R[j], R[j + 1]);
                    };
                    sum(i, q.x, a.x), sum(i + 2, q.y, a.y);
                }
                if (left >= 16) {
#pragma unroll
                    for (int i = 0; i < 8; ++i, row += next) *reinterpret_cast<float *>(const_cast<char *>(row) + at) = R[i];
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i, row += next)
                        if (half * 8 + i < left) *reinterpret_cast<float *>(const_cast<char *>(row) + at) = R[i];
                }
            }
        };
        const auto walk = [&](int c) { walk_chunk<D, ENDS>(n, A, M, M.row0 + c * kChunk, min(kChunk, M.tokens - c * kChunk), M.head, quarter, v, !transition); };
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
            const int st = c & 1;
            wait.warp(&M.row_full[st], c >> 1 & 1, lane);
            const DeltaFactors &f = M.row[st].f;
            if (f.walk) {
                if (owed) {
                    wait.warp(&M.y_done, (live - 1) & 1, lane);
                    tc_fence_after();
                    write_y(c - 1);
                    arrive(&M.row_empty[st ^ 1]);
                    owed = false;
                }
                store_state();
                walk(c);
                load_state(M.to + quarter * kPart * M.to_next + v, M.to_next);
                arrive(&M.row_empty[st]);
                continue;
            }
            const unsigned now = live & 1;
            ++live;
            // the state as an operand
            float most = 0.0f;
#pragma unroll
            for (int i = 0; i < kPart / 2; ++i) most = larger2(most, S[i]);
            M.s_max[quarter][v] = most;
            lane_sync(w4);
            const int es = exponent_of(larger(larger(M.s_max[0][v], M.s_max[1][v], M.s_max[2][v]), M.s_max[3][v], 0.0f));
            const float inv_s = unscale_of(es);
            const unsigned long long by_s = both(scale_of(es));
            unsigned hi[kPart / 2], lo[8];
#pragma unroll
            for (int i = 0; i < kPart / 2; ++i) hi[i] = split_hi(S[i], by_s);
            tmem_write(lanes + kS + quarter * (kPart / 2), hi);
            tmem_written();
            arrive(&M.s_hi);
#pragma unroll
            for (int i = 0; i < kPart / 2; i += 8) {
#pragma unroll
                for (int e = 0; e < 8; ++e) lo[e] = split_lo(S[i + e], by_s, hi[i + e]);
                tmem_write(lanes + kSLo + quarter * (kPart / 2) + i, lo);
            }
            tmem_written();
            arrive(&M.s_ready);
            if (owed) {
                wait.warp(&M.y_done, now ^ 1, lane);
                tc_fence_after();
                write_y(c - 1);
                tc_fence_before();
                arrive(&M.row_empty[st ^ 1]);
            }
            if (!ENDS) arrive(&M.r_free);
            inv_r = inv_s;
            // differences, and as the decays to the chunk's end leave them
            const float *u = M.row[st].u + quarter * 16 * D + (v < D ? v : 0);
            const float by = v < D ? -inv_s : 0.0f;
            float d[16];
            unsigned long long x[8];  // U, before Z is there; with 128 channels that takes registers from the rest, so there after it (3% of the time)
            const auto load_u = [&] {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = ENDS && transition ? 0 : pack2(u[2 * i * D], u[2 * i * D + D]);
            };
            if (kEarlyU) load_u();
            wait.warp(&M.z_done, now, lane);
            if (!kEarlyU) load_u();
            tc_fence_after();
            tmem_read(lanes + kZ + quarter * 16, d);
            float most_d = 0.0f, most_e = 0.0f;
            unsigned long long e[8];
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const ulonglong2 z = *reinterpret_cast<const ulonglong2 *>(f.z + quarter * 16 + i), k = *reinterpret_cast<const ulonglong2 *>(f.k + quarter * 16 + i);
                x[i / 2] = fma2(mul2_rn(pack2(d[i], d[i + 1]), both(by)), z.x, x[i / 2]);
                x[i / 2 + 1] = fma2(mul2_rn(pack2(d[i + 2], d[i + 3]), both(by)), z.y, x[i / 2 + 1]);
                most_d = larger2(larger2(most_d, x[i / 2]), x[i / 2 + 1]);
                e[i / 2] = mul2_rn(x[i / 2], k.x), e[i / 2 + 1] = mul2_rn(x[i / 2 + 1], k.y);
                most_e = larger2(larger2(most_e, e[i / 2]), e[i / 2 + 1]);
            }
            M.d_max[quarter][v] = float2{most_d, most_e};
            tc_fence_before();
            lane_sync(w4);  // Z's lanes have been read, too
            tc_fence_after();
            const float2 m0 = M.d_max[0][v], m1 = M.d_max[1][v], m2 = M.d_max[2][v], m3 = M.d_max[3][v];
            const int ee = exponent_of(larger(larger(m0.y, m1.y, m2.y), m3.y, 0.0f)), ed = exponent_of(larger(larger(m0.x, m1.x, m2.x), m3.x, 0.0f));
            const unsigned long long by_e = both(scale_of(ee));
            unsigned h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = split_hi(e[i], by_e);
            tmem_write(lanes + kE + quarter * 8, h);
            tmem_written();
            arrive(&M.d_hi);
#pragma unroll
            for (int i = 0; i < 8; ++i) lo[i] = split_lo(e[i], by_e, h[i]);
            tmem_write(lanes + kE + 32 + quarter * 8, lo);
            tmem_written();
            arrive(&M.d_ready);
            if (!ENDS) {
#pragma unroll
                for (int i = 0; i < 8; ++i) split2(x[i], both(scale_of(ed)), h[i], lo[i]);
                tmem_write(lanes + kZ + quarter * 8, h);
                tmem_write(lanes + kZ + 32 + quarter * 8, lo);
                tmem_written();
                arrive(&M.y_ready);
                inv_y = unscale_of(ed);
                // A difference that the largest of its channel hides: the chunk is walked, from the state as it was. (While the products run.)
                const float limit = hidden_below(ed);
                const int left = f.counted - quarter * 16;
                float least = limit;
                if (left >= 16) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) least = smaller2(least, x[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float p[2];
                        unpack2(x[i / 2], p[0], p[1]);
                        least = i < left ? smaller(least, p[i & 1], least) : least;
                    }
                }
                const bool closer = least < limit && in && left > 0;
                if (any_work(closer)) {  // mostly a difference near zero beside others
                    bool hidden = false;
                    const float most_s = larger(larger(M.s_max[0][v], M.s_max[1][v], M.s_max[2][v]), M.s_max[3][v], 0.0f);
                    for (unsigned ask = __ballot_sync(0xffffffffu, closer); ask && !hidden; ask &= ask - 1) {
                        const int who = __ffs(ask) - 1;
                        hidden = difference_hidden<D>(A, n.value_heads, M.row0 + c * kChunk, M.head, M.row[st].u + w4 * 32 + who, f,
                                                      __shfl_sync(0xffffffffu, most_s, who), quarter, __shfl_sync(0xffffffffu, limit, who));
                    }
                    if (any_work(hidden)) {
                        wait.warp(&M.d_done, now, lane);
                        wait.warp(&M.y_done, now, lane);
                        tc_fence_after();
                        store_state();
                        walk(c);
                        load_state(M.to + quarter * kPart * M.to_next + v, M.to_next);
                        arrive(&M.row_empty[st]);
                        owed = false;
                        continue;
                    }
                }
            }
            // the new state
            const float inv_e = unscale_of(ee), end = f.end;
#pragma unroll
            for (int i = 0; i < kPart / 2; ++i) S[i] = mul2_rn(S[i], both(end));
            wait.warp(&M.d_done, now, lane);
            tc_fence_after();
#pragma unroll
            for (int i = 0; i < kPart; i += 16) {
                tmem_read(lanes + kNew + quarter * kPart + i, d);
#pragma unroll
                for (int e = 0; e < 16; e += 2) S[(i + e) / 2] = fma2(pack2(d[e], d[e + 1]), both(inv_e), S[(i + e) / 2]);
            }
            tc_fence_before();
            if (ENDS) arrive(&M.row_empty[st]);
            owed = !ENDS;
        }
        if (owed) {
            wait.warp(&M.y_done, (live - 1) & 1, lane);
            tc_fence_after();
            write_y(chunks - 1);
        }
        work_sync();
        if (!*(volatile int *)&M.abort_flag) store_state();
    }
    tc_fence_before();
    __syncthreads();
    settle(&M.abort_flag);
    if (warp == kIssueWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <int D, bool ENDS, bool SORTED = false>
cudaError_t launch_chain(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, const DeltaSlab &slab, cudaStream_t s) {
    const cudaError_t e = mix_shared_memory<k_delta_chain<D, ENDS, SORTED>>(sizeof(ChainSmem<D>));
    if (e != cudaSuccess) return e;
    const int blocks = slab.runs * slab.heads * slab.ratio * (ENDS ? 2 * (slab.parts - 1) : slab.parts);
    return kv8_launch(k_delta_chain<D, ENDS, SORTED>, dim3((unsigned)blocks), dim3(kChainThreads), sizeof(ChainSmem<D>), 1, s, n, a, r, slab);
}

}  // namespace

cudaError_t delta_chain(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, const DeltaSlab &slab, cudaStream_t s) {
    if (slab.sorted) return n.dim <= 64 ? launch_chain<64, false, true>(n, a, r, slab, s) : launch_chain<128, false, true>(n, a, r, slab, s);
    return n.dim <= 64 ? launch_chain<64, false>(n, a, r, slab, s) : launch_chain<128, false>(n, a, r, slab, s);
}
cudaError_t delta_ends(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, const DeltaSlab &slab, cudaStream_t s) {
    return n.dim <= 64 ? launch_chain<64, true>(n, a, r, slab, s) : launch_chain<128, true>(n, a, r, slab, s);
}

}  // namespace strata
