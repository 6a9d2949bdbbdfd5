// Device helpers of the token mixers.
#pragma once
#include <atomic>

#include "kv8.cuh"
#include "mixers.h"

namespace strata {

// What run i works on: its sequence (-1: idle) and tokens.
struct MixRun {
    int sequence, tokens;
};
__device__ __forceinline__ MixRun mix_run(const MixRuns &r, int sequences, int i, unsigned *err) {
    MixRun a{r.sequence ? r.sequence[i] : 0, r.lengths ? r.lengths[i] : r.count};
    if (a.sequence < -1 || (r.sequence && a.sequence >= sequences)) {
        raise_error(err, kErrIndex);
        a.sequence = -1;
    }
    if (a.tokens < 0 || a.tokens > r.count) {
        raise_error(err, kErrIndex);
        a.tokens = a.tokens < 0 ? 0 : r.count;
    }
    return a;
}
// The same where a run changes what its sequence holds, by a whole block: a sequence that an earlier run of the call has
// too is reported, and the later run is idle.
__device__ __forceinline__ MixRun mix_run_alone(const MixRuns &r, int sequences, int i, unsigned *err) {
    MixRun a = mix_run(r, sequences, i, err);
    if (r.once) return a;
    bool twice = false;
    if (a.sequence >= 0)
        for (int j = threadIdx.x; j < i; j += blockDim.x) twice |= r.sequence[j] == a.sequence;
    if (__syncthreads_or(twice)) {
        raise_error(err, kErrIndex);
        a.sequence = -1;
    }
    return a;
}

// Lets a kernel have `bytes` of dynamic shared memory: once a device, from whatever thread.
template <auto kKernel>
cudaError_t mix_shared_memory(size_t bytes) {
    constexpr int kDevices = 64;
    static std::atomic<bool> done[kDevices];
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess || (device < kDevices && done[device].load(std::memory_order_relaxed))) return e;
    e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && device < kDevices) done[device].store(true, std::memory_order_relaxed);
    return e;
}

inline bool mix_aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace strata
