// Internal interface of the token mixers over runs of many sequences: the delta-rule layer's inputs, the gated delta rule, and
// the norms of queries and keys with their rotation (delta_rows.cu; delta_rule.cu with delta_step.cu, delta_prepare.cu, delta_chain.cu and
// delta_join.cu; qk_rope.cu; checked by mixers_api.cu and api.cu). The operators' definitions are in include/strata_cuda.h.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <cstddef>

namespace strata {

// `segments` runs of `count` rows; run i is sequence[i]'s (-1: idle) and has lengths[i] tokens (null: count).
struct MixRuns {
    int segments, count;
    const int *sequence, *lengths;
    bool once = false;  // no sequence is outside or there twice: a kernel of the call has made the list so
};
// Device view of one delta-rule layer.
struct DeltaNet {
    int key_heads, value_heads, dim, taps, sequences;
    float *state;         // [sequences][dim][value_heads][dim]
    float *history;       // [sequences][channels][taps - 1]
    const float *weight;  // [channels][taps]
    void *workspace;      // STRATA_DELTA_WORKSPACE_BYTES
    unsigned *err;        // error word, or null
    __host__ __device__ long long channels() const { return (2LL * key_heads + value_heads) * dim; }
};
struct DeltaInputs {
    const float *x;
    long long row_stride;
    float q_scale, epsilon;
    float *q, *k, *v;
};
struct DeltaRule {
    const float *q, *k, *v, *decay, *beta;
    long long q_stride, k_stride, v_stride;
    float *y;
};
struct QkRope {
    int heads, kv_heads, dim, rotary, cells, sequences;
    const float *q_weight, *k_weight, *cos, *sin;
    unsigned *err;
};
struct QkRopeRows {
    const float *q, *k;
    long long q_stride, q_head_stride, k_stride;
    const int *start;
    float epsilon;
    float *yq, *yk;
};

// Argument checks shared by the handle and the pointer forms; 0 or a status with `msg` filled.
int mix_say(char *msg, size_t cap, int code, const char *text);
int delta_check(int key_heads, int value_heads, int dim, int taps, int sequences, char *msg, size_t cap);
int mix_check_runs(int segments, int count, char *msg, size_t cap);
int mix_check_numbers(float scale, float epsilon, char *msg, size_t cap);
int qk_check(int heads, int kv_heads, int dim, int rotary, int cells, int sequences, char *msg, size_t cap);
int mix_check_stride(const char *what, long long stride, long long width, char *msg, size_t cap);

cudaError_t delta_inputs(const DeltaNet &n, const DeltaInputs &a, const MixRuns &r, cudaStream_t s);
cudaError_t delta_rule(const DeltaNet &n, const DeltaRule &a, const MixRuns &r, cudaStream_t s);
cudaError_t qk_rope(const QkRope &w, const QkRopeRows &a, const MixRuns &r, cudaStream_t s);

}  // namespace strata
