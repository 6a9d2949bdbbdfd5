// Argument checks of the token mixers and their entries on caller-owned device memory (include/strata_cuda.h). The
// handle-based entries are in api.cu and share the checks.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>

#include "../../include/strata_cuda.h"
#include "mixers.h"

namespace strata {

int mix_say(char *msg, size_t cap, int code, const char *text) {
    if (msg && cap) snprintf(msg, cap, "%s", text);
    return code;
}
int delta_check(int key_heads, int value_heads, int dim, int taps, int sequences, char *msg, size_t cap) {
    if (key_heads < 1 || key_heads > 4096) return mix_say(msg, cap, STRATA_ERR_RANGE, "key_heads must be an integer in [1, 4096]");
    if (value_heads < 1 || value_heads > 4096 || value_heads % key_heads)
        return mix_say(msg, cap, STRATA_ERR_RANGE, "value_heads must be a multiple of key_heads, at most 4096");
    if (dim < 1 || dim > 256) return mix_say(msg, cap, STRATA_ERR_RANGE, "dim must be an integer in [1, 256]");
    if (taps < 1 || taps > 8) return mix_say(msg, cap, STRATA_ERR_RANGE, "taps must be an integer in [1, 8]");
    if (sequences < 1) return mix_say(msg, cap, STRATA_ERR_RANGE, "sequences must be an integer >= 1");
    return STRATA_OK;
}
int mix_check_runs(int segments, int count, char *msg, size_t cap) {
    if (segments < 1 || segments > 65535) return mix_say(msg, cap, STRATA_ERR_RANGE, "segments must be an integer in [1, 65535]");
    if (count < 1 || (long long)segments * count > (1 << 24))
        return mix_say(msg, cap, STRATA_ERR_RANGE, "count must be at least 1 and segments * count at most 2^24 rows");
    return STRATA_OK;
}
int mix_check_numbers(float scale, float epsilon, char *msg, size_t cap) {
    if (!std::isfinite(scale)) return mix_say(msg, cap, STRATA_ERR_RANGE, "q_scale must be finite");
    if (!(epsilon >= 0) || !std::isfinite(epsilon)) return mix_say(msg, cap, STRATA_ERR_RANGE, "epsilon must be finite and not negative");
    return STRATA_OK;
}
int qk_check(int heads, int kv_heads, int dim, int rotary, int cells, int sequences, char *msg, size_t cap) {
    if (heads < 1 || heads > 4096) return mix_say(msg, cap, STRATA_ERR_RANGE, "heads must be an integer in [1, 4096]");
    if (kv_heads < 1 || kv_heads > 4096) return mix_say(msg, cap, STRATA_ERR_RANGE, "kv_heads must be an integer in [1, 4096]");
    if (dim < 1 || dim > 256) return mix_say(msg, cap, STRATA_ERR_RANGE, "dim must be an integer in [1, 256]");
    if (rotary < 0 || rotary > dim || rotary % 2) return mix_say(msg, cap, STRATA_ERR_RANGE, "rotary must be even and at most dim");
    if (cells < 1) return mix_say(msg, cap, STRATA_ERR_RANGE, "cells must be an integer >= 1");
    if (sequences < 1) return mix_say(msg, cap, STRATA_ERR_RANGE, "sequences must be an integer >= 1");
    return STRATA_OK;
}
int mix_check_stride(const char *what, long long stride, long long width, char *msg, size_t cap) {
    if (stride >= width && stride <= (1LL << 38)) return STRATA_OK;  // at most 2^24 rows: below 2^63
    if (msg && cap) snprintf(msg, cap, "%s is smaller than a row or out of range", what);
    return STRATA_ERR_LAYOUT;
}

}  // namespace strata

using namespace strata;

namespace {

bool aligned(const void *p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

struct Call {  // where a call's refusals go
    char *msg;
    size_t cap;
    int range(const char *text) const { return mix_say(msg, cap, STRATA_ERR_RANGE, text); }
    int layout(const char *text) const { return mix_say(msg, cap, STRATA_ERR_LAYOUT, text); }
    int done(cudaError_t e) const { return e == cudaSuccess ? STRATA_OK : mix_say(msg, cap, STRATA_ERR_CUDA, cudaGetErrorString(e)); }
    // rows of `width` floats, `stride` apart (0: contiguous); strides are unsigned at the entries
    int rows(const char *what, uint64_t *stride, long long width) const {
        if (!*stride) *stride = (uint64_t)width;
        return mix_check_stride(what, *stride > (1ull << 38) ? -1 : (long long)*stride, width, msg, cap);
    }
    template <typename... P>
    int pointers(P... p) const {
        const void *all[] = {p...};
        for (const void *q : all)
            if (!q) return range("null device pointer");
        for (const void *q : all)
            if (!aligned(q, 4)) return layout("rows and tables must start on 4-byte boundaries");
        return STRATA_OK;
    }
};

int view(const Call &c, const strata_delta_net_dev *net, int segments, int count, const int32_t *sequence, const int32_t *lengths,
         DeltaNet *n, MixRuns *r) {
    if (c.msg && c.cap) c.msg[0] = 0;
    if (!net) return c.range("null net");
    if (int e = delta_check(net->key_heads, net->value_heads, net->dim, net->taps, net->sequences, c.msg, c.cap)) return e;
    if (int e = mix_check_runs(segments, count, c.msg, c.cap)) return e;
    if (int e = c.pointers(sequence)) return e;
    if (!aligned(lengths, 4) || !aligned(net->status, 4)) return c.layout("lengths and status must start on 4-byte boundaries");
    *n = DeltaNet{net->key_heads, net->value_heads, net->dim, net->taps, net->sequences, net->state, net->history, net->weight, net->workspace,
                  net->status};
    *r = MixRuns{segments, count, sequence, lengths};
    return STRATA_OK;
}

}  // namespace

extern "C" int strata_delta_inputs_dev(const strata_delta_inputs_call *a) {
    if (!a) return STRATA_ERR_RANGE;
    const Call c{a->msg, (size_t)a->msg_cap};
    DeltaNet n;
    MixRuns r;
    if (int e = view(c, a->net, a->segments, a->count, a->sequence, a->lengths, &n, &r)) return e;
    if (int e = mix_check_numbers(a->q_scale, a->epsilon, c.msg, c.cap)) return e;
    if (int e = c.pointers(a->x, a->q, a->k, a->v, n.weight)) return e;
    if (n.taps > 1)
        if (int e = c.pointers(n.history)) return e;
    uint64_t stride = a->row_stride;
    if (int e = c.rows("row_stride", &stride, n.channels())) return e;
    return c.done(delta_inputs(n, DeltaInputs{a->x, (long long)stride, a->q_scale, a->epsilon, a->q, a->k, a->v}, r,
                               static_cast<cudaStream_t>(a->stream)));
}

extern "C" int strata_delta_rule_dev(const strata_delta_rule_call *a) {
    if (!a) return STRATA_ERR_RANGE;
    const Call c{a->msg, (size_t)a->msg_cap};
    DeltaNet n;
    MixRuns r;
    if (int e = view(c, a->net, a->segments, a->count, a->sequence, a->lengths, &n, &r)) return e;
    if (int e = c.pointers(a->q, a->k, a->v, a->decay, a->beta, a->y, n.state, n.workspace)) return e;
    if (!aligned(n.workspace, 128)) return c.layout("the workspace must start on a 128-byte boundary");
    uint64_t qs = a->q_stride, ks = a->k_stride, vs = a->v_stride;
    const long long kd = (long long)n.key_heads * n.dim, vd = (long long)n.value_heads * n.dim;
    if (int e = c.rows("q_stride", &qs, kd)) return e;
    if (int e = c.rows("k_stride", &ks, kd)) return e;
    if (int e = c.rows("v_stride", &vs, vd)) return e;
    return c.done(delta_rule(n, DeltaRule{a->q, a->k, a->v, a->decay, a->beta, (long long)qs, (long long)ks, (long long)vs, a->y}, r,
                             static_cast<cudaStream_t>(a->stream)));
}

extern "C" int strata_qk_rope_dev(const strata_qk_rope_call *a) {
    if (!a) return STRATA_ERR_RANGE;
    const Call c{a->msg, (size_t)a->msg_cap};
    if (c.msg && c.cap) c.msg[0] = 0;
    const strata_qk_rope_weights_dev *w = a->weights;
    if (!w) return c.range("null weights");
    // without a list of sequences there is none to be outside of
    if (int e = qk_check(w->heads, w->kv_heads, w->dim, w->rotary, w->cells, a->sequence ? w->sequences : 1, c.msg, c.cap)) return e;
    if (int e = mix_check_runs(a->segments, a->count, c.msg, c.cap)) return e;
    if (int e = mix_check_numbers(0, a->epsilon, c.msg, c.cap)) return e;
    if (int e = c.pointers(a->q, a->k, a->yq, a->yk, a->start, w->q_weight, w->k_weight)) return e;
    if (w->rotary)
        if (int e = c.pointers(w->cos, w->sin)) return e;
    if (!aligned(a->sequence, 4) || !aligned(a->lengths, 4) || !aligned(w->status, 4))
        return c.layout("sequence, lengths and status must start on 4-byte boundaries");
    uint64_t hs = a->q_head_stride, qs = a->q_stride, ks = a->k_stride;
    if (int e = c.rows("q_head_stride", &hs, w->dim)) return e;
    if (hs > (1ull << 24)) return c.layout("q_head_stride is out of range");
    if (int e = c.rows("q_stride", &qs, qs ? (long long)(w->heads - 1) * (long long)hs + w->dim : (long long)w->heads * (long long)hs)) return e;
    if (int e = c.rows("k_stride", &ks, (long long)w->kv_heads * w->dim)) return e;
    const QkRope q{w->heads, w->kv_heads, w->dim, w->rotary, w->cells, w->sequences, w->q_weight, w->k_weight, w->cos, w->sin, w->status};
    return c.done(qk_rope(q, QkRopeRows{a->q, a->k, (long long)qs, (long long)hs, (long long)ks, a->start, a->epsilon, a->yq, a->yk},
                          MixRuns{a->segments, a->count, a->sequence, a->lengths}, static_cast<cudaStream_t>(a->stream)));
}
