// Argument blocks of the token mixers (rope.hip, attn.hip, delta.hip), filled
// and checked by capi.cpp.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#define KV_F16 1
#define KV_BF16 30

struct RopeTable {
    double turns[128];
};

// Rows of n_q + n_k + n_v heads: the first n_q + n_k turn, the n_q go to y, the
// others to the cache entry len[s] + m of row s M + m (len NULL: q heads only).
struct RopeArgs {
    const float *x;
    float *y;
    int64_t ldx, ldy;
    const int32_t *pos, *len;
    const float *freq_factors;
    void *k, *v;
    int64_t capacity, seq_stride, tok_stride, head_stride;
    int n_q, n_k, n_v, head_dim, rot_dim, interleaved, pos0, M, type;
    float mscale;
};

struct AttnArgs {
    const float *q;
    float *out;
    int64_t ldq, ldo;
    const void *k, *v;    // the sequences' own entries
    const void *pk, *pv;  // the shared prefix (P entries; 0: none)
    int64_t capacity, seq_stride, tok_stride, head_stride;
    int64_t P, p_tok_stride, p_head_stride;
    const int32_t *len;
    const uint64_t *mask;  // NULL: causal
    int n_seq, n_q, n_kv, head_dim, M, type;
    float scale;
};

struct DeltaArgs {
    const float *q, *k, *v, *g, *beta;
    int64_t ldq, ldk, ldv, ldg, ldb;
    float *o;
    int64_t ldo;
    const float *state_in;
    float *state_out, *snap;
    const int32_t *len;
    int n_seq, T, n_k, n_v, dk, dv;
    float scale;
    int l2norm;
};
