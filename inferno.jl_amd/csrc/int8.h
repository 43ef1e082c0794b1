// Argument blocks of the 8-bit projections (quant8.hip, gemm8.hip), filled and
// checked by capi.cpp.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#define Q8_PLAIN 0
#define Q8_RMSNORM 1
#define Q8_SILU_MUL 2

// Rows of K values (2 K for Q8_SILU_MUL: gate, then up), ldx between rows. add:
// n_add slices; with x they are summed into it (rows K apart), without x their
// sum is the input (rows ldx apart).
struct Quant8Args {
    float *x;
    const float *norm_w, *add;
    int8_t *q;
    float *scale;
    int64_t ldx, ldq, add_stride;
    int M, K, n_add;
    float eps;
};

// y[m ldy + n] (+)= x_scale[m] w_scale[n] sum_k x[m ldx + k] w[n ldw + k]
struct Gemm8Args {
    const int8_t *x, *w;
    const float *x_scale, *w_scale;
    float *y;
    int64_t ldx, ldw, ldy;
    int M, N, K, accum;
};
