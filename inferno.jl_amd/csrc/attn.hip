// Attention of a batch's new tokens over a shared prefix, their own cached
// entries and each other (src/ModelCPU.jl:730-856).
#include "common.h"
#include "mixer.h"

namespace {

template <int TYPE> __device__ __forceinline__ float kv_at(const void *p, int64_t i) {
    if constexpr (TYPE == KV_F16) return (float)((const _Float16 *)p)[i];
    else return (float)((const __bf16 *)p)[i];
}

// One wave a query row and head, entry by entry with the running maximum m and
// sum l of its softmax; lane i holds values i, i + 64, .. of the head.
template <int TYPE, int D> __global__ __launch_bounds__(64) void attn_row_kernel(AttnArgs a) {
    constexpr int E = D / 64;
    const int64_t row = blockIdx.x;
    const int h = blockIdx.y, lane = threadIdx.x, s = (int)(row / a.M), r = (int)(row - (int64_t)s * a.M);
    const int n = a.len[s];
    if (n < 0) return;
    float *out = a.out + row * a.ldo + (int64_t)h * D;
    if ((int64_t)n + a.M > a.capacity) {
        for (int e = 0; e < E; e++) out[lane + 64 * e] = __builtin_nanf("");
        return;
    }
    const int hk = h / (a.n_q / a.n_kv);
    float q[E], acc[E], m = -__builtin_inff(), l = 0.f;
    for (int e = 0; e < E; e++) {
        q[e] = a.q[row * a.ldq + (int64_t)h * D + lane + 64 * e] * a.scale;
        acc[e] = 0.f;
    }
    auto take = [&](const void *k, const void *v, int64_t at) {
        float z = 0.f;
        for (int e = 0; e < E; e++) z = __builtin_fmaf(q[e], kv_at<TYPE>(k, at + lane + 64 * e), z);
        z = wave_sum(z);
        const float top = fmaxf(m, z);
        const float base = top == -__builtin_inff() ? 0.f : top;
        const float keep = expf(m - base), p = expf(z - base);
        l = l * keep + p;
        for (int e = 0; e < E; e++) acc[e] = acc[e] * keep + p * kv_at<TYPE>(v, at + lane + 64 * e);
        m = top;
    };
    for (int64_t j = 0; j < a.P; j++) take(a.pk, a.pv, j * a.p_tok_stride + hk * a.p_head_stride);
    const int64_t own = s * a.seq_stride + hk * a.head_stride;
    for (int j = 0; j < n; j++) take(a.k, a.v, own + j * a.tok_stride);
    for (int j = 0; j < a.M; j++)
        if (a.mask ? (a.mask[row] >> j) & 1 : j <= r) take(a.k, a.v, own + ((int64_t)n + j) * a.tok_stride);
    for (int e = 0; e < E; e++) out[lane + 64 * e] = l == 0.f ? 0.f : acc[e] / l;
}

}  // namespace

size_t attn_ws(const AttnArgs &) { return 16; }

hipError_t launch_attn(const AttnArgs &a, void *, hipStream_t st) {
    const dim3 grid((unsigned)(a.n_seq * a.M), (unsigned)a.n_q);
#define ROWS(T, D) attn_row_kernel<T, D><<<grid, 64, 0, st>>>(a)
    if (a.type == KV_F16) {
        if (a.head_dim == 64) ROWS(KV_F16, 64);
        else if (a.head_dim == 128) ROWS(KV_F16, 128);
        else ROWS(KV_F16, 256);
    } else {
        if (a.head_dim == 64) ROWS(KV_BF16, 64);
        else if (a.head_dim == 128) ROWS(KV_BF16, 128);
        else ROWS(KV_BF16, 256);
    }
#undef ROWS
    return hipGetLastError();
}
