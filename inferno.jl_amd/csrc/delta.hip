// The gated delta rule (the recurrent layers of the hybrid model,
// src/ModelCPU.jl:476-700).
#include "common.h"
#include "mixer.h"

namespace {

// Token by token: a wave holds 32 columns of one head's state, lane c + 8 g the
// 4 columns 4c .. of rows [g DK / 8, (g + 1) DK / 8). With S the state before
// the token, a = e^g and k, q of unit length where asked for:
//   p = S^T k, r = S^T q (one sum over the row groups for both, and for k.q)
//   u = beta (v - a p); S = a S + k u^T; o = scale (a r + (k.q) u)
template <int DK> __global__ __launch_bounds__(64) void delta_token_kernel(DeltaArgs a) {
    constexpr int R = DK / 8;
    const int lane = threadIdx.x, g = lane >> 3;
    const int hv = blockIdx.y, s = blockIdx.z, hk = hv / (a.n_v / a.n_k);
    const int c0 = blockIdx.x * 32 + (lane & 7) * 4;
    const bool in = c0 < a.dv;
    int n = a.T;
    if (a.len) {
        const int w = a.len[s];
        n = w < 0 ? 0 : w < n ? w : n;
    }
    const int64_t head = ((int64_t)s * a.n_v + hv) * DK * a.dv;
    const int64_t mine = (int64_t)g * R * a.dv + c0;
    f4 S[R];
#pragma unroll
    for (int i = 0; i < R; i++) S[i] = in && a.state_in ? *(const f4 *)(a.state_in + head + mine + (int64_t)i * a.dv) : f4{0, 0, 0, 0};
    for (int t = 0; t < n; t++) {
        const int64_t row = (int64_t)s * a.T + t;
        const f4 *kp = (const f4 *)(a.k + row * a.ldk + (int64_t)hk * DK + g * R);
        const f4 *qp = (const f4 *)(a.q + row * a.ldq + (int64_t)hk * DK + g * R);
        float k[R], q[R];
#pragma unroll
        for (int i = 0; i < R / 4; i++) *(f4 *)(k + 4 * i) = kp[i], *(f4 *)(q + 4 * i) = qp[i];
        const f4 v = in ? *(const f4 *)(a.v + row * a.ldv + (int64_t)hv * a.dv + c0) : f4{0, 0, 0, 0};
        const float decay = expf(a.g[row * a.ldg + hv]), beta = a.beta[row * a.ldb + hv];
        f4 p = {0, 0, 0, 0}, r = {0, 0, 0, 0};
        float kq = 0.f, kk = 0.f, qq = 0.f;
#pragma unroll
        for (int i = 0; i < R; i++) {
            p += S[i] * k[i];
            r += S[i] * q[i];
            kq += k[i] * q[i];
            kk += k[i] * k[i];
            qq += q[i] * q[i];
        }
        for (int o = 8; o < 64; o <<= 1) {
            for (int c = 0; c < 4; c++) p[c] += __shfl_xor(p[c], o), r[c] += __shfl_xor(r[c], o);
            kq += __shfl_xor(kq, o);
            kk += __shfl_xor(kk, o);
            qq += __shfl_xor(qq, o);
        }
        const float nk = a.l2norm ? 1.0f / sqrtf(kk + 1e-6f) : 1.0f, nq = a.l2norm ? 1.0f / sqrtf(qq + 1e-6f) : 1.0f;
        const f4 u = beta * (v - (decay * nk) * p);
#pragma unroll
        for (int i = 0; i < R; i++) S[i] = decay * S[i] + (k[i] * nk) * u;
        if (in && g == 0)
            *(f4 *)(a.o + row * a.ldo + (int64_t)hv * a.dv + c0) = (a.scale * nq) * (decay * r + (kq * nk) * u);
        if (in && a.snap) {
            float *to = a.snap + (row * a.n_v + hv) * DK * a.dv + mine;
#pragma unroll
            for (int i = 0; i < R; i++) *(f4 *)(to + (int64_t)i * a.dv) = S[i];
        }
    }
    if (in && a.state_out) {
#pragma unroll
        for (int i = 0; i < R; i++) *(f4 *)(a.state_out + head + mine + (int64_t)i * a.dv) = S[i];
    }
}

}  // namespace

size_t delta_ws(const DeltaArgs &, bool) { return 16; }

hipError_t launch_delta(const DeltaArgs &a, void *, hipStream_t st) {
    const dim3 grid((unsigned)((a.dv + 31) / 32), (unsigned)a.n_v, (unsigned)a.n_seq);
    if (a.dk == 64) delta_token_kernel<64><<<grid, 64, 0, st>>>(a);
    else delta_token_kernel<128><<<grid, 64, 0, st>>>(a);
    return hipGetLastError();
}
