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

// ---- chunks of 64 tokens ----
//
// With G the running sum of g inside a chunk and S the state before it, the
// chunk's writes X (row i: beta_i (v_i - S_i^T k_i), S_i the state token i
// meets) solve (I + A) X = R, A_ij = beta_i e^(G_i - G_j) k_i.k_j below the
// diagonal, R_i = beta_i (v_i - e^(G_i) S^T k_i); then
//   o_i = scale (e^(G_i) S^T q_i + sum_{j<=i} e^(G_i - G_j) (q_i.k_j) x_j)
//   S'  = e^(G_63) S + sum_j e^(G_63 - G_j) k_j x_j^T
// Every exponent is <= 0 for g <= 0. What does not need the state is prepared
// for all chunks at once (delta_prep_kernel): T = (I + A)^-1 by forward
// substitution (the powers of A that a product form would need can be huge where
// keys repeat), P_ij = e^(G_i - G_j) q_i.k_j, and q, k, T, P as fp16 operands.
// Chunk after chunk (delta_chunk_kernel), a wave carries 16 columns of S in its
// accumulators. The products run on 16x16x32 f16 MFMAs; an fp32 factor is two f16
// limbs (22 bits) times a power of two - a row's for q, k and P, a column's for T
// and for the state, R and X - and a product is hi hi + hi lo + lo hi.

constexpr int CH = 64;
constexpr int TP_BYTES = 6 * 2048;  // T or P: the six 16 x 32 blocks at or below the diagonal, two limbs
constexpr int SCAL = 5 * CH + 16;   // floats: a, b, f, p, d per token, e^(G_63)

__host__ __device__ constexpr int img_bytes(int dk) { return 2 * CH * dk * 2; }  // both limbs of 64 rows

// An image holds a row's values in the order of the operand: 16-byte piece 4 u + q has values 32 u + 4 q .. + 3 and
// 32 u + 16 + 4 q .. + 3, what lane group q takes of 32 values when the other operand is two accumulator tiles side by
// side. Byte of piece c of row r: the pieces of a row are permuted so that neither 16 rows' loads of one piece nor the
// transposing loads of 4 rows' halves of 4 pieces meet in a bank.
template <int DK> __device__ __forceinline__ int img_at(int r, int c) {
    const int x = DK == 64 ? ((r >> 1) & 1) * 4 + ((r >> 2) & 3) : (r & 3) * 4 + ((r >> 2) & 3);
    return r * (DK * 2) + ((c ^ x) << 4);
}
// 16 x 32 block (row tile t, columns 32 u ..) of T or P
__device__ __forceinline__ int tp_block(int t, int u) { return t < 2 ? t : t * 2 - 2 + u; }

// 2^e as a float, e in [-126, 127]
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// 2^x by the one instruction (its argument rounded to fp32 costs |x| 2^-25, as expf's own would)
__device__ __forceinline__ float exp2_of(double x) { return __builtin_amdgcn_exp2f((float)x); }
// exponent of the power of two that brings a largest absolute value to [2^top, 2^(top + 1)); 0 for 0 and non-finite
__device__ __forceinline__ int lift(float most, int top) {
    const int b = (int)((__float_as_uint(most) >> 23) & 255);
    if (b == 0 || b == 255) return 0;
    const int e = top - (b - 127);
    return e < -80 ? -80 : e > 80 ? 80 : e;
}
__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) < __builtin_inff(); }
// the larger of two; not a number if either is not
__device__ __forceinline__ float max_or_nan(float x, float y) { return __builtin_elementwise_maximum(x, y); }
__device__ __forceinline__ float groups_max(float v) {
    const uint32_t x = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    const float m = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const uint32_t y = __float_as_uint(m);
    const auto b = __builtin_amdgcn_permlane16_swap(y, y, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ void split8(const float *x, float up, h8 &hi, h8 &lo) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float v = x[i] * up;
        const _Float16 h = (_Float16)v;
        hi[i] = h;
        lo[i] = (_Float16)(v - (float)h);
    }
}
__device__ __forceinline__ f4 mma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mma3(h8 ah, h8 al, h8 bh, h8 bl, f4 c) { return mma(al, bh, mma(ah, bl, mma(ah, bh, c))); }

struct DeltaWs {
    char *img;    // [seq][key head][chunk]: q image, k image
    char *tp;     // [seq][value head][chunk]: T, P
    float *scal;  // [seq][value head][chunk][SCAL]
    int chunks;
};

__device__ __forceinline__ int tokens_of(const DeltaArgs &a, int s) {
    if (!a.len) return a.T;
    const int w = a.len[s];
    return w < 0 ? 0 : w < a.T ? w : a.T;
}

// One workgroup a chunk of a key head; its value heads two at a time.
template <int DK> __global__ __launch_bounds__(256) void delta_prep_kernel(DeltaArgs a, DeltaWs w) {
    constexpr int IMG = img_bytes(DK), LD = 68, U = DK / 32, PER = DK / 16;  // PER: 16-byte pieces of a row a thread takes
    __shared__ __align__(16) char lds[2 * IMG > 4 * CH * LD * 4 ? 2 * IMG : 4 * CH * LD * 4];
    __shared__ __align__(16) float ck[CH], cq[CH], beta[2][CH], colup[2][CH];
    __shared__ double G[2][CH];
    __shared__ int bad[2][CH];  // rows of A with a value that is not finite
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = blockIdx.x, hk = blockIdx.y, s = blockIdx.z, t0 = c * CH;
    const int rep = a.n_v / a.n_k;

    // running sums of two heads' g log2(e), a wave each, in fp64: a difference of two sums of the chunk keeps its digits however far
    // both have fallen. e^-4096 is 0 in fp32 as is e^g of any g below, -inf among them: such a g counts as -4096, and the
    // sums behind it stay finite and keep their digits.
    auto decays = [&](int h0) __attribute__((always_inline)) {
        if (wave < 2 && h0 + wave < rep) {
            const int hv = hk * rep + h0 + wave;
            const bool at = t0 + lane < a.T;
            const int64_t row = (int64_t)s * a.T + t0 + lane;
            const float gv = at ? a.g[row * a.ldg + hv] : 0.f, bv = at ? a.beta[row * a.ldb + hv] : 0.f;
            const bool in = t0 + lane < tokens_of(a, s);
            double v = !in ? 0.0 : (gv < -4096.f ? -4096.0 : (double)gv) * 1.4426950408889634;
            beta[wave][lane] = in ? bv : 0.f;
            bad[wave][lane] = 0;
            for (int o = 1; o < 64; o <<= 1) {
                const double up = __shfl_up(v, o);
                if (lane >= o) v += up;
            }
            G[wave][lane] = v;
        }
    };
    // rows of q (image 0) and k (image 1) to limbs: 4 threads a row (loaded before it is known how many tokens there are,
    // then taken for zeros past them)
    {
        const int r = tid >> 2, part = tid & 3;
        const bool at = t0 + r < a.T;
        const int64_t row = (int64_t)s * a.T + t0 + r;
        char *out = w.img + (((int64_t)s * a.n_k + hk) * w.chunks + c) * (2 * IMG);
        float x[2][PER / 2][8];
#pragma unroll
        for (int m = 0; m < 2; m++) {
            const float *src = (m ? a.k + row * a.ldk : a.q + row * a.ldq) + (int64_t)hk * DK;
#pragma unroll
            for (int i = 0; i < PER / 2; i++) {
                *(f4 *)(x[m][i]) = at ? *(const f4 *)(src + i * 32 + part * 4) : f4{0, 0, 0, 0};
                *(f4 *)(x[m][i] + 4) = at ? *(const f4 *)(src + i * 32 + 16 + part * 4) : f4{0, 0, 0, 0};
            }
        }
        decays(0);
        const int n = tokens_of(a, s);
        if (t0 >= n) return;
        const bool in = t0 + r < n;
#pragma unroll
        for (int m = 0; m < 2; m++) {
#pragma unroll
            for (int i = 0; i < PER / 2; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) x[m][i][j] = in ? x[m][i][j] : 0.f;
            float sum = 0.f, most = 0.f;
#pragma unroll
            for (int i = 0; i < PER / 2; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) sum = __builtin_fmaf(x[m][i][j], x[m][i][j], sum), most = fmaxf(most, fabsf(x[m][i][j]));
            sum += __shfl_xor(sum, 1);
            most = fmaxf(most, __shfl_xor(most, 1));
            sum += __shfl_xor(sum, 2);
            most = fmaxf(most, __shfl_xor(most, 2));
            const int e = lift(most, 13);
            const float up = pow2(e);
            if (part == 0) (m ? ck : cq)[r] = pow2(-e) * (a.l2norm ? 1.0f / sqrtf(sum + 1e-6f) : 1.0f);
#pragma unroll
            for (int i = 0; i < PER / 2; i++) {
                h8 hi, lo;
                split8(x[m][i], up, hi, lo);
                const int at = m * IMG + img_at<DK>(r, i * 4 + part);
                *(h8 *)(lds + at) = hi;
                *(h8 *)(lds + at + IMG / 2) = lo;
                *(h8 *)(out + at) = hi;
                *(h8 *)(out + at + IMG / 2) = lo;
            }
        }
    }
    __syncthreads();
    // wave t: row tile t of K K^T and Q K^T, columns up to its own tile
    f4 kk[4], qk[4];
    {
        int ra[U];  // (rows 16 apart permute alike)
#pragma unroll
        for (int u = 0; u < U; u++) ra[u] = img_at<DK>(col, 4 * u + g);
        auto rows = [&](int m, int limb, int tile, int u) __attribute__((always_inline)) {
            return *(const h8 *)(lds + m * IMG + limb * (IMG / 2) + ra[u] + tile * 16 * (DK * 2));
        };
#pragma unroll
        for (int j = 0; j < 4; j++) kk[j] = qk[j] = f4{0, 0, 0, 0};
        h8 own[2][2][2], all[2][4][2];  // [set][image][limb], [set][tile][limb]: the next 32 values come in during a product
        auto bring = [&](int u, int set) __attribute__((always_inline)) {
#pragma unroll
            for (int y = 0; y < 2; y++) {
#pragma unroll
                for (int m = 0; m < 2; m++) own[set][m][y] = rows(m, y, wave, u);
#pragma unroll
                for (int j = 0; j < 4; j++) all[set][j][y] = rows(1, y, j, u);
            }
        };
        bring(0, 0);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (u + 1 < U) bring(u + 1, (u + 1) & 1);
            const auto &o = own[u & 1];
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (j <= wave) {
                    const auto &b = all[u & 1][j];
                    kk[j] = mma3(o[1][0], o[1][1], b[0], b[1], kk[j]);
                    qk[j] = mma3(o[0][0], o[0][1], b[0], b[1], qk[j]);
                }
        }
    }
    float *const M = (float *)lds;  // A of two heads, then P of two: [64][LD]
    for (int h0 = 0; h0 < rep; h0 += 2) {
        __syncthreads();  // (the images, or the pair before, are done with)
        if (h0) decays(h0);
        __syncthreads();
#pragma unroll 1
        for (int h = 0; h < 2; h++) {
            if (h0 + h >= rep) break;
            // e^(G_r - G_c): left of the diagonal tile by way of the row tile's first token, a factor a row and one a column
            const int r0 = wave * 16 + 4 * g;
            const double mid = G[h][wave * 16];
            double gr[4], gc[4];
            float kc[4], ec[4];
            const f4 kr = *(const f4 *)(ck + r0), b = *(const f4 *)(beta[h] + r0), qr = *(const f4 *)(cq + r0);
            f4 most = {0, 0, 0, 0}, er;
#pragma unroll
            for (int i = 0; i < 4; i++) gr[i] = G[h][r0 + i], gc[i] = G[h][i * 16 + col], kc[i] = ck[i * 16 + col];
#pragma unroll
            for (int i = 0; i < 4; i++) er[i] = exp2_of(gr[i] - mid);
#pragma unroll
            for (int j = 0; j < 4; j++) ec[j] = j < wave ? exp2_of(mid - gc[j]) * kc[j] : 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (j > wave) continue;
                const int cj = j * 16 + col;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = r0 + i;
                    const float e = j < wave ? er[i] * ec[j] : exp2_of(gr[i] - gc[j]) * kc[j];
                    const float x = cj < r ? b[i] * e * (kk[j][i] * kr[i]) : 0.f;
                    most[i] = max_or_nan(most[i], fabsf(x));
                    M[h * CH * LD + r * LD + cj] = x;
                    M[(2 + h) * CH * LD + r * LD + cj] = cj <= r ? e * (qk[j][i] * (qr[i] * a.scale)) : 0.f;
                }
            }
            // A row of A that is not finite must not reach the rows of T above it (0 times it is not 0): it is taken out here,
            // and the token's own factor then makes its row of R, and with it every later one, not a number.
            if (__any(!is_finite(most[0]) | !is_finite(most[1]) | !is_finite(most[2]) | !is_finite(most[3]))) {
                for (int j = 0; j <= wave; j++)
                    for (int i = 0; i < 4; i++) {
                        const int r = wave * 16 + 4 * g + i;
                        float *x = M + h * CH * LD + r * LD + j * 16 + col;
                        if (!is_finite(*x)) *x = 0.f, bad[h][r] = 1;
                    }
            }
        }
        __syncthreads();
        // T by blocks of 16. On the diagonal, a wave a head: lane 16 b + c has column c of block b, x_i = [i = c] - sum_j
        // A_ij x_j (rows of A read by 16 lanes at once).
        if (wave < 2 && h0 + wave < rep) {
            float *const A = M + wave * CH * LD + (lane >> 4) * (16 * LD + 16);
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float v0 = col == i ? 1.f : 0.f, v1 = 0.f;
#pragma unroll
                for (int j = 0; j < i; j += 4) {
                    const f4 m = *(const f4 *)(A + i * LD + j);
                    v0 = __builtin_fmaf(-m[0], x[j], v0);
                    if (j + 1 < i) v1 = __builtin_fmaf(-m[1], x[j + 1], v1);
                    if (j + 2 < i) v0 = __builtin_fmaf(-m[2], x[j + 2], v0);
                    if (j + 3 < i) v1 = __builtin_fmaf(-m[3], x[j + 3], v1);
                }
                x[i] = v0 + v1;
            }
#pragma unroll
            for (int i = 0; i < 16; i++) A[i * LD + col] = x[i];
        }
        __syncthreads();
        // Below it, block column by block column: T_rc = -T_rr sum_{c<=k<r} A_rk T_kc in fp32 MFMAs, whose accumulators are
        // the B operand of the next product (16 columns, rows 4 g + i by instruction i). Two waves a head: column 0, and
        // columns 1 and 2.
        {
            const int h = wave >> 1, first = wave & 1;
            float *const A = M + h * CH * LD;
            f4 t[3];  // T_10 T_20 T_30 or T_21 T_31 T_32
            if (h0 + h < rep) {
                auto block = [&](int r, int k) __attribute__((always_inline)) { return *(const f4 *)(A + (16 * r + col) * LD + 16 * k + 4 * g); };
                auto times = [&](const f4 &m, const f4 &x, f4 y) __attribute__((always_inline)) {
#pragma unroll
                    for (int i = 0; i < 4; i++) y = __builtin_amdgcn_mfma_f32_16x16x4f32(m[i], x[i], y, 0, 0, 0);
                    return y;
                };
                auto corner = [&](int k) __attribute__((always_inline)) {  // T_kk as accumulators
                    f4 x;
#pragma unroll
                    for (int i = 0; i < 4; i++) x[i] = A[(16 * k + 4 * g + i) * LD + 16 * k + col];
                    return x;
                };
                const f4 zero = {0, 0, 0, 0};
                if (first == 0) {
                    const f4 x0 = corner(0);
                    t[0] = -times(block(1, 1), times(block(1, 0), x0, zero), zero);
                    t[1] = -times(block(2, 2), times(block(2, 1), t[0], times(block(2, 0), x0, zero)), zero);
                    t[2] = -times(block(3, 3), times(block(3, 2), t[1], times(block(3, 1), t[0], times(block(3, 0), x0, zero))), zero);
                } else {
                    const f4 x1 = corner(1), x2 = corner(2);
                    t[0] = -times(block(2, 2), times(block(2, 1), x1, zero), zero);
                    t[1] = -times(block(3, 3), times(block(3, 2), t[0], times(block(3, 1), x1, zero)), zero);
                    t[2] = -times(block(3, 3), times(block(3, 2), x2, zero), zero);
                }
            }
            __syncthreads();  // (A is done with: T takes its place)
            if (h0 + h < rep) {
#pragma unroll
                for (int b = 0; b < 3; b++) {
                    const int r = first == 0 ? b + 1 : b == 0 ? 2 : 3, k = first == 0 ? 0 : b == 2 ? 2 : 1;
#pragma unroll
                    for (int i = 0; i < 4; i++) A[(16 * r + 4 * g + i) * LD + 16 * k + col] = t[b][i];
                }
            }
        }
        __syncthreads();
        // a power of two for each column of T (its largest is at least 1, on the diagonal)
        if (wave < 2 && h0 + wave < rep) {
            const float *const A = M + wave * CH * LD;
            float most = 1.f, t[CH];
#pragma unroll
            for (int i = 0; i < CH; i++) t[i] = A[i * LD + lane];
#pragma unroll
            for (int i = 0; i < CH; i++) most = fmaxf(most, i >= (lane & ~15) ? fabsf(t[i]) : 0.f);
            colup[wave][lane] = pow2(lift(most, 13));
        }
        __syncthreads();
        // operands: wave t takes row tile t of T and P of both heads
#pragma unroll 1
        for (int h = 0; h < 2; h++) {
            if (h0 + h >= rep) break;
            const int64_t unit = ((int64_t)s * a.n_v + hk * rep + h0 + h) * w.chunks + c;
            char *const out = w.tp + unit * (2 * TP_BYTES) + lane * 16;
            const int r = wave * 16 + col;
            const int us = wave < 2 ? 1 : 2;
            f4 t[2][2], p[2][2], cu[2][2];
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const float *src = M + h * CH * LD + r * LD + 32 * u + 16 * y + 4 * g;
                    t[u][y] = *(const f4 *)src;
                    p[u][y] = *(const f4 *)(src + 2 * CH * LD);
                    cu[u][y] = *(const f4 *)(colup[h] + 32 * u + 16 * y + 4 * g);
                }
            float most = 0.f;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        // (past the row's tile nothing was written)
                        const bool there = 2 * u + y <= wave;
                        t[u][y][i] = there ? t[u][y][i] * cu[u][y][i] : 0.f;
                        p[u][y][i] = there ? p[u][y][i] : 0.f;
                        most = fmaxf(most, fabsf(p[u][y][i]));
                    }
            const int e = lift(groups_max(most), 13);
#pragma unroll
            for (int u = 0; u < 2; u++) {
                if (u >= us) continue;
                float x[8];
                h8 hi, lo;
                char *to = out + tp_block(wave, u) * 2048;
                *(f4 *)x = t[u][0], *(f4 *)(x + 4) = t[u][1];
                split8(x, 1.f, hi, lo);
                *(h8 *)to = hi, *(h8 *)(to + 1024) = lo;
                *(f4 *)x = p[u][0], *(f4 *)(x + 4) = p[u][1];
                split8(x, pow2(e), hi, lo);
                *(h8 *)(to + TP_BYTES) = hi, *(h8 *)(to + TP_BYTES + 1024) = lo;
            }
            if (g == 0) {
                float *sc = w.scal + unit * SCAL;
                const float grown = exp2_of(G[h][r]), left = exp2_of(G[h][CH - 1] - G[h][r]);
                const float down = beta[h][r] / colup[h][r];
                sc[r] = bad[h][r] ? __builtin_nanf("") : down;
                sc[CH + r] = down * grown * ck[r];
                sc[2 * CH + r] = a.scale * grown * cq[r];
                sc[3 * CH + r] = pow2(-e);
                sc[4 * CH + r] = left * ck[r];
                if (r == CH - 1) sc[5 * CH] = grown;
            }
        }
    }
}

typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s4 lds_s4;
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(1))) const char g_char;
template <int N> struct Count {
    static constexpr int value = N;
};
// all but the last N of this wave's vector memory operations have completed (they complete in order)
template <int N> __device__ __forceinline__ void wait_vmem() { __builtin_amdgcn_s_waitcnt(0x0F70 | (N & 15) | (N >> 4) << 14); }
// __syncthreads without its wait for every load under way: this wave's LDS stores have completed, and what it loaded to LDS
// is the caller's to wait for
__device__ __forceinline__ void bare_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// nothing is moved across: loads stay ahead of the products that do not need them
#define STAGE() __builtin_amdgcn_sched_barrier(0)

// NS groups of three waves, each group 16 columns of the state. Wave A of a group carries the state: R from K S, X = T R,
// the new state. Wave B forms the outputs from Q S and P X. Wave C brings the chunks' operands to LDS, loaded a chunk
// ahead. The state's limbs and X go from A to B through LDS; two barriers a chunk: B works on Q S while A finds X, and on
// P X while A forms the new state.
template <int DK, int NS> __global__ __launch_bounds__(NS * 192) void delta_chunk_kernel(DeltaArgs a, DeltaWs w) {
    constexpr int IMG = img_bytes(DK), U = DK / 32, R = DK / 16, NB = NS * 64;
    constexpr int NI = IMG / 16 / NB, NTP = TP_BYTES / 16 / NB;  // 16-byte pieces of an image, of T or P, a thread of C brings
    constexpr int NSC = (SCAL / 4 + NB - 1) / NB;
    static_assert(IMG % (16 * NB) == 0 && TP_BYTES % (16 * NB) == 0, "pieces");
    // kbuf 2 x IMG, qbuf IMG, T, P
    constexpr int QB = 2 * IMG, TB = 3 * IMG, PB = TB + TP_BYTES;
    __shared__ __align__(16) char lds[PB + TP_BYTES];
    __shared__ __align__(16) char sbuf[NS][U * 2048], xbuf[NS][4096];
    __shared__ __align__(16) float scal[2][SCAL];
    __shared__ float sdown[NS][64], xdown[NS][64];
    constexpr int LV = 16 * NS + 4;  // floats between rows of v in LDS (a row's pad keeps rows 4 apart in other banks)
    __shared__ __align__(16) float vbuf[CH * LV];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), pair = wave % NS;
    const bool carries = wave < NS, brings = wave >= 2 * NS;
    // consecutive workgroups go to the eight XCDs in turn: a head's column groups, and the heads of a key head, are given
    // to one XCD, whose L2 then fetches the operands once for all of them
    const int groups = (a.dv + 16 * NS - 1) / (16 * NS), heads = a.n_v * a.n_seq, per = (heads + 7) / 8;
    const int unit = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3) / groups, grp = (int)(blockIdx.x >> 3) % groups;
    if (unit >= heads) return;
    const int hv = unit % a.n_v, s = unit / a.n_v, hk = hv / (a.n_v / a.n_k), n = tokens_of(a, s), chunks = (n + CH - 1) / CH;
    const int w0 = (grp * NS + pair) * 16, c0 = w0 + col;
    const bool in = c0 < a.dv;
    const int64_t head = ((int64_t)s * a.n_v + hv) * DK * a.dv + c0;

    const char *img = w.img + ((int64_t)s * a.n_k + hk) * w.chunks * (2 * IMG);
    const char *tp = w.tp + ((int64_t)s * a.n_v + hv) * w.chunks * (2 * TP_BYTES);
    const float *sc = w.scal + ((int64_t)s * a.n_v + hv) * w.chunks * SCAL;

    // Operand of 16 rows, 32 values; of 16 columns as rows, 32 tokens (transposing loads of 4 tokens x 16 values). Rows 16
    // apart permute alike: the lanes' addresses are kept, tiles and limbs are constant offsets.
    int ra[U], ca[U], low_at = lane * 16 + (carries ? TB : PB);
#pragma unroll
    for (int u = 0; u < U; u++) {
        ra[u] = (carries ? 0 : QB) + img_at<DK>(col, 4 * u + g);
        ca[u] = img_at<DK>(4 * g + (col >> 2), 4 * u + (col & 3));
    }
    asm("" : "+v"(low_at));  // (kept as one register: the blocks are constant offsets from it)
    auto rows = [&](int base, int t, int u) __attribute__((always_inline)) {
        return *(const h8 *)(lds + base + ra[u] + t * 16 * (DK * 2));
    };
    auto cols = [&](int base, int r, int u) __attribute__((always_inline)) {
        const char *im = lds + base + ca[r >> 1] + (r & 1) * 8 + 32 * u * (DK * 2);
        const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)im);
        const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(im + 16 * (DK * 2)));
        return __builtin_bit_cast(h8, (s8)__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto per_row = [&](int buf, int which, int t) __attribute__((always_inline)) {
        return *(const f4 *)(&scal[buf][which * CH + t * 16 + 4 * g]);
    };
    // the four tiles of one column to limbs, its largest to [2^13, 2^14); returns what undoes the power of two
    auto largest_of = [&](const f4 (&v)[4]) __attribute__((always_inline)) {
        float most = 0.f;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) most = max_or_nan(most, fabsf(v[t][i]));
        return most;
    };
    auto limbs_of = [&](const f4 (&v)[4], float most, h8 (&l)[2][2]) __attribute__((always_inline)) {
        const int e = lift(groups_max(most), 13);
        const float up = pow2(e);
#pragma unroll
        for (int u = 0; u < 2; u++) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = v[2 * u + (i >> 2)][i & 3];
            split8(x, up, l[u][0], l[u][1]);
        }
        return pow2(-e);
    };
    // A token whose row is not finite must not reach the tokens before it (its 0 in T or P times it is not 0): from the
    // column's first such row on, rows count as 0 in the product, and `spoil` makes them not a number after it. Returns that
    // row, 64 if there is none.
    auto sound = [&](f4 (&v)[4], float &most) __attribute__((always_inline)) {
        int first = CH;
        if (__any(!is_finite(most))) {
#pragma unroll
            for (int t = 3; t >= 0; t--)
#pragma unroll
                for (int i = 3; i >= 0; i--) first = is_finite(v[t][i]) ? first : t * 16 + 4 * g + i;
            first = min(first, __shfl_xor(first, 16));
            first = min(first, __shfl_xor(first, 32));
            most = 0.f;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    v[t][i] = t * 16 + 4 * g + i < first ? v[t][i] : 0.f;
                    most = fmaxf(most, fabsf(v[t][i]));
                }
        }
        return first;
    };
    auto spoil = [&](f4 (&v)[4], int first) __attribute__((always_inline)) {
        if (__any(first < CH)) {
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) v[t][i] = t * 16 + 4 * g + i < first ? v[t][i] : __builtin_nanf("");
        }
    };
    // x[t] = rows of an image (A: K at `base`, B: Q) times the limbs l: the four tiles' products in turn, so that none waits
    // for its own last; the next operands are on their way meanwhile
    auto image_times = [&](int base, const auto &l, f4 (&x)[4]) __attribute__((always_inline)) {
        h8 hi[2][4], lo[2][4];
#pragma unroll
        for (int t = 0; t < 4; t++) hi[0][t] = rows(base, t, 0), lo[0][t] = rows(base + IMG / 2, t, 0);
        STAGE();
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (u + 1 < U) {
#pragma unroll
                for (int t = 0; t < 4; t++) hi[(u + 1) & 1][t] = rows(base, t, u + 1), lo[(u + 1) & 1][t] = rows(base + IMG / 2, t, u + 1);
                STAGE();
            }
#pragma unroll
            for (int t = 0; t < 4; t++) x[t] = mma(hi[u & 1][t], l[u][0], u ? x[t] : f4{0, 0, 0, 0});
#pragma unroll
            for (int t = 0; t < 4; t++) x[t] = mma(hi[u & 1][t], l[u][1], x[t]);
#pragma unroll
            for (int t = 0; t < 4; t++) x[t] = mma(lo[u & 1][t], l[u][0], x[t]);
            STAGE();
        }
    };
    // x[t] += T (A) or P (B) times the limbs l
    auto lower_times = [&](const h8 (&l)[2][2], f4 (&x)[4]) __attribute__((always_inline)) {
        h8 m[6][2];
#pragma unroll
        for (int i = 0; i < 6; i++)
#pragma unroll
            for (int y = 0; y < 2; y++) m[i][y] = *(const h8 *)(lds + low_at + i * 2048 + y * 1024);
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int p = 0; p < 3; p++)
#pragma unroll
                for (int t = 2 * u; t < 4; t++) x[t] = mma(m[tp_block(t, u)][p == 2], l[u][p == 1], x[t]);
    };

    // C: a chunk's operands go straight from memory to LDS, 16 bytes a lane, in two sets: K with P of the chunk before, Q
    // with T. The lines of the next chunk's set are touched meanwhile (a word of each 128 bytes), so that they are in L2
    // when their turn comes.
    const uint32_t ct = (uint32_t)(tid - 2 * NB), c16 = ct * 16;
    const int cw = (wave - 2 * NS) * 1024;
    auto get = [&](int to, const char *from, auto count) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < decltype(count)::value; i++)
            __builtin_amdgcn_global_load_lds((g_char *)(from + i * NB * 16 + c16), (lds_char *)(lds + to + i * NB * 16 + cw), 16, 0, 0);
    };
    typedef Count<NI> Image;
    typedef Count<NTP> Low;
    constexpr int TI = NI / 8, TL = (NTP + 7) / 8;  // touches of an image, of T or P
    uint32_t touched[TI + TL];
    auto touch = [&](const char *image, const char *low) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < TI; i++) touched[i] = *(const uint32_t *)(image + (i * NB + ct) * 128);
#pragma unroll
        for (int i = 0; i < TL; i++) touched[TI + i] = *(const uint32_t *)(low + ((i * NB + ct) * 128 < TP_BYTES ? (i * NB + ct) * 128 : 0));
    };
    auto touch_done = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < TI + TL; i++) asm volatile("" ::"v"(touched[i]));
    };
    u4 fa[NSC];
    auto get_fac = [&](int c) __attribute__((always_inline)) {
        const float *from = sc + (int64_t)(c < chunks ? c : chunks - 1) * SCAL;
#pragma unroll
        for (int i = 0; i < NSC; i++) fa[i] = *(const u4 *)(from + (ct + i * NB < SCAL / 4 ? ct + i * NB : SCAL / 4 - 1) * 4);
    };
    auto put_fac = [&](int c) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NSC; i++)
            if (ct + i * NB < SCAL / 4) *(u4 *)&scal[c & 1][(ct + i * NB) * 4] = fa[i];
    };
    // (past the last chunk the last one again: loads without a branch, never used)
    auto q_of = [&](int c) __attribute__((always_inline)) { return img + (int64_t)(c < chunks ? c : chunks - 1) * (2 * IMG); };
    auto t_of = [&](int c) __attribute__((always_inline)) { return tp + (int64_t)(c < chunks ? c : chunks - 1) * (2 * TP_BYTES); };

    // C: 4 values of 4 rows of v a thread; past the last row that row again (its factor is 0), past the last column the
    // last four (their state is never stored)
    u4 va[4];
    const int vr = (int)ct / (4 * NS), vc = (int)ct % (4 * NS) * 4, vx = grp * NS * 16 + vc;
    const float *const vb = a.v + (int64_t)s * a.T * a.ldv + (int64_t)hv * a.dv + (vx + 4 <= a.dv ? vx : a.dv - 4);
    auto get_v = [&](int c) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int tok = c * CH + i * 16 + vr;
            va[i] = *(const u4 *)(vb + (int64_t)(tok < n ? tok : n - 1) * a.ldv);
        }
    };
    auto put_v = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; i++) *(u4 *)(vbuf + (i * 16 + vr) * LV + vc) = va[i];
    };

    // a lane's values of o: rows 4 g + i of a tile, column c0
    const uint32_t o_at = (uint32_t)(4 * g) * (uint32_t)a.ldo + (uint32_t)c0;
    float *const ob = a.o + (int64_t)s * a.T * a.ldo + (int64_t)hv * a.dv;
    f4 S[R];
    h8 Sl[U][2];
    // The state's limbs: one power of two a column, kept from chunk to chunk while the column's largest stays in
    // [2^3, 2^15) of it (below 2^15 nothing overflows, and 22 bits remain down to 2^-2).
    float Sup = 1.f;
    auto split_tiles = [&](int u) __attribute__((always_inline)) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = S[2 * u + (i >> 2)][i & 3];
        split8(x, Sup, Sl[u][0], Sl[u][1]);
    };
    auto publish = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int x = 0; x < 2; x++) *(h8 *)(sbuf[pair] + (u * 2 + x) * 1024 + lane * 16) = Sl[u][x];
        sdown[pair][lane] = 1.0f / Sup;
    };
    auto largest = [&]() __attribute__((always_inline)) {
        float most = 0.f;
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int i = 0; i < 4; i++) most = fmaxf(most, fabsf(S[r][i]));
        return groups_max(most);
    };
    auto scale_state = [&](float most) __attribute__((always_inline)) {
        Sup = pow2(lift(most, 11));
#pragma unroll
        for (int u = 0; u < U; u++) split_tiles(u);
    };
    // (a loop each, with the same two barriers a turn: no role keeps another's registers)
    if (carries) {
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
            for (int i = 0; i < 4; i++) S[r][i] = in && a.state_in ? a.state_in[head + (int64_t)(r * 16 + 4 * g + i) * a.dv] : 0.f;
        scale_state(largest());
        publish();
        __syncthreads();
        for (int c = 0; c < chunks; c++) {
            const int buf = c & 1, K = buf * IMG;
            f4 x[4];
            h8 l[2][2];
            const float Sdown = 1.0f / Sup;
            f4 v[4], fb[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
#pragma unroll
                for (int i = 0; i < 4; i++) v[t][i] = vbuf[(t * 16 + 4 * g + i) * LV + pair * 16 + col];
                v[t] *= per_row(buf, 0, t), fb[t] = per_row(buf, 1, t) * Sdown;
            }
            image_times(K, Sl, x);
#pragma unroll
            for (int t = 0; t < 4; t++) x[t] = v[t] - fb[t] * x[t];
            float mostR = largest_of(x);
            const int first = sound(x, mostR);
            const float Rdown = limbs_of(x, mostR, l);
#pragma unroll
            for (int t = 0; t < 4; t++) x[t] = f4{0, 0, 0, 0};
            lower_times(l, x);
            spoil(x, first);
#pragma unroll
            for (int t = 0; t < 4; t++) *(f4 *)(xbuf[pair] + t * 1024 + lane * 16) = x[t];  // (in units of R's limbs)
            xdown[pair][lane] = Rdown;
            __syncthreads();
#pragma unroll
            for (int t = 0; t < 4; t++) x[t] *= per_row(buf, 4, t);
            h8 hi[2][2][2], lo[2][2][2];  // [set][tile of the pair][tokens]
            auto bring = [&](int r, int set) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int u = 0; u < 2; u++) hi[set][j][u] = cols(K, r + j, u), lo[set][j][u] = cols(K + IMG / 2, r + j, u);
            };
            bring(0, 0);
            STAGE();
            const float down = limbs_of(x, largest_of(x), l) * Rdown, grown = scal[buf][5 * CH];
            float most = 0.f;
            // a pair of tiles' products while the pair before is added to the state and split
            f4 z[2][2];
            auto add = [&](int r, int set) __attribute__((always_inline)) {
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    S[r + j] = grown * S[r + j] + down * z[set][j];
#pragma unroll
                    for (int i = 0; i < 4; i++) most = fmaxf(most, fabsf(S[r + j][i]));
                }
                split_tiles(r >> 1);
            };
#pragma unroll
            for (int r = 0; r < R; r += 2) {
                const int set = (r >> 1) & 1;
                if (r + 2 < R) bring(r + 2, set ^ 1);
                STAGE();
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int p = 0; p < 3; p++)
#pragma unroll
                        for (int j = 0; j < 2; j++)
                            z[set][j] = mma((p == 2 ? lo : hi)[set][j][u], l[u][p == 1], u || p ? z[set][j] : f4{0, 0, 0, 0});
                if (r) {
                    add(r - 2, set ^ 1);
#pragma unroll
                    for (int i = 0; i < 12; i++) {
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);
                    }
                }
                STAGE();
            }
            add(R - 2, (R / 2 - 1) & 1);
            most = groups_max(most);
            const float big = most * Sup;
            if (__any(!(big < 32768.f && (big >= 8.f || most == 0.f)))) scale_state(most);
            publish();
            __syncthreads();
        }
        if (in && a.state_out) {
#pragma unroll
            for (int r = 0; r < R; r++)
#pragma unroll
                for (int i = 0; i < 4; i++) a.state_out[head + (int64_t)(r * 16 + 4 * g + i) * a.dv] = S[r][i];
        }
    } else if (brings) {
        if (chunks) {
            get(0, q_of(0) + IMG, Image{}), get(QB, q_of(0), Image{}), get(TB, t_of(0), Low{});
            get_fac(0);
            get_v(0);
            put_fac(0);
            put_v();
            get_fac(1);
            wait_stores_done();
        }
        __syncthreads();
        // (LDS is written from registers before the loads to LDS are asked for: the compiler lets no store pass them)
        for (int c = 0; c < chunks; c++) {
            if (c) touch_done();
            put_fac(c + 1);
            STAGE();
            get(PB, t_of(c) + TP_BYTES, Low{}), get(c & 1 ? 0 : IMG, q_of(c + 1) + IMG, Image{});
            STAGE();
            get_v(c + 1);
            touch(q_of(c + 1), t_of(c + 1));
            STAGE();
            wait_vmem<4 + TI + TL>();
            bare_barrier();
            touch_done();
            put_v();
            STAGE();
            get(QB, q_of(c + 1), Image{}), get(TB, t_of(c + 1), Low{});
            STAGE();
            get_fac(c + 2);
            touch(q_of(c + 2) + IMG, t_of(c + 1) + TP_BYTES);
            STAGE();
            wait_vmem<NSC + TI + TL>();
            bare_barrier();
        }
    } else {
        __syncthreads();
        for (int c = 0; c < chunks; c++) {
            const int buf = c & 1;
            f4 x[4], y[4];
            {
                h8 l[U][2];
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int i = 0; i < 2; i++) l[u][i] = *(const h8 *)(sbuf[pair] + (u * 2 + i) * 1024 + lane * 16);
                const float down = sdown[pair][lane];
                image_times(0, l, x);
#pragma unroll
                for (int t = 0; t < 4; t++) x[t] *= per_row(buf, 2, t) * down;
            }
            __syncthreads();
            h8 l[2][2];
#pragma unroll
            for (int t = 0; t < 4; t++) y[t] = *(const f4 *)(xbuf[pair] + t * 1024 + lane * 16);
            float most = largest_of(y);
            const int first = sound(y, most);
            const float down = limbs_of(y, most, l) * xdown[pair][lane];
#pragma unroll
            for (int t = 0; t < 4; t++) y[t] = f4{0, 0, 0, 0};
            lower_times(l, y);
            float *to = ob + (int64_t)c * CH * a.ldo;
#pragma unroll
            for (int t = 0; t < 4; t++) x[t] += y[t] * (per_row(buf, 3, t) * down);
            spoil(x, first);
            if ((c + 1) * CH <= n && w0 + 16 <= a.dv) {
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) (to + (int64_t)(t * 16 + i) * a.ldo)[o_at] = x[t][i];
            } else {
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (in && c * CH + t * 16 + 4 * g + i < n) (to + (int64_t)(t * 16 + i) * a.ldo)[o_at] = x[t][i];
            }
            __syncthreads();
        }
    }
}

// Chunks from 32 tokens on, where no snapshots are asked for.
bool chunked(const DeltaArgs &a, bool snapshots) { return !snapshots && a.T >= 32; }

void ws_of(const DeltaArgs &a, char *ws, DeltaWs &w, size_t &bytes) {
    w.chunks = (a.T + CH - 1) / CH;
    const size_t img = (size_t)a.n_seq * a.n_k * w.chunks * 2 * img_bytes(a.dk);
    const size_t tp = (size_t)a.n_seq * a.n_v * w.chunks * 2 * TP_BYTES;
    w.img = ws, w.tp = ws + img, w.scal = (float *)(ws + img + tp);
    bytes = img + tp + (size_t)a.n_seq * a.n_v * w.chunks * SCAL * sizeof(float);
}

template <int DK> hipError_t launch_chunked(const DeltaArgs &a, void *ws, hipStream_t st) {
    DeltaWs w;
    size_t bytes;
    ws_of(a, (char *)ws, w, bytes);
    delta_prep_kernel<DK><<<dim3((unsigned)w.chunks, (unsigned)a.n_k, (unsigned)a.n_seq), 256, 0, st>>>(a, w);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // one group a workgroup where that leaves no CU with two of them to do; else two, which share the operands in LDS
    const int groups = (a.dv + 15) / 16, heads = a.n_v * a.n_seq;
    const int64_t per = (heads + 7) / 8;
    if ((int64_t)groups * heads <= 256)
        delta_chunk_kernel<DK, 1><<<(unsigned)(8 * per * groups), 192, 0, st>>>(a, w);
    else
        delta_chunk_kernel<DK, 2><<<(unsigned)(8 * per * ((groups + 1) / 2)), 384, 0, st>>>(a, w);
    return hipGetLastError();
}

}  // namespace

size_t delta_ws(const DeltaArgs &a, bool snapshots) {
    if (!chunked(a, snapshots)) return 16;
    DeltaWs w;
    size_t bytes;
    ws_of(a, nullptr, w, bytes);
    return bytes;
}

hipError_t launch_delta(const DeltaArgs &a, void *ws, hipStream_t st) {
    if (chunked(a, a.snap != nullptr)) return a.dk == 64 ? launch_chunked<64>(a, ws, st) : launch_chunked<128>(a, ws, st);
    const dim3 grid((unsigned)((a.dv + 31) / 32), (unsigned)a.n_v, (unsigned)a.n_seq);
    if (a.dk == 64) delta_token_kernel<64><<<grid, 64, 0, st>>>(a);
    else delta_token_kernel<128><<<grid, 64, 0, st>>>(a);
    return hipGetLastError();
}
