// The gated delta rule (the recurrent layers of the hybrid model,
// src/ModelCPU.jl:476-700).
#include "common.h"
#include "mixer.h"

namespace {

// What values whose squares leave fp32's range are multiplied by before they are squared, and l2norm's 1e-6 then: values up to
// 2^90 come to 2^58, and what falls below fp32's range, squares of less than 2^-126, is nothing beside 2^-84.
constexpr float UNDER = 0x1p-32f, UNDER_EPS = 1e-6f * 0x1p-64f;

// Token by token: a wave holds 32 columns of one head's state, lane c + 8 g the
// 4 columns 4c .. of rows [g DK / 8, (g + 1) DK / 8). With S the state before
// the token, a = e^g and k, q of unit length where asked for:
//   p = S^T k, r = S^T q (one sum over the row groups for both, and for k.q)
//   u = beta (v - a p); S = a S + k u^T; o = scale (a r + (k.q) u)
// Bound by the states' bytes where there are many (16 sequences of 5 tokens, 32
// heads of 128 x 128, the state after every token kept: 205 MB in 37.3 us, 5.5
// TB/s), by one pass of loads, sums over the row groups and stores for one token
// of one sequence: 4.8 us.
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
        f4 p, r;
        float kq, kk, qq;
        auto sums = [&]() __attribute__((always_inline)) {
            p = r = f4{0, 0, 0, 0};
            kq = kk = qq = 0.f;
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
        };
        sums();
        float nk = 1.0f, nq = 1.0f;
        if (a.l2norm) {
            nk = 1.0f / sqrtf(kk + 1e-6f), nq = 1.0f / sqrtf(qq + 1e-6f);
            if (__any(!(kk + qq <= 0x1p40f))) {
                // so large that their squares or products may leave fp32's range: brought to unit length first, and taken again
                float k2 = 0.f, q2 = 0.f;
#pragma unroll
                for (int i = 0; i < R; i++) {
                    k[i] *= UNDER, q[i] *= UNDER;
                    k2 += k[i] * k[i];
                    q2 += q[i] * q[i];
                }
                for (int o = 8; o < 64; o <<= 1) k2 += __shfl_xor(k2, o), q2 += __shfl_xor(q2, o);
                nk = 1.0f / sqrtf(k2 + UNDER_EPS), nq = 1.0f / sqrtf(q2 + UNDER_EPS);
#pragma unroll
                for (int i = 0; i < R; i++) k[i] *= nk, q[i] *= nq;
                sums();
                nk = nq = 1.0f;
            }
        }
        const f4 u = beta * (v - (decay * nk) * p);
#pragma unroll
        for (int i = 0; i < R; i++) S[i] = decay * S[i] + (k[i] * nk) * u;
        if (in && g == 0)
            *(f4 *)(a.o + row * a.ldo + (int64_t)hv * a.dv + c0) = (a.scale * nq) * (decay * r + (kq * nk) * u);
        if (in && a.snap) {  // (past the caches: 165 MB would only push each other out, 46.4 us through them, 37.5 so; a few MB,
                                // which what commits one of them could find there, were not timed)
            float *to = a.snap + (row * a.n_v + hv) * DK * a.dv + mine;
#pragma unroll
            for (int i = 0; i < R; i++) __builtin_nontemporal_store(S[i], (f4 *)(to + (int64_t)i * a.dv));
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
// diagonal, R_i = beta_i (v_i - e^(G_i) S^T k_i). With T = (I + A)^-1, X = T R:
//   o_i = scale (e^(G_i) S^T q_i + sum_{j<=i} e^(G_i - G_j) (q_i.k_j) x_j)
//       = scale e^(G_i) S^T q_i + sum_j (P T)_ij r_j
//   S'  = e^(G_63) S + sum_i e^(G_63 - G_i) k_i x_i^T = e^(G_63) S + W R,
//   W   = sum_i e^(G_63 - G_i) k_i T_i.
// Every exponent is <= 0 for g <= 0. What does not need the state is prepared
// for all chunks at once (delta_prep_kernel): T by forward substitution (the
// powers of A that a product form would need can be huge where keys repeat),
// then q, k, W and P T as fp16 operands. What is left to do chunk after chunk
// (delta_chunk_kernel) is two products on the state's way, K S and W R, and two
// beside it, Q S and (P T) R; a workgroup carries 16 columns of S in its
// accumulators. The products run on 16x16x32 f16 MFMAs; an fp32 factor is two f16
// limbs (22 bits) times a power of two - a row's for q, k and P T, a column's for
// W, P T, the state and R - and a product is hi hi + hi lo + lo hi.
//
// What bounds it: the preparation by its bytes and, in a chunk, by steps that few
// waves can share (T's diagonal blocks, its columns); the chunks by the way of the
// state through them. 4096 tokens, 16 key and 32 value heads of 128: 63 us (230
// MB, 3.6 TB/s) and 127 us, 2 us a chunk, in which a CU brings 108 KB of operands
// for its 16 columns (14 TB/s over the chip, from L2, which gives 27 to loads
// alone; without these loads the chunks take 88 us) between two barriers; 178 us
// together. 6 sequences of 333 tokens, 8 heads of 64 x 96: 19 and 17 us, the first
// mostly one chunk's latency, the second 2.7 us a chunk. (Before the state's way
// was cut to two products - X formed for the state too, operands by way of LDS -
// the chunks took 190 us.)

constexpr int CH = 64;
constexpr int PT_BYTES = 6 * 2048;   // P T: the six 16 x 32 blocks at or below the diagonal, two limbs
constexpr int SCAL = 6 * CH + 16;    // floats: b, f, w, p, a, d per token (below), e^(G_63)
// R = b v - f (K S);  state += W (w R);  o = a (Q S) + d ((P T) (p R))
enum { ROW_B, ROW_F, ROW_W, ROW_P, ROW_A, ROW_D };

__host__ __device__ constexpr int img_bytes(int dk) { return 2 * CH * dk * 2; }  // both limbs of 64 rows; W has as many

// An operand in memory: 1 KB blocks of 16 rows and 32 values, limb after limb, 16 bytes a lane in the lanes' order: lane
// 16 q + c has of row c the values 32 u + 4 q .. + 3 and 32 u + 16 + 4 q .. + 3, what lane group q takes of 32 values when
// the other operand is two accumulator tiles side by side. Blocks go row tile, u, limb.
// In the preparation's LDS a row's pieces stay together. Byte of piece 4 u + q of row r: the pieces of a row are permuted so
// that neither 16 rows' loads of one piece nor the transposing loads of 4 rows' halves of 4 pieces meet in a bank.
template <int DK> __device__ __forceinline__ int img_at(int r, int c) {
    const int x = DK == 64 ? ((r >> 1) & 1) * 4 + ((r >> 2) & 3) : (r & 3) * 4 + ((r >> 2) & 3);
    return r * (DK * 2) + ((c ^ x) << 4);
}
// 16 x 32 block (row tile t, columns 32 u ..) of P or P T
__device__ __forceinline__ int pt_block(int t, int u) { return t < 2 ? t : t * 2 - 2 + u; }

// 2^e as a float, e in [-126, 127]
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ int exponent(float p) { return (int)(__float_as_uint(p) >> 23) - 127; }  // of a power of two
// 2^x by the one instruction (its argument rounded to fp32 costs |x| 2^-25, as expf's own would)
__device__ __forceinline__ float exp2_of(double x) { return __builtin_amdgcn_exp2f((float)x); }
// exponent of the power of two that brings a largest absolute value to [2^top, 2^(top + 1)); 0 for 0 and non-finite
__device__ __forceinline__ int lift(float most, int top) {
    const int b = (int)((__float_as_uint(most) >> 23) & 255);
    const int e = top - (b - 127);
    return (e < -80 ? -80 : e > 80 ? 80 : e) & -(int)((uint32_t)(b - 1) < 254u);
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
// (Opaque where they stand: the first limbs packed, else each is rounded a second time on its own for the second; the
// differences in fp32, since the mixed fma to half a register takes half as long again as one to fp32 and the packed rounding.)
__device__ __forceinline__ void split8(const float *x, float up, h8 &hi, h8 &lo) {
    float d[8];
#pragma unroll
    for (int i = 0; i < 8; i++) hi[i] = (_Float16)(x[i] * up);
    asm("" : "+v"(hi));
#pragma unroll
    for (int i = 0; i < 8; i++) {
        d[i] = __builtin_fmaf(x[i], up, -(float)hi[i]);
        asm("" : "+v"(d[i]));
    }
#pragma unroll
    for (int i = 0; i < 8; i++) lo[i] = (_Float16)d[i];
}
__device__ __forceinline__ f4 mma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mma3(h8 ah, h8 al, h8 bh, h8 bl, f4 c) { return mma(al, bh, mma(ah, bl, mma(ah, bh, c))); }

__device__ __forceinline__ void split4(const f4 &x, float up, h4 &hi, h4 &lo) {
#pragma unroll
    for (int i = 0; i < 4; i++) hi[i] = (_Float16)(x[i] * up);
    asm("" : "+v"(hi));
#pragma unroll
    for (int i = 0; i < 4; i++) lo[i] = (_Float16)__builtin_fmaf(x[i], up, -(float)hi[i]);
}

typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;

struct DeltaWs {
    char *img;    // [seq][key head][chunk]: q, k
    char *wpt;    // [seq][value head][chunk]: W, P T
    float *scal;  // [seq][value head][chunk][SCAL]
    int chunks;
};

__device__ __forceinline__ int tokens_of(const DeltaArgs &a, int s) {
    if (!a.len) return a.T;
    const int w = a.len[s];
    return w < 0 ? 0 : w < a.T ? w : a.T;
}

// One workgroup a chunk of a key head and `each` of its value heads, one after the other (a wave: row tile, or column tile,
// `tile`).
template <int DK> __global__ __launch_bounds__(256, 2) void delta_prep_kernel(DeltaArgs a, DeltaWs w, int each) {
    constexpr int IMG = img_bytes(DK), LD = 68, U = DK / 32;
    // k; q, whose place A (then T), P and P's limbs take
    constexpr int AAT = IMG, PAT = AAT + CH * LD * 4, LAT = PAT + CH * LD * 4, END = LAT + PT_BYTES;
    static_assert(END >= 2 * IMG, "q");
    __shared__ __align__(16) char lds[END];
    __shared__ __align__(16) float ck[CH], cq[CH], beta[CH], left[CH];
    __shared__ double G[CH];
    __shared__ int bad[CH];  // rows of A with a value that is not finite
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, col = lane & 15;
    const int tile = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rep = a.n_v / a.n_k, parts = (rep + each - 1) / each;
    const int c = blockIdx.x, hk = blockIdx.y / parts, part0 = (blockIdx.y - hk * parts) * each, s = blockIdx.z, t0 = c * CH;

    // running sums of a head's g log2(e), in fp64: a difference of two sums of the chunk keeps its digits however far
    // both have fallen. e^-4096 is 0 in fp32 as is e^g of any g below, -inf among them: such a g counts as -4096, and the
    // sums behind it stay finite and keep their digits.
    float gv = 0.f, bv = 0.f;
    auto get_decays = [&](int hv) __attribute__((always_inline)) {
        if (tile == 0 && t0 + lane < a.T) {
            const int64_t row = (int64_t)s * a.T + t0 + lane;
            gv = a.g[row * a.ldg + hv], bv = a.beta[row * a.ldb + hv];
        }
    };
    auto sum_decays = [&](int n) __attribute__((always_inline)) {
        if (tile == 0) {
            const bool in = t0 + lane < n;
            double v = !in ? 0.0 : (gv < -4096.f ? -4096.0 : (double)gv) * 1.4426950408889634;
            beta[lane] = in ? bv : 0.f;
            bad[lane] = 0;
            for (int o = 1; o < 64; o <<= 1) {
                const double up = __shfl_up(v, o);
                if (lane >= o) v += up;
            }
            G[lane] = v;
        }
    };
    // rows of q and k to limbs: 4 threads a row (loaded before it is known how many tokens there are, then taken for zeros
    // past them)
    int n;
    {
        const int r = tid >> 2, part = tid & 3;
        const bool at = t0 + r < a.T;
        const int64_t row = (int64_t)s * a.T + t0 + r;
        char *out = w.img + (((int64_t)s * a.n_k + hk) * w.chunks + c) * (2 * IMG);
        float x[2][U][8];
#pragma unroll
        for (int m = 0; m < 2; m++) {
            const float *src = (m ? a.k + row * a.ldk : a.q + row * a.ldq) + (int64_t)hk * DK;
#pragma unroll
            for (int i = 0; i < U; i++) {
                *(f4 *)(x[m][i]) = at ? *(const f4 *)(src + i * 32 + part * 4) : f4{0, 0, 0, 0};
                *(f4 *)(x[m][i] + 4) = at ? *(const f4 *)(src + i * 32 + 16 + part * 4) : f4{0, 0, 0, 0};
            }
        }
        get_decays(hk * rep + part0);
        n = tokens_of(a, s);
        if (t0 >= n) return;
        const bool in = t0 + r < n;
#pragma unroll
        for (int m = 0; m < 2; m++) {
#pragma unroll
            for (int i = 0; i < U; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) x[m][i][j] = in ? x[m][i][j] : 0.f;
            float sum = 0.f, most = 0.f;
#pragma unroll
            for (int i = 0; i < U; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) sum = __builtin_fmaf(x[m][i][j], x[m][i][j], sum), most = fmaxf(most, fabsf(x[m][i][j]));
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                sum += __shfl_xor(sum, o);
                most = fmaxf(most, __shfl_xor(most, o));
            }
            const int e = lift(most, 13);
            const float up = pow2(e);
            float norm = a.l2norm ? 1.0f / sqrtf(sum + 1e-6f) : 1.0f;
            if (a.l2norm && !is_finite(sum)) {  // (the row's four threads alike)
                sum = 0.f;
#pragma unroll
                for (int i = 0; i < U; i++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float y = x[m][i][j] * UNDER;
                        sum = __builtin_fmaf(y, y, sum);
                    }
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) sum += __shfl_xor(sum, o);
                norm = UNDER / sqrtf(sum + UNDER_EPS);
            }
            if (part == 0) (m ? ck : cq)[r] = pow2(-e) * norm;
#pragma unroll
            for (int i = 0; i < U; i++) {
                h8 hi, lo;
                split8(x[m][i], up, hi, lo);
                char *in_lds = lds + (m ? 0 : IMG) + img_at<DK>(r, i * 4 + part);
                *(h8 *)in_lds = hi;
                *(h8 *)(in_lds + IMG / 2) = lo;
                char *to = out + m * IMG + ((r >> 4) * U + i) * 2048 + (part * 16 + (r & 15)) * 16;
                if (part0 == 0) *(h8 *)to = hi, *(h8 *)(to + 1024) = lo;
            }
        }
    }
    __syncthreads();
    // the wave's row tile of K K^T and Q K^T, columns up to its own tile
    f4 kk[4], qk[4];
    {
        int ra[U];  // (rows 16 apart permute alike)
#pragma unroll
        for (int u = 0; u < U; u++) ra[u] = img_at<DK>(col, 4 * u + g);
        auto rows = [&](int m, int limb, int t, int u) __attribute__((always_inline)) {
            return *(const h8 *)(lds + (m ? 0 : IMG) + limb * (IMG / 2) + ra[u] + t * 16 * (DK * 2));
        };
#pragma unroll
        for (int j = 0; j < 4; j++) kk[j] = qk[j] = f4{0, 0, 0, 0};
        h8 own[2][2][2], all[2][4][2];  // [set][image][limb], [set][tile][limb]: the next 32 values come in during a product
        auto bring = [&](int u, int set) __attribute__((always_inline)) {
#pragma unroll
            for (int y = 0; y < 2; y++) {
#pragma unroll
                for (int m = 0; m < 2; m++) own[set][m][y] = rows(m, y, tile, u);
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
                if (j <= tile) {
                    const auto &b = all[u & 1][j];
                    kk[j] = mma3(o[1][0], o[1][1], b[0], b[1], kk[j]);
                    qk[j] = mma3(o[0][0], o[0][1], b[0], b[1], qk[j]);
                }
        }
    }
    sum_decays(n);  // (by the wave with the fewest products)
    float *const A = (float *)(lds + AAT), *const P = (float *)(lds + PAT);  // [64][LD]
    char *const pl = lds + LAT + lane * 16;
    for (int h = part0; h < min(part0 + each, rep); h++) {
        const int64_t unit = ((int64_t)s * a.n_v + hk * rep + h) * w.chunks + c;
        float *const sc = w.scal + unit * SCAL;
        __syncthreads();  // (q's limbs, or the head before, are done with)
        if (h > part0) {
            get_decays(hk * rep + h);
            sum_decays(n);
            __syncthreads();
        }
        {
            // e^(G_r - G_c): left of the diagonal tile by way of the row tile's first token, a factor a row and one a column
            const int r0 = tile * 16 + 4 * g;
            const double mid = G[tile * 16];
            double gr[4], gc[4];
            float kc[4], ec[4];
            const f4 kr = *(const f4 *)(ck + r0), b = *(const f4 *)(beta + r0), qr = *(const f4 *)(cq + r0);
            f4 most = {0, 0, 0, 0}, er;
#pragma unroll
            for (int i = 0; i < 4; i++) gr[i] = G[r0 + i], gc[i] = G[i * 16 + col], kc[i] = ck[i * 16 + col];
#pragma unroll
            for (int i = 0; i < 4; i++) er[i] = exp2_of(gr[i] - mid);
#pragma unroll
            for (int j = 0; j < 4; j++) ec[j] = j < tile ? exp2_of(mid - gc[j]) * kc[j] : 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (j > tile) continue;
                const int cj = j * 16 + col;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = r0 + i;
                    const float e = j < tile ? er[i] * ec[j] : exp2_of(gr[i] - gc[j]) * kc[j];
                    const float x = cj < r ? b[i] * e * (kk[j][i] * kr[i]) : 0.f;
                    most[i] = max_or_nan(most[i], fabsf(x));
                    A[r * LD + cj] = x;
                    P[r * LD + cj] = cj <= r ? e * (qk[j][i] * (qr[i] * a.scale)) : 0.f;
                }
            }
            // A row of A that is not finite must not reach the rows of T above it (0 times it is not 0): it is taken out here,
            // and the token's own factor then makes its row of R, and with it every later one, not a number.
            if (__any(!is_finite(most[0]) | !is_finite(most[1]) | !is_finite(most[2]) | !is_finite(most[3]))) {
                for (int j = 0; j <= tile; j++)
                    for (int i = 0; i < 4; i++) {
                        const int r = tile * 16 + 4 * g + i;
                        float *x = A + r * LD + j * 16 + col;
                        if (!is_finite(*x)) *x = 0.f, bad[r] = 1;
                    }
            }
        }
        __syncthreads();
        // T by blocks of 16. On the diagonal, the first wave: lane 16 b + c has column c of block b, x_i = [i = c] -
        // sum_j A_ij x_j (rows of A read by 16 lanes at once).
        if (tile == 0) {
            float *const D = A + (lane >> 4) * (16 * LD + 16);
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float v0 = col == i ? 1.f : 0.f, v1 = 0.f;
#pragma unroll
                for (int j = 0; j < i; j += 4) {
                    const f4 m = *(const f4 *)(D + i * LD + j);
                    v0 = __builtin_fmaf(-m[0], x[j], v0);
                    if (j + 1 < i) v1 = __builtin_fmaf(-m[1], x[j + 1], v1);
                    if (j + 2 < i) v0 = __builtin_fmaf(-m[2], x[j + 2], v0);
                    if (j + 3 < i) v1 = __builtin_fmaf(-m[3], x[j + 3], v1);
                }
                x[i] = v0 + v1;
            }
#pragma unroll
            for (int i = 0; i < 16; i++) D[i * LD + col] = x[i];
        }
        // The others: P's limbs (row tiles 0 and 1, 2, 3), the factors that need no T.
        if (tile) {
            for (int t = tile == 1 ? 0 : tile; t <= tile; t++) {
                const int us = t < 2 ? 1 : 2, r = t * 16 + col;
                f4 p[2][2];
                float most = 0.f;
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int y = 0; y < 2; y++) p[u][y] = *(const f4 *)(P + r * LD + 32 * u + 16 * y + 4 * g);
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int y = 0; y < 2; y++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            p[u][y][i] = 2 * u + y <= t ? p[u][y][i] : 0.f;  // (past the row's tile nothing was written)
                            most = fmaxf(most, fabsf(p[u][y][i]));
                        }
                const int e = lift(groups_max(most), 13);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    if (u >= us) continue;
                    float x[8];
                    h8 hi, lo;
                    *(f4 *)x = p[u][0], *(f4 *)(x + 4) = p[u][1];
                    split8(x, pow2(e), hi, lo);
                    char *to = pl + pt_block(t, u) * 2048;
                    *(h8 *)to = hi, *(h8 *)(to + 1024) = lo;
                }
                if (g == 0) sc[ROW_D * CH + r] = pow2(-e);
            }
        }
        if (tile == 2) {
            const float grown = exp2_of(G[lane]), b = beta[lane];
            left[lane] = exp2_of(G[CH - 1] - G[lane]) * ck[lane];
            sc[ROW_B * CH + lane] = bad[lane] ? __builtin_nanf("") : b;
            sc[ROW_F * CH + lane] = b * grown * ck[lane];
            sc[ROW_A * CH + lane] = a.scale * grown * cq[lane];
            if (lane == CH - 1) sc[6 * CH] = grown;
        }
        __syncthreads();
        // Below it, block column by block column: T_rc = -T_rr sum_{c<=k<r} A_rk T_kc in fp32 MFMAs, whose accumulators are
        // the B operand of the next product (16 columns, rows 4 g + i by instruction i). Two waves: column 0, and columns 1
        // and 2.
        {
            f4 t[3];  // T_10 T_20 T_30 or T_21 T_31 T_32
            if (tile < 2) {
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
                if (tile == 0) {
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
            if (tile < 2) {
#pragma unroll
                for (int b = 0; b < 3; b++) {
                    const int r = tile == 0 ? b + 1 : b == 0 ? 2 : 3, k = tile == 0 ? 0 : b == 2 ? 2 : 1;
#pragma unroll
                    for (int i = 0; i < 4; i++) A[(16 * r + 4 * g + i) * LD + 16 * k + col] = t[b][i];
                }
            }
        }
        __syncthreads();
        // The wave's column tile of T, transposed, as the operand of two products: with the tokens' e^(G_63 - G_l) for W^T (times
        // K), and for (P T)^T (times P^T). A power of two for each column; the products' accumulators, 2^-19 of them (64 terms
        // below 2^28), are 4 of the 8 values of an operand's lane each.
        {
            f4 t[2][2], tw[2][2];
            float most = 0.f, mostw = 0.f;
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int y = 0; y < 2; y++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) t[u][y][i] = A[(32 * u + 16 * y + 4 * g + i) * LD + tile * 16 + col];
                    tw[u][y] = *(const f4 *)(left + 32 * u + 16 * y + 4 * g);
                }
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int y = 0; y < 2; y++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        t[u][y][i] = 2 * u + y >= tile ? t[u][y][i] : 0.f;  // (above the diagonal tile nothing was written)
                        tw[u][y][i] *= t[u][y][i];
                        most = fmaxf(most, fabsf(t[u][y][i]));
                        mostw = fmaxf(mostw, fabsf(tw[u][y][i]));
                    }
            mostw = groups_max(mostw);
            const int e = lift(groups_max(most), 13), ew = lift(mostw, 13);
            constexpr float DOWN = 1.0f / (1 << 19);
            if (g == 0) {
                // (nothing of a token whose column is gone, whatever its R: it must not set the scale of the others)
                sc[ROW_W * CH + tile * 16 + col] = mostw < 0x1p-126f ? 0.f : pow2(19 - ew);
                sc[ROW_P * CH + tile * 16 + col] = pow2(19 - e);
            }
            h8 l[2][2], lw[2][2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                float x[8];
                *(f4 *)x = t[u][0], *(f4 *)(x + 4) = t[u][1];
                split8(x, pow2(e), l[u][0], l[u][1]);
                *(f4 *)x = tw[u][0], *(f4 *)(x + 4) = tw[u][1];
                split8(x, pow2(ew), lw[u][0], lw[u][1]);
            }
            const int u0 = tile >> 1;  // (columns 32 .. have no rows 0 .. 31)
            char *const wo = w.wpt + unit * (IMG + PT_BYTES) + lane * 16 + (tile & 1) * 8;
            auto cols = [&](int limb, int r, int u) __attribute__((always_inline)) {  // 16 columns of k as rows, 32 tokens
                const char *im = lds + limb * (IMG / 2) + img_at<DK>(4 * g + (col >> 2), 4 * (r >> 1) + (col & 3)) + (r & 1) * 8 + 32 * u * (DK * 2);
                const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)im);
                const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(im + 16 * (DK * 2)));
                return __builtin_bit_cast(h8, (s8)__builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
            };
#pragma unroll
            for (int r = 0; r < DK / 16; r++) {
                f4 z = {0, 0, 0, 0};
                if (u0 == 0) z = mma3(lw[0][0], lw[0][1], cols(0, r, 0), cols(1, r, 0), z);
                z = mma3(lw[1][0], lw[1][1], cols(0, r, 1), cols(1, r, 1), z);
                h4 hi, lo;
                split4(z, DOWN, hi, lo);
                char *to = wo + (r * 2 + u0) * 2048;
                *(h4 *)to = hi, *(h4 *)(to + 1024) = lo;
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {  // row tile r of P T
                if (r + (tile & 1) < tile) continue;
                f4 z = {0, 0, 0, 0};
                if (r >= tile) {
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        if (u < u0 || 2 * u > r) continue;
                        const char *from = pl + pt_block(r, u) * 2048;
                        z = mma3(l[u][0], l[u][1], *(const h8 *)from, *(const h8 *)(from + 1024), z);
                    }
                }
                h4 hi, lo;
                split4(z, DOWN, hi, lo);
                char *to = wo + IMG + pt_block(r, u0) * 2048;
                *(h4 *)to = hi, *(h4 *)(to + 1024) = lo;
            }
        }
    }
}

// __syncthreads without its wait for every load under way: only this wave's LDS accesses have completed
__device__ __forceinline__ void bare_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// nothing is moved across: loads stay ahead of the products that do not need them
#define STAGE() __builtin_amdgcn_sched_barrier(0)

// DK / 32 pairs of waves carry 16 columns of a head's state through its chunks. Waves A have the state, 32 of its rows each: R
// from K S for TT of the four tiles of 16 tokens each, then the new state's rows from W R. Waves B, a chunk behind, form the
// outputs of as many tokens each from Q S and (P T) R, and bring v and the factors to LDS. Each has its operands of the next
// chunk on their way in registers while it works on this one's. The state's limbs (a power of two of its own for each wave's
// part) and R go through LDS; two barriers a chunk, the first behind B's last look at the limbs whose place the next take. (One wave issues a vector instruction in 8 clocks, two on a SIMD one in 4
// to 5: the work between the products, more than the products, is why a head is cut this fine.)
template <int DK> __global__ __launch_bounds__(DK * 4, 2) void delta_chunk_kernel(DeltaArgs a, DeltaWs w) {
    constexpr int IMG = img_bytes(DK), U = DK / 32, TT = 4 / U;
    constexpr int LV = 20;  // floats between rows of v in LDS (a row's pad keeps rows 4 apart in other banks)
    __shared__ __align__(16) char sbuf[2][U * 2048], xbuf[2][4096];
    __shared__ __align__(16) float scal[4][SCAL], vbuf[4][CH * LV], obuf[U][16 * LV];
    __shared__ __align__(16) char lbuf[2][4096];
    __shared__ float sdown[2][U][64];
    __shared__ uint32_t off[2][U];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, col = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), part = wave % U;
    const uint32_t l16 = lane * 16;
    // consecutive workgroups go to the eight XCDs in turn: a head's column groups, and the heads of a key head, are given
    // to one XCD, whose L2 then fetches the operands once for all of them
    const int groups = (a.dv + 15) / 16, heads = a.n_v * a.n_seq, per = (heads + 7) / 8;
    const int unit = (int)(blockIdx.x & 7) * per + (int)(blockIdx.x >> 3) / groups, grp = (int)(blockIdx.x >> 3) % groups;
    if (unit >= heads) return;
    const int hv = unit % a.n_v, s = unit / a.n_v, hk = hv / (a.n_v / a.n_k), n = tokens_of(a, s), chunks = (n + CH - 1) / CH;
    const int c0 = grp * 16 + col;
    const bool in = c0 < a.dv;

    const char *img = w.img + ((int64_t)s * a.n_k + hk) * w.chunks * (2 * IMG);
    const char *wpt = w.wpt + ((int64_t)s * a.n_v + hv) * w.chunks * (IMG + PT_BYTES);
    const float *sc = w.scal + ((int64_t)s * a.n_v + hv) * w.chunks * SCAL;
    // (past the last chunk the last one again: loads without a branch, never used)
    auto q_of = [&](int c) __attribute__((always_inline)) { return img + (int64_t)(c < chunks ? c : chunks - 1) * (2 * IMG); };
    auto w_of = [&](int c) __attribute__((always_inline)) { return wpt + (int64_t)(c < chunks ? c : chunks - 1) * (IMG + PT_BYTES); };

    auto per_row = [&](int c, int which, int t) __attribute__((always_inline)) {
        return *(const f4 *)(&scal[c & 3][which * CH + t * 16 + 4 * g]);
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
    // A token whose row is not finite must not reach the tokens before it (its 0 in P T times it is not 0): from the
    // column's first such row on, rows count as 0 in the product, and are made not a number after it. Returns that
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
    // the wave's rows of an image (K or Q), and the image times the state: each part's limbs have a power of two of their own
    h8 M[U][TT][2];
    auto get_rows = [&](const char *from) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int t = 0; t < TT; t++)
#pragma unroll
                for (int y = 0; y < 2; y++) M[u][t][y] = *(const h8 *)(from + part * (TT * U * 2048) + ((t * U + u) * 2 + y) * 1024 + l16);
    };
    auto image_times = [&](int c, const char *next, f4 (&x)[TT]) __attribute__((always_inline)) {
        h8 l[U][2];
        f4 z[U][TT];
        float down[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
#pragma unroll
            for (int i = 0; i < 2; i++) l[u][i] = *(const h8 *)(sbuf[c & 1] + (u * 2 + i) * 1024 + l16);
            down[u] = sdown[c & 1][u][lane];
        }
#pragma unroll
        for (int p = 0; p < 3; p++)
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int t = 0; t < TT; t++) z[u][t] = mma(M[u][t][p == 2], l[u][p == 1], p ? z[u][t] : f4{0, 0, 0, 0});
        STAGE();
        get_rows(next);
        STAGE();
#pragma unroll
        for (int t = 0; t < TT; t++) {
            x[t] = z[0][t] * down[0];
#pragma unroll
            for (int u = 1; u < U; u++) x[t] += z[u][t] * down[u];
        }
    };
    // (a loop each, with the same two barriers a turn: no role keeps another's registers)
    if (wave < U) {
        // The part is held times a power of two, one a column, kept from chunk to chunk while the column's largest value stays
        // in [2^3, 2^15) (below 2^15 its limbs do not overflow, and 22 bits remain down to 2^-2).
        f4 S[2];
        float Sup = 1.f, Sdown = 1.f;
        const int64_t head = (((int64_t)s * a.n_v + hv) * DK + part * 32) * a.dv + c0;
        auto publish = [&](int c) __attribute__((always_inline)) {
            float x[8];
            h8 hi, lo;
            *(f4 *)x = S[0], *(f4 *)(x + 4) = S[1];
            split8(x, 1.f, hi, lo);
            char *to = sbuf[c & 1] + part * 2048 + l16;
            *(h8 *)to = hi, *(h8 *)(to + 1024) = lo;
        };
        auto largest = [&]() __attribute__((always_inline)) {
            float most = 0.f;
#pragma unroll
            for (int r = 0; r < 2; r++)
#pragma unroll
                for (int i = 0; i < 4; i++) most = fmaxf(most, fabsf(S[r][i]));
            return groups_max(most);
        };
        auto scale_by = [&](int e) __attribute__((always_inline)) {  // (|e| up to 160: in two steps)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int x = h ? e - e / 2 : e / 2;
                Sup *= pow2(x), Sdown *= pow2(-x);
                S[0] *= pow2(x), S[1] *= pow2(x);
            }
        };
        // (the power wanted is found whole and then kept to 2^-80 .. 2^80: a column may come from one end to the other)
        auto scale_state = [&](int c, float most) __attribute__((always_inline)) {
            const int b = (int)((__float_as_uint(most) >> 23) & 255);
            if ((uint32_t)(b - 1) < 254u) {
                const int have = exponent(Sup), want = have + 11 - (b - 127);
                scale_by((want < -80 ? -80 : want > 80 ? 80 : want) - have);
            }
            publish(c);
        };
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
            for (int i = 0; i < 4; i++) S[r][i] = in && a.state_in ? a.state_in[head + (int64_t)(r * 16 + 4 * g + i) * a.dv] : 0.f;
        scale_state(0, largest());
        sdown[0][part][lane] = Sdown;
        h8 W[2][2][2];
        auto get_w = [&](const char *from) __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < 2; r++)
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int y = 0; y < 2; y++) W[r][u][y] = *(const h8 *)(from + part * 8192 + ((r * 2 + u) * 2 + y) * 1024 + l16);
        };
        if (chunks) get_rows(q_of(0) + IMG), get_w(w_of(0));
        // of the wave's tokens: b v, f, w
        f4 v[TT], fb[TT], fw[TT];
        auto get_tokens = [&](int c) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < TT; t++) {
#pragma unroll
                for (int i = 0; i < 4; i++) v[t][i] = vbuf[c & 3][((TT * part + t) * 16 + 4 * g + i) * LV + col];
                v[t] *= per_row(c, ROW_B, TT * part + t), fb[t] = per_row(c, ROW_F, TT * part + t), fw[t] = per_row(c, ROW_W, TT * part + t);
            }
        };
        // R's limbs too are times a power of two, one a column, kept while the column's largest stays in [2^3, 2^15): each wave
        // makes those of its own tokens without waiting to know it. Where a column left it all waves take all of R again.
        float Rup = 1.f, Rdown = 1.f;
        bare_barrier();
        if (chunks) get_tokens(0);
        for (int c = 0; c < chunks; c++) {
            {
                f4 x[TT];
                image_times(c, q_of(c + 1) + IMG, x);
                float most = 0.f;
#pragma unroll
                for (int t = 0; t < TT; t++) {
                    x[t] = v[t] - fb[t] * x[t];
                    *(f4 *)(xbuf[c & 1] + (TT * part + t) * 1024 + l16) = x[t];
                    x[t] *= fw[t];
#pragma unroll
                    for (int i = 0; i < 4; i++) most = max_or_nan(most, fabsf(x[t][i]));
                }
                most *= Rup;
                if constexpr (TT == 2) {
                    float y[8];
                    h8 hi, lo;
                    *(f4 *)y = x[0], *(f4 *)(y + 4) = x[1];
                    split8(y, Rup, hi, lo);
                    char *to = lbuf[c & 1] + part * 2048 + l16;
                    *(h8 *)to = hi, *(h8 *)(to + 1024) = lo;
                } else {
                    h4 hi, lo;
                    split4(x[0], Rup, hi, lo);
                    char *to = lbuf[c & 1] + (part >> 1) * 2048 + l16 + (part & 1) * 8;
                    *(h4 *)to = hi, *(h4 *)(to + 1024) = lo;
                }
                const uint64_t over = __ballot(!(most < 32768.f));
                uint64_t there = __ballot(most >= 8.f);
                there |= there >> 32;
                off[c & 1][part] = over ? ~0u : ~(uint32_t)(there | there >> 16) & 0xffff;
            }
            bare_barrier();
            h8 l[2][2];
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int y = 0; y < 2; y++) l[u][y] = *(const h8 *)(lbuf[c & 1] + (u * 2 + y) * 1024 + l16);
            uint32_t any = off[c & 1][0], all = any;
#pragma unroll
            for (int u = 1; u < U; u++) any |= off[c & 1][u], all &= off[c & 1][u];
            if (__builtin_amdgcn_readfirstlane(any >> 16 | all)) {
                f4 x[4];
#pragma unroll
                for (int t = 0; t < 4; t++) x[t] = *(const f4 *)(xbuf[c & 1] + t * 1024 + l16) * per_row(c, ROW_W, t);
                const int e = lift(groups_max(largest_of(x)), 11);
                Rup = pow2(e), Rdown = pow2(-e);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    float y[8];
                    *(f4 *)y = x[2 * u], *(f4 *)(y + 4) = x[2 * u + 1];
                    split8(y, Rup, l[u][0], l[u][1]);
                }
            }
            // A column of a tiny state (a power up to 2^80) may meet a large write (times up to 2^80 again): its power is brought
            // down first, so that down is at most 2^40 and the sum, with y below 2^37, far from fp32's end.
            if (__any(!(Rdown * Sup <= 0x1p40f))) {
                const int over = exponent(Rdown) + exponent(Sup) - 40;
                scale_by(over > 0 ? -over : 0);
            }
            const float down = Rdown * Sup, grown = scal[c & 3][6 * CH];
            f4 y[2];
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int p = 0; p < 3; p++)
#pragma unroll
                    for (int r = 0; r < 2; r++) y[r] = mma(W[r][u][p == 2], l[u][p == 1], u || p ? y[r] : f4{0, 0, 0, 0});
            STAGE();
            get_w(w_of(c + 1));
            STAGE();
#pragma unroll
            for (int r = 0; r < 2; r++) S[r] = grown * S[r] + down * y[r];
            publish(c + 1);
            const float most = largest();
            if (__any(!(most < 32768.f && (most >= 8.f || most == 0.f)))) scale_state(c + 1, most);
            sdown[(c + 1) & 1][part][lane] = Sdown;
            get_tokens(c + 1);
            bare_barrier();
        }
        if (in && a.state_out) {
#pragma unroll
            for (int r = 0; r < 2; r++)
#pragma unroll
                for (int i = 0; i < 4; i++) a.state_out[head + (int64_t)(r * 16 + 4 * g + i) * a.dv] = S[r][i] * Sdown;
        }
        return;
    }

    constexpr int NB = U * 64, VR = NB / 4;  // threads of B; rows of v they bring at once
    const int ct = tid - NB;
    u4 fa, va[CH / VR];
    auto get_fac = [&](int c) __attribute__((always_inline)) {
        const float *from = sc + (int64_t)(c < chunks ? c : chunks - 1) * SCAL;
        fa = *(const u4 *)(from + (ct < SCAL / 4 ? ct : SCAL / 4 - 1) * 4);
    };
    auto put_fac = [&](int c) __attribute__((always_inline)) {
        if (ct < SCAL / 4) *(u4 *)&scal[c & 3][ct * 4] = fa;
    };
    // 4 values of 1 or 2 rows of v a thread; past the last row that row again (its factor is 0), past the last column the last
    // four (their state is never stored)
    const int vr = ct >> 2, vc = (ct & 3) * 4, vx = grp * 16 + vc;
    const float *const vb = a.v + (int64_t)s * a.T * a.ldv + (int64_t)hv * a.dv + (vx + 4 <= a.dv ? vx : a.dv - 4);
    auto get_v = [&](int c) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < CH / VR; i++) {
            const int tok = c * CH + i * VR + vr;
            va[i] = *(const u4 *)(vb + (int64_t)(tok < n ? tok : n - 1) * a.ldv);
        }
    };
    auto put_v = [&](int c) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < CH / VR; i++) *(u4 *)(&vbuf[c & 3][(i * VR + vr) * LV + vc]) = va[i];
    };
    float *const ob = a.o + (int64_t)s * a.T * a.ldo + (int64_t)hv * a.dv + vx;
    // P T's blocks of the wave's row tiles: of 32 .. 63's columns too where the rows are (the same again, unused, elsewhere)
    const bool low = (part + 1) * TT > 2;
    h8 PT[TT][2][2];
    auto get_pt = [&](int c) __attribute__((always_inline)) {
        const char *from = w_of(c) + IMG;
#pragma unroll
        for (int t = 0; t < TT; t++)
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int y = 0; y < 2; y++) PT[t][u][y] = *(const h8 *)(from + pt_block(TT * part + t, low ? u : 0) * 2048 + y * 1024 + l16);
    };
    // The lines of a chunk some steps ahead are touched (a word of each 128 bytes, a head's column groups and their waves sharing
    // them), so that they are in L2 when their loads come (4096 tokens: 131 -> 127 us; 115 with all
    // operands there).
    constexpr int LQ = 2 * IMG / 128, LINES = LQ + (IMG + PT_BYTES) / 128;
    const int line = (lane * groups + grp) * U + part;
    uint32_t touched = 0;
    auto touch = [&](int c) __attribute__((always_inline)) {
        asm volatile("" ::"v"(touched));
        if (line < LINES) touched = *(const uint32_t *)(line < LQ ? q_of(c) + line * 128 : w_of(c) + (line - LQ) * 128);
    };
    if (chunks) {
        u4 f3[3], v3[3][CH / VR];
#pragma unroll
        for (int i = 0; i < 3; i++) {
            get_fac(i), get_v(i);
            f3[i] = fa;
#pragma unroll
            for (int j = 0; j < CH / VR; j++) v3[i][j] = va[j];
        }
#pragma unroll
        for (int i = 0; i < 3; i++) {
            fa = f3[i];
#pragma unroll
            for (int j = 0; j < CH / VR; j++) va[j] = v3[i][j];
            put_fac(i), put_v(i);
        }
        get_fac(3), get_v(3);
        get_rows(q_of(0)), get_pt(0);
    }
    bare_barrier();
    if (chunks) {
        bare_barrier();
        bare_barrier();
    }
    for (int c = 0; c < chunks; c++) {  // (A works on chunk c + 1)
        f4 x[TT], y[4], o[TT];
        image_times(c, q_of(c + 1), x);
#pragma unroll
        for (int t = 0; t < TT; t++) x[t] *= per_row(c, ROW_A, TT * part + t);
        if (c + 1 < chunks) bare_barrier();
        put_fac(c + 3), put_v(c + 3);  // (4 chunks' places: c to c + 3)
        STAGE();
        get_fac(c + 4), get_v(c + 4), touch(c + 6);
        STAGE();
        h8 l[2][2];
#pragma unroll
        for (int t = 0; t < 4; t++) y[t] = *(const f4 *)(xbuf[c & 1] + t * 1024 + l16) * per_row(c, ROW_P, t);
        float most = largest_of(y);
        const int first = sound(y, most);
        const float down = limbs_of(y, most, l);
#pragma unroll
        for (int p = 0; p < 3; p++)
#pragma unroll
            for (int t = 0; t < TT; t++) o[t] = mma(PT[t][0][p == 2], l[0][p == 1], p ? o[t] : f4{0, 0, 0, 0});
        if (low) {
#pragma unroll
            for (int p = 0; p < 3; p++)
#pragma unroll
                for (int t = 0; t < TT; t++) o[t] = mma(PT[t][1][p == 2], l[1][p == 1], o[t]);
        }
        STAGE();
        get_pt(c + 1);
        STAGE();
#pragma unroll
        for (int t = 0; t < TT; t++) x[t] += o[t] * (per_row(c, ROW_D, TT * part + t) * down);
        if (__any(first < CH)) {
#pragma unroll
            for (int t = 0; t < TT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) x[t][i] = (TT * part + t) * 16 + 4 * g + i < first ? x[t][i] : __builtin_nanf("");
        }
        // by way of LDS to 4 values of a row a lane: one store a tile, not four
#pragma unroll
        for (int t = 0; t < TT; t++) {
#pragma unroll
            for (int i = 0; i < 4; i++) obuf[part][(4 * g + i) * LV + col] = x[t][i];
            const int tok = c * CH + (TT * part + t) * 16 + (lane >> 2);
            const f4 y = *(const f4 *)&obuf[part][(lane >> 2) * LV + (lane & 3) * 4];
            if (tok < n && vx < a.dv) *(f4 *)(ob + (int64_t)tok * a.ldo) = y;
        }
        if (c + 1 < chunks) bare_barrier();
    }
}

// Chunks where no snapshots are asked for and there are tokens enough: a chunk costs as much with one token as with 64, the
// recurrence as many times more as there are tokens. Where the two meet, by the number of 16-column groups there are to carry,
// in microseconds (recurrence, chunks) at dk = dv = 128, 32 heads: 1 sequence (256 groups) 16 tokens 22.9, 19.3; 4 (1024)
// 20 tokens 31.6, 34.9 and 24 tokens 37.0, 35; 16 (4096) 40 tokens 78, 87 and 64 tokens 118, 89. dk = dv = 64, 16 heads: 1
// sequence (64) 16 tokens 17.4, 15.6; 16 (1024) 20 tokens 23.7, 27.2 and 28 tokens 31.5, 27.2. The rule is a line between these.
bool chunked(const DeltaArgs &a, bool snapshots) {
    const int64_t groups = (int64_t)a.n_seq * a.n_v * ((a.dv + 15) / 16);
    return !snapshots && a.T >= 14 + (groups < 4096 ? groups / 128 : 32);
}

void ws_of(const DeltaArgs &a, char *ws, DeltaWs &w, size_t &bytes) {
    w.chunks = (a.T + CH - 1) / CH;
    const size_t img = (size_t)a.n_seq * a.n_k * w.chunks * 2 * img_bytes(a.dk);
    const size_t wpt = (size_t)a.n_seq * a.n_v * w.chunks * (img_bytes(a.dk) + PT_BYTES);
    w.img = ws, w.wpt = ws + img, w.scal = (float *)(ws + img + wpt);
    bytes = img + wpt + (size_t)a.n_seq * a.n_v * w.chunks * SCAL * sizeof(float);
}

template <int DK> hipError_t launch_chunked(const DeltaArgs &a, void *ws, hipStream_t st) {
    DeltaWs w;
    size_t bytes;
    ws_of(a, (char *)ws, w, bytes);
    // A workgroup a value head where that still leaves no CU more than the two that fit at once to do, else one for all value
    // heads of a key head, which then prepares q and k once: in all, 37.2 us against 43.2 at 512 tokens of 16 key and 32 value
    // heads (128 chunks), 84.6 against 93.2 at 2048 (512 chunks, both ways alike); 139 against 128 for 16 sequences of 128
    // tokens (512 chunks, twice as many workgroups as fit).
    const int rep = a.n_v / a.n_k;
    const int each = (int64_t)w.chunks * a.n_k * a.n_seq < 512 ? 1 : rep;
    delta_prep_kernel<DK><<<dim3((unsigned)w.chunks, (unsigned)(a.n_k * ((rep + each - 1) / each)), (unsigned)a.n_seq), 256, 0, st>>>(a, w, each);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t groups = (a.dv + 15) / 16, heads = (int64_t)a.n_v * a.n_seq;
    delta_chunk_kernel<DK><<<(unsigned)(8 * ((heads + 7) / 8) * groups), DK * 4, 0, st>>>(a, w);
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
