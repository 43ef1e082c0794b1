// The product of 8-bit rows with 8-bit weights, a scale for each token and each
// channel:  y[m, n] (+)= x_scale[m] w_scale[n] sum_k x[m, k] w[n, k]
//
// Sums are 32-bit integers and exact (K <= 65536: below 2^30 for codes of +-127,
// 2^30 for -128), so their order has no effect on the result; they are rounded
// to fp32 once and multiplied by the two scales.
#include "common.h"
#include "int8.h"

namespace {

typedef int i4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void global_void;

__device__ const i4 zeros16 = {0, 0, 0, 0};  // what is loaded past K

constexpr int KB = 128;  // bytes of K a tile holds

// Byte of 16-byte chunk c of row r: the chunks of a row are permuted by its number, so that the 16 rows of an operand load
// (one chunk each) do not meet in a bank.
__device__ __forceinline__ int tile_at(int r, int c) { return r * KB + ((c ^ (r & 7)) << 4); }

// One tile of BM tokens x BN channels; WM x WN waves.
template <int BM, int BN, int WM, int WN> __global__ __launch_bounds__(WM *WN * 64) void gemm8_tile(Gemm8Args a, int tiles_m) {
    constexpr int NW = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
    __shared__ char lds[(BM + BN) * KB];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN, g = lane >> 4, col = lane & 15;
    const int m0 = (blockIdx.x % tiles_m) * BM, n0 = (blockIdx.x / tiles_m) * BN;
    i4 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int j = 0; j < TM; j++) acc[i][j] = i4{0, 0, 0, 0};
    const int lr = lane >> 3, lc = (lane & 7) ^ lr;  // this lane's row of 8 and its 16-byte chunk
    for (int k0 = 0; k0 < a.K; k0 += KB) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < (BM + BN) / 8 / NW; i++) {
            const int r = (i * NW + wave) * 8;  // (uniform: rows r .. r + 7 of the tile, tokens first)
            const bool tok = r < BM;
            const int row = (tok ? m0 + r : n0 + r - BM) + lr, last = (tok ? a.M : a.N) - 1;
            const int8_t *p = (tok ? a.x : a.w) + (int64_t)(row < last ? row : last) * (tok ? a.ldx : a.ldw) + k0 + lc * 16;
            const void *src = k0 + lc * 16 < a.K ? (const void *)p : (const void *)&zeros16;
            __builtin_amdgcn_global_load_lds((global_void *)src, (lds_void *)(lds + r * KB), 16, 0, 0);
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; h++) {
            i4 w[TN], x[TM];
#pragma unroll
            for (int i = 0; i < TN; i++) w[i] = *(const i4 *)(lds + tile_at(BM + (wn * TN + i) * 16 + col, 4 * h + g));
#pragma unroll
            for (int j = 0; j < TM; j++) x[j] = *(const i4 *)(lds + tile_at((wm * TM + j) * 16 + col, 4 * h + g));
#pragma unroll
            for (int i = 0; i < TN; i++)
#pragma unroll
                for (int j = 0; j < TM; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], x[j], acc[i][j], 0, 0, 0);
        }
    }
    // a lane's accumulators are 4 channels of one token
    const bool vec = (a.ldy & 3) == 0 && ((uintptr_t)a.y & 15) == 0;
#pragma unroll
    for (int j = 0; j < TM; j++) {
        const int m = m0 + (wm * TM + j) * 16 + col;
        if (m >= a.M) continue;
        const float xs = a.x_scale[m];
#pragma unroll
        for (int i = 0; i < TN; i++) {
            const int n = n0 + (wn * TN + i) * 16 + 4 * g;
            float *y = a.y + (int64_t)m * a.ldy + n;
            if (vec && n + 4 <= a.N) {
                f4 v;
#pragma unroll
                for (int c = 0; c < 4; c++) v[c] = (float)acc[i][j][c] * xs * a.w_scale[n + c];
                if (a.accum) v += *(const f4 *)y;
                *(f4 *)y = v;
            } else {
#pragma unroll
                for (int c = 0; c < 4; c++)
                    if (n + c < a.N) {
                        const float v = (float)acc[i][j][c] * xs * a.w_scale[n + c];
                        y[c] = a.accum ? y[c] + v : v;
                    }
            }
        }
    }
}

}  // namespace

size_t gemm8_ws(const Gemm8Args &) { return 0; }

hipError_t launch_gemm8(const Gemm8Args &a, void *, hipStream_t st) {
    const int tm = (a.M + 63) / 64, tn = (a.N + 127) / 128;
    gemm8_tile<64, 128, 2, 2><<<tm * tn, 256, 0, st>>>(a, tm);
    return hipGetLastError();
}
