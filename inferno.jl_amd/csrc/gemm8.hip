// The product of 8-bit rows with 8-bit weights, a scale for each token and each
// channel:  y[m, n] (+)= x_scale[m] w_scale[n] sum_k x[m, k] w[n, k]
//
// Sums are 32-bit integers and exact (K <= 65536: below 2^30 for codes of +-127,
// 2^30 for -128), so their order has no effect on the result; they are rounded
// to fp32 once and multiplied by the two scales.
//
// What bounds it. Few tokens: reading the weights (gemm8_few: 1 x 24576 x 4096
// in 16.8 us, 6.0 TB/s; 5 x 4096 x 12288 added to y 9.3 us, 5.4). Many: products,
// at the rate of the library's (gemm8_tile: 4096 x 24576 x 4096 in 376 to 382 us,
// the library 382, 2.2 PFLOP/s at 1.9 GHz). Their instructions hold a SIMD's
// matrix core for 393216 cycles, 207 us at that clock and 164 at 2.4 GHz: it is
// busy 56 % of the time, and what fills the rest was not found. Between, what a CU
// takes in, 100 to 125 GB/s, and the rounds of workgroups: 515 x 4096 x 4096 19 us,
// 64 x 12288 x 2048 7.4. Rows that do not begin at multiples of 128 bytes cost the
// tiles 5 to 12 % (2 lines for 1).
#include <type_traits>

#include "common.h"
#include "gemm8_plan.h"
#include "int8.h"

#pragma clang fp contract(off)  // (the addition to y after the product's own rounding, in every kernel)

namespace {

constexpr int KB = GEMM8_KB;

typedef int i4 __attribute__((ext_vector_type(4)));
typedef int i16 __attribute__((ext_vector_type(16)));
typedef f4 f4u __attribute__((aligned(4)));  // (rows of y begin at any value)
typedef __attribute__((address_space(3))) void lds_void;

// Which of the eight 16-byte places of a row its chunk c takes: c ^ turn_of(row). The 16 lanes that LDS serves at once in a
// load of 32 rows' chunk c (lanes 0-7 with 16-23, 8-15 with 24-31: rows) then meet in no bank (no conflicts counted).
__device__ __forceinline__ int turn_of(int row) { return (row & 6) | (row >> 4 & 1); }

// All but the last N loads of this wave are there, its LDS operations are done, and every wave is here.
template <int N> __device__ __forceinline__ void meet() {
    static_assert(N < 64, "the counter's range");
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070 | (N & 15) | (N >> 4) << 14);  // vmcnt N, lgkmcnt 0
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Rows first .. of a matrix, as a buffer that ends behind its last row or behind `most` rows (first is one of its rows).
struct Rows {
    const int8_t *p;
    int bytes;
};
__device__ __forceinline__ Rows rows_at(const int8_t *p, int64_t ld, int first, int rows, int most) {
    const int n = __builtin_amdgcn_readfirstlane(rows - first < most ? rows - first : most);  // (or the loads would loop over lanes)
    return Rows{p + first * ld, n * (int)ld};
}

// The place of workgroup `id` in an order of `total` of which each of the eight XCDs (consecutive workgroups in turn) takes a
// contiguous range.
__device__ __forceinline__ int place_of(int id, int total) {
    const int q = total >> 3, r = total & 7, x = id & 7;
    return x * q + (x < r ? x : r) + (id >> 3);
}

// The tile of workgroup `id`, in groups of GROUP tiles of tokens, so that the tiles in flight on an XCD share rows and channels
// in its L2. (Groups of 4, 8 and 16: 4096 x 24576 x 4096 377, 379 and 400 us.)
constexpr int GROUP = 4;
__device__ __forceinline__ void tile_of(int id, int tiles_m, int tiles_n, int &tm, int &tn) {
    const int t = place_of(id, tiles_m * tiles_n), per = GROUP * tiles_n, group = t / per, first = group * GROUP;
    const int size = tiles_m - first < GROUP ? tiles_m - first : GROUP, in = t - group * per;
    tm = __builtin_amdgcn_readfirstlane(first + in % size), tn = __builtin_amdgcn_readfirstlane(in / size);
}

// How a product is cut: tiles of tokens and channels, `per` of K for each of the launch's y; with several of those their
// sums go to `sums` (rows of ld, a multiple of 4) instead of y.
struct Tiling {
    int m, n, per, ld;
    int *sums;
};

// 4 channels of one token into y
__device__ __forceinline__ void put(const Gemm8Args &a, int m, int n, f4 r) {
    float *y = a.y + (int64_t)m * a.ldy + n;
    if (n + 4 <= a.N) {
        if (a.accum) r += *(const f4u *)y;
        *(f4u *)y = r;
    } else {
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (n + c < a.N) y[c] = a.accum ? y[c] + r[c] : r[c];
    }
}

// A tile of B tokens x B channels; WM x WN waves. H places in LDS, each for the tokens' or the channels' half of a stage: while
// a stage is multiplied, (H - 2) / 2 stages are on their way, straight to LDS (no registers, no LDS stores by the waves).
// Products 32x32x32, which take half the operand reads of 16x16x64; a wave's rows of w are the first operand, so that a lane's
// accumulators are 4 neighbouring channels of one token.
// (4096 x 24576 x 4096: 376 to 382 us in tiles of 256, 573 of 128. In tiles of 256 with stages of 64 bytes 420, four waves of
// 128 x 128 416, workgroups that go on to further tiles 408, as a tile's first wait then includes the last one's stores.)
template <int B, int WM, int WN, int H, int EU>
__global__ __launch_bounds__(WM * WN * 64) __attribute__((amdgpu_waves_per_eu(EU, EU)))
void gemm8_tile(Gemm8Args a, Tiling t) {
#if __HIP_DEVICE_COMPILE__  // (the host's pass over these builtins would leave the kernel without its launch stub)
    constexpr int NW = WM * WN, TM = B / WM / 32, TN = B / WN / 32, NLH = B / 8 / NW, BYTES = B * KB;
    static_assert(B % (8 * NW) == 0 && NW % 4 == 0, "rows of a load");
    static_assert(H % 2 == 1 && H >= 5 && H <= 9 && H * BYTES <= 160 * 1024, "places");
    // (an array each, so that the compiler sees which loads a read has to wait for)
    constexpr int MORE = H > 5 ? BYTES : 16, MOST = H > 7 ? BYTES : 16;
    __shared__ __attribute__((aligned(1024))) char lds0[BYTES], lds1[BYTES], lds2[BYTES], lds3[BYTES], lds4[BYTES];
    __shared__ __attribute__((aligned(1024))) char lds5[MORE], lds6[MORE], lds7[MOST], lds8[MOST];
    auto place = [&](int n) __attribute__((always_inline)) {
        n %= H;
        return n == 0 ? lds0 : n == 1 ? lds1 : n == 2 ? lds2 : n == 3 ? lds3 : n == 4 ? lds4 : n == 5 ? lds5 : n == 6 ? lds6
               : n == 7 ? lds7 : lds8;
    };
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN, g = lane >> 5, col = lane & 31;
    int tm, tn;
    tile_of(blockIdx.x, t.m, t.n, tm, tn);
    const int first = blockIdx.y * t.per, end = first + t.per < a.K ? first + t.per : a.K;  // of K

    // this wave's loads of a stage: rows (i NW + wave) 8 .. + 7 each; a lane brings 16 bytes of one row. Rows past the last and
    // bytes past K are past the buffer's end: they read as zero.
    const int lr = lane >> 3, lc = ((lane & 7) ^ turn_of(wave * 8 + lr)) * 16;
    const Rows x = rows_at(a.x, a.ldx, tm * B, a.M, B), w = rows_at(a.w, a.ldw, tn * B, a.N, B);
    const __amdgpu_buffer_rsrc_t xb = __builtin_amdgcn_make_buffer_rsrc((void *)x.p, 0, x.bytes, 0x00027000);
    const __amdgpu_buffer_rsrc_t wb = __builtin_amdgcn_make_buffer_rsrc((void *)w.p, 0, w.bytes, 0x00027000);
    uint32_t xat[NLH], wat[NLH];
#pragma unroll
    for (int i = 0; i < NLH; i++) {
        xat[i] = (uint32_t)((i * NW + wave) * 8 + lr) * (uint32_t)a.ldx + lc;
        wat[i] = (uint32_t)((i * NW + wave) * 8 + lr) * (uint32_t)a.ldw + lc;
    }
    auto fetch = [&](char *lds, bool tok, int k0) __attribute__((always_inline)) {
        const uint32_t past = k0 + lc < end ? 0u : 1u << 31;
        const int from = k0 < a.K ? k0 : a.K;  // (within a row, and so within the buffer, where all of it is past)
#pragma unroll
        for (int i = 0; i < NLH; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(tok ? xb : wb, (lds_void *)(lds + (i * NW + wave) * 8 * KB), 16,
                                                     (tok ? xat[i] : wat[i]) | past, from, 0, 0);
    };
    i16 acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int j = 0; j < TM; j++) acc[i][j] = i16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    struct Part {  // 32 bytes of K of this wave's rows
        i4 w[TN], x[TM];
    };
    const int ax = (wm * TM * 32 + col) * KB, aw = (wn * TN * 32 + col) * KB, turn = turn_of(col) << 4;
    auto read = [&](const char *lx, const char *lw, int s, Part &p) __attribute__((always_inline)) {
        const int c = ((2 * s + g) << 4) ^ turn;
#pragma unroll
        for (int j = 0; j < TM; j++) p.x[j] = *(const i4 *)(lx + ax + c + j * 32 * KB);
#pragma unroll
        for (int i = 0; i < TN; i++) p.w[i] = *(const i4 *)(lw + aw + c + i * 32 * KB);
    };
    auto multiply = [&](const Part &p) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < TN; i++)
#pragma unroll
            for (int j = 0; j < TM; j++) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(p.w[i], p.x[j], acc[i][j], 0, 0, 0);
    };
    auto spread = [&]() __attribute__((always_inline)) {  // operand loads between the products
#pragma unroll
        for (int i = 0; i < TN * TM; i++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if (i < TN + TM) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
    };
    Part p0, p1;
    // A stage's products in four parts, the operands of each read during the one before. After the third the stage is read and
    // its places are free; the loads into them go between the products of the fourth.
    auto head = [&](const char *cx, const char *cw) __attribute__((always_inline)) {
        read(cx, cw, 1, p1);
        multiply(p0);
        spread();
        read(cx, cw, 2, p0);
        multiply(p1);
        spread();
        read(cx, cw, 3, p1);
        multiply(p0);
        spread();
        meet<(H - 4) * NLH>();  // (the next stage is there; a wave's loads end in the order in which they began)
    };
    auto tail = [&](char *cx, char *cw, const char *nx, const char *nw, int k0) __attribute__((always_inline)) {
        fetch(cx, false, k0 + (H - 1) / 2 * KB);
        fetch(cw, true, k0 + (H + 1) / 2 * KB);
        read(nx, nw, 0, p0);
        multiply(p1);
#pragma unroll
        for (int i = 0; i < TN * TM; i++) {  // (a wave's loads queue behind each other: all at once would hold up its products)
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if (i < TN + TM) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x020, (2 * NLH + TN * TM - 1) / (TN * TM), 0);
        }
    };
#pragma unroll
    for (int h = 0; h < H; h++) fetch(place(h), h % 2 == 0, first + h / 2 * KB);
    meet<(H - 2) * NLH>();
    read(lds0, lds1, 0, p0);
    head(lds0, lds1);
    // (H stages, and each place has held every one of them; written out, for the places have to be known when it is compiled)
    for (int k0 = first;;) {
#define STAGE(i)                                                                          \
    if (k0 + KB >= end) break;                                                            \
    tail(place(2 * (i)), place(2 * (i) + 1), place(2 * (i) + 2), place(2 * (i) + 3), k0); \
    k0 += KB;                                                                             \
    head(place(2 * (i) + 2), place(2 * (i) + 3));
        STAGE(0) STAGE(1) STAGE(2) STAGE(3) STAGE(4)
        if constexpr (H > 5) {
            STAGE(5) STAGE(6)
        }
        if constexpr (H > 7) {
            STAGE(7) STAGE(8)
        }
#undef STAGE
    }
    multiply(p1);
    // the results' places and scales
    const int m0 = tm * B + wm * TM * 32, n0 = tn * B + wn * TN * 32;
    const int er = lane >> 3, en = (lane & 7) * 4;  // this lane's row of 8, its 4 channels
    int *const part = t.sums ? t.sums + (int64_t)blockIdx.y * a.M * t.ld : nullptr;
    float xs[TM][4];
    f4 ws[TN];
#pragma unroll
    for (int j = 0; j < TM; j++)  // (past the ends the last)
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int m = m0 + j * 32 + 8 * u + er;
            xs[j][u] = a.x_scale[m < a.M ? m : a.M - 1];
        }
#pragma unroll
    for (int i = 0; i < TN; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const int n = n0 + i * 32 + en + c;
            ws[i][c] = a.w_scale[n < a.N ? n : a.N - 1];
        }
    // Parts of 32 x 32 through LDS, PB at a time (each wave its own 4 KiB for each): a lane's accumulators are 4 channels of
    // one token, four times; rows of 128 bytes go to memory, 8 of them with an instruction. (Parts of lines cost as much as
    // whole ones. One part at a time 64 x 12288 x 2048 added to y 8.9 us, two 7.9, four spill.)
    constexpr int PB = TN * TM < 2 ? 1 : 2;
    static_assert(2 * PB * 4096 <= BYTES && NW / 2 <= H && TN * TM % PB == 0, "two waves a place");
    auto results = [&](auto adds, auto inside) __attribute__((always_inline)) {  // inside: all of this wave's tile is
        constexpr bool ADDS = decltype(adds)::value, INSIDE = decltype(inside)::value;
        f4 was[PB][4];
        char *const own = place(wave >> 1) + (wave & 1) * (PB * 4096);
#pragma unroll
        for (int p0 = 0; p0 < TN * TM; p0 += PB) {
            if constexpr (ADDS) {  // what is added to, on its way
#pragma unroll
                for (int p = 0; p < PB; p++)
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const int m = m0 + (p0 + p) % TM * 32 + 8 * u + er, n = n0 + (p0 + p) / TM * 32 + en;
                        if constexpr (!INSIDE) was[p][u] = f4{0, 0, 0, 0};
                        if (INSIDE || (m < a.M && n + 4 <= a.N))
                            was[p][u] = *(const f4u *)(a.y + (int64_t)m * a.ldy + n);
                    }
            }
            if (p0 == 0) meet<0>();
#pragma unroll
            for (int p = 0; p < PB; p++) {
                const i16 v = acc[(p0 + p) / TM][(p0 + p) % TM];
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    i4 *const to = (i4 *)(own + p * 4096 + col * 128 + (((2 * q + g) ^ (col & 7)) << 4));
                    *to = i4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
                }
            }
#pragma unroll
            for (int p = 0; p < PB; p++) {
                const int i = (p0 + p) / TM, j = (p0 + p) % TM, n = n0 + i * 32 + en;
                i4 o[4];
#pragma unroll
                for (int u = 0; u < 4; u++)
                    o[u] = *(const i4 *)(own + p * 4096 + (8 * u + er) * 128 + (((lane & 7) ^ er) << 4));
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int m = m0 + j * 32 + 8 * u + er;
                    if constexpr (!INSIDE) {
                        if (m >= a.M) continue;
                        if (part) {
                            if (n < t.ld) *(i4 *)(part + (int64_t)m * t.ld + n) = o[u];
                            continue;
                        }
                    }
                    f4 r;
#pragma unroll
                    for (int c = 0; c < 4; c++) r[c] = (float)o[u][c] * xs[j][u] * ws[i][c];
                    if (INSIDE || n + 4 <= a.N) {
                        if constexpr (ADDS) r += was[p][u];
                        *(f4u *)(a.y + (int64_t)m * a.ldy + n) = r;
                    } else {
                        put(a, m, n, r);
                    }
                }
            }
        }
    };
    if constexpr (TN * TM <= 2) {  // (the largest tile has no registers for a way of its own)
        if (!part && m0 + TM * 32 <= a.M && n0 + TN * 32 <= a.N) {
            if (a.accum) results(std::true_type{}, std::true_type{});
            else results(std::false_type{}, std::true_type{});
            return;
        }
    }
    if (a.accum && !part) results(std::true_type{}, std::false_type{});
    else results(std::false_type{}, std::false_type{});
#endif
}

// The sums of P parts of K, four channels of a token a thread.
template <int P> __global__ __launch_bounds__(256) void gemm8_join(Gemm8Args a, const int *sums, int ld) {
    const int id = blockIdx.x * 256 + threadIdx.x, m = id / (ld / 4), n = (id - m * (ld / 4)) * 4;
    if (m >= a.M) return;
    const int *p = sums + (int64_t)m * ld + n;
    i4 v[P];
#pragma unroll
    for (int i = 0; i < P; i++) v[i] = *(const i4 *)(p + (int64_t)i * a.M * ld);
    const float xs = a.x_scale[m];
    f4 ws, r;
#pragma unroll
    for (int c = 0; c < 4; c++) ws[c] = n + c < a.N ? a.w_scale[n + c] : 0.f;
#pragma unroll
    for (int i = 1; i < P; i++) v[0] += v[i];
#pragma unroll
    for (int c = 0; c < 4; c++) r[c] = (float)v[0][c] * xs * ws[c];
    put(a, m, n, r);
}

template <int B, int WM, int WN, int H, int EU> void tiles(const Gemm8Args &a, int parts, int *sums, hipStream_t st) {
    Tiling t{};
    t.m = (a.M + B - 1) / B, t.n = (a.N + B - 1) / B;
    t.ld = (a.N + 3) / 4 * 4;
    t.per = ((a.K + KB - 1) / KB + parts - 1) / parts * KB;
    t.sums = parts > 1 ? sums : nullptr;
    gemm8_tile<B, WM, WN, H, EU><<<dim3(t.m * t.n, parts), WM * WN * 64, 0, st>>>(a, t);
    const int blocks = (int)(((int64_t)a.M * (t.ld / 4) + 255) / 256);
    if (parts == 2) gemm8_join<2><<<blocks, 256, 0, st>>>(a, sums, t.ld);
    else if (parts == 3) gemm8_join<3><<<blocks, 256, 0, st>>>(a, sums, t.ld);
    else if (parts == 4) gemm8_join<4><<<blocks, 256, 0, st>>>(a, sums, t.ld);
    else if (parts == 6) gemm8_join<6><<<blocks, 256, 0, st>>>(a, sums, t.ld);
    else if (parts == 8) gemm8_join<8><<<blocks, 256, 0, st>>>(a, sums, t.ld);
}

// Few tokens: 16 tokens x 16 channels a workgroup, K over its W waves. A wave brings 128 bytes of K of its 32 rows at a time,
// whole lines (loads of half lines, as the products' registers would take them, reach 40 GB/s a CU, these 112), to places of
// its own in LDS, two ahead; the waves' sums meet at the end. Bound by the weights' bytes where channels are many, else by what
// a CU takes in. (W = 2: 16 x 24576 x 4096 19.9 us, 33 x 4096 x 4096 6.5; with 4 places 22.4 and 6.4, with 8 25.1 and 9.9, as
// fewer workgroups fit on a CU. With 32 tokens a workgroup 64 x 4096 x 4096 6.9 and 16 x 512 x 8192 7.1, with 16 7.8 and 6.2.)
template <int W> __global__ __launch_bounds__(W * 64) void gemm8_few(Gemm8Args a, int tiles_m, int tiles_n) {
#if __HIP_DEVICE_COMPILE__
    // D places a wave, each 16 rows of w, then of x, with turns as a tile's rows; ROWS: bytes of the 8 rows of a load
    constexpr int D = 3, ROWS = 8 * KB, UNIT = 4 * ROWS;
    __shared__ __attribute__((aligned(1024))) char lds[W * D * UNIT];
    __shared__ i4 sums[W][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int g = lane >> 4, col = lane & 15;
    // the tokens of the same channels one after another, on one XCD (50 x 2880 x 5760: 7.9 us, channels first 9.1;
    // 33 x 4096 x 4096: 6.5 and 6.0)
    const int t = place_of(blockIdx.x, tiles_m * tiles_n), tn = __builtin_amdgcn_readfirstlane(t / tiles_m);
    const int n0 = tn * 16, m0 = (t - tn * tiles_m) * 16;
    const Rows x = rows_at(a.x, a.ldx, m0, a.M, 16), w = rows_at(a.w, a.ldw, n0, a.N, 16);
    const __amdgpu_buffer_rsrc_t xb = __builtin_amdgcn_make_buffer_rsrc((void *)x.p, 0, x.bytes, 0x00027000);
    const __amdgpu_buffer_rsrc_t wb = __builtin_amdgcn_make_buffer_rsrc((void *)w.p, 0, w.bytes, 0x00027000);
    const int lr = lane >> 3, lc = ((lane & 7) ^ (lr & 6)) * 16;
    const uint32_t xat = (uint32_t)lr * (uint32_t)a.ldx + lc, wat = (uint32_t)lr * (uint32_t)a.ldw + lc;
    // the first wave's scales and what it adds to, on their way first
    const int m = m0 + col, n = n0 + 4 * g;
    const bool there = m < a.M && n < a.N, whole = n + 4 <= a.N;
    float xs = 0.f;
    f4 ws = {0, 0, 0, 0}, was = {0, 0, 0, 0};
    if (wave == 0 && there) {
        xs = a.x_scale[m];
#pragma unroll
        for (int c = 0; c < 4; c++) ws[c] = a.w_scale[n + c < a.N ? n + c : a.N - 1];
        if (a.accum && whole) was = *(const f4u *)(a.y + (int64_t)m * a.ldy + n);
    }
    const int units = (a.K + KB - 1) / KB, per = (units + W - 1) / W, first = wave * per;
    const int end = first + per < units ? first + per : units;
    char *const own = lds + wave * D * UNIT;
    auto fetch = [&](int at, int u) __attribute__((always_inline)) {
        const int k = u * KB, from = k < a.K ? k : a.K;
        const uint32_t past = u < end && k + lc < a.K ? 0u : 1u << 31;  // (of another wave, or past K: zeros)
        const uint32_t w8 = 8 * (uint32_t)a.ldw, x8 = 8 * (uint32_t)a.ldx;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(wb, (lds_void *)(own + at), 16, wat | past, from, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(wb, (lds_void *)(own + at + ROWS), 16, (wat + w8) | past, from, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(xb, (lds_void *)(own + at + 2 * ROWS), 16, xat | past, from, 0, 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(xb, (lds_void *)(own + at + 3 * ROWS), 16, (xat + x8) | past, from, 0, 0);
    };
    i4 acc = {0, 0, 0, 0};
    const uint32_t row = (uint32_t)(uintptr_t)(lds_void *)own + col * KB, turn = (col & 6) << 4;
    const uint32_t c0 = row + ((uint32_t)(g << 4) ^ turn), c1 = row + ((uint32_t)(64 + (g << 4)) ^ turn);
#pragma unroll
    for (int d = 0; d < D; d++) fetch(d * UNIT, first + d);
    int at = 0;
    for (int u = first; u < end; u++) {
        i4 w0, x0, w1, x1;
        // the oldest place's loads are there; it is read, and free. (A read that the compiler sees it lets wait for all loads.)
        asm volatile("s_waitcnt vmcnt(%6)\n\t"
                     "ds_read_b128 %0, %4\n\t"
                     "ds_read_b128 %1, %4 offset:2048\n\t"
                     "ds_read_b128 %2, %5\n\t"
                     "ds_read_b128 %3, %5 offset:2048\n\t"
                     "s_waitcnt lgkmcnt(0)"
                     : "=&v"(w0), "=&v"(x0), "=&v"(w1), "=&v"(x1)
                     : "v"(c0 + at), "v"(c1 + at), "n"((D - 1) * 4)
                     : "memory");
        fetch(at, u + D);
        at = at == (D - 1) * UNIT ? 0 : at + UNIT;
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(w0, x0, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(w1, x1, acc, 0, 0, 0);
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave || !there) return;
#pragma unroll
    for (int i = 1; i < W; i++) acc += sums[i][lane];
    f4 r;  // (a lane's sums are 4 channels of one token)
#pragma unroll
    for (int c = 0; c < 4; c++) r[c] = (float)acc[c] * xs * ws[c];
    if (whole) {
        if (a.accum) r += was;  // (not without: -0 + 0 is +0)
        *(f4u *)(a.y + (int64_t)m * a.ldy + n) = r;
    } else {
        put(a, m, n, r);
    }
#endif
}

template <int W> void few(const Gemm8Args &a, hipStream_t st) {
    const int tm = (a.M + 15) / 16, tn = (a.N + 15) / 16;
    gemm8_few<W><<<tm * tn, W * 64, 0, st>>>(a, tm, tn);
}

}  // namespace

static size_t sums_bytes(const Gemm8Args &a, const Gemm8Plan &p) {
    return p.parts > 1 ? (size_t)p.parts * a.M * ((a.N + 3) / 4 * 4) * 4 : 0;
}

static Gemm8Plan plan_of(const Gemm8Args &a) { return gemm8_plan(a.M, a.N, a.K, a.accum); }

size_t gemm8_ws(const Gemm8Args &a) { return sums_bytes(a, plan_of(a)); }

// need: the workspace's bytes; with fewer given nothing is launched.
hipError_t launch_gemm8(const Gemm8Args &a, void *ws, size_t ws_bytes, size_t *need, hipStream_t st) {
    const Gemm8Plan p = plan_of(a);
    *need = sums_bytes(a, p);
    if (*need && (!ws || ws_bytes < *need || ((uintptr_t)ws & 15))) return hipErrorInvalidValue;
    if (p.shape < 0) {
        // four waves where half of the CUs or more have no workgroup and K is long (5 x 2048 x 12288: 6.2 us, with two 8.8;
        // 1 x 2048 x 4096: 4.4 and 4.1; 17 x 4096 x 4096: 6.0 and 5.3)
        if ((int64_t)((a.N + 15) / 16) * ((a.M + 15) / 16) <= 128 && a.K >= 8192) few<4>(a, st);
        else few<2>(a, st);
    }
    else if (p.shape == 0) tiles<64, 2, 2, 9, 2>(a, p.parts, (int *)ws, st);
    else if (p.shape == 1) tiles<128, 2, 4, 9, 2>(a, p.parts, (int *)ws, st);
    else if (p.shape == 2) tiles<128, 2, 4, 5, 4>(a, p.parts, (int *)ws, st);
    else tiles<256, 2, 4, 5, 2>(a, p.parts, (int *)ws, st);
    return hipGetLastError();
}
