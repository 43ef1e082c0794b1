// Rows of fp32 values as 8-bit codes with a scale a row: the input of the 8-bit
// products (gemm8.hip), from the residual stream (the residual's addition and
// the RMSNorm of src/ModelCPU.jl:110-122, :870-891), from [gate | up] (:447-473)
// or from rows as they are.
//
//   t = x | x w | silu(gate) up;  top = max |t|;  code = rint(127 t / top)
//   scale = top / 127, times 1 / sqrt(mean(x^2) + eps) for the norm
//
// The norm's factor is one number a row, so it cancels in the codes and enters
// the scale alone: codes need the row's largest |t| and nothing else, and a row
// is read once, held in registers, and its codes written once.
//
// Codes are those of the exact t, not of its fp32 rounding: t and 127 / top are
// formed in fp32, and where 127 t / top comes nearer to a tie than their error
// (a value in ten thousand, four of the gate's) that one value is formed again in
// fp64. So codes do not depend on how the fp32 arithmetic was ordered or contracted.
//
// What bounds it. Many rows: memory. 8190 rows of 4096, the residual added and
// stored, in 71 us (268 MB read, 168 written: 6.1 TB/s; a copy reaches 5.2),
// 4096 plain rows of 12288 in 41 (6.2), 4097 gates of 6144 in 45 (5.1). Few: a
// launch and one row's way, 2 us plain, 3.1 with the norm and the residual, 5.5
// with 12288 gates on one CU. A gate's waves wait 71 % of their time and issue
// vector instructions in 12 % (5 rows of 12288): for their loads, at two barriers,
// and for gate and up read again behind the row's largest, where its exact value or
// a code next to a tie is formed in fp64. One workgroup a row, for a row's largest
// is one exchange through LDS then, and its values wait for it in registers.
#include "common.h"
#include "int8.h"

namespace {

constexpr int WAVES = 16;  // of the largest workgroup

struct Quant8Shared {
    uint32_t top[WAVES];
    float ssq[WAVES];
    uint64_t dtop[WAVES];
    double dssq[WAVES];
    uint64_t most;
};

// The lanes' values joined by op from neighbour to neighbour (DPP, where a shuffle goes by way of LDS), 0 standing for lanes
// that there are not: the 16 of a row of lanes in its last, then the rows in the last of all.
template <int CTRL, class T> __device__ __forceinline__ T from_lane(T v) {
    if constexpr (sizeof(T) == 8) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
        return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
    }
}
template <class T, class Op> __device__ __forceinline__ T join16(T v, Op op) {
    v = op(v, from_lane<0x111>(v));  // (row_shr 1, 2, 4, 8)
    v = op(v, from_lane<0x112>(v));
    v = op(v, from_lane<0x114>(v));
    return op(v, from_lane<0x118>(v));
}
template <class T, class Op> __device__ __forceinline__ T join64(T v, Op op) {
    v = join16(v, op);
    v = op(v, from_lane<0x142>(v));  // (row_bcast 15, 31)
    return op(v, from_lane<0x143>(v));
}
// what lane 15 has
template <class T> __device__ __forceinline__ T of_lane15(T v) {
    if constexpr (sizeof(T) == 8) {
        const uint64_t b = __builtin_bit_cast(uint64_t, v);
        const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, 15);
        const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), 15);
        return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
    } else {
        return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 15));
    }
}

__device__ __forceinline__ uint64_t dbits(double v) { return (uint64_t)__double_as_longlong(fabs(v)); }

__device__ __forceinline__ double silu_mul(double g, double u) { return g / (1.0 + exp(-g)) * u; }

// 4 values at column c of a row as the input has them after its additions
__device__ __forceinline__ f4 input4(const Quant8Args &a, int64_t row, int c) {
    if (a.x) return *(const f4 *)(a.x + row * a.ldx + c);
    f4 v = *(const f4 *)(a.add + row * a.ldx + c);
    for (int s = 1; s < a.n_add; s++) v += *(const f4 *)(a.add + s * a.add_stride + row * a.ldx + c);
    return v;
}

template <int ACT> __device__ __forceinline__ double exact1(float x, float w_or_up) {
    if constexpr (ACT == Q8_PLAIN) return (double)x;
    else if constexpr (ACT == Q8_RMSNORM) return (double)x * (double)w_or_up;
    else return silu_mul((double)x, (double)w_or_up);
}

// the second factor of 4 values at column c (norm_w, up)
template <int ACT> __device__ __forceinline__ f4 second4(const Quant8Args &a, int64_t row, int c) {
    if constexpr (ACT == Q8_RMSNORM) return a.norm_w ? *(const f4 *)(a.norm_w + c) : f4{1, 1, 1, 1};
    else if constexpr (ACT == Q8_SILU_MUL) return input4(a, row, a.K + c);
    else return f4{0, 0, 0, 0};
}

__device__ __forceinline__ float row_scale(double top, double ssq, bool norm, int K, float eps) {
    if (top == 0.0) return 0.f;
    const double s = top / 127.0;
    return (float)(norm ? s / sqrt(ssq / (double)K + (double)eps) : s);
}

// A row whose values leave the range in which fp32 serves: all of it in fp64. (Rows of zeros, of values past most_of or
// below 1e-20, and rows with a value that is not finite or a scale past fp32, whose codes are 0 and whose scale is NaN.)
template <int ACT> __device__ __forceinline__ void wide_row(const Quant8Args &a, int64_t row, Quant8Shared &sh) {
    const int tid = threadIdx.x, n4 = a.K / 4;
    uint64_t top = 0;
    double ssq = 0.0;
    for (int c = tid; c < n4; c += blockDim.x) {
        const f4 x = input4(a, row, 4 * c), w = second4<ACT>(a, row, 4 * c);
        for (int j = 0; j < 4; j++) {
            const uint64_t b = dbits(exact1<ACT>(x[j], w[j]));
            top = top > b ? top : b;
            ssq += (double)x[j] * (double)x[j];
        }
    }
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t w = __shfl_xor((unsigned long long)top, o);
        top = top > w ? top : w;
        ssq += __shfl_xor(ssq, o);
    }
    if ((tid & 63) == 0) sh.dtop[tid >> 6] = top, sh.dssq[tid >> 6] = ssq;
    __syncthreads();
    top = sh.dtop[0], ssq = sh.dssq[0];
    for (int i = 1; i < (int)(blockDim.x >> 6); i++) {
        top = top > sh.dtop[i] ? top : sh.dtop[i];
        ssq += sh.dssq[i];
    }
    const double most = __longlong_as_double((long long)top);
    const float scale = row_scale(most, ssq, ACT == Q8_RMSNORM, a.K, a.eps);
    const bool fine = top < 0x7ff0000000000000ull && scale < __builtin_inff();
    uint32_t *q = (uint32_t *)(a.q + row * a.ldq);
    for (int c = tid; c < n4; c += blockDim.x) {
        uint32_t word = 0;
        if (fine && top) {
            const f4 x = input4(a, row, 4 * c), w = second4<ACT>(a, row, 4 * c);
            for (int j = 0; j < 4; j++) {
                const int code = (int)rint(exact1<ACT>(x[j], w[j]) * 127.0 / most);
                word |= (uint32_t)(code & 255) << (8 * j);
            }
        }
        q[c] = word;
    }
    if (tid == 0) a.scale[row] = fine ? scale : __builtin_nanf("");
}

// Up to which largest |t| fp32 serves. The norm's: its scale top / 127 / sqrt(mean(x^2) + eps) can pass fp32 where the row is all
// but empty and a weight is large, with the sum of squares past 1e-30 and K up to 65536 only from a top of 1.6e23 on.
template <int ACT> constexpr float most_of = ACT == Q8_RMSNORM ? 1e23f : 1e30f;

// how far 127 t / top in fp32 may be off: t to 1 (norm) or 8 (silu: exp 3, 1 + exp 1, reciprocal 2, two products) halves of
// 2^-23, top as much, its reciprocal and the product one each: 127 (1 + 1 + 2) 2^-24 = 3.1e-5, 127 (8 + 8 + 2) 2^-24 = 1.4e-4
template <int ACT> constexpr float NEAR = ACT == Q8_SILU_MUL ? 2e-4f : 4e-5f;

// 4 values at column c of a row, the residual's additions made and stored
template <bool STREAM> __device__ __forceinline__ f4 take4(const Quant8Args &a, int64_t row, int c, bool adds) {
    if constexpr (STREAM) {  // (x and one slice)
        f4 *x = (f4 *)(a.x + row * a.ldx + c);
        const f4 v = __builtin_nontemporal_load(x) + __builtin_nontemporal_load((const f4 *)(a.add + row * a.K + c));
        __builtin_nontemporal_store(v, x);
        return v;
    }
    f4 v = input4(a, row, c);
    if (adds) {
        const float *add = a.add + row * a.K + c;
        f4 s = *(const f4 *)add;
        for (int k = 1; k < a.n_add; k++) s += *(const f4 *)(add + k * a.add_stride);
        v += s;
        *(f4 *)(a.x + row * a.ldx + c) = v;
    }
    return v;
}

// What a thread has found of its row: the sum of squares of x, and the largest |t| in fp32, as bits (as whole numbers NaN is
// the largest); for a norm with weights the largest exact product besides.
struct Found {
    float ssq = 0.f;
    uint32_t top = 0;
    double most = 0.0;
};

// exp(x) for x up to 88: 2^(x log2 e), the exponent's rest (its rounding and log2 e's second part) to first order
__device__ __forceinline__ float exp_to_88(float x) {
    const float y = x * 0x1.715476p+0f;
    const float rest = __builtin_fmaf(x, 0x1.4ae0cp-26f, __builtin_fmaf(x, 0x1.715476p+0f, -y));
    const float e = __builtin_amdgcn_exp2f(y);
    return __builtin_fmaf(e, rest * 0x1.62e43p-1f, e);
}

// x to t in fp32
template <int ACT> __device__ __forceinline__ f4 to_t(f4 x, f4 w, bool weights, Found &f) {
    f4 t = x;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if constexpr (ACT == Q8_RMSNORM) {
            f.ssq = __builtin_fmaf(x[j], x[j], f.ssq);
            t[j] = x[j] * w[j];
            if (weights) f.most = fmax(f.most, fabs((double)x[j] * (double)w[j]));
        } else if constexpr (ACT == Q8_SILU_MUL) {
            const float silu = x[j] * __builtin_amdgcn_rcpf(1.f + exp_to_88(fminf(-x[j], 88.f)));
            t[j] = silu * w[j];
            // (a silu next to nothing has few bits, of a subnormal gate, or none, as exp(-x) stops at 88 and its reciprocal is 0;
            // what is lost counts only beside so large an up)
            if (fabsf(silu) < 1e-30f && fabsf(w[j]) > 1e8f) f.top = 0x7fffffffu;
        }
        const uint32_t b = __float_as_uint(t[j]) & 0x7fffffffu;
        f.top = f.top > b ? f.top : b;
    }
    return t;
}

template <int ACT>
__device__ __forceinline__ void raise_most(const Quant8Args &a, int64_t row, int c, f4 t, float from, Quant8Shared &sh) {
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (fabsf(t[j]) >= from) {
            const f4 x = input4(a, row, c), w = second4<ACT>(a, row, c);
            atomicMax((unsigned long long *)&sh.most, (unsigned long long)dbits(exact1<ACT>(x[j], w[j])));
        }
}

template <int ACT>
__device__ __forceinline__ uint32_t codes4(const Quant8Args &a, int64_t row, int c, f4 t, float inv, double most) {
    constexpr float WHOLE = 0x1.8p23f;  // v + WHOLE: v rounded, ties to even, in the low bits
    uint32_t r[4];
    bool near[4], any = false;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float v = t[j] * inv, n = v + WHOLE;
        near[j] = fabsf(v - (n - WHOLE)) > 0.5f - NEAR<ACT>;
        any |= near[j];
        r[j] = __float_as_uint(n);
    }
    if (any) {
        const f4 x = input4(a, row, c), w = second4<ACT>(a, row, c);
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (near[j]) r[j] = (uint32_t)(int)rint(exact1<ACT>(x[j], w[j]) * 127.0 / most);
    }
    // (bytes 0 of four words: two of the first two, two of the last two, those of both)
    const uint32_t lo = __builtin_amdgcn_perm(r[1], r[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(r[3], r[2], 0x0c0c0400);
    return lo | hi << 16;
}

// One workgroup a row, V x 4 values a thread kept in registers; V = 0: rows of any length, read a second time for the codes.
template <int ACT, int V, bool STREAM = false> __global__ __launch_bounds__(1024) void quant8_kernel(Quant8Args a) {
    __shared__ Quant8Shared sh;
    constexpr int KEPT = V ? V : 1;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, n4 = a.K / 4, nt = blockDim.x;
    const bool adds = ACT != Q8_SILU_MUL && a.x && a.add;
    // (the norm's exact largest: on the way where a row is a workgroup's latency, of the candidates alone where rows are many:
    // 8190 rows of 4096 36.3 us and 34.0)
    constexpr bool DIRECT = ACT == Q8_RMSNORM && (V == 1 || V == 2);
    const bool weights = DIRECT && a.norm_w;
    f4 t[KEPT];
    Found f;
    if constexpr (V > 0) {
        f4 w[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = tid + i * nt;
            t[i] = c < n4 ? take4<STREAM>(a, row, 4 * c, adds) : f4{0, 0, 0, 0};
            w[i] = c < n4 ? second4<ACT>(a, row, 4 * c) : f4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < V; i++) t[i] = to_t<ACT>(t[i], w[i], weights, f);
    } else {
        for (int c = tid; c < n4; c += nt) {
            const f4 x = take4<STREAM>(a, row, 4 * c, adds);
            to_t<ACT>(x, second4<ACT>(a, row, 4 * c), weights, f);
        }
    }
    auto again = [&](int c) __attribute__((always_inline)) {
        Found none;
        return to_t<ACT>(input4(a, row, 4 * c), second4<ACT>(a, row, 4 * c), false, none);
    };
    // the waves' findings, then those of all waves: a lane for each (one row of 4096 3.1 us; by shuffles, and every thread over
    // all waves, 4.3)
    auto umax = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    auto dmax = [](double a, double b) { return fmax(a, b); };
    auto sum = [](float a, float b) { return a + b; };
    f.top = join64(f.top, umax);
    if constexpr (ACT == Q8_RMSNORM) f.ssq = join64(f.ssq, sum);
    if (weights) f.most = join64(f.most, dmax);
    if ((tid & 63) == 63) sh.top[tid >> 6] = f.top, sh.ssq[tid >> 6] = f.ssq, sh.dssq[tid >> 6] = f.most;
    if (tid == 0) sh.most = 0;
    __syncthreads();
    const int wave = tid & 15;
    const bool is = wave < nt >> 6;
    const uint32_t top = of_lane15(join16(is ? sh.top[wave] : 0u, umax));
    float ssq = 0.f;
    if constexpr (ACT == Q8_RMSNORM) ssq = of_lane15(join16(is ? sh.ssq[wave] : 0.f, sum));
    double most = weights ? of_lane15(join16(is ? sh.dssq[wave] : 0.0, dmax)) : 0.0;
    const float ftop = __uint_as_float(top);
    if (!(ftop > 1e-20f && ftop < most_of<ACT>) || (ACT == Q8_RMSNORM && !(ssq > 1e-30f && ssq < 1e30f))) {
        __syncthreads();  // (sh is read)
        wide_row<ACT>(a, row, sh);
        return;
    }
    if (!weights) most = (double)ftop;
    if (ACT == Q8_SILU_MUL || (!DIRECT && ACT == Q8_RMSNORM && a.norm_w)) {
        // the exact largest |t| is among those whose fp32 value is the largest (a product's rounding keeps the order), or
        // within twice the fp32 gate's error of it
        const float from = ACT == Q8_SILU_MUL ? ftop * (1.f - 0x1p-18f) : ftop;
        if constexpr (V > 0) {
#pragma unroll
            for (int i = 0; i < V; i++) raise_most<ACT>(a, row, 4 * (tid + i * nt), t[i], from, sh);
        } else {
            for (int c = tid; c < n4; c += nt) raise_most<ACT>(a, row, 4 * c, again(c), from, sh);
        }
        __syncthreads();
        most = __longlong_as_double((long long)sh.most);
    }
    const float inv = 127.f / ftop;
    uint32_t *q = (uint32_t *)(a.q + row * a.ldq);
    if constexpr (V > 0) {
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int c = tid + i * nt;
            if (c < n4) q[c] = codes4<ACT>(a, row, 4 * c, t[i], inv, most);
        }
    } else {
        for (int c = tid; c < n4; c += nt) q[c] = codes4<ACT>(a, row, 4 * c, again(c), inv, most);
    }
    if (tid == 0) a.scale[row] = row_scale(most, (double)ssq, ACT == Q8_RMSNORM, a.K, a.eps);
}

// How M rows of K values are cut: v times 4 values a thread (0: any number, read twice), nt threads a row.
struct Cut {
    int v, nt;
};
Cut cut_of(int M, int K) {
    const int n4 = K / 4;
    // few values a thread where rows are few and a row's time is latency; four times 4 where they are many (8190 rows of 4096,
    // plain: 34 us, with one 83), as far as a wave has them
    const int v = n4 > 4096 ? 0 : n4 > 2048 ? 4 : M <= 256 ? (n4 > 1024 ? 2 : 1) : n4 > 128 ? 4 : n4 > 64 ? 2 : 1;
    return Cut{v, v ? ((n4 + v - 1) / v + 63) / 64 * 64 : 1024};
}

template <int ACT> void launch(const Quant8Args &a, hipStream_t st) {
    const Cut cut = cut_of(a.M, a.K);
    const int v = cut.v, nt = cut.nt;
    if constexpr (ACT == Q8_RMSNORM) {
        // rows that are read, added to and written past the caches, from 64 MB of them on (8190 of 4096: 75.7 us, 81.4 through
        // them; 515: 9.0 and 8.1)
        if (v == 4 && a.x && a.n_add == 1 && (int64_t)a.M * a.K >= (int64_t)16 << 20) {
            quant8_kernel<ACT, 4, true><<<a.M, nt, 0, st>>>(a);
            return;
        }
    }
    if (v == 1) quant8_kernel<ACT, 1><<<a.M, nt, 0, st>>>(a);
    else if (v == 2) quant8_kernel<ACT, 2><<<a.M, nt, 0, st>>>(a);
    else if (v == 4) quant8_kernel<ACT, 4><<<a.M, nt, 0, st>>>(a);
    else quant8_kernel<ACT, 0><<<a.M, nt, 0, st>>>(a);
}

}  // namespace

bool quant8_fits(int M, int K) { return (int64_t)M * cut_of(M, K).nt < (int64_t)1 << 32; }

hipError_t launch_quant8(const Quant8Args &a, int act, hipStream_t st) {
    if (act == Q8_PLAIN) launch<Q8_PLAIN>(a, st);
    else if (act == Q8_RMSNORM) launch<Q8_RMSNORM>(a, st);
    else launch<Q8_SILU_MUL>(a, st);
    return hipGetLastError();
}
