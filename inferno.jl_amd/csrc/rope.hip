// Rotary positions and the KV-cache append (the reference's partial RoPE and
// cache write: src/ModelCPU.jl:125-231, :245-258).
//
// A pair (a, b) of a head at position p becomes (c a - s b, s a + c b), c + i s
// = mscale e^{i p theta}. The table holds theta in turns (theta / 2 pi, fp64):
// p theta is one fp64 product, its fraction of a turn one fp64 subtraction, and
// only that fraction, in [-1/2, 1/2], is rounded to fp32 for sine and cosine.
//
// One workgroup takes one token (or a part of its heads where tokens are few):
// the pairs' sines and cosines are formed once in LDS and serve every head, so
// beyond that a value is read once, turned and written once, 16 bytes a lane.
// Bound by those bytes where tokens are many, by one pass of loads and stores
// where they are few:
//   8190 rows of 16 q, 4 k and 4 v heads of 256 into fp32 rows and a bf16 cache
//     (369 MB) 73.5 us, 5.0 TB/s; a copy of 1 GiB reaches 5.2. 4 bytes a lane
//     instead of 16: 35.2 us for 29.8 (4096 rows of 48 heads of 128);
//   one row of 32 q, 8 k and 8 v heads of 128: 3.2 us;
//   64 rows of 32 heads of 128: 3.9 us.
#include "common.h"
#include "mixer.h"

namespace {

template <int VEC> struct Vec;
template <> struct Vec<4> { typedef f4 t; };
template <> struct Vec<1> { typedef float t; };

// VEC consecutive values into the cache, rounded once to its type
template <int VEC> __device__ __forceinline__ void put_kv(void *base, int64_t at, int type, const float *v) {
    if (type == KV_F16) {
        _Float16 *p = (_Float16 *)base + at;
        if constexpr (VEC == 4) *(h4 *)p = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
        else p[0] = (_Float16)v[0];
    } else {
        __bf16 *p = (__bf16 *)base + at;
        if constexpr (VEC == 4) *(b4 *)p = b4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
        else p[0] = (__bf16)v[0];
    }
}

// STREAM: rows of fp32 too many for the caches pass them by.
template <int VEC, bool STREAM> __global__ __launch_bounds__(256) void rope_kernel(RopeArgs a, RopeTable tab) {
    __shared__ float2 cs[128];
    typedef typename Vec<VEC>::t vec;
    const int64_t row = blockIdx.x;
    const int D = a.head_dim, half = a.rot_dim / 2, tid = threadIdx.x;
    int s = 0, n = 0;
    bool fits = true;
    if (a.len) {
        s = (int)(row / a.M);
        n = a.len[s];
        if (n < 0) return;
        fits = (int64_t)n + a.M <= a.capacity;
    }
    const int m = a.len ? (int)(row - (int64_t)s * a.M) : 0;
    const double p = a.pos ? (double)a.pos[row] : (double)a.pos0 + (double)n + (double)m;
    if (tid < half) {
        double t = tab.turns[tid];
        if (a.freq_factors) t /= (double)a.freq_factors[tid];
        t *= p;
        const float f = 2.0f * (float)(t - rint(t));
        cs[tid] = float2{cospif(f) * a.mscale, sinpif(f) * a.mscale};
    }
    __syncthreads();
    const float *x = a.x + row * a.ldx;
    float *y = a.y + row * a.ldy;
    // units of a rotating head: `ru` of one or two vectors of pairs, then its copied vectors
    const int ru = a.rot_dim / (VEC == 4 && a.interleaved ? 4 : 2 * VEC);
    const int ut = ru + (D - a.rot_dim) / VEC, uv = D / VEC;
    const int n_turn = (a.n_q + a.n_k) * ut, total = n_turn + a.n_v * uv;
    auto get = [&](int64_t at) __attribute__((always_inline)) {
        if constexpr (STREAM) return __builtin_nontemporal_load((const vec *)(x + at));
        else return *(const vec *)(x + at);
    };
    auto put = [&](int64_t at, const float *v) __attribute__((always_inline)) {
        if constexpr (STREAM) __builtin_nontemporal_store(*(const vec *)v, (vec *)(y + at));
        else *(vec *)(y + at) = *(const vec *)v;
    };
    const int64_t slot = (int64_t)s * a.seq_stride + ((int64_t)n + m) * a.tok_stride;
    for (int i = blockIdx.y * 256 + tid; i < total; i += gridDim.y * 256) {
        const bool turn = i < n_turn;
        const int per = turn ? ut : uv, j = turn ? i : i - n_turn;
        const int hd = j / per, u = j - hd * per;
        const int head = turn ? hd : a.n_q + a.n_k + hd;  // among the row's heads
        int d0, d1 = -1;                                  // the unit's first values (d1: the pairs' other half)
        if (turn && u < ru) {
            d0 = VEC == 4 && a.interleaved ? 4 * u : a.interleaved ? 2 * u : VEC * u;
            if (!a.interleaved) d1 = d0 + half;
            else if (VEC == 1) d1 = d0 + 1;
        } else {
            d0 = turn ? a.rot_dim + (u - ru) * VEC : u * VEC;
        }
        const int64_t src = (int64_t)head * D;
        float v0[VEC], v1[VEC];
        *(vec *)v0 = get(src + d0);
        if (turn && u < ru) {
            if (VEC == 4 && a.interleaved) {
#pragma unroll
                for (int c = 0; c + 1 < VEC; c += 2) {
                    const float2 e = cs[2 * u + c / 2];
                    const float p0 = v0[c], p1 = v0[c + 1];
                    v0[c] = p0 * e.x - p1 * e.y;
                    v0[c + 1] = p1 * e.x + p0 * e.y;
                }
            } else {
                *(vec *)v1 = get(src + d1);
#pragma unroll
                for (int c = 0; c < VEC; c++) {
                    const float2 e = cs[VEC * u + c];
                    const float p0 = v0[c], p1 = v1[c];
                    v0[c] = p0 * e.x - p1 * e.y;
                    v1[c] = p1 * e.x + p0 * e.y;
                }
            }
        }
        if (head < a.n_q) {
            if (!fits) {
#pragma unroll
                for (int c = 0; c < VEC; c++) v0[c] = v1[c] = __builtin_nanf("");
            }
            put(src + d0, v0);
            if (d1 >= 0) put(src + d1, v1);
        } else if (fits) {
            const int kv = turn ? head - a.n_q : hd;
            void *base = turn ? a.k : a.v;
            const int64_t at = slot + (int64_t)kv * a.head_stride;
            put_kv<VEC>(base, at + d0, a.type, v0);
            if (d1 >= 0) put_kv<VEC>(base, at + d1, a.type, v1);
        }
    }
}

}  // namespace

hipError_t launch_rope(const RopeArgs &a, const RopeTable &tab, int64_t rows, bool vec, hipStream_t st) {
    const int per = vec ? 4 : 1;
    const int64_t units = (int64_t)(a.n_q + a.n_k + a.n_v) * (a.head_dim / per);
    // a token's heads over up to 8 workgroups where tokens alone would not fill the chip (us, split and not: 1 row of 80 heads
    // 3.2, 5.3; 512 rows 8.3, 9.6; 16384 rows 246, 239)
    int64_t split = rows >= 1024 ? 1 : (1024 + rows - 1) / rows;
    const int64_t most = (units + 511) / 512;
    split = split < most ? split : most;
    if (split > 8) split = 8;
    const dim3 grid((unsigned)rows, (unsigned)(split < 1 ? 1 : split));
    // past the caches from 32 MB of rows on, what the eight L2s hold: 8190 rows of 201 MB 73.5 us, 77.5 through them (fewer are
    // read again by what comes next; timed by itself, at this size, not with the projection before it and the attention behind)
    const bool stream = rows * units * per * 4 >= (int64_t)32 << 20;
    if (vec && stream) rope_kernel<4, true><<<grid, 256, 0, st>>>(a, tab);
    else if (vec) rope_kernel<4, false><<<grid, 256, 0, st>>>(a, tab);
    else rope_kernel<1, false><<<grid, 256, 0, st>>>(a, tab);
    return hipGetLastError();
}
