// Attention of a batch's new tokens over a shared prefix, their own cached
// entries and each other (src/ModelCPU.jl:730-856).
//
// For a key head, the rows of its query heads (all sequences' for the prefix,
// one sequence's for its own entries) meet a range of keys in one workgroup:
//   S^T = K Q^T, P^T = 2^(S^T c - r), O^T += V^T P^T
// on 16x16x32 MFMAs, 32 keys at a time. Transposed, a lane's accumulators of
// S^T belong to one query row (lane & 15), so the running maximum and sum are a
// number a lane, and they are already the B operand of the second product (its
// sum over keys takes any order of them: lane group g holds keys 4 g .. 4 g + 3
// of either half): P never leaves the registers. V^T is read from the row-major
// tile in LDS with transposing loads.
//
// fp32 accuracy from 16-bit matrix cores: K and V are 16-bit already and enter
// as they are; q (times scale log2 e, and for f16 a power of two per row) and P
// are split into limbs, two of f16 (22 bits) or three of bf16 (24 bits), each
// product summed in fp32.
//
// Ranges of keys (splits) are joined by a last kernel in their order, so results
// do not depend on what runs when.
//
// What bounds it, and what it measured (the parts, then the join):
//   64 sequences of 5 tokens, 32 query heads over 8 of 128, 16384 shared f16
//     entries: the matrix cores and the vector work between their products, 186
//     + 10 us; the limbs' products are 176 GFLOP, 0.95 PFLOP/s (a large f16
//     matrix product reaches 1.17 here), and 4 vector instructions (softmax,
//     limbs) go with each MFMA, two waves a SIMD: about as long to issue;
//   one row of each of 32 query heads over 131072 entries: reading them, 537 MB
//     in 101 + 4 us, 5.3 TB/s;
//   a tree of 64 nodes, 16 query heads over 4 of 256, 6001 bf16 entries: 31 + 7
//     us: three limbs' products at half their rate, and 30 MB of parts written
//     and read (1024 rows of 256 values for each of 27 ranges of keys, 24 of them
//     the prefix's);
//   9 sequences of 5 tokens over 4099 bf16 entries of 64: 11 + 4 us, and one row
//     over 777 entries: 7 + 4 us: two launches, a few tiles one after the other.
#include "common.h"
#include "mixer.h"

namespace {

typedef short s4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;

template <int TYPE> struct Kv;
template <> struct Kv<KV_F16> {
    typedef _Float16 t;
    typedef h8 v8;
    static constexpr int LIMBS = 2;
    static constexpr float BIAS = 8.f;  // the largest P is 2^BIAS: its second limb then reaches 2^-33 of a row's largest
    static __device__ __forceinline__ f4 mfma(v8 a, v8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Kv<KV_BF16> {
    typedef __bf16 t;
    typedef b8 v8;
    static constexpr int LIMBS = 3;
    static constexpr float BIAS = 0.f;
    static __device__ __forceinline__ f4 mfma(v8 a, v8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// x = l[0] + l[1] (+ l[2]), each limb the rest rounded to its type
template <int TYPE> __device__ __forceinline__ void limbs(const float *x, typename Kv<TYPE>::v8 *l) {
    typedef typename Kv<TYPE>::t t;
    if constexpr (TYPE == KV_F16) {
        float one = 1.f;
        asm("" : "+v"(one));  // (x - hi as a mixed fma that rounds to f16 itself: one instruction a value)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const t h = (t)x[i];
            l[0][i] = h;
            l[1][i] = (t)__builtin_fmaf(-(float)h, one, x[i]);
        }
    } else {
        float r[8];
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] = x[i];
#pragma unroll
        for (int n = 0; n < Kv<TYPE>::LIMBS; n++)
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const t h = (t)r[i];
                l[n][i] = h;
                r[i] -= (float)h;
            }
    }
}

__device__ __forceinline__ float max_groups(float v) {  // over the four lane groups of a row
    const uint32_t x = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    const float m = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const uint32_t y = __float_as_uint(m);
    const auto b = __builtin_amdgcn_permlane16_swap(y, y, false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float sum_groups(float v) {
    const uint32_t x = __float_as_uint(v);
    const auto a = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    const float m = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const uint32_t y = __float_as_uint(m);
    const auto b = __builtin_amdgcn_permlane16_swap(y, y, false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Byte of 16-byte chunk c of row r in a tile of D values a row. The chunks of a row are permuted by its number so that
// neither the operand loads of K (16 rows, one chunk each) nor the transposing loads of V (4 rows, two chunks each)
// meet in a bank: a row of 128 or 256 values starts at the same bank as the next.
template <int D> __device__ __forceinline__ int tile_at(int r, int c) {
    const int x = D == 64 ? ((r >> 1) & 3) * 2 : (r & 7) * 2;
    return r * (D * 2) + ((c ^ x) << 4);
}

struct AttnSplit {
    int rows;      // query rows of a key head in this launch's unit (all sequences, or one)
    int blocks;    // row blocks
    int splits;    // ranges of keys
    int first;     // this launch's first part
    int64_t per;   // keys of a split (prefix)
};

// WR x WK waves: wave (wr, wk) takes rows [16 RT wr, ..) of the block and every WK-th 32 keys of a tile of KB keys; the
// next tile goes, in ST parts, through registers to the other buffer in LDS while one is worked on.
template <int RT_, int WR_, int WK_, int KB_, int ST_> struct Shape {
    static constexpr int RT = RT_, WR = WR_, WK = WK_, KB = KB_, ST = ST_, ROWS = WR * RT * 16;
    static_assert(WR * WK == 8, "eight waves");
};
// By the rows of a block: few rows split a tile's keys over the waves, many rows share it. (Two workgroups' worth of
// registers a SIMD, 256 each, and 128 KiB of LDS: one workgroup a CU.)
template <int D, int ID> struct ShapeOf;
template <int D> struct ShapeOf<D, 0> : Shape<1, 2, 4, 128, 1> {};
template <int D> struct ShapeOf<D, 1> : Shape<2, 2, 4, 128, 1> {};
template <int D> struct ShapeOf<D, 2> : Shape<2, 8, 1, 128, 2> {};
template <> struct ShapeOf<256, 1> : Shape<1, 4, 2, 64, 1> {};
template <> struct ShapeOf<256, 2> : Shape<1, 8, 1, 64, 2> {};

struct Shared {
    int bad[2];
    float2 ml[8][32];
};

template <int TYPE, int D, typename SH, bool OWN>
__device__ __forceinline__ void attn_part(const AttnArgs &a, const AttnSplit &sp, int block, char *lds, Shared &sh,
                                          float *__restrict__ opart, float2 *__restrict__ ml) {
    typedef Kv<TYPE> X;
    typedef typename X::t T;
    typedef typename X::v8 v8;
    constexpr int RT = SH::RT, WR = SH::WR, WK = SH::WK, KB = SH::KB, ST = SH::ST;
    constexpr int NT = WR * WK * 64, C = D / 8, STEPS = D / 32, DT = D / 16, ROWS = WR * RT * 16;
    constexpr int TILE = KB * D * 2, NLD = KB * C / NT;
    static_assert(KB % (32 * WK) == 0 && KB * C % NT == 0, "tile shape");
    static_assert(WK == 1 || 4 * TILE >= WR * WK * RT * 16 * D * 4, "the waves' results meet in the tile buffers");
    int *const bad = sh.bad;
    float2(*const wml)[32] = sh.ml;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave / WK, wk = wave % WK, g = lane >> 4, col = lane & 15;
    const int G = a.n_q / a.n_kv;

    // the block's unit: which sequence, key head, rows and keys
    int s = 0, hk, rb, split, n = 0;
    int64_t begin, end;
    const T *K, *V;
    int64_t kstride;
    if constexpr (OWN) {
        int id = block;
        split = id % sp.splits, id /= sp.splits;
        rb = id % sp.blocks, id /= sp.blocks;
        hk = id % a.n_kv, s = id / a.n_kv;
        n = a.len[s];
        if (n < 0 || (int64_t)n + a.M > a.capacity) return;
        const int64_t all = (int64_t)n + a.M, per = ((all + sp.splits - 1) / sp.splits + 31) / 32 * 32;
        begin = split * per;
        end = begin + per < all ? begin + per : all;
        kstride = a.tok_stride;
        K = (const T *)a.k + s * a.seq_stride + hk * a.head_stride;
        V = (const T *)a.v + s * a.seq_stride + hk * a.head_stride;
    } else {
        // row blocks of one range of keys go to one XCD (consecutive workgroups to the eight in turn), whose L2 then
        // holds the range for all of them
        const int id = block, x = id & 7, y = id >> 3;
        rb = y % sp.blocks;
        const int pair = (y / sp.blocks) * 8 + x;
        if (pair >= sp.splits * a.n_kv) return;
        hk = pair / sp.splits, split = pair % sp.splits;
        begin = split * sp.per;
        end = begin + sp.per < a.P ? begin + sp.per : a.P;
        kstride = a.p_tok_stride;
        K = (const T *)a.pk + hk * a.p_head_stride;
        V = (const T *)a.pv + hk * a.p_head_stride;
    }
    const int r0 = rb * ROWS + wr * RT * 16;

    // A tile comes in ST parts through registers, a part ahead: a uniform base and 32-bit lane offsets; past the last key,
    // the last key again (its scores are masked, and its values meet P = 0).
    constexpr int RL = NT / C;  // rows a load of the workgroup covers, a multiple of 8: they permute alike
    static_assert(RL % 8 == 0 && NLD % ST == 0, "rows of a load");
    u4 sk[NLD / ST], sv[NLD / ST];
    const uint32_t lane_at = (uint32_t)(tid / C) * (uint32_t)kstride + (uint32_t)(tid % C) * 8;
    const int put_at = tile_at<D>(tid / C, tid % C);
    auto fetch = [&](int64_t k0, int part) __attribute__((always_inline)) {
        k0 += part * (KB / ST);
        if (k0 + KB / ST <= end) {
            const T *kb = K + k0 * kstride, *vb = V + k0 * kstride;
#pragma unroll
            for (int i = 0; i < NLD / ST; i++) {
                sk[i] = *(const u4 *)(kb + lane_at);
                sv[i] = *(const u4 *)(vb + lane_at);
                kb += RL * kstride, vb += RL * kstride;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NLD / ST; i++) {
                const int64_t r = k0 + tid / C + i * RL, at = (r < end ? r : end - 1) * kstride + (tid % C) * 8;
                sk[i] = *(const u4 *)(K + at);
                sv[i] = *(const u4 *)(V + at);
            }
        }
    };
    auto put = [&](int buf, int part) __attribute__((always_inline)) {
        char *tk = lds + buf * 2 * TILE + part * (TILE / ST) + put_at;
#pragma unroll
        for (int i = 0; i < NLD / ST; i++) {
            *(u4 *)(tk + i * RL * (D * 2)) = sk[i];
            *(u4 *)(tk + TILE + i * RL * (D * 2)) = sv[i];
        }
    };
    if (begin < end) fetch(begin, 0);  // (on its way while the queries are split)

    // this lane's query rows (one a row tile): the token row, its place in the sequence, its head
    auto token = [&](int r) { return (int64_t)s * a.M + r / G; };
    v8 q[RT][STEPS][X::LIMBS];
    float c[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) {
        const int r = r0 + t * 16 + col;
        const bool in = r < sp.rows;
        const float *src = a.q + (in ? token(r) * a.ldq + (int64_t)(hk * G + r % G) * D : 0) + 8 * g;
        float x[STEPS][8], top = 0.f;
        const float k2 = a.scale * 1.44269504088896341f;
#pragma unroll
        for (int u = 0; u < STEPS; u++) {
            *(f4 *)(x[u]) = in ? *(const f4 *)(src + 32 * u) : f4{0, 0, 0, 0};
            *(f4 *)(x[u] + 4) = in ? *(const f4 *)(src + 32 * u + 4) : f4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 8; i++) x[u][i] *= k2, top = fmaxf(top, fabsf(x[u][i]));
        }
        float up = 1.f;
        c[t] = 1.f;
        if constexpr (TYPE == KV_F16) {  // the row's largest to [2^13, 2^14)
            top = max_groups(top);
            int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;
            e = e < -100 ? -100 : e > 127 ? 127 : e;  // (128: a row that is not finite)
            up = __uint_as_float((uint32_t)(127 + 13 - e) << 23);
            c[t] = __uint_as_float((uint32_t)(127 - 13 + e) << 23);
        }
#pragma unroll
        for (int u = 0; u < STEPS; u++) {
#pragma unroll
            for (int i = 0; i < 8; i++) x[u][i] *= up;
            limbs<TYPE>(x[u], q[t][u]);
        }
    }

    // P is 2^(score - ref): ref is 2^BIAS below the row's largest score when it last moved. It is an fp32 number, used as it is
    // by every P, by l and by the join, so that its rounding (8 below a score of 2^27 may be no fp32 number) has no effect.
    f4 o[RT][DT];
    float ref[RT], l[RT];
    auto ref_for = [](float top) __attribute__((always_inline)) {
        const float r = top - X::BIAS;
        return top - r > X::BIAS + 7.f ? top : r;  // (where it was rounded down by 8 or more P would not fit its type)
    };
#pragma unroll
    for (int t = 0; t < RT; t++) {
        ref[t] = -__builtin_inff(), l[t] = 0.f;
#pragma unroll
        for (int d = 0; d < DT; d++) o[t][d] = f4{0, 0, 0, 0};
    }
    // which of the new entries this lane's rows see: those up to `last`, or the bits of a tree node
    uint64_t bits[RT];
    int last[RT];
    if constexpr (OWN) {
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const int r = r0 + t * 16 + col;
            last[t] = r < sp.rows ? r / G : -1;
            bits[t] = a.mask && r < sp.rows ? a.mask[(int64_t)s * a.M + r / G] : 0;
        }
    }
    // (no branches: of entry j behind n, below 0 one of the sequence's own)
    const int tree = OWN && a.mask != nullptr;
    auto sees = [&](int j, int t) __attribute__((always_inline)) {
        const int in_tree = (int)(j < 0) | ((int)(j < a.M) & (int)(bits[t] >> (j & 63) & 1)), before = (int)(j <= last[t]);
        return (tree & in_tree) | ((tree ^ 1) & before);
    };

    // Non-finite values of new entries are taken out of the tile and added for the rows that see them (0 times infinity
    // would reach the others).
    auto sift = [&](int buf) __attribute__((always_inline)) {
        constexpr uint32_t E = TYPE == KV_F16 ? 0x7c00u : 0x7f80u;
        for (int i = 0; i < NLD; i++) {
            u4 *at = (u4 *)(lds + buf * 2 * TILE + TILE + (i * NT + tid) * 16);
            u4 v = *at;
            bool any = false;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t w = v[j];
                if ((w & E) == E) w &= 0xffff0000u, any = true;
                if ((w & (E << 16)) == (E << 16)) w &= 0xffffu, any = true;
                v[j] = w;
            }
            if (any) *at = v, bad[buf] = 1;
        }
    };

    // LDS bytes of this lane's operands. The permutation of a row's chunks touches bits of (4 u + g) and (2 d + vc) that
    // repeat every 16 chunks and is the same for rows 8 apart: a few addresses serve by constant offsets.
    constexpr int KA = STEPS < 4 ? STEPS : 4, VA = DT < 8 ? DT : 8;
    const int vr = (lane & 15) >> 2, vc = (lane & 3) >> 1, vb = (lane & 1) * 8;
    int ka_at[KA], va_at[VA];
#pragma unroll
    for (int u = 0; u < KA; u++) ka_at[u] = tile_at<D>(col, 4 * u + g);
#pragma unroll
    for (int d = 0; d < VA; d++) va_at[d] = TILE + tile_at<D>(4 * g + vr, 2 * d + vc) + vb;

    auto compute = [&](int64_t k0, int buf, int part) __attribute__((always_inline)) {
#pragma unroll 1
        for (int sub = part * (KB / 32 / ST) + wk; sub < (part + 1) * (KB / 32 / ST); sub += WK) {
            const int64_t key0 = k0 + sub * 32;
            if (key0 >= end) break;
            const int base = buf * 2 * TILE + sub * 32 * (D * 2);
            f4 z[RT][2];
#pragma unroll
            for (int t = 0; t < RT; t++) z[t][0] = z[t][1] = f4{0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < STEPS; u++) {
                v8 ka[2];
#pragma unroll
                for (int h = 0; h < 2; h++) ka[h] = *(const v8 *)(lds + base + ka_at[u % KA] + (u / KA) * 256 + h * 16 * (D * 2));
#pragma unroll
                for (int x = 0; x < X::LIMBS; x++)
#pragma unroll
                    for (int t = 0; t < RT; t++)
#pragma unroll
                        for (int h = 0; h < 2; h++) z[t][h] = X::mfma(ka[h], q[t][u][x], z[t][h]);
            }
            // (the operand loads two steps ahead of the products)
            __builtin_amdgcn_sched_group_barrier(0x100, STEPS < 2 ? 2 : 4, 0);
#pragma unroll
            for (int u = 0; u + 2 < STEPS; u++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 2 * RT * X::LIMBS, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, 4 * RT * X::LIMBS, 0);
            const bool partial = OWN ? key0 + 32 > n : key0 + 32 > end;
            if (partial) {
                const int there = (int)(end - key0 < 32 ? end - key0 : 32), j0 = OWN ? (int)(key0 - n) : 0;
#pragma unroll
                for (int t = 0; t < RT; t++)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const int at = (i >> 2) * 16 + 4 * g + (i & 3);
                        int on = (int)(at < there);
                        if constexpr (OWN) on &= sees(j0 + at, t);
                        z[t][i >> 2][i & 3] = on ? z[t][i >> 2][i & 3] : -__builtin_inff();
                    }
            }
            float top[RT];
            bool past = false;
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const f4 x = z[t][0], y = z[t][1];
                top[t] = c[t] * fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])));
                past |= top[t] - ref[t] > X::BIAS + 7.f;  // (a difference of near numbers is exact, a sum with 7 is not)
            }
            // the reference point moves only when a row's maximum passes it by 2^7 more (P then still fits its type)
            if (__any(past)) {
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    const float to = fmaxf(ref[t], ref_for(max_groups(top[t])));
                    const float keep = ref[t] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ref[t] - to);
                    ref[t] = to;
                    l[t] *= keep;
#pragma unroll
                    for (int d = 0; d < DT; d++) o[t][d] *= keep;
                }
            }
            v8 p[RT][X::LIMBS];
            float pf[RT][8];
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const float off = ref[t] == -__builtin_inff() ? 0.f : -ref[t];
#pragma unroll
                for (int i = 0; i < 8; i++) pf[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[t][i >> 2][i & 3], c[t], off));
                l[t] += ((pf[t][0] + pf[t][1]) + (pf[t][2] + pf[t][3])) + ((pf[t][4] + pf[t][5]) + (pf[t][6] + pf[t][7]));
                limbs<TYPE>(pf[t], p[t]);
            }
            // transposing loads: 16 lanes read 4 keys x 16 values, lane i gets value i of the four
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const char *at = lds + base + va_at[d % VA] + (d / VA) * 256;
                const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)at);
                const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(at + 16 * (D * 2)));
                const v8 va = __builtin_bit_cast(v8, (s8)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                for (int x = 0; x < X::LIMBS; x++)
#pragma unroll
                    for (int t = 0; t < RT; t++) o[t][d] = X::mfma(va, p[t][x], o[t][d]);
            }
            __builtin_amdgcn_sched_group_barrier(0x100, 6, 1);
#pragma unroll
            for (int d = 0; d + 3 < DT; d++) {
                __builtin_amdgcn_sched_group_barrier(0x008, RT * X::LIMBS, 1);
                __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, 3 * RT * X::LIMBS, 1);
            if constexpr (OWN) {
                if (k0 + KB > n && bad[buf]) {
                    for (int j = 0; j < 32; j++) {
                        const int64_t key = key0 + j;
                        if (key >= end) break;
#pragma unroll
                        for (int t = 0; t < RT; t++) {
                            float mine = 0.f;
#pragma unroll
                            for (int i = 0; i < 8; i++)
                                if ((i >> 2) == (j >> 4) && (i & 3) == (j & 3)) mine = pf[t][i];
                            const float w = __shfl(mine, ((j >> 2) & 3) * 16 + col);
                            const int on = sees((int)(key - n), t);
#pragma unroll
                            for (int d = 0; d < DT; d++)
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    const float v = (float)V[key * kstride + d * 16 + 4 * g + i];
                                    if (on && !(fabsf(v) < __builtin_inff())) o[t][d][i] += w * v;
                                }
                        }
                    }
                }
            }
        }
    };

    if (tid < 2) bad[tid] = 0;
    if (begin < end) {
#pragma unroll
        for (int part = 0; part < ST; part++) {
            if (part) fetch(begin, part);
            put(0, part);
        }
        fetch(begin + KB < end ? begin + KB : begin, 0);
    }
    int buf = 0;
    for (int64_t k0 = begin; k0 < end; k0 += KB, buf ^= 1) {
        __syncthreads();
        if constexpr (OWN) {
            if (k0 + KB > n) {
                sift(buf);
                __syncthreads();
            }
        }
        // (the last tiles' loads and stores of a tile that is not there repeat the first: no branch, but a range of one tile
        // waits for such a load before its products)
        const int64_t k1 = k0 + KB < end ? k0 + KB : begin, k2 = k0 + 2 * KB < end ? k0 + 2 * KB : begin;
#pragma unroll
        for (int part = 0; part < ST; part++) {
            put(buf ^ 1, part);
            if (part + 1 < ST) fetch(k1, part + 1);
            else fetch(k2, 0);
            if (r0 < sp.rows) compute(k0, buf, part);
        }
    }
    if constexpr (WK > 1) __syncthreads();
#pragma unroll
    for (int t = 0; t < RT; t++) l[t] = sum_groups(l[t]);

    const int64_t all_rows = (int64_t)a.n_seq * a.M * a.n_q, part = (int64_t)(sp.first + split) * all_rows;
    auto place = [&](int r) { return part + token(r) * a.n_q + hk * G + r % G; };
    if constexpr (WK == 1) {
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const int r = r0 + t * 16 + col;
            if (r < sp.rows) {
                const int64_t at = place(r);
                if (g == 0) ml[at] = float2{ref[t], l[t]};
#pragma unroll
                for (int d = 0; d < DT; d++) *(f4 *)(opart + at * D + d * 16 + 4 * g) = o[t][d];
            }
        }
    } else {
        // the waves of a row block that took different keys meet in LDS: [wave][row][value], 16-byte pieces permuted
        f4 *const meet = (f4 *)lds;
        constexpr int Q = D / 4;
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const int r = t * 16 + col;
            if (g == 0) wml[wave][r] = float2{ref[t], l[t]};
#pragma unroll
            for (int d = 0; d < DT; d++) meet[(wave * RT * 16 + r) * Q + ((d * 4 + g) ^ (r & 7))] = o[t][d];
        }
        __syncthreads();
        for (int i = tid; i < ROWS * Q; i += NT) {
            const int r = i / Q, ch = i % Q, w = r / (RT * 16), rr = r % (RT * 16), at_row = rb * ROWS + r;
            if (at_row >= sp.rows) break;
            float top = -__builtin_inff(), sum = 0.f;
#pragma unroll
            for (int x = 0; x < WK; x++) top = fmaxf(top, wml[w * WK + x][rr].x);
            f4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int x = 0; x < WK; x++) {
                const float2 e = wml[w * WK + x][rr];
                const float keep = e.x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(e.x - top);
                sum += keep * e.y;
                acc += keep * meet[((w * WK + x) * RT * 16 + rr) * Q + (ch ^ (rr & 7))];
            }
            const int64_t at = place(at_row);
            if (ch == 0) ml[at] = float2{top, sum};
            *(f4 *)(opart + at * D + ch * 4) = acc;
        }
    }
}

// The prefix's blocks, then the sequences' own: one launch, so that the short ones fill the gaps of the long.
template <int TYPE, int D, int PRE, int SELF>
__global__ __launch_bounds__(512) void attn_part_kernel(AttnArgs a, AttnSplit pre, AttnSplit own, int n_pre,
                                                      float *__restrict__ opart, float2 *__restrict__ ml) {
    typedef ShapeOf<D, PRE> P;
    typedef ShapeOf<D, SELF> S;
    constexpr int KB = P::KB > S::KB ? P::KB : S::KB;
    __shared__ __align__(16) char lds[4 * KB * D * 2];  // two of (K tile, V tile)
    __shared__ Shared sh;
    if ((int)blockIdx.x < n_pre) attn_part<TYPE, D, P, false>(a, pre, (int)blockIdx.x, lds, sh, opart, ml);
    else attn_part<TYPE, D, S, true>(a, own, (int)blockIdx.x - n_pre, lds, sh, opart, ml);
}

// Ranges of keys that a prefix and a sequence's own entries are cut into at most.
constexpr int MOST_PRE = 128, MOST_OWN = 64;

// The parts' results of a row, each times 2^(its reference - the largest), over their sum: W waves a row, each taking every W-th
// part, four loads in flight. Bound by reading the parts (256 rows of a tree, 256 wide, 64 parts: 67 MB). With W = 4 and 1
// (us, the whole call, 8 heads of D = 128): 16 query heads and 4 parts 10.4, 10.2, 16 parts 11.1, 12.8; 1024 and 4 25.3, 24.1,
// 16 31.7, 32.2: four from 9 parts on.
template <int D, int W> __global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, int parts, const float *__restrict__ opart,
                                                                              const float2 *__restrict__ ml) {
    constexpr int E = D / 64, ROWS = 4 / W, LANES = W * 64;
    __shared__ float weight[ROWS][MOST_PRE + MOST_OWN];
    __shared__ float4 red[4][64];
    __shared__ float tops[4], sums[4];
    typedef float ve __attribute__((ext_vector_type(E)));
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, slot = wave / W, ws = wave % W;
    const int64_t rows = (int64_t)a.n_seq * a.M * a.n_q;
    int64_t row = (int64_t)blockIdx.x * ROWS + slot;
    const bool real = row < rows;
    if (!real) row = rows - 1;
    const int64_t tok = row / a.n_q;
    const int h = (int)(row - tok * a.n_q), n = a.len[tok / a.M];
    const float *src = opart + row * D + lane * E;
    ve v[4];
    auto four = [&](int i) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = *(const ve *)(src + (int64_t)(i + j * W < parts ? i + j * W : parts - 1) * rows * D);
    };
    four(ws);  // (on their way while the weights are found)
    float top = -__builtin_inff(), sum = 0.f;
    for (int i = ws * 64 + lane; i < parts; i += LANES) top = fmaxf(top, ml[(int64_t)i * rows + row].x);
    top = wave_max(top);
    if constexpr (W > 1) {
        if (lane == 0) tops[wave] = top;
        __syncthreads();
        top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    }
    for (int i = ws * 64 + lane; i < parts; i += LANES) {
        const float2 e = ml[(int64_t)i * rows + row];
        const float keep = e.x == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(e.x - top);
        weight[slot][i] = keep;
        sum += keep * e.y;
    }
    sum = wave_sum(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if constexpr (W > 1) sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    ve acc = (ve)0.f;
    for (int i = ws; i < parts; i += 4 * W) {
        if (i != ws) four(i);
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i + j * W < parts) acc += weight[slot][i + j * W] * v[j];
    }
    if constexpr (W > 1) {
        *(ve *)&red[wave][lane] = acc;
        __syncthreads();
        if (wave) return;
        acc = (*(ve *)&red[0][lane] + *(ve *)&red[1][lane]) + (*(ve *)&red[2][lane] + *(ve *)&red[3][lane]);
    }
    if (!real || n < 0) return;
    if ((int64_t)n + a.M > a.capacity) acc = (ve)__builtin_nanf("");  // (its parts were not written)
    else acc = sum == 0.f ? (ve)0.f : acc / sum;
    *(ve *)(a.out + tok * a.ldo + (int64_t)h * D + lane * E) = acc;
}

// ---- launch shapes ----

// The shape for `rows` query rows that meet `keys` keys in each of `units` heads (of sequences), and its rows a block. Blocks
// of 32 rows are the quickest to finish, and where they are many take the fewest ranges of keys, whose results cost a pass of
// their own; blocks of 64 and 256 (D = 256: 64 and 128) read less LDS for a product. Measured over a prefix in 2 or 8 heads,
// rows / 4 sequences of one token and 4 query heads a key head, with 20 own entries each, whose workgroups (1024 rows, 8 heads:
// 2048) are in the times (us: blocks of 32, 64, 256; f16, D = 128): 256 rows, 4000 keys, 2 heads (2^21) 16.2, 19.6, 25.6; 512
// rows, 4000, 8 (2^24) 58.5, 57.5, 61.2; 1024, 4000, 8 (2^25) 105.5, 97.5, 99.3; 2048, 16000, 8 (2^28) 455, 361, 327; 2048,
// 1000, 2 (2^22) 51.6, 44.2, 52.0. Of sequences' own entries (D = 64, bf16): 16 heads of 256 rows, 2064 keys 19.7, -, 28.9; 128
// of 48 rows, 2012 keys 32.3, 25.9. D = 256 (blocks of 64, 128): 256 rows, 4000 keys, 2 heads (2^21) 25.6, 29.7; 16 heads of
// 256 rows, 2064 keys (2^23) 59.6, 50.2. With what 256 rows leave empty counted (f16, D = 128, 32000 keys, 8 heads; one
// sequence of 64 tokens, 16 and 32 of 5, 300 own entries each; blocks of 64, 256): 256 rows 135, 112, 320 rows 174, 202, 640
// rows 190, 172. Sizes between these were not measured. bf16 at D = 128 spills registers in blocks of 64: 1024 rows, 4000, 8
// 113, 117, 111.
int shape_for(const AttnArgs &a, int64_t rows, int64_t units, int64_t keys) {
    const double work = (double)rows * (double)units * (double)keys;
    if (a.head_dim == 256) return rows <= 64 || work <= 1 << 22 ? 1 : 2;
    const bool spills = a.head_dim == 128 && a.type == KV_BF16;
    if (rows <= (spills ? 64 : 32) || (rows <= 1024 && work <= 1 << 24 && (rows + 31) / 32 * units < 256)) return 0;
    const bool padded = (rows + 255) / 256 * 256 * 3 > rows * 4;
    return !spills && (rows <= 64 || work <= 3 << 24 || padded) ? 1 : 2;
}
int shape_rows(int D, int id) { return id == 0 ? 32 : id == 1 ? 64 : D == 256 ? 128 : 256; }

struct AttnPlan {
    AttnSplit pre, own;
    int parts, pre_shape, own_shape;
};

// One workgroup fills a CU. The sequences' own entries: ranges of 128 keys or more, up to 256 workgroups (5 tokens, 4 heads of
// 4 rows each, D = 128: 16 sequences of 4000 entries 29.5 us, 56.9 unsplit, 38.0 with up to 512; 4 of 200 12.7, 13.1, 21.3),
// half that beside a prefix. The prefix: as many ranges (of 128 keys or more) as fill the chip beside them, or once over where
// they are many. Half and all of the chip for the own entries (us, 8 heads of D = 128, 4 rows a token, 1024 to 4096 entries of
// capacity): 4 sequences of 5 tokens, 777 shared entries 14.4, 21.0; 8, 1500 17.7, 23.6; 9, 4099 25.7, 29.8; 16 of one token,
// 8000 23.5, 27.8; 16 of 5, 8000 55, 49. The host knows capacities, not lengths: a cache with room to spare gives its own
// entries ranges that are empty, and the prefix as many workgroups fewer. Ranges of 128 and of 64: one row a head over 777
// entries 10.6, 11.1, at D = 256 over 3000 14.8, 17.0.
AttnPlan plan_of(const AttnArgs &a) {
    AttnPlan p{};
    const int64_t G = a.n_q / a.n_kv, own_rows = a.M * G;
    p.own_shape = shape_for(a, own_rows, (int64_t)a.n_kv * a.n_seq, a.capacity);
    const int own_block = shape_rows(a.head_dim, p.own_shape);
    p.own.rows = (int)own_rows;
    p.own.blocks = (int)((own_rows + own_block - 1) / own_block);
    const int64_t units = (int64_t)p.own.blocks * a.n_kv * a.n_seq;
    int64_t splits = (a.P > 0 ? 128 : 256) / units;
    splits = splits < 1 ? 1 : splits > MOST_OWN ? MOST_OWN : splits;
    const int64_t most = (a.capacity + 127) / 128;
    p.own.splits = (int)(splits < most ? splits : most);
    p.pre_shape = p.own_shape;
    if (a.P > 0) {
        const int64_t rows = (int64_t)a.n_seq * own_rows;
        const int shape = shape_for(a, rows, a.n_kv, a.P);
        p.pre_shape = shape > p.own_shape ? shape : p.own_shape;
        const int block = shape_rows(a.head_dim, p.pre_shape);
        p.pre.rows = (int)rows;
        p.pre.blocks = (int)((rows + block - 1) / block);
        const int64_t beside = units * p.own.splits, room = beside <= 128 ? 256 - beside : 256;
        int64_t n = room / ((int64_t)p.pre.blocks * a.n_kv);
        n = n < 1 ? 1 : n > MOST_PRE ? MOST_PRE : n;
        const int64_t top = (a.P + 127) / 128;
        n = n < top ? n : top;
        p.pre.per = ((a.P + n - 1) / n + 31) / 32 * 32;
        p.pre.splits = (int)((a.P + p.pre.per - 1) / p.pre.per);
    }
    p.own.first = p.pre.splits;
    p.parts = p.pre.splits + p.own.splits;
    return p;
}

template <int TYPE, int D, int PRE, int SELF>
hipError_t launch_part(const AttnArgs &a, const AttnPlan &p, float *opart, float2 *ml, hipStream_t st) {
    const int64_t n_pre = a.P > 0 ? ((int64_t)p.pre.splits * a.n_kv + 7) / 8 * 8 * p.pre.blocks : 0;
    const int64_t grid = n_pre + (int64_t)p.own.splits * p.own.blocks * a.n_kv * a.n_seq;
    if (grid > 0x7fffffff) return hipErrorInvalidValue;
    attn_part_kernel<TYPE, D, PRE, SELF><<<(unsigned)grid, 512, 0, st>>>(a, p.pre, p.own, (int)n_pre, opart, ml);
    return hipGetLastError();
}

template <int TYPE, int D> hipError_t launch_all(const AttnArgs &a, const AttnPlan &p, void *ws, hipStream_t st) {
    const int64_t rows = (int64_t)a.n_seq * a.M * a.n_q;
    float2 *ml = (float2 *)ws;
    float *opart = (float *)((char *)ws + ((size_t)p.parts * rows * sizeof(float2) + 255) / 256 * 256);
    hipError_t e = hipErrorInvalidValue;
    const int shapes = p.pre_shape * 3 + p.own_shape;  // (own_shape <= pre_shape)
    if constexpr (D < 256) {
        if (shapes == 0) e = launch_part<TYPE, D, 0, 0>(a, p, opart, ml, st);
        if constexpr (!(D == 128 && TYPE == KV_BF16))
            if (shapes == 3) e = launch_part<TYPE, D, 1, 0>(a, p, opart, ml, st);
        if (shapes == 6) e = launch_part<TYPE, D, 2, 0>(a, p, opart, ml, st);
    }
    if constexpr (!(D == 128 && TYPE == KV_BF16)) {
        if (shapes == 4) e = launch_part<TYPE, D, 1, 1>(a, p, opart, ml, st);
        if (shapes == 7) e = launch_part<TYPE, D, 2, 1>(a, p, opart, ml, st);
    }
    if (shapes == 8) e = launch_part<TYPE, D, 2, 2>(a, p, opart, ml, st);
    if (e != hipSuccess) return e;
    if (p.parts > 8) attn_join_kernel<D, 4><<<(unsigned)rows, 256, 0, st>>>(a, p.parts, opart, ml);
    else attn_join_kernel<D, 1><<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(a, p.parts, opart, ml);
    return hipGetLastError();
}

}  // namespace

size_t attn_ws(const AttnArgs &a) {
    const AttnPlan p = plan_of(a);
    const size_t rows = (size_t)a.n_seq * a.M * a.n_q;
    return (p.parts * rows * sizeof(float2) + 255) / 256 * 256 + p.parts * rows * a.head_dim * sizeof(float);
}

hipError_t launch_attn(const AttnArgs &a, void *ws, hipStream_t st) {
    const AttnPlan p = plan_of(a);
    if (a.type == KV_F16)
        return a.head_dim == 64    ? launch_all<KV_F16, 64>(a, p, ws, st)
               : a.head_dim == 128 ? launch_all<KV_F16, 128>(a, p, ws, st)
                                   : launch_all<KV_F16, 256>(a, p, ws, st);
    return a.head_dim == 64    ? launch_all<KV_BF16, 64>(a, p, ws, st)
           : a.head_dim == 128 ? launch_all<KV_BF16, 128>(a, p, ws, st)
                               : launch_all<KV_BF16, 256>(a, p, ws, st);
}
