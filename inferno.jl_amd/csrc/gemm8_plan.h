// Which kernel of gemm8.hip takes a product of 8-bit codes. Plain C++ for the host,
// so that the choice can be looked at without a GPU.
#pragma once
#include <stdint.h>

#include <initializer_list>

#define GEMM8_KB 128  // bytes of K that a stage holds: a line of each row

// Which kernel, and into how many parts K goes: the one whose time comes out shortest. A launch is rounds of workgroups. A
// round takes `fill` for its first loads, for each stage `alone` where it leaves most of the chip's memory paths to few
// workgroups and `full` where it fills the chip, and the time of its results, by a CU's rate or by the chip's. (us, fitted to
// 60 products of 1 to 4096 tokens, 17 to 24576 channels, K 128 to 12288; there the choice is mostly within 5% of the best of
// these kernels, at worst 13% behind it.)
struct Gemm8Shape {
    int tile, at_once;
    double fill, alone, full;
    bool late;  // (nears `full` with the square of the round's part)
};
constexpr Gemm8Shape gemm8_shapes[] = {
    {64, 512, 1.2, 0.18, 0.39, false},   // 9 places of 8 KiB, two workgroups a CU
    {128, 256, 2.0, 0.36, 0.56, true},   // 9 places of 16 KiB
    {128, 512, 1.2, 0.50, 1.09, false},  // 5 places of 16 KiB, two workgroups a CU
    {256, 256, 5.0, 0.95, 1.60, false},  // 5 places of 32 KiB
};
struct Gemm8Plan {
    int shape, parts;  // shape -1: gemm8_few
};
inline Gemm8Plan gemm8_plan(int M, int N, int K, int accum) {
    const double weights = 1.0 + (double)N * K / 5.0e6;  // reading them, at 5 TB/s
    const int64_t few_wgs = (int64_t)((N + 15) / 16) * ((M + 15) / 16);
    // a CU takes in 98 GB/s; weights that several workgroups take come more slowly (a launch holds 2^32 threads)
    const double a_cu = (few_wgs > 256 ? (double)few_wgs : 256.0) / 256.0;
    const double few_us = 2.5 + a_cu * (0.2 + (16.0 + (M < 16 ? M : 16)) * K / 98e3);
    const double few_weights = weights + (M > 16 ? 0.7 * a_cu : 0.0);
    Gemm8Plan best{-1, 1};
    double best_us = few_wgs > 1 << 24 ? 1e9 : few_us > few_weights ? few_us : few_weights;
    if (best_us <= weights) return best;  // (no other is faster than reading the weights)
    for (int i = 0; i < 4; i++)
        for (const int parts : {1, 2, 3, 4, 6, 8}) {
            const Gemm8Shape &s = gemm8_shapes[i];
            const int64_t wgs = (int64_t)((M + s.tile - 1) / s.tile) * ((N + s.tile - 1) / s.tile) * parts;
            const int stages = ((K + GEMM8_KB - 1) / GEMM8_KB + parts - 1) / parts;
            const double y = 4.0 * M * ((N + 3) / 4 * 4), touched = accum ? 2.0 : 1.0;
            if (parts > 1 && (stages < 8 || parts * y > (double)(64 << 20))) break;
            const double bytes = 4.0 * s.tile * s.tile * (parts > 1 ? 1.0 : touched);
            const double one = bytes / 60e3, all = s.at_once * bytes / 5.0e6;
            auto round = [&](double part) {
                const double results = part < 1 ? one + (all > one ? all - one : 0.0) * part : all;
                return s.fill + results + stages * (s.alone + (s.full - s.alone) * (s.late ? part * part : part));
            };
            const double rest = (double)(wgs % s.at_once) / s.at_once;
            double us = 2.0 + (double)(wgs / s.at_once) * round(1.0) + (rest > 0 ? round(rest) : 0.0);
            if (us < weights) us = weights;
            if (parts > 1) us += 2.5 + y * (parts + touched) / 8.0e6;  // (the sums read again, and a launch more)
            if (us < best_us) best_us = us, best = Gemm8Plan{i, parts};
        }
    return best;
}
