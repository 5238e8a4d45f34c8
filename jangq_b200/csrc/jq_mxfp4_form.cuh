// Which form of the product of two MXFP4 operands takes a size (host code without CUDA; jq_mxfp4_gemm4.cu has the kernels).
#pragma once

#include <algorithm>
#include <cstdint>

namespace jq {

struct Gemm4Form {
    int ks;                  // CTAs that split K of a tile of 128 weight rows, 0: CTA pairs on 256
    int tn;                  // activation rows per tile, a multiple of 16
    int64_t mt, tiles;       // tiles along M, and in all
};

// The form with the shortest estimated time (us on B200; K stages of 256 codes, weights from HBM).
//   one CTA per tile   0.7 once, per wave of tiles 3.3 and 0.28 + 0.0001 tn per stage; a split of K adds 0.1 + 0.018 tn; the weights
//                      at 3.4 TB/s at best
//   CTA pairs          7.0 once, then 0.275 + 0.00065 tn per stage and round; the weights at 4.25 TB/s at best
// Up to 128 activation rows a tile holds them all, so both forms read a weight once and a pair saves nothing.
// Measured (us, one CTA, split by 2, by 4, pairs): 16 rows 4096x4096 7.9 6.4 6.2 11.2, 14336x8192 16.0 20.7 27.1 20.8; 128 rows
// 2048x8192 12.7 11.0 8.9 15.7; 256 rows 4096x4096 9.0 9.1 15.3 12.2, 4096x14336 19.0 15.5 23.2 25.2; 512 rows 14336x8192 47.6 72 111
// 34.8; 1024 rows 4096x4096 16.0 30.7 53.3 14.2; 4096 rows 14336x4096 210 - - 100.  Over 361 sizes (1 .. 4096 rows, weights of
// 512x1024 .. 28672x8192) the form taken is 0.3 % slower than the best one in the mean, 12 % at most (1 row of 512x1024).
inline Gemm4Form gemm4_form(int64_t M, int64_t N, int64_t nblk, int64_t sms) {
    const int64_t stages = (nblk + 7) / 8;
    const double mbytes = 17e-6 * (double)N * (double)nblk;
    Gemm4Form f = {0, 0, 0, 0};
    double best = 1e300;
    const auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    {
        const int64_t tn = up(up(M, up(M, 128)), 16) * 16, mt = up(M, tn), tiles = mt * up(N, 128);
        for (int k : {1, 2, 4}) {
            if (mt >= 65536 || (k > 1 && stages < 4 * k)) continue;
            // clusters at once: one of four stays within a GPC (32 on 148 SMs, not 37)
            const int64_t slots = std::max<int64_t>(1, k == 4 ? sms * 8 / 37 : sms / k);
            const double wave = 3.3 + (double)up(stages, k) * (0.28 + 0.0001 * (double)tn) + (k > 1 ? 0.1 + 0.018 * (double)tn : 0.0);
            const double t = 0.7 + std::max((double)up(tiles, slots) * wave, mbytes * 0.295);
            if (t < best) { best = t; f = {k, (int)tn, mt, tiles}; }
        }
    }
    if (M > 128) {
        const int64_t least = up(M, 256), slots = std::max<int64_t>(1, sms / 2);
        for (int64_t nt = least; nt <= least + 3; ++nt) {
            const int64_t tn = up(up(M, nt), 16) * 16, mt = up(M, tn), tiles = mt * up(N, 256);
            const double t = 7.0 + std::max((double)up(tiles, slots) * (double)stages * (0.275 + 0.00065 * (double)tn), mbytes * 0.235);
            if (t < best) { best = t; f = {0, (int)tn, mt, tiles}; }
        }
    }
    return f;
}

}  // namespace jq
