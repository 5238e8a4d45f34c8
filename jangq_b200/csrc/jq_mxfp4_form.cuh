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

// The form with the shortest estimated time (us on B200; K stages of 256 codes).  One CTA per tile: 2 once, then per wave of tiles 2.2
// and 0.205 + 0.00085 tn per stage; a split of K adds 0.7 + 0.011 tn.  CTA pairs: 7.2 once, then 0.04 + 0.0015 tn per stage and round.
// Measured: 16 rows 4096x4096 7.6 unsplit, 6.5 by 2, 6.0 by 4, 10.2 in pairs; 128 rows 2048x8192 12.7, 11.0, 9.0, 15.4; 256 rows
// 4096x4096 9.0, 9.0, 15.4, 12.3; 1024 rows 4096x4096 16.0, 30.6, 53.5, 14.3; 4096 rows 14336x4096 181 unsplit, 96 to 98 in pairs.
inline Gemm4Form gemm4_form(int64_t M, int64_t N, int64_t nblk, int64_t sms) {
    const int64_t stages = (nblk + 7) / 8;
    Gemm4Form f = {0, 0, 0, 0};
    double best = 1e300;
    const auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    {
        const int64_t tn = up(up(M, up(M, 128)), 16) * 16, mt = up(M, tn), tiles = mt * up(N, 128);
        for (int k : {1, 2, 4}) {
            if (mt >= 65536 || (k > 1 && stages < 4 * k)) continue;
            // clusters at once: one of four stays within a GPC (32 on 148 SMs, not 37)
            const int64_t slots = std::max<int64_t>(1, k == 4 ? sms * 8 / 37 : sms / k);
            const double wave = 2.2 + (double)up(stages, k) * (0.205 + 0.00085 * (double)tn) + (k > 1 ? 0.7 + 0.011 * (double)tn : 0.0);
            const double t = 2.0 + (double)up(tiles, slots) * wave;
            if (t < best) { best = t; f = {k, (int)tn, mt, tiles}; }
        }
    }
    {
        const int64_t least = up(M, 256), slots = std::max<int64_t>(1, sms / 2);
        for (int64_t nt = least; nt <= least + 3; ++nt) {
            const int64_t tn = up(up(M, nt), 16) * 16, mt = up(M, tn), tiles = mt * up(N, 256);
            const double t = 7.2 + (double)up(tiles, slots) * (double)stages * (0.04 + 0.0015 * (double)tn);
            if (t < best) { best = t; f = {0, (int)tn, mt, tiles}; }
        }
    }
    return f;
}

}  // namespace jq
