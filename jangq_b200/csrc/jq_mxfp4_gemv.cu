// Mat-vecs over MXFP4 weights with 16-bit activations: y[m, n] = sum_k x[m, k] * deq(w)[n, k] for up to 16 rows, and the
// same for the (token, slot) pairs of routed experts.
//
// Bound: the weights' 17/32 byte each from HBM on paper, and the issue of their expansion: integer instructions run at half
// rate, and eight codes put together by permutes or shifts take 28 cycles of a scheduler, eight cycles with the conversion
// instruction to f16 pairs.  So the operands of the warp MMAs (m16n8k16, the weights as the 16-row operand) are f16: the codes'
// plain values, and activations scaled per block of 32 by a power of two (none for f16 activations, which are exact; a
// bf16 one is exact unless it is below 2^-29 of the largest of its block, and off by 2^-39 of that at most).  Each block's
// sums, 32 products, leave the MMA in f32 and are multiplied by the two powers of two on their way into the row's sum, the
// activations' first: it is held 2^10 smaller and the weight's 2^10 larger, so that the first product, up to 2^136 for the largest
// activations, stays finite; it is exact at the lower end too, a multiple of 2^-144.
//   up to 2 rows   the MMA's eight columns are four blocks of two tokens: a lane reads one whole block, its activations stand
//                  in that block's column alone, and one multiplication per two columns and row puts in the scales
//   up to 8 rows   the columns are tokens, block after block; more rows take further launches
// One CTA of 16 warps per SM takes an even share of the row tiles (16 x RG weight rows of one matrix); the warps are RG row
// groups of KS warps that share the rows in stretches of 256 codes.  Every warp keeps its own ring of stretches in shared
// memory, codes and scale bytes copied asynchronously across the tiles' ends, so the weights stream without a pause.  A warp
// goes through a batch of tiles with one stretch of k, whose activations stay in registers, and then with its next one; its
// sums stand in shared memory until the CTA meets at the end of the batch to add them, KS to a row, in an order that does not
// change.
//
// Measured (bf16, copies in turn beyond L2): one row of 14336 x 4096 11.0 us = 2.8 TB/s, 11008 x 4096 9.3, 4096 x 4096 6.2,
// 2048 x 2048 4.1; eight rows 16.7, 14.4, 9.5, 5.8.  The large ones are bound by issue (half of the scheduler's slots, no pipe
// above a third) in four warps per scheduler, the small ones by some 3 us of launch, staging and the meeting at the end.
#include <algorithm>

#include "jq_launch.cuh"
#include "jq_mxfp4.cuh"

namespace jq {

struct MxGemvArgs {
    const uint16_t* x;
    const uint8_t* codes;
    const uint8_t* scales;
    uint16_t* y;
    int64_t ldx, ldy, N;
    int64_t scale_bytes;                 // of all matrices
    int nblk;                            // blocks of 32 codes per row
    int M;
    int ks_log2;                         // KS = 1 << ks_log2 warps share a row
    uint32_t tiles, items;               // row tiles of one matrix, and of all pairs
    // pairs of routed experts: row p of y is x[p / x_div] . w[pair_expert[p] - expert_base], items p * tiles + tile
    const int32_t* pair_expert;
    int x_div, num_experts, expert_base;
};

constexpr int MXV_WARPS = 16, MXV_UNIT = 8, MXV_STAGES = 3;            // UNIT: blocks of a stretch
// a stretch of 16 rows: 128 bytes of codes each, and the three aligned words around its eight scale bytes (16 bytes apart)
constexpr int MXV_CODES = 16 * 128, MXV_STAGE = MXV_CODES + 16 * 16;
constexpr int MXV_RING = MXV_WARPS * MXV_STAGES * MXV_STAGE;
constexpr int MXV_MAX_SMEM = 226 * 1024;
constexpr int MXV_EXTRA = 128;                                          // a row of zeros, and what tokens past the last read
constexpr int MXV_PAD = 32;                                             // halves between activation rows, past whole stretches
constexpr int MXV_SHIFT = 10;                                           // powers of two between the activations' scales and the weights'

// COLS: one or two tokens (the columns are blocks); else up to eight
template <bool COLS> __host__ __device__ constexpr int mxv_tokens() { return COLS ? 2 : 8; }
template <bool COLS> __host__ __device__ constexpr int mxv_batch() { return COLS ? 8 : 4; }      // tiles between two meetings of the CTA
template <bool COLS> __host__ __device__ constexpr int mxv_part() { return mxv_batch<COLS>() * MXV_WARPS * mxv_tokens<COLS>() * 17 * 4; }
// bytes of one activation row in shared memory, with its blocks' powers of two where it has them
__host__ __device__ __forceinline__ int mxv_row_bytes(int nunit, bool scaled) {
    return (nunit * MXV_UNIT * 32 + MXV_PAD) * 2 + (scaled ? nunit * MXV_UNIT * 4 : 0);
}
// a row that always fits beside the ring and the largest partial sums
constexpr int MXV_MAX_K = 36864;
static_assert(MXV_RING + mxv_part<false>() + MXV_EXTRA + (MXV_MAX_K + MXV_PAD) * 2 + MXV_MAX_K / 8 <= MXV_MAX_SMEM, "one row");
// The 16-byte chunk of block b of a row: rows 128 bytes apart, so that eight rows read together, or two with four blocks
// each, fall into eight bank groups.
__device__ __forceinline__ int mxv_chunk(int b, int row) { return b ^ ((row & 1) << 2 | (row >> 1 & 3)); }

// 2^(byte - 127) of byte I of a word; the other form also of bytes 0 (a subnormal) and 255 (not a number)
template <int I> __device__ __forceinline__ float mx_scale(uint32_t w) {
    return __uint_as_float((I < 3 ? w << (23 - 8 * I) : w >> 1) & 0x7F800000u);
}
template <int I> __device__ __forceinline__ float mx_scale_any(uint32_t w) {
    const uint32_t f = __float_as_uint(mx_scale<I>(w));
    return __uint_as_float(f == 0u ? 0x00400000u : (f == 0x7F800000u ? 0x7FC00000u : f));
}
// The four of a word, times 2^SHIFT where fast.  fast: none of the warp's bytes leaves the normal numbers then (0 and 255 without a
// shift; with one a zero byte is in range, and those from 255 - SHIFT on are not).
template <int SHIFT> __device__ __forceinline__ void mx_scales4(uint32_t w, bool fast, float (&f)[4]) {
    if (fast) {
        w += SHIFT * 0x01010101u;
        f[0] = mx_scale<0>(w); f[1] = mx_scale<1>(w); f[2] = mx_scale<2>(w); f[3] = mx_scale<3>(w);
    } else {
        f[0] = mx_scale_any<0>(w); f[1] = mx_scale_any<1>(w); f[2] = mx_scale_any<2>(w); f[3] = mx_scale_any<3>(w);
    }
}
// bit 7 of every byte that is out of the fast form's range
template <int SHIFT> __device__ __forceinline__ uint32_t mx_slow_bytes(uint32_t w) {
    const uint32_t low = w & 0x7F7F7F7Fu, high = (low + (SHIFT + 1) * 0x01010101u) & w;
    return (SHIFT > 0 ? high : high | ~((low + 0x7F7F7F7Fu) | w)) & 0x80808080u;
}
// One activation row into shared memory as f16, zeros from K to the end of its last stretch.  bf16: block b is multiplied by
// 2^-e and scales[b * stride] = 2^(e - MXV_SHIFT), e such that the block's largest is in [2^14, 2^15), but not below -109: from
// there on every bf16 number, a multiple of 2^-133, is one of f16's smallest step.  A block with an infinity or a NaN keeps those as
// they are and nothing else: the products are the same.
// Threads 4i .. 4i + 3 share a block.
template <typename AT>
__device__ __forceinline__ void stage_row(const uint16_t* __restrict__ src, int nblk, int nunit, uint16_t* dst, float* scales, int stride,
                                          int tid, int threads) {
    for (int c = tid; c < nunit * MXV_UNIT * 4; c += threads) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (c < nblk * 4) v = *reinterpret_cast<const uint4*>(src + c * 8);
        if constexpr (umma_fmt<AT>() == 1u) {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) m = max(m, max(w[i] & 0x7FFFu, w[i] >> 16 & 0x7FFFu));
            const uint32_t four = 0xFu << (threadIdx.x & 28);
            m = max(m, __shfl_xor_sync(four, m, 1));
            m = max(m, __shfl_xor_sync(four, m, 2));
            const int ex = (int)(m >> 7), e = ex == 255 ? 0 : max(ex - 141, -109);
            const float mult = __uint_as_float((uint32_t)(127 - e) << 23);
            uint32_t o[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float lo = Act<__nv_bfloat16>::lo_f32(w[i]), hi = Act<__nv_bfloat16>::hi_f32(w[i]);
                if (ex == 255) {
                    lo = fabsf(lo) < INFINITY ? 0.f : lo;
                    hi = fabsf(hi) < INFINITY ? 0.f : hi;
                }
                o[i] = Act<__half>::pack_hi(lo * mult, hi * mult);
            }
            v = make_uint4(o[0], o[1], o[2], o[3]);
            if ((c & 3) == 0) scales[(c >> 2) * stride] = __uint_as_float((uint32_t)(127 - MXV_SHIFT + e) << 23);
        }
        *reinterpret_cast<uint4*>(dst + c * 8) = v;
    }
}

// The next stretch that a warp copies: tile `item` (of all pairs'), stretch u of its rows.  The tiles of a batch take turns with
// one stretch before the next.
template <bool COLS, bool GATHER> struct MxvAhead {
    uint32_t item, base, stop;           // of the batch [base, stop)
    int u, left;                         // left: N - 1 - first of the 16 weight rows; rows past it repeat the last one
    bool none;                           // no expert of the bank takes the pair
    int bytes;                           // of scales from there to the end of the array, at most 2^30
    const uint8_t *codes, *scales;       // of the first of the 16 rows
    __device__ __forceinline__ uint32_t batch_end(const MxGemvArgs& a, uint32_t end) const {
        return min(base + mxv_batch<COLS>(), GATHER ? min(end, (base / a.tiles + 1) * a.tiles) : end);
    }
    __device__ __forceinline__ void enter(const MxGemvArgs& a, int rg, int rows) {
        uint32_t tile = item;
        int64_t row = 0;
        none = false;
        if constexpr (GATHER) {
            const uint32_t p = item / a.tiles;
            tile = item - p * a.tiles;
            const int e = a.pair_expert[p] - a.expert_base;
            none = e < 0 || e >= a.num_experts;
            row = none ? 0 : e * a.N;
        }
        const int64_t n0 = (int64_t)tile * rows + rg * 16;
        left = (int)(a.N - 1 - n0);
        codes = a.codes + (row + n0) * a.nblk * 16;
        scales = a.scales + (row + n0) * a.nblk;
        bytes = (int)min(a.scale_bytes - (row + n0) * a.nblk, (int64_t)1 << 30);
    }
    __device__ __forceinline__ void next(const MxGemvArgs& a, uint32_t end, int nunit, int ks, int KS, int rg, int rows) {
        if (++item < stop) {
            left -= rows;
            codes += (int64_t)rows * a.nblk * 16;
            scales += (int64_t)rows * a.nblk;
            bytes = (int)min(a.scale_bytes - (scales - a.scales), (int64_t)1 << 30);
            return;
        }
        if ((u += KS) >= nunit) {
            u = ks;
            base = stop;
            stop = batch_end(a, end);
        }
        item = base;
        if (item < end) enter(a, rg, rows);
    }
};

// COLS: up to two rows (or one row per pair), else up to eight
template <typename AT, bool COLS, bool GATHER>
__global__ void __launch_bounds__(32 * MXV_WARPS, 1)
mxfp4_gemv_kernel(const MxGemvArgs a) {
    using H = Act<__half>;
    extern __shared__ __align__(16) uint8_t mxv_smem[];
    constexpr bool SCALED = umma_fmt<AT>() == 1u;
    constexpr int TOK = mxv_tokens<COLS>(), SHIFT = SCALED ? MXV_SHIFT : 0;
    overlap_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int KS = 1 << a.ks_log2, ks = warp & (KS - 1), rg = warp >> a.ks_log2, rows = 16 * (MXV_WARPS >> a.ks_log2);
    const int nunit = (a.nblk + MXV_UNIT - 1) / MXV_UNIT, M = GATHER ? 1 : a.M;
    uint8_t* ring = mxv_smem + warp * MXV_STAGES * MXV_STAGE;
    float* part = reinterpret_cast<float*>(mxv_smem + MXV_RING);
    uint8_t* zero = mxv_smem + MXV_RING + mxv_part<COLS>();              // 64 bytes that the lanes of no token read
    const int xpitch = nunit * MXV_UNIT * 32 + MXV_PAD, nb = nunit * MXV_UNIT;
    uint16_t* sx = reinterpret_cast<uint16_t*>(zero + 64);
    float* se = reinterpret_cast<float*>(sx + M * xpitch);                // [row][block], or [block][row] with columns of tokens
    const int crow = a.nblk * 16;
    const uint32_t begin = (uint32_t)((uint64_t)a.items * blockIdx.x / gridDim.x), end = (uint32_t)((uint64_t)a.items * (blockIdx.x + 1) / gridDim.x);

    const bool three = a.nblk & 3;
    // one stretch into a slot of the ring; codes of zero past the row's end and without an expert
    MxvAhead<COLS, GATHER> ahead{};
    const uint32_t cdst = smem_u32(ring) + (uint32_t)((lane >> 3) * 128), sdst = smem_u32(ring) + MXV_CODES;
    auto copy = [&](int slot) {
        if (ahead.item < end) {
            const int c0 = ahead.u * MXV_UNIT + (lane & 7);
            const bool in = c0 < a.nblk && !(GATHER && ahead.none);
            const uint8_t* src = ahead.codes + (in ? c0 * 16 : 0);
            const uint32_t at = (uint32_t)(slot * MXV_STAGE);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int r = (lane >> 3) + 4 * c;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                             ::"r"(cdst + at + (uint32_t)(c * 512 + mxv_chunk(lane & 7, r) * 16)),
                               "l"(src + (int64_t)min(r, ahead.left) * crow), "r"(in ? 16 : 0) : "memory");
            }
            // the aligned words around a row's eight bytes (two where rows are whole words); the array's last one may be short
            const int off = min(lane & 15, ahead.left) * a.nblk + ahead.u * MXV_UNIT + (lane >> 4) * 4;
            const int low = (int)(reinterpret_cast<uintptr_t>(ahead.scales) + off) & 3, have = ahead.bytes - (off - low);
            const uint8_t* word = ahead.scales + (off - low);
            const uint32_t wdst = sdst + at + (uint32_t)((lane & 15) * 16 + (lane >> 4) * 4);
            if (have > 0)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(wdst), "l"(word), "r"(min(have, 4)) : "memory");
            if (three && lane < 16 && have > 8)
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(wdst + 8), "l"(word + 8), "r"(min(have - 8, 4)) : "memory");
            ahead.next(a, end, nunit, ks, KS, rg, rows);
        }
        cp_async_commit();
    };
    ahead.base = ahead.item = begin;
    ahead.u = ks;
    ahead.stop = ahead.batch_end(a, end);
    ahead.enter(a, rg, rows);
#pragma unroll
    for (int i = 0; i < MXV_STAGES - 1; ++i) copy(i);
    if (threadIdx.x < 16) reinterpret_cast<uint32_t*>(zero)[threadIdx.x] = 0u;
    uint32_t xrow = 0;                                     // GATHER: the row in shared memory
    if constexpr (GATHER) {
        xrow = begin / a.tiles / (uint32_t)a.x_div;
        stage_row<AT>(a.x + (int64_t)xrow * a.ldx, a.nblk, nunit, sx, se, 1, threadIdx.x, 32 * MXV_WARPS);
    } else {
        // a group of warps per row; a row's threads are whole warps, so four of them share a block
        const int per = MXV_WARPS / M;
        for (int m = warp / per; m < M; m += MXV_WARPS / per)
            stage_row<AT>(a.x + m * a.ldx, a.nblk, nunit, sx + m * xpitch, COLS ? se + m * nb : se + m, COLS ? 1 : M,
                          (warp % per) * 32 + lane, per * 32);
    }
    __syncthreads();

    // where this lane's activations are, byte offsets masked to nothing for a lane of no token
    const int tok = COLS ? g >> 2 : g;
    const bool live = tok < M && (!COLS || (g & 3) == t);
    const uint32_t mask = live ? 0xFFFFFFFFu : 0u;
    const uint8_t* xl = live ? reinterpret_cast<const uint8_t*>(sx + tok * xpitch) : zero;
    const float* sel = COLS ? se + min(t >> 1, M - 1) * nb + 2 * (t & 1) : se + 2 * t;
    // offset of this lane's codes, and of the scale bytes of its rows, in a slot
    const uint8_t* codes0 = ring + g * 128;
    const uint32_t pick = t & 1 ? 0x7632u : 0x5410u;       // this lane's two of four blocks, in two rows' words

    int slot = 0;
    for (uint32_t item = begin; item < end;) {
        // a batch of tiles, of one pair
        const uint32_t pair = GATHER ? item / a.tiles : 0u, first = item - pair * a.tiles;
        const int batch = (int)min((uint32_t)mxv_batch<COLS>(), (GATHER ? min(end, (pair + 1) * a.tiles) : end) - item);
        int64_t mat = 0;                                   // first row of the pair's matrix
        bool none = false;                                 // no expert: zeros, whatever the activations and scales are
        if constexpr (GATHER) {
            const int e = a.pair_expert[pair] - a.expert_base;
            none = e < 0 || e >= a.num_experts;
            mat = none ? 0 : e * a.N;
        }
        // where row g's bytes stand in the aligned words around them: tiles and row groups are 16 rows apart, g + 8 is 8
        const int sh = (int)((mat + g) * a.nblk & 3) * 8;
        for (int u = ks; u < nunit; u += KS) {
            const int b0 = u * MXV_UNIT;
            uint4 xv[8];                                   // the stretch's activations: (half, word), or blocks
            float2 xe[COLS ? 2 : 8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                xv[i] = *reinterpret_cast<const uint4*>(
                    xl + (COLS ? ((uint32_t)((b0 + 4 * (i >> 2) + t) * 64) & mask) + (i & 3) * 16 : (uint32_t)((b0 + i) * 64 + t * 16) & mask));
            if constexpr (SCALED) {
#pragma unroll
                for (int i = 0; i < (COLS ? 2 : 8); ++i) {
                    // tokens past the last: whatever stands there, in columns that are not stored
                    if constexpr (COLS) xe[i] = *reinterpret_cast<const float2*>(sel + b0 + 4 * i);
                    else xe[i] = make_float2(sel[(b0 + i) * M], sel[(b0 + i) * M + 1]);
                }
            }
            for (int ti = 0; ti < batch; ++ti) {
                cp_async_wait<MXV_STAGES - 2>();
                __syncwarp();                              // this stretch is there, the slot of the last one is free
                copy(slot == 0 ? MXV_STAGES - 1 : slot - 1);
                const uint8_t* st = codes0 + slot * MXV_STAGE;
                // the eight scale bytes of rows g and g + 8
                const uint4 z0 = *reinterpret_cast<const uint4*>(ring + slot * MXV_STAGE + MXV_CODES + g * 16);
                const uint4 z1 = *reinterpret_cast<const uint4*>(ring + slot * MXV_STAGE + MXV_CODES + (g + 8) * 16);
                uint32_t p0[2] = {__funnelshift_r(z0.x, z0.y, sh), __funnelshift_r(z0.y, z0.z, sh)};
                uint32_t p1[2] = {__funnelshift_r(z1.x, z1.y, sh), __funnelshift_r(z1.y, z1.z, sh)};
                if (b0 + MXV_UNIT > a.nblk) {              // past the row's end: the next row's bytes, or none; codes are zero
                    const int n = a.nblk - b0;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int k = n - 4 * i;
                        const uint32_t keep = k >= 4 ? 0xFFFFFFFFu : k <= 0 ? 0u : (1u << (8 * k)) - 1u;
                        p0[i] = (p0[i] & keep) | (0x7F7F7F7Fu & ~keep);
                        p1[i] = (p1[i] & keep) | (0x7F7F7F7Fu & ~keep);
                    }
                }
                // a byte among them that needs the other form, whose sums are 2^SHIFT smaller (and whole multiples of 2^-139, far
                // below the smallest numbers of the results): the four lanes of a row pair look at a word each
                const uint32_t mine = t & 2 ? (t & 1 ? p1[1] : p1[0]) : (t & 1 ? p0[1] : p0[0]);
                const bool fast = !__any_sync(0xFFFFFFFFu, mx_slow_bytes<SHIFT>(mine));
                float* out = part + (ti * MXV_WARPS + warp) * (TOK * 17);
                if constexpr (COLS) {
                    float d[2][4], v0 = 0.f, v1 = 0.f;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {          // four blocks: lane t has block t of them
                        const uint4 w0 = *reinterpret_cast<const uint4*>(st + mxv_chunk(4 * h + t, g) * 16);
                        const uint4 w1 = *reinterpret_cast<const uint4*>(st + 8 * 128 + mxv_chunk(4 * h + t, g + 8) * 16);
                        const uint32_t q0[4] = {w0.x, w0.y, w0.z, w0.w}, q1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            uint32_t e0[4], e1[4];
                            mx_values8(q0[j], e0);
                            mx_values8(q1[j], e1);
                            const uint32_t fa[4] = {e0[0], e1[0], e0[1], e1[1]}, fb[4] = {e0[2], e1[2], e0[3], e1[3]};
                            const uint4 x4 = xv[4 * h + j];
                            if (j == 0) H::mma0(d[h], fa, x4.x, x4.y);
                            else H::mma(d[h], fa, x4.x, x4.y);
                            H::mma(d[h], fb, x4.z, x4.w);
                        }
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        // columns 2t, 2t + 1: blocks 2 (t & 1), + 1 of the four, token t / 2
                        if constexpr (SCALED) {
                            d[h][0] *= xe[h].x; d[h][1] *= xe[h].y; d[h][2] *= xe[h].x; d[h][3] *= xe[h].y;
                        }
                        float f[4];                        // rows g and g + 8 of the two blocks
                        mx_scales4<SHIFT>(prmt(p0[h], p1[h], pick), fast, f);
                        v0 = fmaf(d[h][1], f[1], fmaf(d[h][0], f[0], v0));
                        v1 = fmaf(d[h][3], f[3], fmaf(d[h][2], f[2], v1));
                    }
                    if (SCALED && !fast) { v0 *= (float)(1 << SHIFT); v1 *= (float)(1 << SHIFT); }
                    // the two column pairs of a token
                    v0 += __shfl_xor_sync(0xFFFFFFFFu, v0, 1);
                    v1 += __shfl_xor_sync(0xFFFFFFFFu, v1, 1);
                    if ((t & 1) == 0) {
                        float* o = out + (t >> 1) * 17 + g;
                        o[0] = u == ks ? v0 : o[0] + v0;
                        o[8] = u == ks ? v1 : o[8] + v1;
                    }
                } else {
                    float acc[4] = {0.f, 0.f, 0.f, 0.f}, f0[MXV_UNIT], f1[MXV_UNIT];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float f[4];
                        mx_scales4<SHIFT>(p0[i], fast, f);
                        f0[4 * i] = f[0]; f0[4 * i + 1] = f[1]; f0[4 * i + 2] = f[2]; f0[4 * i + 3] = f[3];
                        mx_scales4<SHIFT>(p1[i], fast, f);
                        f1[4 * i] = f[0]; f1[4 * i + 1] = f[1]; f1[4 * i + 2] = f[2]; f1[4 * i + 3] = f[3];
                    }
#pragma unroll
                    for (int b = 0; b < MXV_UNIT; ++b) {   // lane t has eight codes of block b
                        uint32_t e0[4], e1[4];
                        mx_values8(*reinterpret_cast<const uint32_t*>(st + mxv_chunk(b, g) * 16 + t * 4), e0);
                        mx_values8(*reinterpret_cast<const uint32_t*>(st + 8 * 128 + mxv_chunk(b, g + 8) * 16 + t * 4), e1);
                        const uint32_t fa[4] = {e0[0], e1[0], e0[1], e1[1]}, fb[4] = {e0[2], e1[2], e0[3], e1[3]};
                        float d[4];
                        H::mma0(d, fa, xv[b].x, xv[b].y);
                        H::mma(d, fb, xv[b].z, xv[b].w);
                        if constexpr (SCALED) {
                            d[0] *= xe[b].x; d[1] *= xe[b].y; d[2] *= xe[b].x; d[3] *= xe[b].y;
                        }
                        acc[0] = fmaf(d[0], f0[b], acc[0]);
                        acc[1] = fmaf(d[1], f0[b], acc[1]);
                        acc[2] = fmaf(d[2], f1[b], acc[2]);
                        acc[3] = fmaf(d[3], f1[b], acc[3]);
                    }
                    if (SCALED && !fast) { acc[0] *= (float)(1 << SHIFT); acc[1] *= (float)(1 << SHIFT); acc[2] *= (float)(1 << SHIFT); acc[3] *= (float)(1 << SHIFT); }
                    // rows g, g + 8 of tokens 2t, 2t + 1
                    float* o = out + 2 * t * 17 + g;
                    o[0] = u == ks ? acc[0] : o[0] + acc[0];
                    o[17] = u == ks ? acc[1] : o[17] + acc[1];
                    o[8] = u == ks ? acc[2] : o[8] + acc[2];
                    o[25] = u == ks ? acc[3] : o[25] + acc[3];
                }
                if (++slot == MXV_STAGES) slot = 0;
            }
        }
        __syncthreads();
        // rows of the batch x tokens, the row's KS sums in warp order
        const int nrow = batch * rows;
        for (int q = threadIdx.x; q < nrow * M; q += 32 * MXV_WARPS) {
            const int m = q / nrow, r = q - m * nrow, ti = r / rows, n = r - ti * rows;
            const float* src = part + (ti * MXV_WARPS + (n >> 4) * KS) * (TOK * 17) + m * 17 + (n & 15);
            float v = 0.f;
#pragma unroll 4
            for (int w = 0; w < KS; ++w) v += src[w * (TOK * 17)];
            const int64_t col = (int64_t)first * rows + r;
            if (col < a.N) a.y[(int64_t)(GATHER ? pair : (uint32_t)m) * a.ldy + col] = Act<AT>::from_f32(none ? 0.f : v);
        }
        item += (uint32_t)batch;
        if (item >= end) break;
        if constexpr (GATHER)                              // the next pair's row; everyone is done with this one's
            if (item / a.tiles / (uint32_t)a.x_div != xrow) {
                xrow = item / a.tiles / (uint32_t)a.x_div;
                stage_row<AT>(a.x + (int64_t)xrow * a.ldx, a.nblk, nunit, sx, se, 1, threadIdx.x, 32 * MXV_WARPS);
            }
        __syncthreads();
    }
    cp_async_wait<0>();
}

template <typename AT, bool COLS, bool GATHER>
static int launch_mxv(const MxGemvArgs& a, int row_bytes, cudaStream_t st) {
    auto kernel = mxfp4_gemv_kernel<AT, COLS, GATHER>;
    const size_t smem = (size_t)MXV_RING + mxv_part<COLS>() + MXV_EXTRA + (size_t)a.M * row_bytes;
    static bool attr_done[64] = {};
    int dev = 0;
    JQ_CUDA_OK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        JQ_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MXV_MAX_SMEM));
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    JQ_CUDA_OK(launch_overlapped(kernel, dim3((unsigned)std::min<uint32_t>(a.items, (uint32_t)sm_count())), 32 * MXV_WARPS, smem, st, a));
    return JQ_OK;
}

static int mx_gemv_common(const void* x, int x_dtype, int64_t ldx, const uint32_t* codes, const uint8_t* scales, int64_t N,
                          int64_t K, void* y, int64_t ldy, MxGemvArgs& a) {
    int rc = check_mxfp4_shape(N, K);
    if (rc != JQ_OK) return rc;
    JQ_REQUIRE(K <= MXV_MAX_K, JQ_EUNSUPPORTED, "the mat-vec takes rows of up to %d activations, got %lld", MXV_MAX_K, (long long)K);
    JQ_REQUIRE(x_dtype == JQ_BF16 || x_dtype == JQ_F16, JQ_EINVAL, "activations must be bf16 or f16");
    JQ_REQUIRE(K > 0, JQ_EINVAL, "K must be positive");
    JQ_REQUIRE(x && codes && scales && y, JQ_EINVAL, "null pointer");
    JQ_REQUIRE(aligned(x, 16) && ldx % 8 == 0 && ldx >= K, JQ_EINVAL, "x must be 16-byte aligned with ldx %% 8 == 0");
    JQ_REQUIRE(aligned(codes, 16) && aligned(scales, 4), JQ_EINVAL, "codes must be 16-byte aligned, scales 4-byte");
    JQ_REQUIRE(ldy >= N, JQ_EINVAL, "ldy too small");
    a.x = (const uint16_t*)x; a.codes = (const uint8_t*)codes; a.scales = scales; a.y = (uint16_t*)y;
    a.ldx = ldx; a.ldy = ldy; a.N = N; a.nblk = (int)(K / MX_BLOCK);
    a.scale_bytes = N * a.nblk;
    // as many warps on a row as it has stretches, up to all of them
    const int nunit = (a.nblk + MXV_UNIT - 1) / MXV_UNIT;
    a.ks_log2 = 0;
    while (a.ks_log2 < 4 && (2 << a.ks_log2) <= nunit) ++a.ks_log2;
    const int64_t rows = 16 * (MXV_WARPS >> a.ks_log2);
    a.tiles = a.items = (uint32_t)((N + rows - 1) / rows);
    a.pair_expert = nullptr; a.x_div = 1; a.num_experts = 0; a.expert_base = 0;
    return JQ_OK;
}

}  // namespace jq

extern "C" {

int jq_mxfp4_gemv(const void* x, int x_dtype, int64_t M, int64_t ldx, const uint32_t* codes, const uint8_t* scales, int64_t N,
                  int64_t K, void* y, int64_t ldy, jq_stream_t stream) {
    using namespace jq;
    JQ_REQUIRE(M >= 0 && M <= 16, JQ_EINVAL, "jq_mxfp4_gemv takes up to 16 rows, got %lld", (long long)M);
    if (M == 0 || N == 0) return check_mxfp4_shape(N, K);
    MxGemvArgs a;
    int rc = mx_gemv_common(x, x_dtype, ldx, codes, scales, N, K, y, ldy, a);
    if (rc != JQ_OK) return rc;
    // as many rows per launch as fit beside the ring, in even parts
    const int row_bytes = mxv_row_bytes((a.nblk + MXV_UNIT - 1) / MXV_UNIT, x_dtype == JQ_BF16);
    const int64_t fit = std::min<int64_t>(8, (MXV_MAX_SMEM - MXV_RING - mxv_part<false>() - MXV_EXTRA) / row_bytes);
    const int64_t parts = (M + fit - 1) / fit;
    for (int64_t i = 0; i < parts && rc == JQ_OK; ++i) {
        const int64_t m0 = i * M / parts;
        a.M = (int)((i + 1) * M / parts - m0);
        a.x = (const uint16_t*)x + m0 * ldx;
        a.y = (uint16_t*)y + m0 * ldy;
        JQ_DISPATCH_DTYPE16(x_dtype, AT, rc = a.M <= 2 ? launch_mxv<AT, true, false>(a, row_bytes, (cudaStream_t)stream)
                                                       : launch_mxv<AT, false, false>(a, row_bytes, (cudaStream_t)stream))
    }
    return rc;
}

int jq_mxfp4_gather_gemv(const void* x, int x_dtype, int64_t ldx, int x_div, const int32_t* pair_expert, int64_t P,
                         const uint32_t* codes, const uint8_t* scales, int num_experts, int expert_base, int64_t N, int64_t K,
                         void* y, int64_t ldy, jq_stream_t stream) {
    using namespace jq;
    JQ_REQUIRE(P >= 0 && x_div >= 1 && num_experts >= 1, JQ_EINVAL, "P >= 0, x_div >= 1 and num_experts >= 1");
    JQ_REQUIRE(P <= 65535, JQ_EUNSUPPORTED, "jq_mxfp4_gather_gemv takes up to 65535 pairs, got %lld", (long long)P);
    if (P == 0 || N == 0) return check_mxfp4_shape(N, K);
    MxGemvArgs a;
    int rc = mx_gemv_common(x, x_dtype, ldx, codes, scales, N, K, y, ldy, a);
    if (rc != JQ_OK) return rc;
    JQ_REQUIRE(pair_expert, JQ_EINVAL, "null pointer");
    a.M = 1;
    a.pair_expert = pair_expert; a.x_div = x_div; a.num_experts = num_experts; a.expert_base = expert_base;
    a.scale_bytes *= num_experts;
    JQ_REQUIRE((int64_t)a.tiles * P < (1ll << 31), JQ_EUNSUPPORTED, "too many rows for one launch");
    a.items = a.tiles * (uint32_t)P;
    const int row_bytes = mxv_row_bytes((a.nblk + MXV_UNIT - 1) / MXV_UNIT, x_dtype == JQ_BF16);
    JQ_DISPATCH_DTYPE16(x_dtype, AT, return launch_mxv<AT, true, true>(a, row_bytes, (cudaStream_t)stream))
    return JQ_OK;
}

}  // extern "C"
