// Product of two MXFP4 operands on the block-scaled tensor-core path: Y[M, N] = deq(X)[M, K] . deq(W)[N, K]^T.
//
// Bound: tensor throughput of kind::mxf4 for many rows (four times the 16-bit rate, so the copies from L2 are the next
// wall), the packed weights from HBM for few.  Codes go from global memory to the MMA as they are: weight rows are the A
// operand, activation rows the B operand (a short batch costs no padded work), 256 codes of each per stage in 128-byte-
// swizzled rows.  The scale bytes of a stage are laid out by the loader warps as the 32-lane pattern that tcgen05.cp copies
// to tensor memory (row r of a 128-row group: lane r % 32, column r / 32, one byte per block of 32), and an MMA of 64 codes
// names its two bytes by the scale id.  Products and sums are f32 in the tensor core.
//   warp 0        TMA producer of both code tiles
//   warp 1        allocates the tensor memory, copies the scales there and issues the MMAs (one elected lane)
//   warps 2 .. 7  scale loaders, four rows per lane and four stages at a time
//   epilogue      warps 4 .. 7 once the loading is done, or warps 8 .. 15 of the form for CTA pairs
// Every mbarrier wait is bounded; a wait that runs out sets the library's status word and the CTA leaves through the
// common exit (tensor memory is always released).
#include <algorithm>

#include "jq_mxfp4.cuh"
#include "jq_mxfp4_form.cuh"

namespace jq {

struct Gemm4Args {
    const uint8_t *wscales, *xscales;
    void* y;
    int64_t M, N, ldy;
    int nblk;                // blocks of 32 per row
    int tn;                  // activation rows per tile, a multiple of 16
    int mt, tiles;           // CTA pairs: tiles along M, and in all (activation rows vary fastest)
    int vec;                 // every row's scales are whole 16-byte vectors
    int y_pair_ok, y_vec_ok;         // rows of y are 4-byte, 16-byte aligned
    int* status;
};

constexpr int G4_LOADERS = 6;                     // warps 2 .. 7
constexpr int G4_GS = 4;                          // stages of a scale group: 32 scale bytes per row
constexpr int G4_A = 128 * 128;                   // bytes of 128 rows of 256 codes
constexpr int G4_NCOLS = 512;

// A and B e2m1, scales ue8m0, both K-major, M = 128, dense K = 64; N at run time, scale ids added per MMA
// CG CTAs share the product: 128 rows of A each
template <int CG> __device__ __forceinline__ uint32_t umma_idesc_mxf4(int n) {
    return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(CG * 128 >> 4) << 24);
}
template <int CG>
__device__ __forceinline__ void umma_mxf4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                          uint32_t sfb, uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}
// 32 rows of 16 bytes -> 4 columns of 32 lanes, repeated in the four lane quarters (of both CTAs, from their own memory)
template <int CG> __device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
    if constexpr (CG == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// descriptor of scale rows: no swizzle, 8-row groups of 128 bytes back to back; the low half is the address >> 4
constexpr uint32_t ROWS16_HI = (128u >> 4) | (1u << 14);
__device__ __forceinline__ uint64_t rows16_join(uint32_t lo) { return ((uint64_t)ROWS16_HI << 32) | lo; }

// 32 scale bytes of a row from block b on (past the row's end: 1.0).  `total`: bytes of the whole array, which starts at a
// 4-byte boundary; rows that are not whole vectors are read as the aligned words around them and shifted.
__device__ __forceinline__ void load_scales32(const uint8_t* base, int64_t total, int64_t row_at, int b, int nblk, bool vec,
                                              uint32_t (&v)[8]) {
    constexpr uint32_t ONE = 0x7F7F7F7Fu;
    if (vec) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint4 q = make_uint4(ONE, ONE, ONE, ONE);
            if (b + 16 * h < nblk) q = __ldg(reinterpret_cast<const uint4*>(base + row_at + b + 16 * h));
            v[4 * h] = q.x; v[4 * h + 1] = q.y; v[4 * h + 2] = q.z; v[4 * h + 3] = q.w;
        }
        return;
    }
    const int64_t at = row_at + b, w0 = at & ~(int64_t)3;
    const int sh = (int)(at & 3) * 8, left = nblk - b;                 // bytes of the row left
    uint32_t w[9];
#pragma unroll
    for (int i = 0; i < 9; ++i) {
        const int64_t p = w0 + 4 * i;
        w[i] = 0;
        if (4 * i < left + 3) {                                        // words past the row are not read
            if (p + 4 <= total) w[i] = __ldg(reinterpret_cast<const uint32_t*>(base + p));
            else for (int j = 0; j < 3; ++j) if (p + j < total) w[i] |= (uint32_t)base[p + j] << (8 * j);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int n = left - 4 * i;
        const uint32_t mask = n >= 4 ? 0xFFFFFFFFu : (n <= 0 ? 0u : (1u << (8 * n)) - 1u);
        v[i] = (__funnelshift_r(w[i], w[i + 1], sh) & mask) | (ONE & ~mask);
    }
}

// One stage's MMAs: its scales (from descriptor `sc` on: two chunks of the weights', then GROUPS per chunk of the
// activations') to tensor memory at `sf`, then four steps of 64 codes.  A warp alone on its scheduler issues an instruction
// every few cycles, so what is computed here per stage is kept to single additions: with it spread out a stage took 330 ns
// to issue, more than its MMAs run.
template <int CG, int GROUPS>
__device__ __forceinline__ void mma_stage(uint32_t dcol, uint32_t sf, uint32_t sc, uint32_t ad, uint32_t bd, uint32_t idesc,
                                          uint32_t accumulate) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        tmem_cp_scales<CG>(sf + c * 4, rows16_join(sc + c * 32));
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
            tmem_cp_scales<CG>(sf + 8 + (c * GROUPS + g) * 4, rows16_join(sc + 64 + (c * GROUPS + g) * 32));
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)                                           // scale bytes 0, 1 or 2, 3 of the column
        umma_mxf4<CG>(dcol, umma_desc_join(ad + k * 2), umma_desc_join(bd + k * 2), k & 1 ? idesc | (2u << 4) | (2u << 29) : idesc,
                      sf + (k >> 1) * 4, sf + 8 + (k >> 1) * GROUPS * 4, k > 0 ? 1u : accumulate);
}

// The scales of one 128-row group (the weight rows, or 128 of the activation rows) on their way to tensor memory: a lane
// holds rows lane + 32 j, whose bytes of a chunk of four blocks stand side by side in the 16 bytes of that lane.  A warp reads
// a group of four stages at once (eight chunks) and has the time of as many groups as there are sets of loader warps for
// it: every set fills its own two slots.  With one set and a slot ahead,
// the latency of the reads set the pace of the kernel.
struct ScaleGroup {
    int64_t row[4];
    uint32_t v[4][8];
    __device__ __forceinline__ void init(int64_t r0, int64_t last, int nblk, int lane) {
#pragma unroll
        for (int j = 0; j < 4; ++j) row[j] = min(r0 + lane + 32 * j, last) * nblk;
    }
    // from block b on, a multiple of 16
    __device__ __forceinline__ void fetch(const uint8_t* base, int64_t total, int b, int nblk, bool vec) {
#pragma unroll
        for (int j = 0; j < 4; ++j) load_scales32(base, total, row[j], b, nblk, vec, v[j]);
    }
    // chunk c of stage i: to slot + i * STAGE + c * GAP
    template <int STAGE, int GAP> __device__ __forceinline__ void store(uint8_t* slot, int lane) const {
#pragma unroll
        for (int i = 0; i < G4_GS; ++i)
#pragma unroll
            for (int c = 0; c < 2; ++c)
                *reinterpret_cast<uint4*>(slot + i * STAGE + c * GAP + lane * 16) =
                    make_uint4(v[0][2 * i + c], v[1][2 * i + c], v[2][2 * i + c], v[3][2 * i + c]);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
};

// 32 accumulator columns (activation rows of y from yb on, `rows` of them valid) of weight row nn per lane
template <typename OT>
__device__ __forceinline__ void store_tile32(const Gemm4Args& a, const uint32_t (&v)[32], OT* yb, int rows, int64_t nn, bool pairs,
                                             int lane) {
    if constexpr (sizeof(OT) == 2) {
        if (pairs) {
            // neighbouring lanes swap halves: an even lane stores columns (n, n+1) of the even rows, an odd lane (n-1, n) of
            // the odd ones, 4 bytes each
            const bool odd = lane & 1;
            OT* yl = yb + (odd ? a.ldy : 0) + (nn & ~1ll);
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
                const float keep = __uint_as_float(odd ? v[j + 1] : v[j]);
                const float got = __uint_as_float(__shfl_xor_sync(0xFFFFFFFFu, odd ? v[j] : v[j + 1], 1));
                const uint32_t pk = odd ? Act<OT>::pack_hi(got, keep) : Act<OT>::pack_hi(keep, got);
                if (j + (odd ? 1 : 0) < rows) *reinterpret_cast<uint32_t*>(yl + j * a.ldy) = pk;
            }
            return;
        }
    }
    if (nn < a.N) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (j < rows) yb[j * a.ldy + nn] = Elt<OT>::from_f32(__uint_as_float(v[j]));
    }
}

// ---- tiles of 128 weight rows x up to 128 activation rows, one per CTA ----------------------------------------
// KS: CTAs of a cluster (along blockIdx.z) that split K where the tiles would leave most SMs idle: each leaves its sums as
// float32 in its (by then idle) shared memory; after a cluster barrier CTA r adds and stores the activation rows of its share,
// in rank order.  Both cluster barriers are reached by every thread on every path.
constexpr int G4S_RA = 5, G4S_SF = 2 * 1024, G4S_THREADS = 256, G4S_DCOLS = 128, G4S_SFCOLS = 16, G4S_SETS = 3, G4S_SLOTS = 2 * G4S_SETS;
constexpr size_t G4S_SMEM = 1024 + (size_t)G4S_RA * 2 * G4_A + G4S_SLOTS * G4_GS * G4S_SF + (2 * G4S_RA + 2 * G4S_SLOTS + 1) * 8 + 16;
static_assert(G4S_SMEM <= 227 * 1024, "shared memory of one CTA");
static_assert(G4S_DCOLS + 2 * G4_GS * G4S_SFCOLS <= G4_NCOLS, "tensor memory");

template <typename OT, int KS>
__global__ void __launch_bounds__(G4S_THREADS, 1)
mxfp4_gemm4_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Gemm4Args a) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sA = smem, *sB = sA + G4S_RA * G4_A, *sS = sB + G4S_RA * G4_A;
    uint64_t* full = reinterpret_cast<uint64_t*>(sS + G4S_SLOTS * G4_GS * G4S_SF);
    uint64_t* empty = full + G4S_RA;
    uint64_t* sfull = empty + G4S_RA;                      // slots of scale groups
    uint64_t* sempty = sfull + G4S_SLOTS;
    uint64_t* accfull = sempty + G4S_SLOTS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accfull + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t n0 = (int64_t)blockIdx.x * 128, m0 = (int64_t)blockIdx.y * a.tn;
    const int rows = (int)min((int64_t)a.tn, a.M - m0);
    // this CTA's stages [st0, st0 + nst): all, or its share of a split K, from an even one on (scales are read by 16 bytes)
    const int all = (a.nblk + 7) / 8, rank = KS > 1 ? (int)blockIdx.z : 0;
    const int st0 = rank * all / KS & ~1, nst = (rank == KS - 1 ? all : (rank + 1) * all / KS & ~1) - st0;

    if (threadIdx.x == 0) {
        for (int i = 0; i < G4S_RA; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
        for (int i = 0; i < G4S_SLOTS; ++i) { mbar_init(sfull + i, G4_LOADERS / G4S_SETS); mbar_init(sempty + i, 1); }
        mbar_init(accfull, 1);
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc(tmem_slot, G4_NCOLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    bool ok = true;

    // the producer and the issuer are one thread each, which alone learns of a wait that ran out
    if (warp == 0) {
        if (elect_one()) {
            int s = 0;
            uint32_t ph = 1u;
            const uint32_t bytes = (uint32_t)(G4_A + a.tn * 128);
            for (int i = 0; i < nst && ok; ++i) {
                ok = ts_wait(empty + s, ph);
                if (!ok) break;
                mbar_expect_tx(full + s, bytes);                              // parts outside the matrices read as zeros
                tma_load_2d(sA + s * G4_A, &wmap, (st0 + i) * 128, (int)n0, full + s);
                tma_load_2d(sB + s * G4_A, &xmap, (st0 + i) * 128, (int)m0, full + s);
                if (++s == G4S_RA) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            const uint32_t idesc = umma_idesc_mxf4<1>(a.tn), sc0 = smem_u32(sS) >> 4;
            const uint32_t a_lo = umma_desc_sw128_lo(smem_u32(sA)), b_lo = umma_desc_sw128_lo(smem_u32(sB));
            int s = 0;
            uint32_t ph = 0u, slot = 0u, sph = 0u;
            for (int i0 = 0; i0 < nst && ok; i0 += G4_GS) {
                ok = ts_wait(sfull + slot, sph);
#pragma unroll
                for (int j = 0; j < G4_GS; ++j) {
                    if (!ok || i0 + j >= nst) break;
                    ok = ts_wait(full + s, ph);
                    if (!ok) break;
                    tc_fence_after();
                    mma_stage<1, 1>(tmem_base, tmem_base + G4S_DCOLS + ((slot & 1u) * G4_GS + j) * G4S_SFCOLS,
                                    sc0 + (slot * G4_GS + j) * (G4S_SF >> 4), a_lo + (uint32_t)s * (G4_A >> 4),
                                    b_lo + (uint32_t)s * (G4_A >> 4), idesc, (uint32_t)(i0 + j));
                    umma_commit(empty + s);
                    if (++s == G4S_RA) { s = 0; ph ^= 1u; }
                }
                umma_commit(sempty + slot);
                if (++slot == G4S_SLOTS) { slot = 0u; sph ^= 1u; }
            }
            if (ok) umma_commit(accfull);
        }
    } else {
        // warps (2, 3), (4, 5), (6, 7): weight and activation rows, every third group of stages
        const int ngrp = (nst + G4_GS - 1) / G4_GS, set = (warp - 2) >> 1, part = warp & 1;
        const uint8_t* base = part ? a.xscales : a.wscales;
        const int64_t count = part ? a.M : a.N;
        ScaleGroup sg;
        sg.init(part ? m0 : n0, count - 1, a.nblk, lane);
        uint32_t ph = 1u;
        int slot = set;
        if (set < ngrp) sg.fetch(base, count * a.nblk, st0 * 8 + set * 32, a.nblk, a.vec);
        for (int g = set; g < ngrp; g += G4S_SETS) {
            ok = __all_sync(0xFFFFFFFFu, ts_wait(sempty + slot, ph));
            if (!ok) break;
            sg.store<G4S_SF, 512>(sS + slot * G4_GS * G4S_SF + part * 1024, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive(sfull + slot);
            if ((slot += G4S_SETS) >= G4S_SLOTS) { slot = set; ph ^= 1u; }
            if (g + G4S_SETS < ngrp) sg.fetch(base, count * a.nblk, st0 * 8 + (g + G4S_SETS) * 32, a.nblk, a.vec);
        }
        if (warp >= 4) {
            if (ok) ok = __all_sync(0xFFFFFFFFu, ts_wait(accfull, 0));
            if (ok) {
                tc_fence_after();
                const int quarter = warp & 3;
                const uint32_t src = tmem_base + ((uint32_t)(quarter * 32) << 16);
                OT* y = reinterpret_cast<OT*>(a.y) + m0 * a.ldy;
#pragma unroll 1
                for (int c0 = 0; c0 < rows; c0 += 32) {
                    uint32_t v[32];
                    tmem_ld32(src + (uint32_t)c0, v);
                    if constexpr (KS > 1) {
                        float* out = reinterpret_cast<float*>(smem) + c0 * 128 + quarter * 32 + lane;
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (c0 + j < rows) out[j * 128] = __uint_as_float(v[j]);
                        continue;
                    }
                    store_tile32<OT>(a, v, y + c0 * a.ldy, rows - c0, n0 + quarter * 32 + lane, a.y_pair_ok && n0 + 128 <= a.N, lane);
                }
            }
        }
    }
    __syncwarp();
    if constexpr (KS > 1) {
        static_assert(128 * 128 * 4 <= G4S_RA * 2 * G4_A, "staged sums fit");
        ts_cluster_sync();                               // the staged sums are complete
        const int t0 = rank * rows / KS, t1 = (rank + 1) * rows / KS;
        for (int q = threadIdx.x + t0 * 32; q < t1 * 32; q += G4S_THREADS) {        // four neighbouring weight rows
            const int tok = q >> 5, nl = (q & 31) * 4;
            const float* src = reinterpret_cast<const float*>(smem) + tok * 128 + nl;
            float4 f = ld_cluster_f32x4(src, 0);
#pragma unroll
            for (int r = 1; r < KS; ++r) {
                const float4 o = ld_cluster_f32x4(src, (uint32_t)r);
                f.x += o.x; f.y += o.y; f.z += o.z; f.w += o.w;
            }
            OT* yp = reinterpret_cast<OT*>(a.y) + (m0 + tok) * a.ldy + n0 + nl;
            if (a.y_vec_ok && n0 + nl + 4 <= a.N) {
                if constexpr (sizeof(OT) == 4) *reinterpret_cast<float4*>(yp) = f;
                else *reinterpret_cast<uint2*>(yp) = make_uint2(Act<OT>::pack_hi(f.x, f.y), Act<OT>::pack_hi(f.z, f.w));
                continue;
            }
            const float fv[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n0 + nl + j < a.N) yp[j] = Elt<OT>::from_f32(fv[j]);
        }
        ts_cluster_sync();                               // every CTA keeps its shared memory until all have read it
    }
    if (!ok) atomicOr(a.status, JQ_STATUS_LOCAL_WAIT);
    tc_fence_before();
    const int gave_up = __syncthreads_or(ok ? 0 : 1);
    if (warp == 1) {
        // after a wait that gave up, copies and MMAs of this CTA may still be in flight: give them a millisecond
        // to land before the tensor memory goes back and the CTA's shared memory is reused
        if (gave_up)
            for (int i = 0; i < 1000; ++i) __nanosleep(1000);
        tc_fence_after();
        tmem_dealloc(tmem_base, G4_NCOLS);
    }
}

// ---- more rows: CTA pairs walk tiles of 256 weight rows x up to 256 activation rows ---------------------------
// Each CTA copies its 128 weight rows and half of the activation rows; the MMAs of the first CTA (cta_group::2) read both
// halves from both CTAs' shared memory, so a code byte is copied from L2 half as often as with one CTA per tile -- those
// copies are the bound: tiles of 224 rows with two whole accumulators were slower (115 us for 4096 rows x 14336 x 4096; this form 96 to 98 = 4.9 PFLOP/s, 12.8 TB/s out of L2).
// Tensor memory holds two accumulators of 256 columns that share 48: the epilogue warps read those first, and the next
// tile's MMAs run into the other one while they take and store the rest (with a single accumulator the MMAs stood still for
// 1.7 of 7.4 us per tile).  The remaining 48 columns are the scales of two stages: a stage's are copied once the MMAs of the
// stage before the last are done.
//   full[s], sfull   in the first CTA: the code bytes of both CTAs; the scale loaders of both
//   empty[s], sempty, accfull   in each CTA: the MMAs' commits
//   accempty   in the first CTA, once per tile: the epilogue warps of both have read the tile before and the shared columns
constexpr int G4P_RA = 5, G4P_TN = 256, G4P_SF = 3 * 1024, G4P_THREADS = 512, G4P_SFCOLS = 24, G4P_EPI = 8;
constexpr int G4P_SETS = 2, G4P_SLOTS = 2 * G4P_SETS, G4P_SHARE = 48, G4P_D1 = G4P_TN - G4P_SHARE, G4P_DCOLS = G4P_D1 + G4P_TN;
constexpr int G4P_STORE = G4P_RA * 2 * G4_A + G4P_SLOTS * G4_GS * G4P_SF;          // 2 KB per epilogue warp
constexpr size_t G4P_SMEM = 1024 + (size_t)G4P_STORE + G4P_EPI * 2048 + (2 * G4P_RA + 2 * G4P_SLOTS + 3) * 8 + 16;
static_assert(G4P_SMEM <= 227 * 1024, "shared memory of one CTA");
static_assert(G4P_DCOLS + 2 * G4P_SFCOLS <= G4_NCOLS, "tensor memory");

// the address in the shared memory of the pair's first CTA
__device__ __forceinline__ uint32_t in_first_cta(const void* p) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(0));
    return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// For warps that only read tensor memory.  Their reads are over (tcgen05.wait::ld), fence::before_thread_sync and the __syncwarp
// put them before lane 0's arrive, and the issuer's fence::after_thread_sync puts the MMAs behind its wait; no write of these
// warps is read there, so nothing is to be released (the releasing form takes a microsecond).
__device__ __forceinline__ void mbar_arrive_cluster_relaxed(uint32_t addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// a copy into this CTA's shared memory whose bytes count on a barrier of the pair's first CTA
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// arrive on the barrier at this offset in both CTAs once the MMAs issued so far have completed
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(smem_u32(bar)), "h"((uint16_t)3)
                 : "memory");
}
// ts_wait that acquires what the other CTA released (a fence after the wait took most of a microsecond, every stage)
__device__ __forceinline__ bool pair_wait(uint64_t* bar, uint32_t parity) {
    const uint32_t addr = smem_u32(bar);
    unsigned long long t0 = 0;
    for (uint32_t i = 0;; ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(addr), "r"(parity), "r"(20000u)
            : "memory");
        if (done) return true;
        const unsigned long long now = wall_ns();
        if (t0 == 0) t0 = now;
        else if (i >= 4096u && now - t0 > MBAR_WAIT_NS) return false;
    }
}

template <typename OT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(G4P_THREADS, 1)
mxfp4_gemm4_pair_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Gemm4Args a) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sA = smem, *sB = sA + G4P_RA * G4_A, *sS = sB + G4P_RA * G4_A;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + G4P_STORE + G4P_EPI * 2048);
    uint64_t* empty = full + G4P_RA;
    uint64_t* sfull = empty + G4P_RA;
    uint64_t* sempty = sfull + G4P_SLOTS;
    uint64_t* accfull = sempty + G4P_SLOTS;
    uint64_t* accempty = accfull + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accempty + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x & 1;                       // clusters are pairs of neighbouring blocks
    const int nst = (a.nblk + 7) / 8, half = a.tn / 2;
    const uint32_t mt = (uint32_t)a.mt, tiles = (uint32_t)a.tiles, first = blockIdx.x >> 1, step = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int i = 0; i < G4P_RA; ++i) { mbar_init(full + i, 1); mbar_init(empty + i, 1); }
        for (int i = 0; i < G4P_SLOTS; ++i) { mbar_init(sfull + i, 2 * G4_LOADERS / G4P_SETS); mbar_init(sempty + i, 1); }
        for (int i = 0; i < 2; ++i) mbar_init(accfull + i, 1);
        mbar_init(accempty, 2 * G4P_EPI);
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(G4_NCOLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    ts_cluster_sync();                                     // the other CTA's barriers and tensor memory are there
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    bool ok = true;

    if (warp == 0) {
        // ---------------- TMA producer: one thread ----------------
        if (elect_one()) {
            int s = 0;
            uint32_t ph = 1u;
            const uint32_t bytes = (uint32_t)(2 * (G4_A + half * 128)), bars = in_first_cta(full);
            for (uint32_t tile = first; tile < tiles && ok; tile += step) {
                const int n0 = (int)(tile / mt * 256u) + rank * 128, m0 = (int)(tile % mt * (uint32_t)a.tn) + rank * half;
                for (int i = 0; i < nst; ++i) {
                    ok = pair_wait(empty + s, ph);
                    if (!ok) break;
                    if (rank == 0) mbar_expect_tx(full + s, bytes);           // parts outside the matrices read as zeros
                    tma_load_2d_pair(sA + s * G4_A, &wmap, i * 128, n0, bars + (uint32_t)s * 8u);
                    tma_load_2d_pair(sB + s * G4_A, &xmap, i * 128, m0, bars + (uint32_t)s * 8u);
                    if (++s == G4P_RA) { s = 0; ph ^= 1u; }
                }
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer: one thread of the first CTA ----------------
        if (rank == 0 && elect_one()) {
            const uint32_t idesc = umma_idesc_mxf4<2>(a.tn), sc0 = smem_u32(sS) >> 4;
            const uint32_t a_lo = umma_desc_sw128_lo(smem_u32(sA)), b_lo = umma_desc_sw128_lo(smem_u32(sB));
            int s = 0, s2 = 0;
            uint32_t ph = 0u, ph2 = 0u, d = 0u, dph = 1u, slot = 0u, sph = 0u, at = 0u, behind = 0u;
            for (uint32_t tile = first; tile < tiles && ok; tile += step) {
                ok = pair_wait(accempty, dph);
                dph ^= 1u;
                for (int i0 = 0; i0 < nst && ok; i0 += G4_GS) {
                    ok = pair_wait(sfull + slot, sph);
#pragma unroll
                    for (int j = 0; j < G4_GS; ++j) {
                        if (!ok || i0 + j >= nst) break;
                        if (behind == 2u) {                // the MMAs that read the scales this stage replaces are done
                            ok = pair_wait(empty + s2, ph2);
                            if (++s2 == G4P_RA) { s2 = 0; ph2 ^= 1u; }
                        } else {
                            ++behind;
                        }
                        if (ok) ok = pair_wait(full + s, ph);
                        if (!ok) break;
                        tc_fence_after();
                        mma_stage<2, 2>(tmem_base + d * G4P_D1, tmem_base + G4P_DCOLS + at * G4P_SFCOLS,
                                        sc0 + (slot * G4_GS + j) * (G4P_SF >> 4), a_lo + (uint32_t)s * (G4_A >> 4),
                                        b_lo + (uint32_t)s * (G4_A >> 4), idesc, (uint32_t)(i0 + j));
                        umma_commit_pair(empty + s);
                        at ^= 1u;
                        if (++s == G4P_RA) { s = 0; ph ^= 1u; }
                    }
                    umma_commit_pair(sempty + slot);
                    if (++slot == G4P_SLOTS) { slot = 0u; sph ^= 1u; }
                }
                if (ok) umma_commit_pair(accfull + d);
                d ^= 1u;
            }
        }
    } else if (warp < 8) {
        // ---------------- scale loaders: warps 2 .. 4 and 5 .. 7 take every other group of stages, counted over the tiles;
        // the first of a set the weight rows, the others 128 activation rows each ----------------
        const int ngrp = (nst + G4_GS - 1) / G4_GS, set = (warp - 2) / 3, part = (warp - 2) % 3;
        const uint8_t* base = part ? a.xscales : a.wscales;
        const int64_t count = part ? a.M : a.N;
        uint8_t* dst = sS + (part ? 1024 + (part - 1) * 512 : 0);
        const uint32_t bars = in_first_cta(sfull);
        ScaleGroup sg;
        auto read = [&](uint32_t tile, int g, bool fresh) {
            if (fresh)
                sg.init(part ? (int64_t)(tile % mt) * a.tn + (part - 1) * 128 : (int64_t)(tile / mt) * 256 + rank * 128, count - 1,
                        a.nblk, lane);
            sg.fetch(base, count * a.nblk, g * 32, a.nblk, a.vec);
        };
        uint32_t tile = first;
        int g = set;
        while (g >= ngrp) { g -= ngrp; tile += step; }
        if (tile < tiles) read(tile, g, true);
        uint32_t ph = 1u;
        int slot = set;
        while (tile < tiles) {
            ok = __all_sync(0xFFFFFFFFu, pair_wait(sempty + slot, ph));
            if (!ok) break;
            if (part) sg.store<G4P_SF, 1024>(dst + slot * G4_GS * G4P_SF, lane);
            else sg.store<G4P_SF, 512>(dst + slot * G4_GS * G4P_SF, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(bars + (uint32_t)slot * 8u);
            if ((slot += G4P_SETS) >= G4P_SLOTS) { slot = set; ph ^= 1u; }
            const uint32_t before = tile;
            g += G4P_SETS;
            while (g >= ngrp) { g -= ngrp; tile += step; }
            if (tile < tiles) read(tile, g, tile != before);
        }
    } else {
        // ---------------- epilogue: lane = weight row, column = activation row; a warp takes half of the columns ----------------
        constexpr int COLS = G4P_TN / 2;
        const int quarter = warp & 3, hf = (warp - 8) >> 2;
        const uint32_t src0 = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(hf * COLS), done = in_first_cta(accempty);
        uint32_t d = 0u, dph = 0u;
        for (uint32_t tile = first; tile < tiles && ok; tile += step) {
            const int64_t n0 = (int64_t)(tile / mt) * 256 + rank * 128, nn = n0 + quarter * 32 + lane;
            const int64_t t0 = (int64_t)(tile % mt) * a.tn, row0 = t0 + hf * COLS;
            const int rows = (int)min(min((int64_t)a.tn, a.M - t0) - hf * COLS, (int64_t)COLS);
            OT* y = reinterpret_cast<OT*>(a.y) + row0 * a.ldy;
            ok = __all_sync(0xFFFFFFFFu, pair_wait(accfull + d, dph));
            if (!ok) break;
            tc_fence_after();
            const uint32_t src = src0 + d * G4P_D1;
            bool stored = false;
            if constexpr (sizeof(OT) == 2) {
                if (a.y_vec_ok && n0 + 128 <= a.N) {
                    // rounded to pairs of neighbouring activation rows, the columns that the other accumulator shares first
                    // (the last 48 of the first accumulator, the first 48 of the second)
                    uint32_t pk[COLS / 2];
                    auto take = [&](int c) {
                        uint32_t v[16];
                        tmem_ld16(src + (uint32_t)(c * 16), v);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            pk[c * 8 + j] = Act<OT>::pack_hi(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
                    };
                    auto hand_back = [&] {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster_relaxed(done);
                    };
                    if (hf == 1 && d == 0u) {
#pragma unroll
                        for (int c = COLS / 16 - 3; c < COLS / 16; ++c) take(c);
                        hand_back();
#pragma unroll
                        for (int c = 0; c < COLS / 16 - 3; ++c) take(c);
                    } else if (hf == 0 && d == 1u) {
#pragma unroll
                        for (int c = 0; c < 3; ++c) take(c);
                        hand_back();
#pragma unroll
                        for (int c = 3; c < COLS / 16; ++c) take(c);
                    } else {
                        hand_back();                       // none of this warp's columns is shared
#pragma unroll
                        for (int c = 0; c < COLS / 16; ++c) take(c);
                    }
                    stored = true;
                    // 32 activation rows at a time through the warp's 2 KB: four lanes store 64 bytes of a row (4 bytes per lane,
                    // straight from the registers: 1024 rows x 4096 x 4096 16.1 us, now 14.3)
                    uint16_t* sw = reinterpret_cast<uint16_t*>(smem + G4P_STORE) + (warp - 8) * 1024;
                    OT* yl = y + (nn & ~31ll) + (lane & 3) * 8;
#pragma unroll
                    for (int c = 0; c < COLS / 32; ++c) {
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            sw[2 * j * 32 + lane] = (uint16_t)pk[c * 16 + j];
                            sw[(2 * j + 1) * 32 + lane] = (uint16_t)(pk[c * 16 + j] >> 16);
                        }
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int j = c * 32 + 8 * i + (lane >> 2);
                            if (j < rows) *reinterpret_cast<uint4*>(yl + j * a.ldy) = reinterpret_cast<const uint4*>(sw)[i * 32 + lane];
                        }
                    }
                }
            }
            if (!stored) {
#pragma unroll 1
                for (int c0 = 0; c0 < rows; c0 += 16) {
                    uint32_t v[16];
                    tmem_ld16(src + (uint32_t)c0, v);
                    if (nn < a.N) {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            if (c0 + j < rows) y[(int64_t)(c0 + j) * a.ldy + nn] = Elt<OT>::from_f32(__uint_as_float(v[j]));
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster_relaxed(done);
            }
            d ^= 1u;
            dph ^= d ^ 1u;
        }
    }
    __syncwarp();
    if (!ok) atomicOr(a.status, JQ_STATUS_LOCAL_WAIT);
    tc_fence_before();
    const int gave_up = __syncthreads_or(ok ? 0 : 1);
    // after a wait that gave up, copies and MMAs may still be in flight: give them a millisecond to land before the tensor
    // memory goes back and the shared memory is reused; neither CTA leaves before the other is done
    if (gave_up)
        for (int i = 0; i < 1000; ++i) __nanosleep(1000);
    ts_cluster_sync();
    tc_fence_after();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(G4_NCOLS) : "memory");
}

static int encode_codes(CUtensorMap* map, const void* codes, int64_t rows, int64_t K, int box_rows) {
    EncodeTiledFn enc = encode_tiled_fn();
    JQ_REQUIRE(enc != nullptr, JQ_ECUDA, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t gdim[2] = {(cuuint64_t)K / 2, (cuuint64_t)rows};
    const cuuint64_t gstride[1] = {(cuuint64_t)K / 2};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    CUresult cr = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), gdim, gstride, box, estr,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    JQ_REQUIRE(cr == CUDA_SUCCESS, JQ_ECUDA, "cuTensorMapEncodeTiled failed with code %d", (int)cr);
    return JQ_OK;
}

// KS: CTAs that split K of a tile, 0: CTA pairs
template <typename OT, int KS>
static int launch_gemm4(const CUtensorMap& wmap, const CUtensorMap& xmap, const Gemm4Args& a, cudaStream_t st) {
    constexpr bool PAIR = KS == 0;
    void (*kernel)(CUtensorMap, CUtensorMap, Gemm4Args);
    if constexpr (PAIR) kernel = mxfp4_gemm4_pair_kernel<OT>;
    else kernel = mxfp4_gemm4_kernel<OT, KS>;
    constexpr size_t smem = PAIR ? G4P_SMEM : G4S_SMEM;
    static bool attr_done[64] = {};
    int dev = 0;
    JQ_CUDA_OK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        JQ_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    if constexpr (PAIR) {
        kernel<<<(unsigned)(2 * std::min(a.tiles, sm_count() / 2)), G4P_THREADS, smem, st>>>(wmap, xmap, a);
        return check_launch("mxfp4_gemm4");
    } else {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)((a.N + 127) / 128), (unsigned)((a.M + a.tn - 1) / a.tn), KS);
        cfg.blockDim = dim3(G4S_THREADS);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 1; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = KS;
        cfg.attrs = attr;
        cfg.numAttrs = KS > 1 ? 1 : 0;
        JQ_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, wmap, xmap, a));
        return JQ_OK;
    }
}

}  // namespace jq

extern "C" int jq_mxfp4_gemm4(const uint32_t* xcodes, const uint8_t* xscales, int64_t M, const uint32_t* wcodes,
                              const uint8_t* wscales, int64_t N, int64_t K, void* y, int y_dtype, int64_t ldy,
                              jq_stream_t stream) {
    using namespace jq;
    int rc = check_mxfp4_shape(N, K);
    if (rc != JQ_OK) return rc;
    rc = check_mxfp4_shape(M, K);
    if (rc != JQ_OK) return rc;
    JQ_REQUIRE(valid_dtype(y_dtype), JQ_EINVAL, "bad dtype id %d", y_dtype);
    if (M == 0 || N == 0) return JQ_OK;
    JQ_REQUIRE(K > 0, JQ_EINVAL, "K must be positive");
    JQ_REQUIRE(xcodes && xscales && wcodes && wscales && y, JQ_EINVAL, "null pointer");
    JQ_REQUIRE(aligned(xcodes, 16) && aligned(wcodes, 16) && aligned(xscales, 4) && aligned(wscales, 4), JQ_EINVAL,
               "codes must be 16-byte aligned, scales 4-byte");
    JQ_REQUIRE(aligned(y, dtype_size(y_dtype)) && ldy >= N, JQ_EINVAL, "y must be aligned to its type, ldy at least N");
    Gemm4Args a;
    a.wscales = wscales; a.xscales = xscales; a.y = y;
    a.M = M; a.N = N; a.ldy = ldy;
    a.nblk = (int)(K / MX_BLOCK);
    const Gemm4Form f = gemm4_form(M, N, a.nblk, sm_count());
    const bool pair = f.ks == 0;
    JQ_REQUIRE(!pair || f.tiles < (1ll << 30), JQ_EUNSUPPORTED, "too many tiles for one launch (%lld)", (long long)f.tiles);
    a.tn = f.tn; a.mt = (int)f.mt; a.tiles = (int)f.tiles;
    a.vec = a.nblk % 16 == 0 && aligned(wscales, 16) && aligned(xscales, 16);
    a.y_pair_ok = (aligned(y, 4) && ldy % 2 == 0) ? 1 : 0;
    a.y_vec_ok = (aligned(y, 16) && ldy % 8 == 0) ? 1 : 0;
    a.status = status_word();
    JQ_REQUIRE(a.status != nullptr, JQ_ECUDA, "could not locate the device status word");
    CUtensorMap wmap, xmap;
    rc = encode_codes(&wmap, wcodes, N, K, 128);
    if (rc != JQ_OK) return rc;
    rc = encode_codes(&xmap, xcodes, M, K, pair ? a.tn / 2 : a.tn);
    if (rc != JQ_OK) return rc;
    JQ_DISPATCH_DTYPE(y_dtype, OT,
        if (f.ks == 1) return launch_gemm4<OT, 1>(wmap, xmap, a, (cudaStream_t)stream);
        if (f.ks == 2) return launch_gemm4<OT, 2>(wmap, xmap, a, (cudaStream_t)stream);
        if (f.ks == 4) return launch_gemm4<OT, 4>(wmap, xmap, a, (cudaStream_t)stream);
        return launch_gemm4<OT, 0>(wmap, xmap, a, (cudaStream_t)stream))
    return JQ_OK;
}
