// Product of two MXFP4 operands on the block-scaled tensor-core path: Y[M, N] = deq(X)[M, K] . deq(W)[N, K]^T.
//
// Bound: tensor throughput of kind::mxf4 for many rows (four times the 16-bit rate, so the copies from L2 are the next
// wall), the packed weights from HBM for few.  Codes go from global memory to the MMA as they are: 128 weight rows are the A
// operand, up to 256 activation rows the B operand (a short batch costs no padded work), 256 codes of each per stage in
// 128-byte-swizzled rows.  The scale bytes of a stage are laid out by the loader warps as the 32-lane pattern that
// tcgen05.cp copies to tensor memory (row r of a 128-row group: lane r % 32, column r / 32, one byte per block of 32), and
// an MMA of 64 codes names its two bytes by the scale id.  Products and sums are f32 in the tensor core.
//   warp 0        TMA producer of both code tiles
//   warp 1        allocates the tensor memory, copies the scales there and issues the MMAs (one elected lane)
//   warps 2 .. 7  scale loaders, two rows per thread; warps 4 .. 7 then store the tile
// Every mbarrier wait is bounded; a wait that runs out sets the library's status word and the CTA leaves through the
// common exit (tensor memory is always released).
#include <algorithm>

#include "jq_mxfp4.cuh"

namespace jq {

struct Gemm4Args {
    const uint8_t *wscales, *xscales;
    void* y;
    int64_t M, N, ldy;
    int nblk;                // blocks of 32 per row
    int tn;                  // activation rows per tile, a multiple of 16
    int vec;                 // scale bytes per aligned load: 8, 4 or 1
    int y_pair_ok;
    int* status;
};

constexpr int G4_RA = 4, G4_TN = 256;
constexpr int G4_A = 128 * 128, G4_B = G4_TN * 128, G4_SF = 3 * 1024, G4_STAGE = G4_A + G4_B + G4_SF;
constexpr int G4_THREADS = 256, G4_LOADERS = 192;
constexpr int G4_DCOLS = G4_TN, G4_SFCOLS = 24, G4_NCOLS = 512;
constexpr size_t G4_SMEM = 1024 + (size_t)G4_RA * G4_STAGE + (2 * G4_RA + 1) * 8 + 16;
static_assert(G4_SMEM <= 227 * 1024, "shared memory of one CTA");
static_assert(G4_DCOLS + G4_RA * G4_SFCOLS <= G4_NCOLS, "tensor memory");

// A and B e2m1, scales ue8m0, both K-major, M = 128, dense K = 64; N at run time, scale ids added per MMA
__device__ __forceinline__ uint32_t umma_idesc_mxf4(int n) {
    return (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void umma_mxf4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa,
                                          uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
// 32 rows of 16 bytes -> 4 columns of 32 lanes, repeated in the four lane quarters
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// no swizzle, 8-row groups of 128 bytes back to back
__device__ __forceinline__ uint64_t umma_desc_rows16(uint32_t smem_addr) {
    return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)(128u >> 4) << 32) | (1ull << 46);
}

// eight scale bytes from block b on (one past the row's end: 1.0)
__device__ __forceinline__ uint2 load_scales8(const uint8_t* row, int b, int nblk, int vec) {
    uint2 v = make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu);
    if (vec == 8) {
        if (b < nblk) v = *reinterpret_cast<const uint2*>(row + b);
    } else if (vec == 4) {
        if (b < nblk) v.x = *reinterpret_cast<const uint32_t*>(row + b);
        if (b + 4 < nblk) v.y = *reinterpret_cast<const uint32_t*>(row + b + 4);
    } else {
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i >> 2] |= (uint32_t)(b + i < nblk ? row[b + i] : 0x7F) << (8 * (i & 3));
        v = make_uint2(w[0], w[1]);
    }
    return v;
}

template <typename OT> __device__ __forceinline__ uint32_t pack_out(float a, float b) { return Act<OT>::pack_hi(a, b); }

template <typename OT>
__global__ void __launch_bounds__(G4_THREADS, 1)
mxfp4_gemm4_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, const Gemm4Args a) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sA = smem, *sB = sA + G4_RA * G4_A, *sS = sB + G4_RA * G4_B;
    uint64_t* full = reinterpret_cast<uint64_t*>(sS + G4_RA * G4_SF);
    uint64_t* empty = full + G4_RA;
    uint64_t* accfull = empty + G4_RA;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(accfull + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t n0 = (int64_t)blockIdx.x * 128, m0 = (int64_t)blockIdx.y * a.tn;
    const int rows = (int)min((int64_t)a.tn, a.M - m0);
    const int n_mma = (rows + 15) & ~15;
    const int nst = (a.nblk + 7) / 8;

    if (threadIdx.x == 0) {
        for (int i = 0; i < G4_RA; ++i) { mbar_init(full + i, 1 + G4_LOADERS / 32); mbar_init(empty + i, 1); }
        mbar_init(accfull, 1);
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc(tmem_slot, G4_NCOLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    bool ok = true;

    if (warp == 0) {
        int s = 0;
        uint32_t ph = 1u;
        const uint32_t bytes = (uint32_t)(G4_A + a.tn * 128);
        for (int i = 0; i < nst; ++i) {
            ok = __all_sync(0xFFFFFFFFu, ts_wait(empty + s, ph));
            if (!ok) break;
            if (elect_one()) {
                mbar_expect_tx(full + s, bytes);                              // parts outside the matrices read as zeros
                tma_load_2d(sA + s * G4_A, &wmap, i * 128, (int)n0, full + s);
                tma_load_2d(sB + s * G4_B, &xmap, i * 128, (int)m0, full + s);
            }
            __syncwarp();
            if (++s == G4_RA) { s = 0; ph ^= 1u; }
        }
    } else if (warp == 1) {
        const uint32_t idesc = umma_idesc_mxf4(n_mma);
        const uint32_t a_lo = umma_desc_sw128_lo(smem_u32(sA)), b_lo = umma_desc_sw128_lo(smem_u32(sB));
        int s = 0;
        uint32_t ph = 0u;
        for (int i = 0; i < nst; ++i) {
            ok = __all_sync(0xFFFFFFFFu, ts_wait(full + s, ph));
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
                const uint32_t sf = tmem_base + (uint32_t)(G4_DCOLS + s * G4_SFCOLS);
                const uint32_t src = smem_u32(sS) + (uint32_t)(s * G4_SF);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    tmem_cp_scales(sf + c * 4, umma_desc_rows16(src + c * 512));
                    tmem_cp_scales(sf + 8 + c * 8, umma_desc_rows16(src + 1024 + c * 1024));
                    if (n_mma > 128) tmem_cp_scales(sf + 12 + c * 8, umma_desc_rows16(src + 1536 + c * 1024));
                }
                const uint32_t ad = a_lo + (uint32_t)s * (G4_A >> 4), bd = b_lo + (uint32_t)s * (G4_B >> 4);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t id = (uint32_t)(k & 1) * 2u;               // scale bytes 0, 1 or 2, 3 of the column
                    umma_mxf4(tmem_base, umma_desc_join(ad + k * 2), umma_desc_join(bd + k * 2), idesc | (id << 4) | (id << 29),
                              sf + (k >> 1) * 4, sf + 8 + (k >> 1) * 8, (i > 0 || k > 0) ? 1u : 0u);
                }
                umma_commit(empty + s);
                if (i == nst - 1) umma_commit(accfull);
            }
            __syncwarp();
            if (++s == G4_RA) { s = 0; ph ^= 1u; }
        }
    } else {
        // rows l and l + 192 of the tile's 128 weight and 256 activation rows
        const int l = threadIdx.x - 64;
        const uint8_t* row[2];
        uint32_t dst[2], gap[2];
        bool need[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = l + j * G4_LOADERS;
            if (r < 128) {
                row[j] = a.wscales + min(n0 + r, a.N - 1) * a.nblk;
                dst[j] = (uint32_t)((r & 31) * 16 + (r >> 5) * 4);
                gap[j] = 512;
                need[j] = true;
            } else {
                const int b = r - 128;
                row[j] = a.xscales + min(m0 + b, a.M - 1) * a.nblk;
                dst[j] = (uint32_t)(1024 + (b >> 7) * 512 + (b & 31) * 16 + ((b & 127) >> 5) * 4);
                gap[j] = 1024;
                need[j] = b < ((n_mma + 127) & ~127);
            }
        }
        uint2 next[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
            if (need[j]) next[j] = load_scales8(row[j], 0, a.nblk, a.vec);
        int s = 0;
        uint32_t ph = 1u;
        for (int i = 0; i < nst; ++i) {
            const uint2 cur[2] = {next[0], next[1]};
            if (i + 1 < nst) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (need[j]) next[j] = load_scales8(row[j], (i + 1) * 8, a.nblk, a.vec);
            }
            ok = __all_sync(0xFFFFFFFFu, ts_wait(empty + s, ph));
            if (!ok) break;
            uint8_t* base = sS + s * G4_SF;
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (need[j]) {
                    *reinterpret_cast<uint32_t*>(base + dst[j]) = cur[j].x;
                    *reinterpret_cast<uint32_t*>(base + dst[j] + gap[j]) = cur[j].y;
                }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(full + s);
            if (++s == G4_RA) { s = 0; ph ^= 1u; }
        }
        if (warp >= 4) {
            if (ok) ok = __all_sync(0xFFFFFFFFu, ts_wait(accfull, 0));
            if (ok) {
                tc_fence_after();
                const int quarter = warp & 3;
                const int64_t nn = n0 + quarter * 32 + lane;
                const uint32_t src = tmem_base + ((uint32_t)(quarter * 32) << 16);
                const bool whole = n0 + 128 <= a.N;
                OT* yt = reinterpret_cast<OT*>(a.y) + m0 * a.ldy;
#pragma unroll 1
                for (int c0 = 0; c0 < rows; c0 += 32) {
                    uint32_t v[32];
                    tmem_ld32(src + (uint32_t)c0, v);
                    OT* yb = yt + c0 * a.ldy;
                    if constexpr (sizeof(OT) == 2) {
                        if (a.y_pair_ok && whole) {
                            // neighbouring lanes swap halves: an even lane stores columns (n, n+1) of the even rows, an odd
                            // lane (n-1, n) of the odd ones, 4 bytes each
                            const bool odd = lane & 1;
                            OT* yl = yb + (odd ? a.ldy : 0) + (nn & ~1ll);
#pragma unroll
                            for (int j = 0; j < 32; j += 2) {
                                const float keep = __uint_as_float(odd ? v[j + 1] : v[j]);
                                const float got = __uint_as_float(__shfl_xor_sync(0xFFFFFFFFu, odd ? v[j] : v[j + 1], 1));
                                const uint32_t pk = odd ? pack_out<OT>(got, keep) : pack_out<OT>(keep, got);
                                if (c0 + j + (odd ? 1 : 0) < rows) *reinterpret_cast<uint32_t*>(yl + j * a.ldy) = pk;
                            }
                            continue;
                        }
                    }
                    if (nn < a.N) {
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (c0 + j < rows) yb[j * a.ldy + nn] = Elt<OT>::from_f32(__uint_as_float(v[j]));
                    }
                }
            }
        }
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

template <typename OT>
static int launch_gemm4(const CUtensorMap& wmap, const CUtensorMap& xmap, const Gemm4Args& a, cudaStream_t st) {
    auto kernel = mxfp4_gemm4_kernel<OT>;
    static bool attr_done[64] = {};
    int dev = 0;
    JQ_CUDA_OK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        JQ_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)G4_SMEM));
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    const dim3 grid((unsigned)((a.N + 127) / 128), (unsigned)((a.M + a.tn - 1) / a.tn));
    kernel<<<grid, G4_THREADS, G4_SMEM, st>>>(wmap, xmap, a);
    return check_launch("mxfp4_gemm4");
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
    JQ_REQUIRE(aligned(xcodes, 16) && aligned(wcodes, 16), JQ_EINVAL, "codes must be 16-byte aligned");
    JQ_REQUIRE(aligned(y, dtype_size(y_dtype)) && ldy >= N, JQ_EINVAL, "y must be aligned to its type, ldy at least N");
    Gemm4Args a;
    a.wscales = wscales; a.xscales = xscales; a.y = y;
    a.M = M; a.N = N; a.ldy = ldy;
    a.nblk = (int)(K / MX_BLOCK);
    const int64_t nt = (M + G4_TN - 1) / G4_TN;
    a.tn = (int)(((M + nt - 1) / nt + 15) / 16 * 16);
    JQ_REQUIRE((M + a.tn - 1) / a.tn < 65536, JQ_EUNSUPPORTED, "too many row tiles for one launch");
    a.vec = a.nblk % 8 == 0 && aligned(wscales, 8) && aligned(xscales, 8) ? 8
          : a.nblk % 4 == 0 && aligned(wscales, 4) && aligned(xscales, 4) ? 4 : 1;
    a.y_pair_ok = (aligned(y, 4) && ldy % 2 == 0) ? 1 : 0;
    a.status = status_word();
    JQ_REQUIRE(a.status != nullptr, JQ_ECUDA, "could not locate the device status word");
    CUtensorMap wmap, xmap;
    rc = encode_codes(&wmap, wcodes, N, K, 128);
    if (rc != JQ_OK) return rc;
    rc = encode_codes(&xmap, xcodes, M, K, a.tn);
    if (rc != JQ_OK) return rc;
    JQ_DISPATCH_DTYPE(y_dtype, OT, return launch_gemm4<OT>(wmap, xmap, a, (cudaStream_t)stream));
    return JQ_OK;
}
