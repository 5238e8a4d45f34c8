// Mat-vecs over MXFP4 weights with 16-bit activations: y[m, n] = sum_k x[m, k] * deq(w)[n, k] for up to 16 rows, and the
// same for the (token, slot) pairs of routed experts.
//
// Bound: the weights' 17/32 byte each from HBM on paper; at 2 weights per byte the issue of their expansion is about as
// long.  Warp MMAs (m16n8k16) with the weights as the 16-row operand: eight codes of a word become four pairs by byte
// permutes over the block's scaled magnitudes (MxTable), so every product of the row goes into one f32 accumulator.
// The sum over k does not care which k an MMA slot stands for: a lane takes two whole blocks (32 consecutive bytes) of
// its row, and the activations are read in the same order.  A CTA owns 16 weight rows; its warps take every eighth
// stretch of 256 codes and their sums meet in shared memory in warp order, so results do not depend on timing.
// The weight is exact in bf16; in f16 it is rounded once (scales below 2^-23 or above 2^13).
#include <algorithm>

#include "jq_launch.cuh"
#include "jq_mxfp4.cuh"

namespace jq {

struct MxGemvArgs {
    const uint16_t* x;
    const uint8_t* codes;
    const uint8_t* scales;
    uint16_t* y;
    int64_t ldx, ldy, N, nblk;           // nblk: blocks of 32 codes per row
    int M;
    int even;                            // two scale bytes of neighbouring blocks are one aligned 16-bit load
    // pairs of routed experts: row blockIdx.y of y is x[pair / x_div] . w[pair_expert[pair] - expert_base]
    const int32_t* pair_expert;
    int x_div, num_experts, expert_base;
};

constexpr int MXV_WARPS = 8;
constexpr int MXV_UNIT = 8;              // blocks per warp step

// this lane's two blocks of one weight row
struct MxTile {
    uint4 q[4];
    uint32_t s;                          // scale bytes, low first
    __device__ __forceinline__ void load(const MxGemvArgs& a, const uint8_t* crow, const uint8_t* srow, int64_t b) {
        // blocks past the row's end: codes of zero, scale 1
        const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
        const bool in0 = b < a.nblk, in1 = b + 1 < a.nblk;
        const uint4* p = reinterpret_cast<const uint4*>(crow + b * 16);
        q[0] = in0 ? __ldg(p) : zero;
        q[1] = in1 ? __ldg(p + 1) : zero;
        if (a.even) {
            s = in0 ? *reinterpret_cast<const uint16_t*>(srow + b) : 0x7F7Fu;
        } else {
            s = (in0 ? srow[b] : 0x7Fu) | (in1 ? srow[b + 1] : 0x7Fu) << 8;
        }
    }
};

template <typename AT, int NT, bool GATHER>
__global__ void __launch_bounds__(32 * MXV_WARPS)
mxfp4_gemv_kernel(const MxGemvArgs a) {
    using A = Act<AT>;
    __shared__ float part[MXV_WARPS][NT * 8][16 + 1];
    overlap_enter();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const int64_t crow_bytes = a.nblk * 16;
    const uint8_t *codes = a.codes, *scales = a.scales;
    const uint16_t* x = a.x;
    uint16_t* y = a.y;
    int M = a.M;
    if constexpr (GATHER) {
        const int64_t p = blockIdx.y;
        const int e = a.pair_expert[p] - a.expert_base;
        y += p * a.ldy;
        if (e < 0 || e >= a.num_experts) {                 // another rank's expert: a row of zeros
            if (threadIdx.x < 16 && n0 + threadIdx.x < a.N) y[n0 + threadIdx.x] = 0;
            return;
        }
        codes += (int64_t)e * a.N * crow_bytes;
        scales += (int64_t)e * a.N * a.nblk;
        x += p / a.x_div * a.ldx;
        M = 1;
    }
    // rows past N repeat the last one and are never stored
    const int64_t r0 = min(n0 + g, a.N - 1), r1 = min(n0 + g + 8, a.N - 1);
    const uint8_t *c0 = codes + r0 * crow_bytes, *c1 = codes + r1 * crow_bytes;
    const uint8_t *s0 = scales + r0 * a.nblk, *s1 = scales + r1 * a.nblk;
    const uint16_t* xr[NT];
    bool live[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        live[i] = g + 8 * i < M;
        xr[i] = x + (live[i] ? (g + 8 * i) * a.ldx : 0);
    }

    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;

    MxTile w0, w1;
    int64_t b = (int64_t)warp * MXV_UNIT + 2 * t;
    if (warp * MXV_UNIT < a.nblk) { w0.load(a, c0, s0, b); w1.load(a, c1, s1, b); }
    for (int64_t u = (int64_t)warp * MXV_UNIT; u < a.nblk; u += MXV_WARPS * MXV_UNIT) {
        const MxTile v0 = w0, v1 = w1;
        const int64_t at = b;
        b += MXV_WARPS * MXV_UNIT;
        if (u + MXV_WARPS * MXV_UNIT < a.nblk) { w0.load(a, c0, s0, b); w1.load(a, c1, s1, b); }
        const bool fast = __all_sync(0xFFFFFFFFu, max(max(v0.s & 255u, v0.s >> 8), max(v1.s & 255u, v1.s >> 8)) <= Mx<AT>::FAST_MAX);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            MxTable<AT> t0, t1;
            t0.build(h ? v0.s >> 8 : v0.s & 255u, fast);
            t1.build(h ? v1.s >> 8 : v1.s & 255u, fast);
            const uint32_t q0[4] = {v0.q[h].x, v0.q[h].y, v0.q[h].z, v0.q[h].w};
            const uint32_t q1[4] = {v1.q[h].x, v1.q[h].y, v1.q[h].z, v1.q[h].w};
            const bool in = at + h < a.nblk;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t e0[4], e1[4];
                t0.expand(q0[j], e0);
                t1.expand(q1[j], e1);
                const uint32_t fa[4] = {e0[0], e1[0], e0[1], e1[1]}, fb[4] = {e0[2], e1[2], e0[3], e1[3]};
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    uint4 xv = make_uint4(0u, 0u, 0u, 0u);
                    if (live[i] && in) xv = *reinterpret_cast<const uint4*>(xr[i] + (at + h) * 32 + j * 8);
                    A::mma(acc[i], fa, xv.x, xv.y);
                    A::mma(acc[i], fb, xv.z, xv.w);
                }
            }
        }
    }
    // lane (g, t) holds rows g, g + 8 of tokens 2t, 2t + 1 of every token tile
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        part[warp][8 * i + 2 * t][g] = acc[i][0];
        part[warp][8 * i + 2 * t + 1][g] = acc[i][1];
        part[warp][8 * i + 2 * t][g + 8] = acc[i][2];
        part[warp][8 * i + 2 * t + 1][g + 8] = acc[i][3];
    }
    __syncthreads();
    for (int q = threadIdx.x; q < M * 16; q += 32 * MXV_WARPS) {
        const int m = q >> 4, n = q & 15;
        float s = part[0][m][n];
#pragma unroll
        for (int w = 1; w < MXV_WARPS; ++w) s += part[w][m][n];
        if (n0 + n < a.N) y[m * a.ldy + n0 + n] = A::from_f32(s);
    }
}

static int mx_gemv_common(const void* x, int x_dtype, int64_t ldx, const uint32_t* codes, const uint8_t* scales, int64_t N,
                          int64_t K, void* y, int64_t ldy, MxGemvArgs& a) {
    int rc = check_mxfp4_shape(N, K);
    if (rc != JQ_OK) return rc;
    JQ_REQUIRE(x_dtype == JQ_BF16 || x_dtype == JQ_F16, JQ_EINVAL, "activations must be bf16 or f16");
    JQ_REQUIRE(K > 0, JQ_EINVAL, "K must be positive");
    JQ_REQUIRE(x && codes && scales && y, JQ_EINVAL, "null pointer");
    JQ_REQUIRE(aligned(x, 16) && ldx % 8 == 0 && ldx >= K, JQ_EINVAL, "x must be 16-byte aligned with ldx %% 8 == 0");
    JQ_REQUIRE(aligned(codes, 16) && aligned(scales, 2), JQ_EINVAL, "codes must be 16-byte aligned, scales 2-byte");
    JQ_REQUIRE(ldy >= N, JQ_EINVAL, "ldy too small");
    a.x = (const uint16_t*)x; a.codes = (const uint8_t*)codes; a.scales = scales; a.y = (uint16_t*)y;
    a.ldx = ldx; a.ldy = ldy; a.N = N; a.nblk = K / MX_BLOCK;
    a.even = a.nblk % 2 == 0;
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
    a.M = (int)M;
    const dim3 grid((unsigned)((N + 15) / 16));
    cudaStream_t st = (cudaStream_t)stream;
    JQ_DISPATCH_DTYPE16(x_dtype, AT,
        JQ_CUDA_OK(launch_overlapped(M <= 8 ? mxfp4_gemv_kernel<AT, 1, false> : mxfp4_gemv_kernel<AT, 2, false>, grid,
                                     32 * MXV_WARPS, 0, st, a)))
    return JQ_OK;
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
    a.even = a.nblk % 2 == 0;
    const dim3 grid((unsigned)((N + 15) / 16), (unsigned)P);
    JQ_DISPATCH_DTYPE16(x_dtype, AT,
        JQ_CUDA_OK(launch_overlapped(mxfp4_gemv_kernel<AT, 1, true>, grid, 32 * MXV_WARPS, 0, (cudaStream_t)stream, a)))
    return JQ_OK;
}

}  // extern "C"
