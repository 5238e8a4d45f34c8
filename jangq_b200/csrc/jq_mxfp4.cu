// MXFP4 quantizer and dequantizer.
//
//   e = floor(log2(max |w|)) - 2 of a block of 32, from -127 on;  byte = e + 127;  code = e2m1(w * 2^-e), nearest, ties to
//   the even code, 6 and above to 6.  A block with an infinity or a NaN gets byte 255 (not a number) and codes of zero.
//
// Bound: HBM, 2 + 17/32 bytes per 16-bit weight either way.  Rows are whole blocks, so a matrix is one stream: four lanes
// share a block, each reads eight numbers (16 bytes of a 16-bit type) and writes one word of codes; the block's maximum
// takes two shuffles.  The product with 2^-e is exact in f32, so the conversion instruction's rounding is the only one.
#include <algorithm>

#include "jq_launch.cuh"
#include "jq_mxfp4.cuh"

namespace jq {

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 q = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = Act<T>::lo_f32(w[i]); v[2 * i + 1] = Act<T>::hi_f32(w[i]); }
    }
}

__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// A thread takes U words, a CTA's width apart.  words is a multiple of 4 and the steps are multiples of 32, so the four lanes
// of a block are in range together.
template <typename T, int U>
__global__ void __launch_bounds__(256) mxfp4_quantize_kernel(const T* __restrict__ w, int64_t words, uint32_t* __restrict__ codes,
                                                             uint8_t* __restrict__ scales) {
    overlap_enter();
    const int64_t i0 = (int64_t)blockIdx.x * (256 * U) + threadIdx.x;
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (i0 + u * 256 < words) load8(w + (i0 + u * 256) * 8, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t i = i0 + u * 256;
        if (i >= words) break;
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[u][j]) & 0x7FFFFFFFu);
        const uint32_t four = 0xFu << (threadIdx.x & 28);
        m = max(m, __shfl_xor_sync(four, m, 1));
        m = max(m, __shfl_xor_sync(four, m, 2));
        const uint32_t ex = m >> 23;                       // biased exponent of the maximum; 255: not finite
        const uint32_t byte = ex == 255u ? 255u : (ex > 2u ? ex - 2u : 0u);
        const float inv = __uint_as_float((254u - min(byte, 253u)) << 23);     // 2^-e; 2^127 at byte 0
#pragma unroll
        for (int j = 0; j < 8; ++j) v[u][j] *= inv;
        codes[i] = byte == 255u ? 0u : e2m1x8(v[u]);
        if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)byte;
    }
}

template <typename T, int U>
__global__ void __launch_bounds__(256) mxfp4_dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                               int64_t words, T* __restrict__ out) {
    overlap_enter();
    const int64_t i0 = (int64_t)blockIdx.x * (256 * U) + threadIdx.x;
    uint32_t ws[U], bs[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (i0 + u * 256 < words) {
            ws[u] = codes[i0 + u * 256];
            bs[u] = scales[(i0 + u * 256) >> 2];
        }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t i = i0 + u * 256;
        if (i >= words) break;
        const uint32_t w = ws[u], b = bs[u];
        // 2^(b - 127) as f32: byte 0 is a subnormal, 255 not a number
        const float s = __uint_as_float(b == 0u ? 0x00400000u : (b == 255u ? 0x7FC00000u : b << 23));
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            // the fields as f16 are the values times 2^-14; the product with 2^14 is exact
            const uint32_t f = j == 0 ? mx_field<__half, 0>(w) : j == 1 ? mx_field<__half, 1>(w)
                             : j == 2 ? mx_field<__half, 2>(w) : mx_field<__half, 3>(w);
            v[j] = Act<__half>::lo_f32(f) * 16384.f * s;
            v[j + 4] = Act<__half>::hi_f32(f) * 16384.f * s;
        }
        if constexpr (sizeof(T) == 4) {
            reinterpret_cast<float4*>(out + i * 8)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(out + i * 8)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            using A = Act<T>;
            *reinterpret_cast<uint4*>(out + i * 8) = make_uint4(A::pack_hi(v[0], v[1]), A::pack_hi(v[2], v[3]),
                                                                A::pack_hi(v[4], v[5]), A::pack_hi(v[6], v[7]));
        }
    }
}

int check_mxfp4_shape(int64_t rows, int64_t K) {
    JQ_REQUIRE(rows >= 0 && K >= 0, JQ_EINVAL, "negative shape rows=%lld K=%lld", (long long)rows, (long long)K);
    JQ_REQUIRE(K % MX_BLOCK == 0, JQ_EINVAL, "input dimension %lld is not divisible by the block of 32", (long long)K);
    JQ_REQUIRE(rows < (1ll << 31) && K < (1ll << 31), JQ_EUNSUPPORTED, "dimension too large");
    return JQ_OK;
}

// Words per thread: four where that still leaves every SM a full set of threads, one below.
static bool four_words(int64_t words) { return words >= (int64_t)sm_count() * 2048 * 4; }
static int check_words(int64_t words) {
    JQ_REQUIRE(words / 256 < (1ll << 31) - 1, JQ_EUNSUPPORTED, "too many elements for one launch");
    return JQ_OK;
}

}  // namespace jq

extern "C" {

int jq_mxfp4_quantize(const void* w, int w_dtype, int64_t rows, int64_t K, uint32_t* codes, uint8_t* scales, jq_stream_t stream) {
    using namespace jq;
    int rc = check_mxfp4_shape(rows, K);
    if (rc != JQ_OK) return rc;
    JQ_REQUIRE(valid_dtype(w_dtype), JQ_EINVAL, "bad dtype id %d", w_dtype);
    if (rows == 0 || K == 0) return JQ_OK;
    JQ_REQUIRE(w && codes && scales, JQ_EINVAL, "null pointer");
    JQ_REQUIRE(aligned(w, 16) && aligned(codes, 4), JQ_EINVAL, "w must be 16-byte aligned, codes 4-byte");
    const int64_t words = rows * (K / 8);
    rc = check_words(words);
    if (rc != JQ_OK) return rc;
    const bool four = four_words(words);
    const dim3 grid((unsigned)((words + (four ? 1023 : 255)) / (four ? 1024 : 256)));
    JQ_DISPATCH_DTYPE(w_dtype, T, JQ_CUDA_OK(launch_overlapped(four ? mxfp4_quantize_kernel<T, 4> : mxfp4_quantize_kernel<T, 1>, grid, 256,
                                                               0, (cudaStream_t)stream, (const T*)w, words, codes, scales)))
    return JQ_OK;
}

int jq_mxfp4_dequantize(const uint32_t* codes, const uint8_t* scales, int64_t rows, int64_t K, void* out, int out_dtype,
                        jq_stream_t stream) {
    using namespace jq;
    int rc = check_mxfp4_shape(rows, K);
    if (rc != JQ_OK) return rc;
    JQ_REQUIRE(valid_dtype(out_dtype), JQ_EINVAL, "bad dtype id %d", out_dtype);
    if (rows == 0 || K == 0) return JQ_OK;
    JQ_REQUIRE(codes && scales && out, JQ_EINVAL, "null pointer");
    JQ_REQUIRE(aligned(out, 16) && aligned(codes, 4), JQ_EINVAL, "out must be 16-byte aligned, codes 4-byte");
    const int64_t words = rows * (K / 8);
    rc = check_words(words);
    if (rc != JQ_OK) return rc;
    const bool four = four_words(words);
    const dim3 grid((unsigned)((words + (four ? 1023 : 255)) / (four ? 1024 : 256)));
    JQ_DISPATCH_DTYPE(out_dtype, T, JQ_CUDA_OK(launch_overlapped(four ? mxfp4_dequantize_kernel<T, 4> : mxfp4_dequantize_kernel<T, 1>, grid,
                                                                 256, 0, (cudaStream_t)stream, codes, scales, words, (T*)out)))
    return JQ_OK;
}

}  // extern "C"
