// MXFP4 quantizer and dequantizer.
//
//   e = floor(log2(max |w|)) - 2 of a block of 32, from -127 on;  byte = e + 127;  code = e2m1(w * 2^-e), nearest, ties to
//   the even code, 6 and above to 6.  A block with an infinity or a NaN gets byte 255 (not a number) and codes of zero.
//
// Bound: HBM, 2 + 17/32 bytes per 16-bit weight either way.  Rows are whole blocks, so a matrix is one stream: four lanes
// share a block, each reads eight numbers (16 bytes of a 16-bit type) and writes one word of codes; the block's maximum
// takes two shuffles.  The product with 2^-e is exact in f32, so the conversion instruction's rounding is the only one.
// The numbers stay packed until they are used: 39 registers at four words per thread (50 before, 12.4 us for the first figure).
// Measured (f16, copies in turn beyond L2): quantizer 4096 x 4096 8.6 us = 4.9 TB/s, 14336 x 4096 24.7 = 6.0 TB/s (0.92 of a
// copy); dequantizer 8.5 and 25.6; f32 14336 x 4096 39.9 and 46.4.
#include <type_traits>

#include "jq_launch.cuh"
#include "jq_mxfp4.cuh"

namespace jq {

// Eight numbers as they stand in memory, their largest magnitude as f32 bits, and themselves as f32.
template <typename T> struct Eight {
    uint4 q;
    __device__ __forceinline__ void load(const T* p) { q = *reinterpret_cast<const uint4*>(p); }
    // of the four lanes of a block
    __device__ __forceinline__ uint32_t largest(uint32_t four) const {
        const uint32_t m = 0x7FFF7FFFu;
        uint32_t v = __vmaxu2(__vmaxu2(q.x & m, q.y & m), __vmaxu2(q.z & m, q.w & m));
        v = __vmaxu2(v, __shfl_xor_sync(four, v, 1));
        v = __vmaxu2(v, __shfl_xor_sync(four, v, 2));
        return __float_as_uint(Act<T>::lo_f32(max(v & 0xFFFFu, v >> 16)));
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = Act<T>::lo_f32(w[i]); v[2 * i + 1] = Act<T>::hi_f32(w[i]); }
    }
};
template <> struct Eight<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) {
        a = reinterpret_cast<const float4*>(p)[0];
        b = reinterpret_cast<const float4*>(p)[1];
    }
    __device__ __forceinline__ uint32_t largest(uint32_t four) const {
        float v[8];
        get(v);
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7FFFFFFFu);
        m = max(m, __shfl_xor_sync(four, m, 1));
        return max(m, __shfl_xor_sync(four, m, 2));
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};

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
    Eight<T> in[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (i0 + u * 256 < words) in[u].load(w + (i0 + u * 256) * 8);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t i = i0 + u * 256;
        if (i >= words) break;
        const uint32_t m = in[u].largest(0xFu << (threadIdx.x & 28));
        const uint32_t ex = m >> 23;                       // biased exponent of the maximum; 255: not finite
        const uint32_t byte = ex == 255u ? 255u : (ex > 2u ? ex - 2u : 0u);
        float v[8];
        in[u].get(v);
        const float inv = __uint_as_float((254u - min(byte, 253u)) << 23);     // 2^-e; 2^127 at byte 0
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= inv;
        codes[i] = byte == 255u ? 0u : e2m1x8(v);
        if ((threadIdx.x & 3) == 0) scales[i >> 2] = (uint8_t)byte;
    }
}

// A thread writes U units of 16 bytes, a CTA's width apart, so that a warp's stores are whole lines in every type; a unit is a
// word of codes, or half of one for f32.
template <typename T, int U>
__global__ void __launch_bounds__(256) mxfp4_dequantize_kernel(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                               int64_t units, T* __restrict__ out) {
    overlap_enter();
    constexpr int NUM = 16 / sizeof(T), PER = MX_BLOCK / NUM;              // numbers of a unit, units of a block
    using Word = std::conditional_t<NUM == 8, uint32_t, uint16_t>;
    const int64_t i0 = (int64_t)blockIdx.x * (256 * U) + threadIdx.x;
    uint32_t ws[U], bs[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (i0 + u * 256 < units) {
            ws[u] = reinterpret_cast<const Word*>(codes)[i0 + u * 256];
            bs[u] = scales[(i0 + u * 256) / PER];
        }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t i = i0 + u * 256;
        if (i >= units) break;
        const uint32_t w = ws[u], b = bs[u];
        const float scale = mx_scale_f32(b);
        float v[NUM];
#pragma unroll
        for (int j = 0; j < NUM / 2; ++j) {                                // two codes of a byte, as f16 numbers
            uint32_t f;
            asm("{\n\t.reg .b8 c;\n\tcvt.u8.u32 c, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, c;\n\t}" : "=r"(f) : "r"(w >> (8 * j)));
            v[2 * j] = Act<__half>::lo_f32(f) * scale;
            v[2 * j + 1] = Act<__half>::hi_f32(f) * scale;
        }
        if constexpr (NUM == 4) {
            reinterpret_cast<float4*>(out)[i] = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            using A = Act<T>;
            reinterpret_cast<uint4*>(out)[i] = make_uint4(A::pack_hi(v[0], v[1]), A::pack_hi(v[2], v[3]), A::pack_hi(v[4], v[5]),
                                                          A::pack_hi(v[6], v[7]));
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
    const int64_t words = rows * (K / 8), units = words * (out_dtype == JQ_F32 ? 2 : 1);
    rc = check_words(units);
    if (rc != JQ_OK) return rc;
    const bool four = four_words(units);
    const dim3 grid((unsigned)((units + (four ? 1023 : 255)) / (four ? 1024 : 256)));
    JQ_DISPATCH_DTYPE(out_dtype, T, JQ_CUDA_OK(launch_overlapped(four ? mxfp4_dequantize_kernel<T, 4> : mxfp4_dequantize_kernel<T, 1>, grid,
                                                                 256, 0, (cudaStream_t)stream, codes, scales, units, (T*)out)))
    return JQ_OK;
}

}  // extern "C"
