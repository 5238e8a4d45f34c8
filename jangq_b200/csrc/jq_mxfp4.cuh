// Shared by the MXFP4 kernels.  Microscaled 4-bit floating point (OCP MX): 32 numbers share a power of two 2^(byte - 127), a number is e2m1: sign, two
// exponent bits, one mantissa bit, values 0 .5 1 1.5 2 3 4 6.  Byte 255 marks a block that is not a number.
#pragma once

#include "jq_mma.cuh"
#include "jq_ts.cuh"

namespace jq {

constexpr int MX_BLOCK = 32;

int check_mxfp4_shape(int64_t rows, int64_t K);

// ---- expansion to a 16-bit float type -----------------------------------------------------------------
// eight codes -> four f16 pairs of their plain values, in order
__device__ __forceinline__ void mx_values8(uint32_t w, uint32_t (&o)[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
        : "r"(w));
}
// 2^(byte - 127) as f32: byte 0 is a subnormal, 255 not a number
__device__ __forceinline__ float mx_scale_f32(uint32_t byte) {
    return __uint_as_float(byte == 0u ? 0x00400000u : (byte == 255u ? 0x7FC00000u : byte << 23));
}

// One product per pair puts the scale in, rounded once where the type does not hold the weight.  FAST_MIN .. FAST_MAX: the bytes
// whose factor is a number of the type.
template <typename AT> struct Mx;
// bf16: the three low bits of a code placed at the top of the mantissa and the bottom of the exponent read as the code's value
// times 2^-126, zero and the subnormal 0.5 included.  A multiplication by 2^6 + 2^12 places them and the sign (the copies of a
// code do not touch), so eight codes take 11 logic and permute instructions (at half rate) and eight of the multiply pipe; shifts
// took the logic pipe for 23, byte tables with the scale built in for 15 and 10 per block.  f16 takes the conversion instruction:
// eight in all.  GEMM of 512 rows x 11008 x 4096: tables bf16 47.3 us, f16 49.2; now 42.2 and 38.2; 16 rows x 14336 x 4096: 21.7 and
// 22.6; now 19.4 and 16.3.
template <> struct Mx<__nv_bfloat16> {
    static constexpr uint32_t FAST_MIN = 0, FAST_MAX = 128;
    __device__ static __forceinline__ uint32_t factor(uint32_t b) { return ((b + 126u) << 7) * 0x00010001u; }      // 2^(byte - 1), twice
    __device__ static __forceinline__ void fields8(uint32_t w, uint32_t (&o)[4]) {
        const uint32_t even = w & 0x0F0F0F0Fu, odd = w >> 4 & 0x0F0F0F0Fu;
        o[0] = prmt(even, odd, 0x8480); o[1] = prmt(even, odd, 0x8581);
        o[2] = prmt(even, odd, 0x8682); o[3] = prmt(even, odd, 0x8783);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = o[i] * 0x1040u & 0x81C081C0u;
    }
};
template <> struct Mx<__half> {
    static constexpr uint32_t FAST_MIN = 103, FAST_MAX = 142;                                   // 2^-24 .. 2^15
    __device__ static __forceinline__ uint32_t factor(uint32_t b) {
        return (b >= 113u ? (b - 112u) << 10 : 1u << (b - 103u)) * 0x00010001u;                 // 2^(byte - 127), twice
    }
    __device__ static __forceinline__ void fields8(uint32_t w, uint32_t (&o)[4]) { mx_values8(w, o); }
};
// the 32 codes of a block; fast: the byte is in the type's range (in all lanes of the warp, which branch together)
template <typename AT> __device__ __forceinline__ void mx_expand32(const uint32_t (&w)[4], uint32_t byte, bool fast, uint32_t* out) {
    if (fast) {
        const uint32_t factor = Mx<AT>::factor(byte);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t f[4];
            Mx<AT>::fields8(w[i], f);
#pragma unroll
            for (int j = 0; j < 4; ++j) out[4 * i + j] = P2<AT>::fma(f[j], factor, 0x80008000u);
        }
    } else {
        const float scale = mx_scale_f32(byte);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t f[4];
            mx_values8(w[i], f);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                out[4 * i + j] = Act<AT>::pack_hi(Act<__half>::lo_f32(f[j]) * scale, Act<__half>::hi_f32(f[j]) * scale);
        }
    }
}

}  // namespace jq
