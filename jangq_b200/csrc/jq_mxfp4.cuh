// Shared by the MXFP4 kernels.  Microscaled 4-bit floating point (OCP MX): 32 numbers share a power of two 2^(byte - 127), a number is e2m1: sign, two
// exponent bits, one mantissa bit, values 0 .5 1 1.5 2 3 4 6.  Byte 255 marks a block that is not a number.
#pragma once

#include "jq_mma.cuh"
#include "jq_ts.cuh"

namespace jq {

constexpr int MX_BLOCK = 32;

int check_mxfp4_shape(int64_t rows, int64_t K);

// ---- expansion to a 16-bit float type -----------------------------------------------------------------
// The three low bits of a code placed at the top of the type's mantissa and the bottom of its exponent read as the code's
// value times 2^-126 (bf16) or 2^-14 (f16), zero and the subnormal 0.5 included, so the scale goes in with the multiply
// that lifts them: one product per two weights, and nothing is rounded where the type holds the weight.
template <typename AT> struct Mx;
template <> struct Mx<__nv_bfloat16> {
    static constexpr int POS = 6;                        // bit of the code's mantissa bit
    static constexpr int FAST_MAX = 128;                 // largest byte whose lift is a bf16 number
    // 2^(byte - 1), twice
    __device__ static __forceinline__ uint32_t lift(uint32_t b) { return ((b + 126u) << 7) * 0x00010001u; }
    // the product for any byte: up to 2^127, then the rest
    __device__ static __forceinline__ uint32_t any(uint32_t field, uint32_t b) {
        if (b <= FAST_MAX) return P2<__nv_bfloat16>::fma(field, lift(b), 0x80008000u);
        const uint32_t rest = b == 255u ? 0x7FC0u : (b - 1u) << 7;                       // 2^(b - 128)
        return P2<__nv_bfloat16>::fma(P2<__nv_bfloat16>::fma(field, lift(128u), 0x80008000u), rest * 0x00010001u, 0x80008000u);
    }
};
template <> struct Mx<__half> {
    static constexpr int POS = 9;
    static constexpr int FAST_MAX = 128;
    // 2^(byte - 113), twice; zero below 2^-24, where no weight of the block reaches half of f16's smallest number
    __device__ static __forceinline__ uint32_t lift(uint32_t b) {
        const uint32_t h = b >= 99u ? (b - 98u) << 10 : (b >= 89u ? 1u << (b - 89u) : 0u);
        return h * 0x00010001u;
    }
    __device__ static __forceinline__ uint32_t any(uint32_t field, uint32_t b) {
        if (b <= FAST_MAX) return P2<__half>::fma(field, lift(b), 0x80008000u);
        const uint32_t one = P2<__half>::fma(field, lift(128u), 0x80008000u);             // twice the code's value
        const uint32_t e1 = min(b - 128u, 15u), e2 = min(b - 128u - e1, 15u);             // 2^30 overflows every weight
        const uint32_t m1 = b == 255u ? 0x7E00u : (e1 + 15u) << 10, m2 = (e2 + 15u) << 10;
        return P2<__half>::fma(P2<__half>::fma(one, m1 * 0x00010001u, 0x80008000u), m2 * 0x00010001u, 0x80008000u);
    }
};

// The eight magnitudes of a block, scaled, as the byte tables of two byte permutes: a code's three low bits are a permute
// selector as they stand, so four codes cost a look-up of their high and one of their low bytes, and the scale is
// multiplied in once per block instead of once per pair.  15 instructions per eight codes and 10 per block; fields shifted
// into place and multiplied took 23 to the same order.
template <typename AT> struct MxTable {
    uint32_t h0, h1, l0, l1;
    // fast: the byte is at most FAST_MAX (in all lanes of the warp, which branch together)
    __device__ __forceinline__ void build(uint32_t byte, bool fast) {
        constexpr uint32_t one = 0x00010001u << Mx<AT>::POS;                 // codes (0, 1), (2, 3), (4, 5), (6, 7) as fields
        uint32_t t[4];
        const uint32_t lift = Mx<AT>::lift(byte);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t f = one * (2u * i) + (0x00010000u << Mx<AT>::POS);
            t[i] = fast ? P2<AT>::fma(f, lift, 0x80008000u) : Mx<AT>::any(f, byte);
        }
        h0 = prmt(t[0], t[1], 0x7531); h1 = prmt(t[2], t[3], 0x7531);
        l0 = prmt(t[0], t[1], 0x6420); l1 = prmt(t[2], t[3], 0x6420);
    }
    // eight codes -> four pairs in order
    __device__ __forceinline__ void expand(uint32_t w, uint32_t* o) const {
        const uint32_t s = w & 0x77777777u, s2 = s >> 16, up = w << 4;
        // sign bytes: bit 3 of a code is the top bit of its byte in w (odd codes) or w << 4 (even ones)
        const uint32_t a = and_or(prmt(up, w, 0xD9C8), 0x80808080u, prmt(h0, h1, s)), la = prmt(l0, l1, s);
        const uint32_t b = and_or(prmt(up, w, 0xFBEA), 0x80808080u, prmt(h0, h1, s2)), lb = prmt(l0, l1, s2);
        o[0] = prmt(la, a, 0x5140); o[1] = prmt(la, a, 0x7362);
        o[2] = prmt(lb, b, 0x5140); o[3] = prmt(lb, b, 0x7362);
    }
};

}  // namespace jq
