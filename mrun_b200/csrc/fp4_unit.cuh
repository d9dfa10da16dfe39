// The 4-bit key/value cache's unit: 16 tokens of one kv head, their keys and their values.
//
// Sixteen neighbouring features of a token share a scale; a value is scale * code.  The code is a
// 4-bit float (E2M1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign: the bit of 8, set for values below zero, also where they
// round to zero; a zero of either sign is code 0), two to a byte, the even feature in the low half; the scale is an
// unsigned byte of 5 exponent and 3 mantissa bits, which are bits 7 to 14 of the half of the same value (byte << 7 is that half).  The largest scale that is written is
// 10,240: every value is then a half and a bfloat16 exactly.  A group that holds a value that is not finite has
// the scale byte 0xFF, a NaN.
//
// A unit is [key codes | value codes | key scales | value scales], each in the order in which the 32
// lanes 4 g + t of a warp hold it in products of 16 x 8 x 16, so that a lane's share is one 4- to 16-byte
// load without bank conflicts:
//   key codes     row by row; lane 4 g + t takes features D/4 * t .. of tokens g and g + 8
//   value codes   lane 4 g + t takes features D/8 * g .. of tokens 2 t, 2 t + 1, and of 2 t + 8, 2 t + 9
//   scales        of the same
#pragma once

namespace mrun {

constexpr int FP4_TOKENS = 16;         // tokens of a unit
constexpr int FP4_GROUP = 16;          // features that share a scale
constexpr int FP4_MAX_SCALE = 226;     // the byte of 10,240
constexpr int FP4_NAN_SCALE = 255;

template <int D> struct Fp4Unit {
    static_assert(D == 64 || D == 128, "head sizes 64 and 128");
    static constexpr int K_CODES = 0, V_CODES = 8 * D, K_SCALES = 16 * D, V_SCALES = 17 * D, BYTES = 18 * D;
    static constexpr int PIECE = D / 16;          // bytes of value codes that a lane takes of a token
    static constexpr int PER = D / 64;            // key scales that a lane takes of a token
    // Offsets in a unit, for token r: the byte of features 2 * pair and 2 * pair + 1; the scale of group s.
    static __host__ __device__ constexpr int k_code(int r, int pair) { return K_CODES + r * (D / 2) + pair; }
    static __host__ __device__ constexpr int v_code(int r, int pair) {
        return V_CODES + (r >> 3) * (4 * D) + ((pair / PIECE * 4 + ((r >> 1) & 3)) * 2 + (r & 1)) * PIECE + pair % PIECE;
    }
    static __host__ __device__ constexpr int k_scale(int r, int s) {
        return K_SCALES + ((r & 7) * 4 + s / PER) * (2 * PER) + (r >> 3) * PER + s % PER;
    }
    static __host__ __device__ constexpr int v_scale(int r, int s) {
        return V_SCALES + (s * 4 + ((r >> 1) & 3)) * 4 + (r >> 3) * 2 + (r & 1);
    }
};

// The eight codes of a word as four pairs of halves.
__device__ __forceinline__ void halves_of(unsigned word, unsigned (&h)[4]) {
    asm("{\n.reg .b8 c0, c1, c2, c3;\nmov.b32 {c0, c1, c2, c3}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, c0;\ncvt.rn.f16x2.e2m1x2 %1, c1;\ncvt.rn.f16x2.e2m1x2 %2, c2;\ncvt.rn.f16x2.e2m1x2 %3, c3;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(word));
}

}  // namespace mrun
