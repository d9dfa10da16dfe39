// Writing the 4-bit key/value cache and reading it back (the format: fp4_unit.cuh).
#include <cuda_fp16.h>

#include "common.cuh"
#include "fp4_unit.cuh"

namespace {

using namespace mrun;
using bf16 = __nv_bfloat16;

// ------------------------------------------------------------------------------------------
// Per head of every token: q = rotate(rmsnorm(q) * w_q) in bfloat16, in place or into rows of its own; k the
// same and v as it is into the unit that the token's slot names.  The arithmetic of q is that of
// qk_norm_rope_cache.
//
// A key is quantised from its unrounded value, and which side of a border between two codes a value
// falls on decides a whole step of the code.  So that the codes are those of the formula and do not depend on
// the order of a sum, a key is computed in 32 bits with a bound of its error, quantised at both ends of the bound, and where
// the two differ (about one head in a hundred) computed again in 64 bits.  In 64 bits throughout a step of one
// token took 10.5 us with its read back, 4.2 so.
// A value is a bfloat16: its quotient by a scale of 4 bits is a border (at most 3 bits) exactly or 2^-9 away from it.
//
// D / 8 lanes take a run of heads of a token, eight features a lane, with the token's cosines and sines loaded once and the features of
// the next three heads on their way into shared memory, where a lane reads what it copied itself.  What bounds it is the chain of a head
// (sum over the lanes, root, rotation across lanes) and its instructions, with 28 warps a multiprocessor to hide it: 14.3 us for 2,048 tokens of 32 + 8 + 8 heads
// of 128 in runs of 6, of which the queries alone take 9.4 (the bytes take 6.8, the write of bfloat16 pages 13.7); a copy to every two heads, in
// registers, took 21.7.  Longer runs save instructions and leave fewer lanes at work, hence as long as the step has
// heads for them (us in runs of 2 / 4 / 6 / 12: 512 tokens 8.3 / 8.1 / 8.5 / 9.9; 2,048 18.8 / 14.9 / 14.3 / 14.8; 8,192 72.5 / 55.5 / 50.5 / 47.1).
// ------------------------------------------------------------------------------------------
constexpr int STORE_THREADS = 256;
constexpr int RUN_THREADS = 128, RUN_DEPTH = 4;
constexpr unsigned MOST_A_RUN = 12;
constexpr unsigned HEADS_A_RUN = 16384;    // a run gets a head more for every so many heads of the step

// The byte of the scale nearest to `wanted` (0 .. 10,240), ties to the even byte.  `wanted` has a bit set below
// its 24 wherever something was cut off, so that this is the only rounding.
__device__ __forceinline__ unsigned scale_byte(float wanted) {
    const unsigned bits = __float_as_uint(wanted);
    const unsigned normal = ((bits + 0x7FFFFu + ((bits >> 20) & 1u)) >> 20) - (112u << 3);
    const unsigned byte = wanted < 6.103515625e-05f ? __float2uint_rn(wanted * 131072.f) : normal;
    return min(byte, (unsigned)FP4_MAX_SCALE);
}
__device__ __forceinline__ float scale_value(unsigned byte) {
    return __half2float(__ushort_as_half((unsigned short)(byte << 7)));
}

// Eight 4-bit floats, the first in the lowest bits: nearest, ties to the even code, at most 6.
__device__ __forceinline__ unsigned codes_of(const float2 (&f)[4]) {
    unsigned out;
    asm("{\n.reg .b8 c0, c1, c2, c3;\ncvt.rn.satfinite.e2m1x2.f32 c0, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 c1, %4, %3;\n"
        "cvt.rn.satfinite.e2m1x2.f32 c2, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 c3, %8, %7;\nmov.b32 %0, {c0, c1, c2, c3};\n}"
        : "=r"(out) : "f"(f[0].x), "f"(f[0].y), "f"(f[1].x), "f"(f[1].y), "f"(f[2].x), "f"(f[2].y), "f"(f[3].x), "f"(f[3].y));
    return out;
}

// `v` cut to 32 bits with the last bit set where something was cut off.
__device__ __forceinline__ float cut_sticky(double v) {
    const float f = __double2float_rz(v);
    return (double)f == v ? f : __uint_as_float(__float_as_uint(f) | 1u);
}

// Magnitudes as their bits, whose order is theirs; those of NaN and the infinities lie above.
constexpr unsigned INFINITE = 0x7F800000u;
__device__ __forceinline__ unsigned magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// The codes (8 features a lane, four bytes) and the scale of the 16 features that two neighbouring lanes hold: of any doubles,
__device__ __forceinline__ unsigned quantise(const double (&x)[8], unsigned mask, unsigned& scale) {
    double largest = 0.0;
    bool finite = true;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        finite = finite && fabs(x[e]) < INFINITY;
        largest = fmax(largest, fabs(x[e]));
    }
    largest = fmax(largest, __shfl_xor_sync(mask, largest, 1));
    finite = __shfl_xor_sync(mask, (int)finite, 1) && finite;
    scale = finite ? scale_byte(cut_sticky(fmin(largest / 6.0, 10240.0))) : (unsigned)FP4_NAN_SCALE;
    if (!finite) return 0u;
    const double s = scale_value(scale);
    // A shade more than 1 / s, so that a quotient that is a border exactly is not cut below it.  Under a scale of zero any quotient rounds to zero.
    const double inverse = s > 0.0 ? 1.0 / s * (1.0 + 8.8817841970012523e-16) : 1.0;
    float2 f[4];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float& part = e % 2 ? f[e / 2].y : f[e / 2].x;
        part = __double2float_rz(__fma_rn(x[e], inverse, 0.0));          // -0 + 0 is 0: only what is below zero keeps a sign
        if ((double)part * s != x[e]) part = __uint_as_float(__float_as_uint(part) | 1u);
    }
    return codes_of(f);
}

__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }

// To 12 bits, by two subtractions (4,097 = 2^12 + 1): of a quotient that is a number of few bits exactly, and was off by some of its last
// of 24, that number; any quotient that is 2^-10 away from it stays on its side.  One by one: the compiler makes one operation of
// a product of pairs and the sum behind it.
__device__ __forceinline__ float to_12_bits(float v) {
    const float wide = __fmul_rn(v, 4097.f);
    return __fsub_rn(wide, __fsub_rn(wide, v));
}

// The largest magnitude of the 16 features that two neighbouring lanes hold, as its bits.
__device__ __forceinline__ unsigned largest_of(const float2 (&x)[4], unsigned mask) {
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, max(magnitude(x[e].x), magnitude(x[e].y)));
    return max(top, __shfl_xor_sync(mask, top, 1));
}

// of floats that hold bfloat16 values,
__device__ __forceinline__ unsigned quantise(const float2 (&x)[4], unsigned mask, unsigned& scale) {
    const unsigned top = largest_of(x, mask);
    if (top >= INFINITE) {
        scale = FP4_NAN_SCALE;
        return 0u;
    }
    scale = scale_byte(to_12_bits(fminf(__uint_as_float(top) * (1.f / 6.f), 10240.f)));
    const float s = scale_value(scale), inverse = s > 0.f ? __fdividef(1.f, s) : 1.f;
    float2 f[4];                                       // -0 + 0 is 0: only what is below zero keeps a sign
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = make_float2(to_12_bits(__fmaf_rn(x[e].x, inverse, 0.f)), to_12_bits(__fmaf_rn(x[e].y, inverse, 0.f)));
    return codes_of(f);
}

// and of floats that are within `off` of the values meant.  `sure`: neither the scale nor a code depends on where within.
__device__ __forceinline__ unsigned quantise(const float2 (&x)[4], float off, unsigned mask, unsigned& scale, bool& sure) {
    const unsigned top = largest_of(x, mask);
    const float largest = __uint_as_float(top);
    scale = scale_byte(fminf((largest + off) * (1.f / 6.f) * 1.000001f, 10240.f));
    sure = top < INFINITE && off < INFINITY && scale == scale_byte(fminf(fmaxf(largest - off, 0.f) * (1.f / 6.f) * 0.999999f, 10240.f));
    const float s = scale_value(scale), inverse = s > 0.f ? __fdividef(1.f, s) : 0.f;
    // the quotients are at most 6.4 where they are not far beyond the last border, and off by 2^-21 of them
    const float away = fmaf(off, inverse * 1.000001f, 4e-6f);
    float2 low[4], high[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        low[e] = __ffma2_rn(x[e], twice(inverse), twice(-away));
        high[e] = __ffma2_rn(x[e], twice(inverse), twice(away));
    }
    const unsigned codes = codes_of(low);
    sure = sure && codes == codes_of(high);
    return codes;
}

// Eight floats of `src`, on 16 bytes.
__device__ __forceinline__ void load8(float2 (&v)[4], const float* __restrict__ src) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(src)), b = __ldg(reinterpret_cast<const float4*>(src) + 1);
    v[0] = make_float2(a.x, a.y); v[1] = make_float2(a.z, a.w); v[2] = make_float2(b.x, b.y); v[3] = make_float2(b.z, b.w);
}

// What a lane needs of the rotation of its eight features.  Pairs (j, j + half): with a half of a multiple of eight a
// lane's partners are the eight features of another lane, and it holds their cosines and sines (these with their sign).
struct Turn {
    int partner;            // the lane of the group, itself where nothing turns
    bool turns;
    float2 c[4], s[4];
};

__device__ __forceinline__ float squares(const float2 (&v)[4]) {
    float2 two = __fmul2_rn(v[0], v[0]);
#pragma unroll
    for (int e = 1; e < 4; ++e) two = __ffma2_rn(v[e], v[e], two);
    return two.x + two.y;
}
__device__ __forceinline__ void scale_by(float2 (&v)[4], float inv, const float2 (&weight)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __fmul2_rn(__fmul2_rn(v[e], twice(inv)), weight[e]);
}

// The norm in 32 bits, two features an instruction; returns the sum of squares.
template <int D> __device__ __forceinline__ float norm(float2 (&v)[4], const float2 (&weight)[4], float eps, unsigned mask) {
    float ss = squares(v);
#pragma unroll
    for (int o = D / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
    scale_by(v, rsqrtf(ss * (1.f / D) + eps), weight);
    return ss;
}
template <int D> __device__ __forceinline__ void norm(double (&v)[8], const float2 (&weight)[4], float eps, unsigned mask) {
    double ss = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += v[e] * v[e];
#pragma unroll
    for (int o = D / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
    const double inv = rsqrt(ss / D + (double)eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] * inv * (double)(e % 2 ? weight[e / 2].y : weight[e / 2].x);
}

// With WIDEST returns the largest |first| + |second| of the two products that are added, whatever the size of the cosines and sines.
template <bool WIDEST> __device__ __forceinline__ float rotate(float2 (&v)[4], const Turn& turn, unsigned mask, int part) {
    const int from = (int)(threadIdx.x & 31) - part + turn.partner;
    float widest = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 other = make_float2(__shfl_sync(mask, v[e].x, from), __shfl_sync(mask, v[e].y, from));
        if (turn.turns) {
            const float2 second = __fmul2_rn(other, turn.s[e]);
            if constexpr (WIDEST)
                widest = fmaxf(widest, fmaxf(fmaf(fabsf(v[e].x), fabsf(turn.c[e].x), fabsf(second.x)), fmaf(fabsf(v[e].y), fabsf(turn.c[e].y), fabsf(second.y))));
            v[e] = __ffma2_rn(v[e], turn.c[e], second);
        } else if constexpr (WIDEST) {
            widest = fmaxf(widest, fmaxf(fabsf(v[e].x), fabsf(v[e].y)));
        }
    }
    return widest;
}
__device__ __forceinline__ void rotate(double (&v)[8], const Turn& turn, unsigned mask, int part) {
    const int from = (int)(threadIdx.x & 31) - part + turn.partner;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const double other = __shfl_sync(mask, v[e], from);
        if (turn.turns)
            v[e] = v[e] * (double)(e % 2 ? turn.c[e / 2].y : turn.c[e / 2].x) + other * (double)(e % 2 ? turn.s[e / 2].y : turn.s[e / 2].x);
    }
}

// The rotation with the partners fetched one by one through `stage`, a row of D of the group's own.
template <typename F>
__device__ __forceinline__ void rotate_staged(F (&v)[8], const float2* __restrict__ cs, int half, unsigned mask, int part, F* stage) {
    __syncwarp(mask);
#pragma unroll
    for (int e = 0; e < 8; ++e) stage[part * 8 + e] = v[e];
    __syncwarp(mask);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int j = part * 8 + e;
        if (j < half) v[e] = v[e] * (F)cs[j].x - stage[j + half] * (F)cs[j].y;
        else if (j < 2 * half) v[e] = v[e] * (F)cs[j - half].x + stage[j - half] * (F)cs[j - half].y;
    }
}

// What the lanes of a token need of it.
template <int D> struct Token {
    int part;                           // of the D / 8 lanes of a head
    unsigned mask;                      // theirs
    Turn turn;
    bool turned, normed, writes;        // writes: its slot lies in the cache
    int off_row;                        // its row of a unit
    unsigned char* units;               // its unit of the first kv head
    int head_bytes;                     // from a kv head to the next
};

template <int D, bool STAGED>
__device__ __forceinline__ Token<D> token_of(const float* q_weight, const float2* __restrict__ cs, int half, bool turned, int slot,
                                             unsigned char* cache, int kv_heads, int page_size, long pages) {
    using Unit = Fp4Unit<D>;
    constexpr int LANES = D / 8;
    Token<D> t;
    t.part = threadIdx.x % LANES;
    t.mask = ((1u << LANES) - 1u) << (threadIdx.x & 31 & ~(unsigned)(LANES - 1));
    t.normed = q_weight != nullptr;
    t.turned = turned;
    if (!STAGED && turned) {
        const int away = half / 8;
        const bool low = t.part < away;
        t.turn.turns = t.part < 2 * away;
        t.turn.partner = t.turn.turns ? (low ? t.part + away : t.part - away) : t.part;
        if (t.turn.turns) {
            float2 two[2][4];                                      // (cosine, sine) of a pair each
            const float* src = reinterpret_cast<const float*>(cs + (low ? t.part : t.turn.partner) * 8);
            load8(two[0], src);
            load8(two[1], src + 8);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 a = two[e / 2][e % 2 * 2], b = two[e / 2][e % 2 * 2 + 1];
                t.turn.c[e] = make_float2(a.x, b.x);
                t.turn.s[e] = low ? make_float2(-a.y, -b.y) : make_float2(a.y, b.y);
            }
        }
    }
    const int page = slot >= 0 ? slot / page_size : -1, off = slot - page * page_size;
    t.writes = page >= 0 && page < pages;
    t.off_row = off & (FP4_TOKENS - 1);
    t.units = cache + ((size_t)page * kv_heads * (page_size / FP4_TOKENS) + off / FP4_TOKENS) * Unit::BYTES;
    t.head_bytes = page_size / FP4_TOKENS * Unit::BYTES;
    return t;
}

__device__ __forceinline__ void unpack(float2 (&x)[4], const uint4& raw) {
    const __nv_bfloat162* pairs = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = __bfloat1622float2(pairs[e]);
}

template <int D, bool STAGED>
__device__ __forceinline__ void store_query(const uint4& raw, const float2 (&weight)[4], const Token<D>& t, float eps,
                                            const float2* __restrict__ cs, int half, float* stage, bf16* out) {
    float2 x[4];
    unpack(x, raw);
    if (t.normed) norm<D>(x, weight, eps, t.mask);
    if (t.turned) {
        if constexpr (STAGED) {
            float y[8] = {x[0].x, x[0].y, x[1].x, x[1].y, x[2].x, x[2].y, x[3].x, x[3].y};
            rotate_staged(y, cs, half, t.mask, t.part, stage);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = make_float2(y[2 * e], y[2 * e + 1]);
        } else {
            rotate<false>(x, t.turn, t.mask, t.part);
        }
    }
    uint4 packed;
    __nv_bfloat162* pairs = reinterpret_cast<__nv_bfloat162*>(&packed);
#pragma unroll
    for (int e = 0; e < 4; ++e) pairs[e] = __floats2bfloat162_rn(x[e].x, x[e].y);
    *reinterpret_cast<uint4*>(out + t.part * 8) = packed;
}

// A key, or a value, of kv head `head`.
template <int D, bool STAGED>
__device__ __forceinline__ void store_held(const uint4& raw, bool is_k, int head, const float2 (&weight)[4], const Token<D>& t, float eps,
                                           const float2* __restrict__ cs, int half, double* stage) {
    using Unit = Fp4Unit<D>;
    float2 x[4];
    unpack(x, raw);
    unsigned scale, codes;
    if (is_k && (t.normed || t.turned)) {
        bool sure = false;
        if constexpr (!STAGED) {
            float2 y[4] = {x[0], x[1], x[2], x[3]};
            // a sum of squares outside these bounds may have lost digits to the ends of the range (eps hides a small one)
            bool kept = true;
            if (t.normed) {
                const float ss = norm<D>(y, weight, eps, t.mask);
                kept = ss < 1e36f && (ss > 1e-30f || eps > 1e-20f);
            }
            float widest = 0.f;
            if (t.turned) {
                widest = rotate<true>(y, t.turn, t.mask, t.part);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) widest = fmaxf(widest, fmaxf(fabsf(y[e].x), fabsf(y[e].y)));
            }
            widest = fmaxf(widest, __shfl_xor_sync(t.mask, widest, 1));
            // The sum of squares is off by 12 roundings at most and half of that under the root, the root by 2^-22, the two products and the
            // two of the rotation by one each: less than 2^-20 of |first| + |second|.
            codes = quantise(y, widest * 1.9073486328125e-06f, t.mask, scale, sure);
            sure = __all_sync(t.mask, sure && kept);
        }
        if (!sure) {
            double y[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = e % 2 ? x[e / 2].y : x[e / 2].x;
            if (t.normed) norm<D>(y, weight, eps, t.mask);
            if (t.turned) {
                if constexpr (STAGED) rotate_staged(y, cs, half, t.mask, t.part, stage);
                else rotate(y, t.turn, t.mask, t.part);
            }
            codes = quantise(y, t.mask, scale);
        }
    } else {
        codes = quantise(x, t.mask, scale);
    }
    unsigned char* unit = t.units + (size_t)head * t.head_bytes;
    const int part = t.part, r = t.off_row;
    // eight features are four bytes of one piece: D = 128 has pieces of eight bytes, D = 64 of four
    *reinterpret_cast<unsigned*>(unit + (is_k ? Unit::k_code(r, part * 4) : Unit::v_code(r, part * 4))) = codes;
    if ((part & 1) == 0) unit[is_k ? Unit::k_scale(r, part / 2) : Unit::v_scale(r, part / 2)] = (unsigned char)scale;
}

// A head to every D / 8 lanes.  STAGED: rotary sizes that are no multiple of 16, and weights or tables off 16 bytes; keys in 64 bits throughout (2,048
// tokens of 32 + 8 + 8 heads of 128 under a rotary size of 20 / 126: 32.7 / 46.5 us; 64 tokens 4.5 / 4.7, 3.6 by the other).
template <int D, bool STAGED>
__global__ void __launch_bounds__(STORE_THREADS, STAGED ? 1 : 4)
qk_norm_rope_cache_fp4_kernel(const bf16* qkv, bf16* q_out /* may be qkv */, long q_stride,
                              const float* __restrict__ q_weight, const float* __restrict__ k_weight, float eps,
                              const float2* __restrict__ rot, int half, const int* __restrict__ slots, unsigned char* __restrict__ cache,
                              unsigned groups, int heads, int kv_heads, int page_size, long pages) {
    constexpr int LANES = D / 8;
    __shared__ double stage_all[STAGED ? STORE_THREADS / LANES * D : 1];
    const int per_token = heads + 2 * kv_heads;
    const unsigned group = blockIdx.x * (STORE_THREADS / LANES) + threadIdx.x / LANES;
    if (group >= groups) return;                                   // all lanes of a head together
    const int t = (int)(group / per_token), head = (int)(group - t * per_token), part = threadIdx.x % LANES;
    const uint4 raw = *reinterpret_cast<const uint4*>(qkv + (size_t)group * D + part * 8);
    const bool is_q = head < heads, is_k = !is_q && head < heads + kv_heads;
    // a slot outside the cache (a padding row's -1) writes nothing
    const int slot = is_q || slots == nullptr ? -1 : slots[t];
    const float2* cs = rot + (size_t)t * half;
    const Token<D> token = token_of<D, STAGED>(q_weight, cs, half, half > 0 && (is_q || is_k), slot, cache, kv_heads, page_size, pages);
    double* stage = stage_all + (STAGED ? threadIdx.x / LANES * D : 0);
    if (!is_q && !token.writes) return;
    float2 weight[4];
    if (token.normed && (is_q || is_k)) {
        const float* weights = is_q ? q_weight : k_weight;
        if constexpr (STAGED) {
#pragma unroll
            for (int e = 0; e < 4; ++e) weight[e] = make_float2(weights[part * 8 + 2 * e], weights[part * 8 + 2 * e + 1]);
        } else {
            load8(weight, weights + part * 8);
        }
    }
    if (is_q) store_query<D, STAGED>(raw, weight, token, eps, cs, half, reinterpret_cast<float*>(stage), q_out + (size_t)t * q_stride + (size_t)head * D);
    else store_held<D, STAGED>(raw, is_k, is_k ? head - heads : head - heads - kv_heads, weight, token, eps, cs, half, stage);
}

// `run` heads of a token, one after the other, to every D / 8 lanes; a lane copies its own features of the next heads into shared memory
// meanwhile.  The lanes of a warp have the same heads of several tokens, so that they go the same way; those that quantise begin first.
template <int D>
__global__ void __launch_bounds__(RUN_THREADS, 7)
qk_norm_rope_cache_fp4_runs_kernel(const bf16* qkv, bf16* q_out /* may be qkv */, long q_stride,
                                   const float* __restrict__ q_weight, const float* __restrict__ k_weight, float eps,
                                   const float2* __restrict__ rot, int half, const int* __restrict__ slots, unsigned char* __restrict__ cache,
                                   unsigned tokens, unsigned runs, int run, int heads, int kv_heads, int page_size, long pages) {
    constexpr int LANES = D / 8;
    __shared__ uint4 ring[RUN_DEPTH][RUN_THREADS];
    const int per_token = heads + 2 * kv_heads;
    const unsigned group = blockIdx.x * (RUN_THREADS / LANES) + threadIdx.x / LANES;
    if (group >= tokens * runs) return;                            // all lanes of a run together
    const unsigned before = group / tokens, t = group - before * tokens, part = threadIdx.x % LANES;
    const int first = (int)(runs - 1 - before) * run, end = min(first + run, per_token);
    const bf16* row = qkv + (size_t)t * per_token * D + part * 8;
    auto ask = [&](int head) {
        const unsigned dst = (unsigned)__cvta_generic_to_shared(&ring[(head - first) % RUN_DEPTH][threadIdx.x]);
        if (head < end) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(row + (size_t)head * D) : "memory");
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < RUN_DEPTH - 1; ++i) ask(first + i);
    const int slot = end <= heads || slots == nullptr ? -1 : slots[t];
    const Token<D> token = token_of<D, false>(q_weight, rot + (size_t)t * half, half, half > 0 && first < heads + kv_heads, slot, cache, kv_heads,
                                              page_size, pages);
    float2 weight[4];
    if (token.normed && first < heads + kv_heads) load8(weight, (first < heads ? q_weight : k_weight) + part * 8);
    for (int head = first; head < end; ++head) {
        if (head >= heads && !token.writes) break;                 // keys and values lie behind the queries
        asm volatile("cp.async.wait_group %0;\n" ::"n"(RUN_DEPTH - 2) : "memory");
        const uint4 raw = ring[(head - first) % RUN_DEPTH][threadIdx.x];
        ask(head + RUN_DEPTH - 1);                                 // into the place of the head before, whose features are used
        if (head < heads) {
            store_query<D, false>(raw, weight, token, eps, nullptr, 0, nullptr, q_out + (size_t)t * q_stride + (size_t)head * D);
        } else {
            const bool is_k = head < heads + kv_heads;
            if (token.normed && head == heads) load8(weight, k_weight + part * 8);
            store_held<D, false>(raw, is_k, is_k ? head - heads : head - heads - kv_heads, weight, token, eps, nullptr, 0, nullptr);
        }
    }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
}

// ------------------------------------------------------------------------------------------
// Reading back into rows [page, kv head, row, :] of bfloat16 keys and values (exact: a value has at most 6
// significant bits).  A block takes 16 rows of one kv head, a thread eight features of two keys and two values.
//   ids      output page i is cache page ids[i]
//   spans    the output pages hold the tokens of spans of requests, one span's pages after the other's: tokens `first` .. `end` (a
//            span begins with an output page's first row) of the request in block-table row `row`; rows behind `end`
//            are zeros.  The blocks of the first kv head also write the spans' own block tables ([spans, table_width], -1 in front of
//            `first`) and, for the rows row0 .. row0 + rows of the step, which span they belong to.
// A page outside the cache gives zeros.  What bounds it: 64 pages of 64 rows of 8 heads of 128 (21 MB) take 4.6 us, of which the bytes
// take 3.3; the launch and three latencies (page number, codes, stores) the rest.  Two rows a thread, so that the lanes' 16-byte stores
// are whole rows: a thread with 16 neighbouring features stores half sectors and took 6.8.
// ------------------------------------------------------------------------------------------
constexpr int MAX_SPANS = 64;               // of one launch: they are given by value, so that no copy to the device goes before it
struct Span {
    int row, first, end, page0, row0, rows;  // page0: its first output page
};
struct Spans {
    int n, index0;                          // index0: of the first of them among the call's
    Span span[MAX_SPANS];
    int* table;                             // null: neither is written
    int table_width;
    int* span_of_row;
};

template <int D>
__global__ void __launch_bounds__(D)
fp4_rows_kernel(const unsigned char* __restrict__ cache, const int* __restrict__ ids, const __grid_constant__ Spans spans,
                const int* __restrict__ block_tables, int table_rows, int max_blocks, bf16* __restrict__ k_out, bf16* __restrict__ v_out,
                int kv_heads, int page_size, int out_page, long pages) {
    using Unit = Fp4Unit<D>;
    constexpr int LANES = D / 8;
    const int units_out = out_page / FP4_TOKENS, units_in = page_size / FP4_TOKENS;
    int i = blockIdx.x / units_out;
    const int unit_out = blockIdx.x - i * units_out, kv_head = blockIdx.y;
    const int part = threadIdx.x % LANES, r = threadIdx.x / LANES;
    long page = -1;
    int unit_in = unit_out, rows = FP4_TOKENS;
    if (ids) {
        page = ids[i];
    } else {
        i += spans.span[0].page0;
        int s = 0;
        while (s + 1 < spans.n && spans.span[s + 1].page0 <= i) ++s;
        const Span& span = spans.span[s];
        const int in_span = i - span.page0, unit = span.first / FP4_TOKENS + in_span * units_out + unit_out, block = unit / units_in;
        unit_in = unit - block * units_in;
        rows = span.end - unit * FP4_TOKENS;
        if (rows > 0 && span.row >= 0 && span.row < table_rows && block < max_blocks) page = block_tables[(size_t)span.row * max_blocks + block];
        if (spans.table && kv_head == 0 && unit_out == 0) {
            int* table = spans.table + (size_t)(spans.index0 + s) * spans.table_width;
            const int before = span.first / out_page;
            if (threadIdx.x == 0) table[before + in_span] = i;
            if (in_span == 0) {
                for (int b = threadIdx.x; b < before; b += D) table[b] = -1;
                for (int b = before + (span.end - span.first + out_page - 1) / out_page + threadIdx.x; b < spans.table_width; b += D) table[b] = -1;
                for (int r0 = threadIdx.x; r0 < span.rows; r0 += D) spans.span_of_row[span.row0 + r0] = spans.index0 + s;
            }
        }
    }
    uint4 out[2][2] = {};                          // rows r and r + 8: the key's features, the value's
    if (page >= 0 && page < pages) {
        const unsigned char* unit = cache + ((size_t)(page * kv_heads + kv_head) * units_in + unit_in) * Unit::BYTES;
        unsigned codes[2][2];
        unsigned char bytes[2][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            codes[h][0] = *reinterpret_cast<const unsigned*>(unit + Unit::k_code(r + 8 * h, part * 4));
            codes[h][1] = *reinterpret_cast<const unsigned*>(unit + Unit::v_code(r + 8 * h, part * 4));
            bytes[h][0] = unit[Unit::k_scale(r + 8 * h, part / 2)];
            bytes[h][1] = unit[Unit::v_scale(r + 8 * h, part / 2)];
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (r + 8 * h >= rows) continue;
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                const __half2 scale = __half2half2(__ushort_as_half((unsigned short)(bytes[h][kv] << 7)));
                __nv_bfloat162* pairs = reinterpret_cast<__nv_bfloat162*>(&out[h][kv]);
                unsigned two[4];
                halves_of(codes[h][kv], two);
#pragma unroll
                for (int e = 0; e < 4; ++e)                        // scale times code is a half and a bfloat16
                    pairs[e] = __float22bfloat162_rn(__half22float2(__hmul2(*reinterpret_cast<const __half2*>(&two[e]), scale)));
            }
        }
    }
    const size_t row = ((size_t)i * kv_heads + kv_head) * out_page + unit_out * FP4_TOKENS + r;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        *reinterpret_cast<uint4*>(k_out + (row + 8 * h) * D + part * 8) = out[h][0];
        *reinterpret_cast<uint4*>(v_out + (row + 8 * h) * D + part * 8) = out[h][1];
    }
}

template <int D>
cudaError_t launch_store(const void* qkv, void* q_out, long q_stride, const float* q_weight, const float* k_weight, float eps,
                         const float* rot, int rotary_dim, const int* slots, void* cache, int tokens, int heads, int kv_heads,
                         int page_size, long pages, cudaStream_t stream) {
    const unsigned per_token = (unsigned)(heads + 2 * kv_heads), groups = (unsigned)tokens * per_token;
    const bool staged = rotary_dim % 16 || (((uintptr_t)q_weight | (uintptr_t)k_weight | (uintptr_t)rot) & 15);
    const unsigned run = (groups + HEADS_A_RUN - 1) / HEADS_A_RUN < MOST_A_RUN ? (groups + HEADS_A_RUN - 1) / HEADS_A_RUN : MOST_A_RUN;
    if (!staged && run > 1) {
        constexpr unsigned GROUPS = RUN_THREADS / (D / 8);
        const unsigned runs = (per_token + run - 1) / run;
        return launch_kernel(qk_norm_rope_cache_fp4_runs_kernel<D>, dim3(((unsigned)tokens * runs + GROUPS - 1) / GROUPS), dim3(RUN_THREADS), 0, stream,
                             (const bf16*)qkv, (bf16*)q_out, q_stride, q_weight, k_weight, eps, (const float2*)rot, rotary_dim / 2, slots,
                             (unsigned char*)cache, (unsigned)tokens, runs, (int)run, heads, kv_heads, page_size, pages);
    }
    constexpr unsigned GROUPS = STORE_THREADS / (D / 8);
    return launch_kernel(staged ? qk_norm_rope_cache_fp4_kernel<D, true> : qk_norm_rope_cache_fp4_kernel<D, false>,
                         dim3((groups + GROUPS - 1) / GROUPS), dim3(STORE_THREADS), 0, stream, (const bf16*)qkv, (bf16*)q_out, q_stride,
                         q_weight, k_weight, eps, (const float2*)rot, rotary_dim / 2, slots, (unsigned char*)cache, groups, heads, kv_heads,
                         page_size, pages);
}

int launch_rows(const void* cache, const int* ids, const Spans& spans, const int* block_tables, int table_rows, int max_blocks, void* k_out,
                void* v_out, int n, int kv_heads, int head_dim, int page_size, int out_page, long pages, const char* name, cudaStream_t stream) {
    MRUN_REQUIRE(n >= 0 && kv_heads > 0 && kv_heads < 65536 && pages >= 0, "%s: bad sizes", name);
    MRUN_REQUIRE((((uintptr_t)cache | (uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0, "%s: pages start on 16 bytes", name);
    if (n == 0) return 0;
    const long blocks = (long)n * (out_page / FP4_TOKENS);
    MRUN_REQUIRE(blocks < (1L << 31), "%s: %d pages are more than a launch takes", name, n);
    const dim3 grid((unsigned)blocks, (unsigned)kv_heads);
    const auto launch = [&](auto kernel) {
        return launch_kernel(kernel, grid, dim3(head_dim), 0, stream, (const unsigned char*)cache, ids, spans, block_tables, table_rows,
                             max_blocks, (bf16*)k_out, (bf16*)v_out, kv_heads, page_size, out_page, pages);
    };
    MRUN_CHECK_CUDA(head_dim == 64 ? launch(fp4_rows_kernel<64>) : launch(fp4_rows_kernel<128>), name);
    MRUN_CHECK_LAUNCH(name);
    return 0;
}

}  // namespace

#define MRUN_REQUIRE_FP4(head_dim, page_size, name)                                                                   \
    MRUN_REQUIRE((head_dim) == 64 || (head_dim) == 128, "%s: head_dim=%d: the 4-bit cache takes heads of 64 or 128 features", name, head_dim); \
    MRUN_REQUIRE((page_size) > 0 && (page_size) % mrun::FP4_TOKENS == 0, "%s: page_size=%d is not a multiple of 16", name, page_size)

MRUN_API int mrun_qk_norm_rope_cache_fp4(const void* qkv, void* q_out, long q_stride, const float* q_weight, const float* k_weight,
                                         float eps, const float* rot, int rotary_dim, const int* slots, void* cache, int tokens,
                                         int heads, int kv_heads, int head_dim, int page_size, long pages, cudaStream_t stream) {
    const char* name = "qk_norm_rope_cache_fp4";
    MRUN_REQUIRE(tokens >= 0 && heads > 0 && kv_heads > 0 && pages >= 0, "%s: bad sizes", name);
    MRUN_REQUIRE_FP4(head_dim, page_size, name);
    MRUN_REQUIRE(rotary_dim >= 0 && rotary_dim <= head_dim && rotary_dim % 2 == 0,
                 "%s: rotary_dim=%d must be even and at most head_dim=%d", name, rotary_dim, head_dim);
    MRUN_REQUIRE(rotary_dim == 0 || rot, "%s: rotary_dim=%d without a table", name, rotary_dim);
    MRUN_REQUIRE((q_weight == nullptr) == (k_weight == nullptr), "%s: q and k norm weights come together", name);
    MRUN_REQUIRE(slots == nullptr || cache, "%s: slots without a cache", name);
    MRUN_REQUIRE(((uintptr_t)qkv & 15) == 0 && ((uintptr_t)q_out & 15) == 0 && q_stride % 8 == 0 && ((uintptr_t)cache & 15) == 0,
                 "%s: rows and pages start on 16 bytes", name);
    MRUN_REQUIRE(((uintptr_t)rot & 7) == 0, "%s: the table starts on 8 bytes", name);
    if (tokens == 0) return 0;
    MRUN_REQUIRE((long)tokens * (heads + 2 * kv_heads) < (1L << 31), "%s: %d tokens of %d heads are more than a launch takes", name, tokens, heads);
    auto launch = head_dim == 64 ? launch_store<64> : launch_store<128>;
    MRUN_CHECK_CUDA(launch(qkv, q_out, q_stride, q_weight, k_weight, eps, rot, rotary_dim, slots, cache, tokens, heads, kv_heads, page_size,
                           pages, stream), name);
    MRUN_CHECK_LAUNCH(name);
    return 0;
}

// Output page i is cache page ids[i].
MRUN_API int mrun_fp4_pages(const void* cache, const int* ids, void* k_out, void* v_out, int n, int kv_heads, int head_dim,
                            int page_size, long pages, cudaStream_t stream) {
    const char* name = "fp4_pages";
    MRUN_REQUIRE_FP4(head_dim, page_size, name);
    return launch_rows(cache, ids, Spans{}, nullptr, 0, 0, k_out, v_out, n, kv_heads, head_dim, page_size, page_size, pages, name, stream);
}

// `spans` (host memory): int [n, 6], see Span, in ascending order of their pages and without a gap between them; out_page: rows of an output page.
MRUN_API int mrun_fp4_spans(const void* cache, const int* spans, int n, const int* block_tables, int table_rows, int max_blocks,
                            void* k_out, void* v_out, int* table, int table_width, int* span_of_row, int kv_heads, int head_dim,
                            int page_size, int out_page, long pages, cudaStream_t stream) {
    const char* name = "fp4_spans";
    MRUN_REQUIRE_FP4(head_dim, page_size, name);
    MRUN_REQUIRE(out_page > 0 && out_page % FP4_TOKENS == 0, "%s: out_page=%d", name, out_page);
    MRUN_REQUIRE(n >= 0 && spans && block_tables && (table == nullptr) == (span_of_row == nullptr), "%s: %d spans", name, n);
    int next = 0;
    for (int s = 0; s < n; ++s) {
        const int* v = spans + 6 * s;
        MRUN_REQUIRE(v[1] >= 0 && v[1] % out_page == 0 && v[2] > v[1] && v[3] == next && v[4] >= 0 && v[5] >= 0, "%s: span %d is [%d, %d) at page %d", name, s,
                     v[1], v[2], v[3]);
        next += (v[2] - v[1] + out_page - 1) / out_page;
        MRUN_REQUIRE(table == nullptr || v[1] / out_page + (v[2] - v[1] + out_page - 1) / out_page <= table_width, "%s: table_width=%d", name, table_width);
    }
    for (int first = 0; first < n; first += MAX_SPANS) {
        Spans part = {};
        part.n = n - first < MAX_SPANS ? n - first : MAX_SPANS;
        part.index0 = first;
        part.table = table;
        part.table_width = table_width;
        part.span_of_row = span_of_row;
        for (int s = 0; s < part.n; ++s) {
            const int* v = spans + 6 * (first + s);
            part.span[s] = Span{v[0], v[1], v[2], v[3], v[4], v[5]};
        }
        const int end = first + part.n < n ? spans[6 * (first + part.n) + 3] : next;
        if (int rc = launch_rows(cache, nullptr, part, block_tables, table_rows, max_blocks, k_out, v_out, end - part.span[0].page0, kv_heads,
                                 head_dim, page_size, out_page, pages, name, stream))
            return rc;
    }
    return 0;
}
