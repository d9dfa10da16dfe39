// Attention of single tokens over the 4-bit key/value cache (the format: fp4_unit.cuh).
//
//   o_h = sum_j p_j v_j / sum_j p_j,   p_j = exp2(scale_log2 q_h . k_j - m_h),   j the visible keys whose page is held
//
// What bounds it: a key and its value are 2.25 D / 2 bytes of DRAM, a quarter of their bfloat16 size, so the
// work on them counts.  At 6.5 TB/s a multiprocessor gets a key and value of 128 features every 6 clocks, 42
// codes a clock.  Turned into halves by cvt.e2m1x2 (two codes an instruction, full rate: 21 words of eight codes
// a clock and multiprocessor measured; integer codes by mask and subtraction 9.6) and times their scale
// (exact), they are operands of mma.m16n8k16, whose 16 rows are keys or features and whose 8 columns are the
// query heads of a kv head:
//   S^T [16 keys x 8 heads]     = K Q^T      A = the keys as they lie in the page, B = the queries (registers)
//   O^T [32 features x 8 heads] += V^T P^T   A = the values as they lie in the page: a register holds two
//                                            neighbouring features of one key, not two keys of one feature.
// The second product gets its sum over keys all the same: its k index is (key, parity of the feature), and P is
// given twice, once with zeros in the places of the odd parity (giving the even features) and once
// with zeros in those of the even one.  That is twice the products (24 for 16 keys, a quarter of the tensor
// pipe's time at the memory's rate) and no permutation of the values.
// P comes out of the first product by rows and goes into the second by columns: one movmatrix for 8 keys.
// Queries are scaled by a power of two into a half's range (exact for 24 binary digits below the largest);
// P carries a factor of 32, so that a half keeps its digits down to 2^-19 of the running maximum, which is raised
// only when a score passes it by 8 (base 2).
//
// A block is four warps; each copies its own units (16 keys) with cp.async into a ring of its own, several
// ahead, across pairs: no barrier but where a pair's pieces meet.  Every warp of a block works on the same
// (token, kv head, group of heads) pair.  The tiles (4 units) of all pairs lie in one list, cut evenly among the
// blocks that the device holds at once; a pair that lies in several blocks leaves its pieces in scratch, and
// a second kernel adds them in block order.
#include <cuda_fp16.h>

#include "attention_paging.cuh"
#include "common.cuh"
#include "fp4_unit.cuh"

namespace {

using namespace mrun;
using bf16 = __nv_bfloat16;

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int RING = 4;                 // units that a warp has under way or in work
constexpr int UNITS_A_TILE = WARPS;
constexpr int TILE_KEYS = UNITS_A_TILE * FP4_TOKENS;
constexpr int MAX_TOKENS = 512;         // tokens of one launch (their prefix lies in shared memory beside the rings of four blocks)
constexpr float LIFT = 5.f;             // log2 of the factor that P carries
constexpr float SLACK = 8.f;            // how far a score may pass the running maximum (base 2)

__device__ __forceinline__ unsigned smem_addr(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async_16(unsigned dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_f16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transposed(unsigned rows) {
    unsigned out;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(out) : "r"(rows));
    return out;
}
__device__ __forceinline__ unsigned mul_h2(unsigned a, unsigned b) {
    unsigned out;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(out) : "r"(a), "r"(b));
    return out;
}
__device__ __forceinline__ unsigned pack_h2(float lo, float hi) {
    unsigned out;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(out) : "f"(hi), "f"(lo));
    return out;
}
__device__ __forceinline__ float exp2_fast(float v) {
    float out;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(out) : "f"(v));
    return out;
}
// The eight codes of a word as four pairs of halves.
__device__ __forceinline__ void halves_of(unsigned word, unsigned (&h)[4]) {
    asm("{\n.reg .b8 c0, c1, c2, c3;\nmov.b32 {c0, c1, c2, c3}, %4;\n"
        "cvt.rn.f16x2.e2m1x2 %0, c0;\ncvt.rn.f16x2.e2m1x2 %1, c1;\ncvt.rn.f16x2.e2m1x2 %2, c2;\ncvt.rn.f16x2.e2m1x2 %3, c3;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(word));
}
// Byte `i` of `bytes`, a scale, as the same half twice.
template <int I> __device__ __forceinline__ unsigned scale_twice(unsigned bytes) {
    return __byte_perm(bytes, 0u, (I << 12) | (4 << 8) | (I << 4) | 4) >> 1;
}

// Tiles of a token that sees the keys from the first visible one to its own position.
__device__ __forceinline__ int tiles_of(int pos, int window) {
    if (pos < 0) return 0;
    const int units = pos / FP4_TOKENS - first_visible(pos, window) / FP4_TOKENS + 1;
    return (units + UNITS_A_TILE - 1) / UNITS_A_TILE;
}

// One (token, kv head, group of heads) pair's part of a block's range.
struct Piece {
    int tok, kvh, hg;            // the pair
    int tile0, tiles;            // its first tile here and their number
    bool complete;               // all of the pair's tiles
};
struct Cursor {
    int tok, rest;               // token, and the tile inside the token's tiles over all its kv heads and head groups
};

// The piece that begins at `at` and holds at most `left` tiles; `at` is moved behind it.
__device__ __forceinline__ Piece next_piece(Cursor& at, int left, const int* prefix, int kv_heads, int head_groups) {
    while (true) {
        const int tiles = prefix[at.tok + 1] - prefix[at.tok];
        if (at.rest < tiles * kv_heads * head_groups) {
            Piece p;
            p.tok = at.tok;
            const int pair = at.rest / tiles;
            p.kvh = pair / head_groups;
            p.hg = pair - p.kvh * head_groups;
            p.tile0 = at.rest - pair * tiles;
            p.tiles = min(left, tiles - p.tile0);
            p.complete = p.tiles == tiles;
            at.rest += p.tiles;
            return p;
        }
        at.rest -= tiles * kv_heads * head_groups;
        ++at.tok;
    }
}

template <int D, int NT>
struct Shared {
    static constexpr int ROW = D + 4;                                            // a head's values, maximum, sum
    static constexpr int RING_BYTES = WARPS * RING * Fp4Unit<D>::BYTES;
    static constexpr int MERGE_BYTES = WARPS * 8 * NT * ROW * 4;
    static size_t bytes(int tokens) { return RING_BYTES + MERGE_BYTES + (size_t)(tokens + 1) * 4; }
};

// Sums tiles_of over the tokens into prefix[0 .. tokens]; all threads of the block, `scratch` of 33 ints.
__device__ __forceinline__ void make_prefix(int* prefix, const int* __restrict__ positions, int tokens, int window, int* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int carried = 0;
    if (threadIdx.x == 0) prefix[0] = 0;
    for (int first = 0; first < tokens; first += THREADS) {
        const int t = first + threadIdx.x;
        int sum = t < tokens ? tiles_of(positions[t], window) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int below = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += below;
        }
        if (lane == 31) scratch[warp] = sum;
        __syncthreads();
        int before = carried;
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) before += scratch[w];
            carried += scratch[w];
        }
        if (t < tokens) prefix[t + 1] = before + sum;
        __syncthreads();
    }
    __syncthreads();
}

// Tiles that a block takes.
__device__ __forceinline__ int tiles_a_block(long total, int blocks) { return (int)((total + blocks - 1) / blocks); }

struct Step {
    const int* block_tables;
    const int* token_slot;
    const int* positions;
    const int* rows;             // the rows of q and out that the tokens are, or null: the first ones
    int max_blocks, table_rows, tokens, heads, kv_heads, page_size, window;
    long pages, q_stride;
    float scale_log2;
};

template <int D, int NT>
__global__ void __launch_bounds__(THREADS, NT == 1 ? 4 : 3)
decode_fp4_kernel(const bf16* __restrict__ q, bf16* __restrict__ out, const unsigned char* __restrict__ cache, const Step step,
                  float* __restrict__ part_o, float2* __restrict__ part_ml) {
    using Unit = Fp4Unit<D>;
    using Sh = Shared<D, NT>;
    constexpr int HEADS = 8 * NT, WORDS_K = D / 32, WORDS_V = D / 64, TILES_M = D / 32;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ int scratch[WARPS];
    float* merge = reinterpret_cast<float*>(smem + Sh::RING_BYTES);              // [WARPS][HEADS][ROW]
    int* prefix = reinterpret_cast<int*>(smem + Sh::RING_BYTES + Sh::MERGE_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = smem + warp * RING * Unit::BYTES;
    const int group = step.heads / step.kv_heads, head_groups = (group + HEADS - 1) / HEADS;
    const int units_a_page = step.page_size / FP4_TOKENS;

    make_prefix(prefix, step.positions, step.tokens, step.window, scratch);
    // padding rows come out as zeros
    for (int tok = blockIdx.x; tok < step.tokens; tok += gridDim.x)
        if (step.positions[tok] < 0)
            for (int i = threadIdx.x; i < step.heads * D / 2; i += THREADS)
                reinterpret_cast<unsigned*>(out + (size_t)(step.rows ? step.rows[tok] : tok) * step.heads * D)[i] = 0u;

    const long total = (long)prefix[step.tokens] * step.kv_heads * head_groups;
    const int per = tiles_a_block(total, gridDim.x);
    const long begin = (long)blockIdx.x * per;
    if (begin >= total) return;
    const int count = (int)min((long)per, total - begin);
    Cursor start;
    {   // the token whose tiles hold the block's first one
        int low = 0, high = step.tokens - 1;
        while (low < high) {
            const int mid = (low + high) / 2;
            if ((long)prefix[mid + 1] * step.kv_heads * head_groups <= begin) low = mid + 1;
            else high = mid;
        }
        start.tok = low;
        start.rest = (int)(begin - (long)prefix[low] * step.kv_heads * head_groups);
    }

    // ---- the copies: this warp's unit of every tile, RING - 1 ahead of the work
    Cursor ahead = start;
    Piece ap = {};
    int ap_tile = 0, issued = 0;
    int a_pos = -1, a_first = 0;                       // of the token whose units are copied
    const int* a_table = nullptr;
    unsigned held = 0;                                 // bit i: the unit in stage i is there
    auto issue = [&]() {
        const int s = issued % RING;
        held &= ~(1u << s);
        if (issued < count) {
            if (ap_tile == ap.tiles) {
                ap = next_piece(ahead, count - issued, prefix, step.kv_heads, head_groups);
                ap_tile = 0;
                a_pos = step.positions[ap.tok];
                a_first = first_visible(a_pos, step.window) / FP4_TOKENS;
                const int slot = step.token_slot[ap.tok];
                a_table = slot >= 0 && slot < step.table_rows ? step.block_tables + (size_t)slot * step.max_blocks : nullptr;
            }
            const int unit = a_first + (ap.tile0 + ap_tile) * UNITS_A_TILE + warp;
            const int block = unit / units_a_page;
            if (unit <= a_pos / FP4_TOKENS && a_table && block < step.max_blocks) {
                const int page = a_table[block];
                if (page >= 0 && page < step.pages) {
                    const unsigned char* src = cache + (((size_t)page * step.kv_heads + ap.kvh) * units_a_page + (unit - block * units_a_page)) * Unit::BYTES;
                    const unsigned dst = smem_addr(ring + s * Unit::BYTES);
#pragma unroll
                    for (int c = 0; c < Unit::BYTES / 512; ++c) cp_async_16(dst + (c * 32 + lane) * 16, src + (c * 32 + lane) * 16);
                    if (lane < Unit::BYTES % 512 / 16)
                        cp_async_16(dst + (Unit::BYTES / 512 * 32 + lane) * 16, src + (Unit::BYTES / 512 * 32 + lane) * 16);
                    held |= 1u << s;
                }
            }
            ++ap_tile;
        }
        cp_async_commit();
        ++issued;
    };
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) issue();

    Cursor at = start;
    for (int done = 0, seg = 0; done < count; ++seg) {
        const Piece p = next_piece(at, count - done, prefix, step.kv_heads, head_groups);
        const int pos = step.positions[p.tok], lo = first_visible(pos, step.window), first_unit = lo / FP4_TOKENS;
        const size_t row = step.rows ? step.rows[p.tok] : p.tok;
        const int head0 = p.kvh * group + p.hg * HEADS, heads_here = min(HEADS, group - p.hg * HEADS);

        // the queries: lane 4 g + t has features D/4 t .. of head g, as halves with the largest of the head in [128, 256)
        unsigned qf[NT][D / 16][2];
        float scale[NT][2];                                // of the scores of heads 2 t and 2 t + 1
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int h = nt * 8 + g;
            const bf16* src = q + row * step.q_stride + (size_t)(head0 + h) * D + t * (D / 4);
            uint4 raw[D / 32];
            float largest = 0.f;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                raw[c] = make_uint4(0, 0, 0, 0);
                if (h < heads_here) raw[c] = *reinterpret_cast<const uint4*>(src + c * 8);
                const __nv_bfloat162* pairs = reinterpret_cast<const __nv_bfloat162*>(&raw[c]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = __bfloat1622float2(pairs[e]);
                    largest = fmaxf(largest, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
            }
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
            // 2^(7 - exponent) and its inverse; a head of zeros or with an infinity stays as it is
            int ex = (int)(__float_as_uint(largest) >> 23);
            ex = ex == 255 || largest == 0.f ? 134 : max(ex, 8);
            const float up = __uint_as_float((unsigned)(261 - ex) << 23), down = __uint_as_float((unsigned)(ex - 7) << 23);
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                const __nv_bfloat162* pairs = reinterpret_cast<const __nv_bfloat162*>(&raw[c]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = __bfloat1622float2(pairs[e]);
                    qf[nt][c * 2 + (e >> 1)][e & 1] = pack_h2(f.x * up, f.y * up);
                }
            }
            scale[nt][0] = __shfl_sync(0xffffffffu, down, 8 * t) * step.scale_log2;
            scale[nt][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4) * step.scale_log2;
        }

        float m[NT][2], l[NT][2], o[NT][TILES_M][2][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < TILES_M; ++i)
#pragma unroll
                for (int e = 0; e < 2; ++e) o[nt][i][e][0] = o[nt][i][e][1] = o[nt][i][e][2] = o[nt][i][e][3] = 0.f;
        }

        for (int tile = p.tile0; tile < p.tile0 + p.tiles; ++tile, ++done) {
            __syncwarp();                                  // the stage that is filled next was read by all lanes
            issue();
            const int s = done % RING;
            cp_async_wait<RING - 1>();
            __syncwarp();
            if (!((held >> s) & 1u)) continue;
            const unsigned char* unit = ring + s * Unit::BYTES;
            const int key0 = (first_unit + tile * UNITS_A_TILE + warp) * FP4_TOKENS;

            // ---- scores
            float c[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.f;
            {
                unsigned kw[2][WORDS_K];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const unsigned char* src = unit + Unit::k_code(r * 8 + g, t * (D / 8));
                    if constexpr (D == 128) *reinterpret_cast<uint4*>(kw[r]) = *reinterpret_cast<const uint4*>(src);
                    else *reinterpret_cast<uint2*>(kw[r]) = *reinterpret_cast<const uint2*>(src);
                }
                unsigned ks;                               // bytes: D = 128 [token g: 2, token g + 8: 2], D = 64 [1, 1]
                if constexpr (D == 128) ks = *reinterpret_cast<const unsigned*>(unit + Unit::K_SCALES + lane * 4);
                else ks = *reinterpret_cast<const unsigned short*>(unit + Unit::K_SCALES + lane * 2);
                unsigned sc[2][Unit::PER];
                if constexpr (D == 128) {
                    sc[0][0] = scale_twice<0>(ks); sc[0][Unit::PER - 1] = scale_twice<1>(ks);
                    sc[1][0] = scale_twice<2>(ks); sc[1][Unit::PER - 1] = scale_twice<3>(ks);
                } else {
                    sc[0][0] = scale_twice<0>(ks); sc[1][0] = scale_twice<1>(ks);
                }
#pragma unroll
                for (int w = 0; w < WORDS_K; ++w) {
                    unsigned a[2][4];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        halves_of(kw[r][w], a[r]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) a[r][i] = mul_h2(a[r][i], sc[r][w / 2]);
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma_f16(c[nt], a[0][2 * j], a[1][2 * j], a[0][2 * j + 1], a[1][2 * j + 1], qf[nt][2 * w + j][0], qf[nt][2 * w + j][1]);
                }
            }
            const bool whole = key0 >= lo && key0 + FP4_TOKENS - 1 <= pos;
            bool raise = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = c[nt][e] * scale[nt][e & 1];
                    if (!whole) {
                        const int key = key0 + g + (e >> 1) * 8;
                        if (key > pos || key < lo) v = -INFINITY;
                    }
                    c[nt][e] = v;
                    raise = raise || v > m[nt][e & 1] + SLACK;
                }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float mx = fmaxf(c[nt][h], c[nt][h + 2]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        mx = fmaxf(mx, m[nt][h]);
                        const float corr = m[nt][h] == -INFINITY ? 0.f : exp2_fast(m[nt][h] - mx);
                        m[nt][h] = mx;
                        l[nt][h] *= corr;
#pragma unroll
                        for (int i = 0; i < TILES_M; ++i)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                o[nt][i][e][h] *= corr;
                                o[nt][i][e][h + 2] *= corr;
                            }
                    }
            }
            unsigned pt[NT][2];                            // lane 4 g + t: keys 2 t and 2 t + 1 (then + 8) of head g
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float base[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) base[h] = m[nt][h] == -INFINITY ? 0.f : m[nt][h] - LIFT;
                float pr[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) pr[e] = exp2_fast(c[nt][e] - base[e & 1]);
                l[nt][0] += pr[0] + pr[2];
                l[nt][1] += pr[1] + pr[3];
                pt[nt][0] = transposed(pack_h2(pr[0], pr[1]));
                pt[nt][1] = transposed(pack_h2(pr[2], pr[3]));
            }

            // ---- values
            unsigned vs = *reinterpret_cast<const unsigned*>(unit + Unit::V_SCALES + (D == 128 ? lane : (g >> 1) * 4 + t) * 4);
            if (!whole) {
                // a key that is not seen may lie in memory that nothing has written: 0 times its value must be 0
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const int key = key0 + (b >> 1) * 8 + 2 * t + (b & 1);
                    if (key > pos || key < lo) vs &= ~(0xFFu << (8 * b));
                }
            }
            const unsigned sv[4] = {scale_twice<0>(vs), scale_twice<1>(vs), scale_twice<2>(vs), scale_twice<3>(vs)};
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                unsigned vw[2][WORDS_V];                   // of tokens 2 t and 2 t + 1 (+ 8 half)
                const unsigned char* src = unit + Unit::V_CODES + half * (4 * D) + lane * 2 * Unit::PIECE;
                if constexpr (D == 128) *reinterpret_cast<uint4*>(vw) = *reinterpret_cast<const uint4*>(src);
                else *reinterpret_cast<uint2*>(vw) = *reinterpret_cast<const uint2*>(src);
                unsigned be[NT][2], bo[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    be[nt][0] = pt[nt][half] & 0xffffu; be[nt][1] = pt[nt][half] >> 16;
                    bo[nt][0] = pt[nt][half] << 16;     bo[nt][1] = pt[nt][half] & 0xffff0000u;
                }
#pragma unroll
                for (int w = 0; w < WORDS_V; ++w) {
                    unsigned a[2][4];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        halves_of(vw[r][w], a[r]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) a[r][i] = mul_h2(a[r][i], sv[half * 2 + r]);
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma_f16(o[nt][2 * w + j][0], a[0][2 * j], a[0][2 * j + 1], a[1][2 * j], a[1][2 * j + 1], be[nt][0], be[nt][1]);
                            mma_f16(o[nt][2 * w + j][1], a[0][2 * j], a[0][2 * j + 1], a[1][2 * j], a[1][2 * j + 1], bo[nt][0], bo[nt][1]);
                        }
                }
            }
        }

        // ---- the four warps' results meet
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], 4);
                l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], 8);
                l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], 16);
                const int head = nt * 8 + 2 * t + h;
                float* dst = merge + (warp * HEADS + head) * Sh::ROW;
                if (head < heads_here) {
#pragma unroll
                    for (int i = 0; i < TILES_M; ++i)      // features D/8 g + 4 i ..
                        *reinterpret_cast<float4*>(dst + g * (D / 8) + 4 * i) =
                            make_float4(o[nt][i][0][h], o[nt][i][1][h], o[nt][i][0][h + 2], o[nt][i][1][h + 2]);
                    if (g == 0) {
                        dst[D] = m[nt][h];
                        dst[D + 1] = l[nt][h];
                    }
                }
            }
        __syncthreads();
        const size_t my = (size_t)blockIdx.x * 2 + (seg == 0 ? 0 : 1);
        for (int i = threadIdx.x; i < heads_here * (D / 4); i += THREADS) {
            const int head = i / (D / 4), d = (i - head * (D / 4)) * 4;
            float mm = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, merge[(w * HEADS + head) * Sh::ROW + D]);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            float ll = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float* src = merge + (w * HEADS + head) * Sh::ROW;
                const float f = src[D] == -INFINITY ? (src[D + 1] == 0.f ? 0.f : 1.f) : exp2f(src[D] - mm);
                const float4 v = *reinterpret_cast<const float4*>(src + d);
                acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
                ll += src[D + 1] * f;
            }
            if (p.complete) {
                const float inv = ll == 0.f ? 0.f : 1.f / ll;
                __nv_bfloat162 pair[2] = {__floats2bfloat162_rn(acc.x * inv, acc.y * inv), __floats2bfloat162_rn(acc.z * inv, acc.w * inv)};
                *reinterpret_cast<uint2*>(out + row * step.heads * D + (size_t)(head0 + head) * D + d) = *reinterpret_cast<uint2*>(pair);
            } else {
                *reinterpret_cast<float4*>(part_o + (my * HEADS + head) * D + d) = acc;
                if (d == 0) part_ml[my * HEADS + head] = make_float2(mm, ll);
            }
        }
        __syncthreads();
    }
    cp_async_wait<0>();
}

// Adds the pieces of the pairs that lie in several blocks, in block order.  A block takes a pair.
template <int D, int NT>
__global__ void __launch_bounds__(THREADS)
merge_fp4_kernel(bf16* __restrict__ out, const Step step, const float* __restrict__ part_o, const float2* __restrict__ part_ml, int blocks) {
    constexpr int HEADS = 8 * NT;
    __shared__ int scratch[WARPS];
    extern __shared__ int prefix[];
    wait_for_kernel_before();
    make_prefix(prefix, step.positions, step.tokens, step.window, scratch);
    const int group = step.heads / step.kv_heads, head_groups = (group + HEADS - 1) / HEADS;
    const int pairs = step.kv_heads * head_groups;
    const int tok = blockIdx.x / pairs, pair = blockIdx.x - tok * pairs;
    const long total = (long)prefix[step.tokens] * pairs;
    const int per = tiles_a_block(total, blocks), tiles = prefix[tok + 1] - prefix[tok];
    if (tiles == 0) return;
    const long start = (long)prefix[tok] * pairs + (long)pair * tiles;
    const int first = (int)(start / per), last = (int)((start + tiles - 1) / per);
    if (first == last) return;
    const int kvh = pair / head_groups, hg = pair - kvh * head_groups;
    const int heads_here = min(HEADS, group - hg * HEADS);
    const size_t row = step.rows ? step.rows[tok] : tok;
    // a block's piece of this pair is its first one where its range begins inside the pair
    auto slot = [&](int b) { return (size_t)b * 2 + ((long)b * per >= start ? 0 : 1); };
    for (int i = threadIdx.x; i < heads_here * (D / 4); i += THREADS) {
        const int head = i / (D / 4), d = (i - head * (D / 4)) * 4;
        float mm = -INFINITY;
        for (int b = first; b <= last; ++b) mm = fmaxf(mm, part_ml[slot(b) * HEADS + head].x);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float ll = 0.f;
        for (int b = first; b <= last; ++b) {
            const float2 ml = part_ml[slot(b) * HEADS + head];
            const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : exp2f(ml.x - mm);
            const float4 v = *reinterpret_cast<const float4*>(part_o + (slot(b) * HEADS + head) * D + d);
            acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
            ll += ml.y * f;
        }
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        __nv_bfloat162 two[2] = {__floats2bfloat162_rn(acc.x * inv, acc.y * inv), __floats2bfloat162_rn(acc.z * inv, acc.w * inv)};
        *reinterpret_cast<uint2*>(out + row * step.heads * D + (size_t)(kvh * group + hg * HEADS + head) * D + d) = *reinterpret_cast<uint2*>(two);
    }
}

template <int D, int NT>
cudaError_t launch_decode(const bf16* q, bf16* out, const unsigned char* cache, const Step& step, float* part_o, float* part_ml, int blocks,
                          cudaStream_t stream) {
    const size_t smem = Shared<D, NT>::bytes(step.tokens);
    cudaError_t err = cudaFuncSetAttribute(decode_fp4_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shared<D, NT>::bytes(MAX_TOKENS));
    if (err != cudaSuccess) return err;
    err = launch_kernel(decode_fp4_kernel<D, NT>, dim3(blocks), dim3(THREADS), smem, stream, q, out, cache, step, part_o, (float2*)part_ml);
    if (err != cudaSuccess) return err;
    const int group = step.heads / step.kv_heads, head_groups = (group + 8 * NT - 1) / (8 * NT);
    return launch_kernel_overlapped(merge_fp4_kernel<D, NT>, dim3(step.tokens * step.kv_heads * head_groups), dim3(THREADS),
                                    (size_t)(step.tokens + 1) * 4, stream, out, step, part_o, (const float2*)part_ml, blocks);
}

template <int D, int NT> int occupancy() {
    int n = 0;
    cudaFuncSetAttribute(decode_fp4_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shared<D, NT>::bytes(MAX_TOKENS));
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, decode_fp4_kernel<D, NT>, THREADS, Shared<D, NT>::bytes(MAX_TOKENS)) != cudaSuccess) return 0;
    return n;
}

}  // namespace

// Blocks of the decode kernel that a multiprocessor holds at once; 0: the device refuses.
MRUN_API int mrun_attn_fp4_occupancy(int head_dim, int group) {
    return head_dim == 64 ? (group <= 8 ? occupancy<64, 1>() : occupancy<64, 2>()) : (group <= 8 ? occupancy<128, 1>() : occupancy<128, 2>());
}

// part_o: float [blocks, 2, heads a block, head_dim]; part_ml: float [blocks, 2, heads a block, 2].
MRUN_API int mrun_attn_fp4_decode(const void* q, long q_stride, void* out, const void* cache, const int* block_tables, int table_rows,
                                  int max_blocks, const int* token_slot, const int* positions, const int* rows, int tokens, int heads,
                                  int kv_heads, int head_dim, int page_size, long pages, float scale, int window, float* part_o,
                                  float* part_ml, int blocks, cudaStream_t stream) {
    const char* name = "paged_attention_fp4";
    MRUN_REQUIRE(tokens >= 0 && tokens <= MAX_TOKENS, "%s: %d tokens, a launch takes up to %d", name, tokens, MAX_TOKENS);
    MRUN_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && blocks > 0 && pages >= 0 && max_blocks >= 0 && table_rows >= 0,
                 "%s: bad sizes", name);
    MRUN_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim=%d: the 4-bit cache takes heads of 64 or 128 features", name, head_dim);
    MRUN_REQUIRE(page_size > 0 && page_size % FP4_TOKENS == 0, "%s: page_size=%d is not a multiple of 16", name, page_size);
    MRUN_REQUIRE((((uintptr_t)q | (uintptr_t)out | (uintptr_t)cache | (uintptr_t)part_o) & 15) == 0 && q_stride % 8 == 0,
                 "%s: rows and pages start on 16 bytes", name);
    if (tokens == 0) return 0;
    Step step = {block_tables, token_slot, positions, rows, max_blocks, table_rows, tokens, heads, kv_heads, page_size, window,
                 pages, q_stride, scale * 1.4426950408889634f};
    auto launch = head_dim == 64 ? (heads / kv_heads <= 8 ? launch_decode<64, 1> : launch_decode<64, 2>)
                                 : (heads / kv_heads <= 8 ? launch_decode<128, 1> : launch_decode<128, 2>);
    MRUN_CHECK_CUDA(launch((const bf16*)q, (bf16*)out, (const unsigned char*)cache, step, part_o, part_ml, blocks, stream), name);
    MRUN_CHECK_LAUNCH(name);
    return 0;
}
