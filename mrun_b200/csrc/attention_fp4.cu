// Attention of single tokens over the 4-bit key/value cache (the format: fp4_unit.cuh).
//
//   o_h = sum_j p_j v_j / sum_j p_j,   p_j = exp2(scale_log2 q_h . k_j - m_h),   j the visible keys whose page is held
//
// What bounds it: a key and its value are 9/8 D bytes of DRAM, 3.6 times fewer than in bfloat16, so the
// work on them counts.  At 6.5 TB/s a multiprocessor gets a key and value of 128 features every 6 clocks, 42
// codes a clock.  cvt.e2m1x2 makes two halves of a byte in one instruction of the integer pipe (two a clock and
// multiprocessor; integer codes by mask and subtraction take three times as many); times their scale (exact) they are
// operands of mma.m16n8k16, whose 16 rows are keys or features and whose 8 columns are query heads of a kv head:
//   S^T [16 keys x 8]     = K Q^T      A = the keys as they lie in the page, B = the queries (registers)
//   O^T [32 features x 8] += V^T P^T   A = the values as they lie in the page: a register holds two
//                                      neighbouring features of one key, not two keys of one feature.
// The second product gets its sum over keys all the same: its k index is (key, parity of the feature), and a column
// of P has zeros in the places of one parity, so that it gives the features of the other.  A group of up to four query
// heads has both columns of a head in one product (the tensor pipe is 28 % busy); a wider one takes two products, one a parity, and
// no permutation of the values.
// P comes out of the first product by rows and goes into the second by columns: one movmatrix for 8 keys.
// Queries are scaled by a power of two into a half's range (exact for 24 binary digits below the largest);
// P carries a factor of 32, so that a half keeps its digits down to 2^-19 of the running maximum, which is raised
// only when a score passes it by 8 (base 2).
//
// A block is four warps; each copies its own units (two at a time, 32 keys) with cp.async into a ring of its own while it
// works on the two before, across pairs: no barrier but where a pair's pieces meet.  Every warp of a block works on the same
// (token, kv head, group of heads) pair.  The tiles (8 units) of short contexts are cut among the one to eight blocks of a pair's
// cluster, which add their pieces through distributed shared memory.  Those of long ones lie in one list, cut evenly among the
// blocks that the device holds at once (by whole pairs, where that is nearly even, 64 requests of 8,192 keys take 115 us and not 107); a pair that
// lies in several blocks leaves its pieces in scratch, and a second kernel, whose launch overlaps the first one's end, adds them in block order.
//
// Measured (B200): 64 requests of up to 8,192 keys, 32 heads over 8 of 128 (456 MB): 81 us at 1,965 MHz, 5.6 TB/s, the start (positions, pages, first keys)
// and the second launch among them.  267 instructions a unit, 64 of them conversions (the integer pipe
// is 48 % busy) and 64 multiplications.  In a run of seconds the power cap brings the clock to 1,600 MHz.
// One request of 1,024 keys: 5.6 us, a chain of latencies.  A ring of three stages, twelve warps a multiprocessor instead of sixteen, pages of 64
// or 256 keys: the same within 2 %.
#include <atomic>
#include <cfloat>
#include <cuda_fp16.h>

#include "attention_paging.cuh"
#include "common.cuh"
#include "fp4_unit.cuh"

namespace {

using namespace mrun;
using bf16 = __nv_bfloat16;

constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int UNITS = 2;                // units that a warp takes at a time
constexpr int STAGES = 2;
constexpr int UNITS_A_TILE = WARPS * UNITS;
constexpr int MAX_TOKENS = 256;         // tokens of one launch (their plan lies in shared memory beside the rings of four blocks)
constexpr int MERGE_THREADS = 128;
constexpr int MAX_CLUSTER = 8;          // blocks of a cluster that every device takes
constexpr float LIFT = 5.f;             // log2 of the factor that P carries
constexpr float SLACK = 8.f;            // how far a score may pass the running maximum (base 2)

__device__ __forceinline__ unsigned smem_addr(const void* p) { return (unsigned)__cvta_generic_to_shared(p); }
// 16 bytes, or with bytes = 0 zeros, the source not read
__device__ __forceinline__ void cp_async_16(unsigned dst, const void* src, unsigned bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma_f16(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with nothing to add to.
__device__ __forceinline__ void mma_f16_first(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ unsigned transposed(unsigned rows) {
    unsigned out;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(out) : "r"(rows));
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
// Bytes I and I + 1 of `bytes`, scales, as halves.
template <int I> __device__ __forceinline__ __half2 two_scales(unsigned bytes) {
    const unsigned bits = __byte_perm(bytes, 0u, ((I + 1) << 12) | (4 << 8) | (I << 4) | 4) >> 1;
    return *reinterpret_cast<const __half2*>(&bits);
}
// Both halves of `codes` times one of two scales, which the multiplication picks itself.
__device__ __forceinline__ unsigned scaled(unsigned codes, __half2 scales, int which) {
    const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&codes), which ? __high2half2(scales) : __low2half2(scales));
    return *reinterpret_cast<const unsigned*>(&v);
}

// A score less the maximum it is taken against.  The product is rounded as the maximum's was: fused, the difference of a huge
// score and its own rounding would stand in the exponent.
__device__ __forceinline__ float against(float product, float scale, float nbase) { return __fadd_rn(__fmul_rn(product, scale), nbase); }

// The weight of a part whose maximum is m beside one of maximum `top`.  A part without keys has m = -inf and l = 0; one whose
// scores are all NaN has m = -inf and l = NaN, and keeps it.
__device__ __forceinline__ float weight_of(float m, float l, float top) {
    return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : exp2_fast(m - top);
}

__device__ __forceinline__ void store_row(bf16* dst, float4 acc, float l) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    __nv_bfloat162 two[2] = {__floats2bfloat162_rn(acc.x * inv, acc.y * inv), __floats2bfloat162_rn(acc.z * inv, acc.w * inv)};
    *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(two);
}

// Powers of two that bring a head's queries, the largest of them `largest`, into [128, 256) and its scores back; a head of zeros or with an
// infinity stays as it is.
struct Powers {
    float up, down;
};
__device__ __forceinline__ Powers powers_of(float largest) {
    int ex = (int)(__float_as_uint(largest) >> 23);
    ex = ex == 255 || largest == 0.f ? 134 : max(ex, 8);
    return {__uint_as_float((unsigned)(261 - ex) << 23), __uint_as_float((unsigned)(ex - 7) << 23)};
}

// What a product with such queries is multiplied by.  Never 0, which would make NaN of a hidden key's score (a head that small has scores of 0
// either way), nor infinite, which would make NaN of a key of zeros (any other score of such a head is beyond 32 bits either way).
__device__ __forceinline__ float score_scale(float down, float scale_log2) { return fminf(fmaxf(down * scale_log2, FLT_MIN), FLT_MAX); }

// Tiles of a token that sees the keys from the first visible one to its own position, as far as its block table goes.
__device__ __forceinline__ int tiles_of(int pos, int window, int table_units) {
    if (pos < 0) return 0;
    const int units = min(pos / FP4_TOKENS, table_units - 1) - first_visible(pos, window) / FP4_TOKENS + 1;
    return units <= 0 ? 0 : (units + UNITS_A_TILE - 1) / UNITS_A_TILE;
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
            p.kvh = head_groups == 1 ? pair : pair / head_groups;
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

// FOUR: up to four query heads, each with both of its columns in one product; else up to eight.
template <int D, bool FOUR>
struct Shape {
    static constexpr int HEADS = FOUR ? 4 : 8;
    static constexpr int MINE = FOUR ? 1 : 2;                                    // heads whose scores a lane holds
    static constexpr int ROW = D + 4;                                            // a head's values, maximum, sum
    static constexpr int RING_BYTES = WARPS * STAGES * UNITS * Fp4Unit<D>::BYTES;
    static constexpr int MERGE_BYTES = WARPS * HEADS * ROW * 4;
    // ... and per token its prefix of tiles, position and block-table row
    static size_t bytes(int tokens) { return RING_BYTES + MERGE_BYTES + (size_t)(3 * tokens + 1) * 4; }        // a cluster's blocks: 0 tokens
};

// Which rows of the step a launch's tokens are: the first ones, or (listed) these, given by value so that no copy
// to the device goes before the launch.
struct Rows {
    int listed;
    int row[MAX_TOKENS];
    __device__ __forceinline__ int of(int tok) const { return listed ? row[tok] : tok; }
};

// Sums tiles_of over the tokens into prefix[0 .. tokens], positions into held[0 .. tokens) and block-table rows into
// held[tokens .. 2 tokens); all threads of the block.
__device__ __forceinline__ void make_plan(int* prefix, int* held, const int* __restrict__ positions, const int* __restrict__ token_slot,
                                          const Rows& rows, int tokens, int window, int table_units, int* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int carried = 0;
    if (threadIdx.x == 0) prefix[0] = 0;
    for (int first = 0; first < tokens; first += THREADS) {
        const int t = first + threadIdx.x;
        int pos = -1, table_row = -1;
        if (t < tokens) {
            const int row = rows.of(t);
            pos = positions[row];
            table_row = token_slot[row];
            held[t] = pos;
            held[tokens + t] = table_row;
        }
        int sum = tiles_of(pos, window, table_units);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int below = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += below;
        }
        if (first + THREADS >= tokens && tokens - first <= 32) {       // few tokens left: the first warp has them all
            if (t < tokens) prefix[t + 1] = carried + sum;
            break;
        }
        if (lane == 31) scratch[warp] = sum;
        __syncthreads();
        int before = carried;
#pragma unroll
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
__device__ __forceinline__ int tiles_a_block(int total, int blocks) { return (total + blocks - 1) / blocks; }

struct Step {
    const int* block_tables;
    const int* token_slot;
    const int* positions;
    int max_blocks, table_rows, tokens, heads, kv_heads, page_size, unit_shift, window;     // unit_shift: of the units of a page, or -1
    int pages;
    unsigned page_bytes;         // of all kv heads
    long q_stride;
    float scale_log2;
    float* part_o;               // [blocks, 2, HEADS, D]
    float2* part_ml;             // [blocks, 2, HEADS]: maximum, sum
    int* plan;                   // [tokens + 1]: the prefix of tiles
};

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// Values at `own`, an address of this block's shared memory, in block `rank` of the cluster.
__device__ __forceinline__ unsigned in_block(const void* own, unsigned rank) {
    unsigned out;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(out) : "r"(smem_addr(own)), "r"(rank));
    return out;
}
__device__ __forceinline__ float4 load4_in(unsigned address) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(address));
    return v;
}
__device__ __forceinline__ float2 load2_in(unsigned address) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0,%1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "r"(address));
    return v;
}

// CLUSTERED: grid (blocks of a cluster, tokens * pairs), a cluster a pair: its tiles are cut evenly among its blocks, whose pieces the first
// block adds through distributed shared memory.  Neither plan nor scratch nor a second kernel.
template <int D, bool FOUR, bool CLUSTERED>
__global__ void __launch_bounds__(THREADS, FOUR ? 4 : 3)     // eight heads: 150 registers a thread without spills, 31 us where four blocks took 32
decode_fp4_kernel(const bf16* __restrict__ q, bf16* __restrict__ out, const unsigned char* __restrict__ cache, const Step step,
                  const __grid_constant__ Rows rows) {
    using Unit = Fp4Unit<D>;
    using Sh = Shape<D, FOUR>;
    constexpr int HEADS = Sh::HEADS, MINE = Sh::MINE, WORDS_K = D / 32, WORDS_V = D / 64, TILES_M = D / 32;
    constexpr int COLUMNS = FOUR ? 1 : 2;              // products that give 32 features of the heads
    extern __shared__ __align__(128) unsigned char smem[];      // on 16 bytes the copies took 64 requests of up to 8,192 keys from 81 to 90 us
    __shared__ int scratch[WARPS];
    float* merge = reinterpret_cast<float*>(smem + Sh::RING_BYTES);              // [WARPS][HEADS][ROW]
    int* prefix = reinterpret_cast<int*>(smem + Sh::RING_BYTES + Sh::MERGE_BYTES);
    int* held_pos = prefix + step.tokens + 1;
    const int* held_row = held_pos + step.tokens;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = smem + warp * STAGES * UNITS * Unit::BYTES;
    const int group = step.heads / step.kv_heads, head_groups = (group + HEADS - 1) / HEADS;
    const int units_a_page = step.page_size / FP4_TOKENS, table_units = step.max_blocks * units_a_page, pairs = step.kv_heads * head_groups;

    Piece p = {};
    Cursor at = {};
    int count, my_pos = -1, my_row = -1;               // CLUSTERED: of the pair's token
    if constexpr (CLUSTERED) {
        p.tok = blockIdx.y / pairs;
        const int pair = blockIdx.y - p.tok * pairs;
        p.kvh = head_groups == 1 ? pair : pair / head_groups;
        p.hg = pair - p.kvh * head_groups;
        my_pos = step.positions[rows.of(p.tok)];
        my_row = step.token_slot[rows.of(p.tok)];
        const int tiles = tiles_of(my_pos, step.window, table_units);
        if (tiles == 0) {                              // the whole cluster leaves
            const int heads_here = min(HEADS, group - p.hg * HEADS);
            if (blockIdx.x == 0)
                for (int i = threadIdx.x; i < heads_here * D / 2; i += THREADS)
                    reinterpret_cast<unsigned*>(out + ((size_t)rows.of(p.tok) * step.heads + p.kvh * group + p.hg * HEADS) * D)[i] = 0u;
            return;
        }
        const int base = tiles / (int)gridDim.x, more = tiles - base * (int)gridDim.x, rank = blockIdx.x;
        p.tile0 = rank * base + min(rank, more);
        count = p.tiles = base + (rank < more ? 1 : 0);
    } else {
        make_plan(prefix, held_pos, step.positions, step.token_slot, rows, step.tokens, step.window, table_units, scratch);
        if (blockIdx.x == 0)
            for (int i = threadIdx.x; i <= step.tokens; i += THREADS) step.plan[i] = prefix[i];
        // rows without a tile (padding) come out as zeros
        for (int tok = blockIdx.x; tok < step.tokens; tok += gridDim.x)
            if (prefix[tok] == prefix[tok + 1])
                for (int i = threadIdx.x; i < step.heads * D / 2; i += THREADS)
                    reinterpret_cast<unsigned*>(out + (size_t)rows.of(tok) * step.heads * D)[i] = 0u;

        const int total = prefix[step.tokens] * pairs, per = tiles_a_block(total, gridDim.x), begin = blockIdx.x * per;
        if (begin >= total) return;
        count = min(per, total - begin);
        int low = 0, high = step.tokens - 1;           // the token whose tiles hold the block's first one
        while (low < high) {
            const int mid = (low + high) / 2;
            if (prefix[mid + 1] * pairs <= begin) low = mid + 1;
            else high = mid;
        }
        at.tok = low;
        at.rest = begin - prefix[low] * pairs;
    }
    auto position = [&](const Piece& of) { return CLUSTERED ? my_pos : held_pos[of.tok]; };

    // ---- the copies: this warp's units of every tile, one tile ahead of the work.  The pages of 16 tiles' units are asked for
    // together, one a lane, a tile before the first of them is copied.
    Cursor ahead = at;
    Piece ap = {};
    int ap_tile = 0, issued = 0;
    int a_unit = 0;                                    // this warp's first unit of the piece that is copied
    const unsigned char* a_head = cache;               // the kv head's part of page 0
    int window = -1;                                   // lane l: the page of unit l % 2 of tile ap_tile / 16 * 16 + l / 2 of the piece
    unsigned arriving = 0;                             // bit u: unit u of the stage that was filled last is there
    static_assert(UNITS == 2, "a lane a unit of 16 tiles");
    auto ask_pages = [&]() {                           // for the tile that is copied next
        if (issued >= count) return;
        if (ap_tile == ap.tiles) {
            ap = CLUSTERED ? p : next_piece(ahead, count - issued, prefix, step.kv_heads, head_groups);
            ap_tile = 0;
            a_unit = first_visible(position(ap), step.window) / FP4_TOKENS + ap.tile0 * UNITS_A_TILE + warp * UNITS;
            a_head = cache + (size_t)ap.kvh * units_a_page * Unit::BYTES + lane * 16;
        }
        if (ap_tile % 16 == 0) {
            const int table_row = CLUSTERED ? my_row : held_row[ap.tok], last = min(position(ap) / FP4_TOKENS, table_units - 1);
            const int unit = a_unit + (ap_tile + lane / 2) * UNITS_A_TILE + lane % 2;
            window = -1;
            if (unit <= last && table_row >= 0 && table_row < step.table_rows)
                window = __ldg(step.block_tables + (size_t)table_row * step.max_blocks + (step.unit_shift >= 0 ? unit >> step.unit_shift : unit / units_a_page));
        }
    };
    auto issue = [&]() {                               // copies the next tile's units, one that is not there as zeros
        const unsigned dst = smem_addr(ring + (issued % STAGES) * (UNITS * Unit::BYTES)) + lane * 16;
        arriving = 0;
        if (issued < count) {
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                const int page = __shfl_sync(0xffffffffu, window, ap_tile % 16 * 2 + u), unit = a_unit + ap_tile * UNITS_A_TILE + u;
                const bool there = (unsigned)page < (unsigned)step.pages;
                const int in_page = step.unit_shift >= 0 ? unit & (units_a_page - 1) : unit % units_a_page;
                const unsigned char* src = a_head + (size_t)(there ? (unsigned)page : 0u) * step.page_bytes + in_page * Unit::BYTES;
                const unsigned bytes = there ? 16u : 0u;
#pragma unroll
                for (int c = 0; c < Unit::BYTES / 512; ++c) cp_async_16(dst + u * Unit::BYTES + c * 512, src + c * 512, bytes);
                if (lane < Unit::BYTES % 512 / 16) cp_async_16(dst + u * Unit::BYTES + Unit::BYTES / 512 * 512, src + Unit::BYTES / 512 * 512, bytes);
                arriving |= (there ? 1u : 0u) << u;
            }
            ++ap_tile;
            ++issued;
        }
        cp_async_commit();
        ask_pages();
    };
    // The queries of a piece: lane 4 g + t has features D/4 t .. of the head of column g.
    uint4 raw[D / 32];
    auto ask_queries = [&](const Piece& p) {
        const int h = FOUR ? g >> 1 : g;
        const size_t row = rows.of(p.tok);
        const bf16* src = q + row * step.q_stride + (size_t)(p.kvh * group + p.hg * HEADS + h) * D + t * (D / 4);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
            raw[c] = make_uint4(0, 0, 0, 0);
            if (h < group - p.hg * HEADS) raw[c] = *reinterpret_cast<const uint4*>(src + c * 8);
        }
    };
    if constexpr (!CLUSTERED) p = next_piece(at, count, prefix, step.kv_heads, head_groups);
    ask_pages();
    ask_queries(p);
    issue();

    int done = 0, seg = 0;
    do {
        const int pos = position(p), lo = first_visible(pos, step.window), first_unit = lo / FP4_TOKENS;
        const size_t row = rows.of(p.tok);
        const int head0 = p.kvh * group + p.hg * HEADS, heads_here = min(HEADS, group - p.hg * HEADS);

        unsigned qf[D / 16][2];                            // as halves with the largest of the head in [128, 256)
        float scale[MINE];                                 // of the scores of the lane's heads
        {
            float largest = 0.f;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                const __nv_bfloat162* two = reinterpret_cast<const __nv_bfloat162*>(&raw[c]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = __bfloat1622float2(two[e]);
                    largest = fmaxf(largest, fmaxf(fabsf(f.x), fabsf(f.y)));
                }
            }
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
            largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
            const auto [up, down] = powers_of(largest);
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                const __nv_bfloat162* two = reinterpret_cast<const __nv_bfloat162*>(&raw[c]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = __bfloat1622float2(two[e]);
                    qf[c * 2 + (e >> 1)][e & 1] = pack_h2(f.x * up, f.y * up);
                }
            }
#pragma unroll
            for (int h = 0; h < MINE; ++h) scale[h] = score_scale(__shfl_sync(0xffffffffu, down, 8 * t + 4 * h), step.scale_log2);
        }

        float m[MINE], nbase[MINE], l[MINE], o[TILES_M][COLUMNS][4];         // nbase: LIFT less the maximum
#pragma unroll
        for (int h = 0; h < MINE; ++h) {
            m[h] = -INFINITY;
            nbase[h] = FLT_MAX;                            // any score raises it; one of -inf stays -inf
            l[h] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < TILES_M; ++i)
#pragma unroll
            for (int e = 0; e < COLUMNS; ++e) o[i][e][0] = o[i][e][1] = o[i][e][2] = o[i][e][3] = 0.f;

        for (int tile = p.tile0; tile < p.tile0 + p.tiles; ++tile, ++done) {
            __syncwarp();                                  // the stage that is filled next was read by all lanes
            const unsigned here = arriving;                // which units of this stage are there
            const unsigned char* stage = ring + (done % STAGES) * (UNITS * Unit::BYTES);
            issue();
            cp_async_wait<1>();
            __syncwarp();
            if (here == 0) continue;
            const int key0 = (first_unit + tile * UNITS_A_TILE + warp * UNITS) * FP4_TOKENS;
            const bool whole = here == (1u << UNITS) - 1 && key0 >= lo && key0 + UNITS * FP4_TOKENS - 1 <= pos;

            // ---- scores
            float c[UNITS][4];
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                const unsigned char* unit = stage + u * Unit::BYTES;
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
                // of token g's and token g + 8's groups: D = 128 two each, D = 64 one each in one pair
                const __half2 sc[2] = {two_scales<0>(ks), two_scales<(D == 128 ? 2 : 0)>(ks)};
#pragma unroll
                for (int w = 0; w < WORDS_K; ++w) {
                    unsigned a[2][4];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        halves_of(kw[r][w], a[r]);
#pragma unroll
                        for (int i = 0; i < 4; ++i) a[r][i] = scaled(a[r][i], sc[r], D == 128 ? w / 2 : r);
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        if (w == 0 && j == 0) mma_f16_first(c[u], a[0][0], a[1][0], a[0][1], a[1][1], qf[0][0], qf[0][1]);
                        else mma_f16(c[u], a[0][2 * j], a[1][2 * j], a[0][2 * j + 1], a[1][2 * j + 1], qf[2 * w + j][0], qf[2 * w + j][1]);
                    }
                }
            }
            // Score of the lane's head h with key g or g + 8 (r) of unit u: c[u][h + 2 r].
            unsigned seen[UNITS];                          // of the value scales, which a lane holds of keys 2 t, 2 t + 1, 2 t + 8 and 2 t + 9
#pragma unroll
            for (int u = 0; u < UNITS; ++u) seen[u] = 0xffffffffu;
            if (!whole) {
                // A key that is not seen may lie in memory that nothing has written: its score is -inf, and its value's scale 0.
                auto hidden = [&](int u, int r) {
                    const int key = key0 + u * FP4_TOKENS + r;
                    return key > pos || key < lo || !((here >> u) & 1u);
                };
#pragma unroll
                for (int u = 0; u < UNITS; ++u) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (hidden(u, g + (e >> 1) * 8)) c[u][e] = -INFINITY;
#pragma unroll
                    for (int b = 0; b < 4; ++b)
                        if (hidden(u, (b >> 1) * 8 + 2 * t + (b & 1))) seen[u] &= ~(0xFFu << (8 * b));
                }
            }
            float x[MINE][UNITS][2];                       // score + nbase, what P is the power of
            bool raise = false;
#pragma unroll
            for (int h = 0; h < MINE; ++h)
#pragma unroll
                for (int u = 0; u < UNITS; ++u)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        x[h][u][r] = against(c[u][h + 2 * r], scale[h], nbase[h]);
                        raise = raise || x[h][u][r] > LIFT + SLACK;
                    }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int h = 0; h < MINE; ++h) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int u = 0; u < UNITS; ++u)
#pragma unroll
                        for (int r = 0; r < 2; ++r) mx = fmaxf(mx, __fmul_rn(c[u][h + 2 * r], scale[h]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    mx = fmaxf(mx, m[h]);
                    const float corr = m[h] == -INFINITY ? 0.f : exp2_fast(m[h] - mx);
                    m[h] = mx;
                    if (mx > -INFINITY) nbase[h] = LIFT - mx;
                    l[h] *= corr;
#pragma unroll
                    for (int i = 0; i < TILES_M; ++i)
#pragma unroll
                        for (int e = 0; e < COLUMNS; ++e)
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if (FOUR || (k & 1) == h) o[i][e][k] *= corr;
#pragma unroll
                    for (int u = 0; u < UNITS; ++u)
#pragma unroll
                        for (int r = 0; r < 2; ++r) x[h][u][r] = against(c[u][h + 2 * r], scale[h], nbase[h]);
                }
            }
#pragma unroll
            for (int h = 0; h < MINE; ++h)
#pragma unroll
                for (int u = 0; u < UNITS; ++u)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        x[h][u][r] = exp2_fast(x[h][u][r]);
                        l[h] += x[h][u][r];
                    }

            // ---- values
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                const unsigned char* unit = stage + u * Unit::BYTES;
                const unsigned vs = *reinterpret_cast<const unsigned*>(unit + Unit::V_SCALES + (D == 128 ? lane : (g >> 1) * 4 + t) * 4) & seen[u];
                const __half2 sv[2] = {two_scales<0>(vs), two_scales<2>(vs)};       // of tokens 2 t and 2 t + 1, then + 8
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    unsigned vw[2][WORDS_V];               // of tokens 2 t and 2 t + 1 (+ 8 half)
                    const unsigned char* src = unit + Unit::V_CODES + half * (4 * D) + lane * 2 * Unit::PIECE;
                    if constexpr (D == 128) *reinterpret_cast<uint4*>(vw) = *reinterpret_cast<const uint4*>(src);
                    else *reinterpret_cast<uint2*>(vw) = *reinterpret_cast<const uint2*>(src);
                    unsigned b[COLUMNS][2];                // P of tokens 2 t and 2 t + 1 for the head of column g
                    const unsigned pt = transposed(pack_h2(x[0][u][half], x[MINE - 1][u][half]));
                    if constexpr (FOUR) {                  // column g is of head g / 2 and of the features of parity g % 2
                        b[0][0] = __byte_perm(pt, 0u, g & 1 ? 0x1044u : 0x4410u);
                        b[0][1] = __byte_perm(pt, 0u, g & 1 ? 0x3244u : 0x4432u);
                    } else {
                        b[0][0] = pt & 0xffffu; b[0][1] = pt >> 16;
                        b[COLUMNS - 1][0] = pt << 16; b[COLUMNS - 1][1] = pt & 0xffff0000u;
                    }
#pragma unroll
                    for (int w = 0; w < WORDS_V; ++w) {
                        unsigned a[2][4];
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            halves_of(vw[r][w], a[r]);
#pragma unroll
                            for (int i = 0; i < 4; ++i) a[r][i] = scaled(a[r][i], sv[half], r);
                        }
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int e = 0; e < COLUMNS; ++e)
                                mma_f16(o[2 * w + j][e], a[0][2 * j], a[0][2 * j + 1], a[1][2 * j], a[1][2 * j + 1], b[e][0], b[e][1]);
                    }
                }
            }
        }

        // ---- the four warps' results meet; the next piece's queries are on their way meanwhile
        Piece next = p;
        if constexpr (!CLUSTERED) {
            if (done < count) next = next_piece(at, count - done, prefix, step.kv_heads, head_groups);
            ask_queries(next);
        }
#pragma unroll
        for (int h = 0; h < MINE; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 4);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 8);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 16);
            const int head = FOUR ? t : 2 * t + h;
            float* dst = merge + (warp * HEADS + head) * Sh::ROW;
            if (head < heads_here) {
#pragma unroll
                for (int i = 0; i < TILES_M; ++i)          // features D/8 g + 4 i ..
                    *reinterpret_cast<float4*>(dst + g * (D / 8) + 4 * i) =
                        FOUR ? make_float4(o[i][0][0], o[i][0][1], o[i][0][2], o[i][0][3])
                             : make_float4(o[i][0][h], o[i][COLUMNS - 1][h], o[i][0][h + 2], o[i][COLUMNS - 1][h + 2]);
                if (g == 0) {
                    dst[D] = m[h];
                    dst[D + 1] = l[h];
                }
            }
        }
        __syncthreads();
        const size_t my = (size_t)blockIdx.x * 2 + (seg == 0 ? 0 : 1);
        constexpr int ITEMS = (HEADS * (D / 4) + THREADS - 1) / THREADS;         // four values of a head each
        float4 sums[ITEMS];
        float2 tops[ITEMS];
#pragma unroll
        for (int item = 0; item < ITEMS; ++item) {
            const int i = item * THREADS + threadIdx.x;
            if (i >= heads_here * (D / 4)) break;
            const int head = i / (D / 4), d = (i - head * (D / 4)) * 4;
            float mm = -INFINITY;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, merge[(w * HEADS + head) * Sh::ROW + D]);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            float ll = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float* src = merge + (w * HEADS + head) * Sh::ROW;
                const float f = weight_of(src[D], src[D + 1], mm);
                const float4 v = *reinterpret_cast<const float4*>(src + d);
                acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
                ll += src[D + 1] * f;
            }
            sums[item] = acc;
            tops[item] = make_float2(mm, ll);
            if constexpr (CLUSTERED) continue;
            if (p.complete) {
                store_row(out + row * step.heads * D + (size_t)(head0 + head) * D + d, acc, ll);
            } else {
                *reinterpret_cast<float4*>(step.part_o + (my * HEADS + head) * D + d) = acc;
                if (d == 0) step.part_ml[my * HEADS + head] = make_float2(mm, ll);
            }
        }
        __syncthreads();
        if constexpr (CLUSTERED) {
#pragma unroll
            for (int item = 0; item < ITEMS; ++item) {
                const int i = item * THREADS + threadIdx.x, head = i / (D / 4), d = (i - head * (D / 4)) * 4;
                if (i >= heads_here * (D / 4)) break;
                *reinterpret_cast<float4*>(merge + head * Sh::ROW + d) = sums[item];
                if (d == 0) *reinterpret_cast<float2*>(merge + head * Sh::ROW + D) = tops[item];
            }
            cluster_sync();
            if (blockIdx.x == 0)
                for (int i = threadIdx.x; i < heads_here * (D / 4); i += THREADS) {
                    const int head = i / (D / 4), d = (i - head * (D / 4)) * 4;
                    float2 ml[MAX_CLUSTER];
                    float mm = -INFINITY;
#pragma unroll
                    for (int b = 0; b < MAX_CLUSTER; ++b) {
                        ml[b] = b < (int)gridDim.x ? load2_in(in_block(merge + head * Sh::ROW + D, b)) : make_float2(-INFINITY, 0.f);
                        mm = fmaxf(mm, ml[b].x);
                    }
                    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
                    float ll = 0.f;
#pragma unroll
                    for (int b = 0; b < MAX_CLUSTER; ++b) {
                        if (b >= (int)gridDim.x) break;
                        const float f = weight_of(ml[b].x, ml[b].y, mm);
                        const float4 v = load4_in(in_block(merge + head * Sh::ROW + d, b));
                        acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
                        ll += ml[b].y * f;
                    }
                    store_row(out + row * step.heads * D + (size_t)(head0 + head) * D + d, acc, ll);
                }
            cluster_sync();                                // the pieces are read
        }
        p = next;
        ++seg;
    } while (!CLUSTERED && done < count);
    cp_async_wait<0>();
}

// Adds the pieces of the pairs that lie in several blocks.  Four values of a head a thread; the groups of D / 4 threads of a block take a head each
// (grid: pairs, heads / groups), or with `deep`, where pairs are few and their pieces many, every so-manieth piece of
// one head (grid: pairs, heads), added in the groups' order at the end.
template <int D, bool FOUR>
__global__ void __launch_bounds__(MERGE_THREADS)
merge_fp4_kernel(bf16* __restrict__ out, const Step step, const __grid_constant__ Rows rows, int blocks, int deep) {
    constexpr int HEADS = Shape<D, FOUR>::HEADS, LANES = D / 4, GROUPS = MERGE_THREADS / LANES;
    __shared__ float4 sums[GROUPS][LANES];
    __shared__ float2 tops[GROUPS];
    const int group = step.heads / step.kv_heads, head_groups = (group + HEADS - 1) / HEADS, pairs = step.kv_heads * head_groups;
    const int tok = blockIdx.x / pairs, pair = blockIdx.x - tok * pairs, kvh = pair / head_groups, hg = pair - kvh * head_groups;
    const int part = threadIdx.x / LANES, d = threadIdx.x % LANES;
    const int head = deep ? blockIdx.y : blockIdx.y * GROUPS + part, slice = deep ? part : 0, slices = deep ? GROUPS : 1;
    wait_for_kernel_before();
    const int before = __ldcg(step.plan + tok), tiles = __ldcg(step.plan + tok + 1) - before;
    const int total = __ldcg(step.plan + step.tokens) * pairs;
    if (tiles == 0) return;
    const int per = tiles_a_block(total, blocks), start = before * pairs + pair * tiles;
    const int first = start / per, last = (start + tiles - 1) / per;
    if (first == last) return;
    // a block's piece of this pair is its first one where its range begins inside the pair
    auto slot = [&](int b) { return ((size_t)b * 2 + (b * per >= start ? 0 : 1)) * HEADS + head; };
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (head < group - hg * HEADS && head < HEADS)
        for (int b0 = first + slice; b0 <= last; b0 += 4 * slices) {
            float2 ml[4];
            float4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {                  // all asked for before any is used
                ml[k] = make_float2(-INFINITY, 0.f);
                v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                const int b = b0 + k * slices;
                if (b <= last) {
                    ml[k] = __ldcg(step.part_ml + slot(b));
                    v[k] = __ldcg(reinterpret_cast<const float4*>(step.part_o + slot(b) * D) + d);
                }
            }
            float mm = m;
#pragma unroll
            for (int k = 0; k < 4; ++k) mm = fmaxf(mm, ml[k].x);
            const float old = weight_of(m, l, mm);
            acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
            l *= old;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float f = weight_of(ml[k].x, ml[k].y, mm);
                acc.x += v[k].x * f; acc.y += v[k].y * f; acc.z += v[k].z * f; acc.w += v[k].w * f;
                l += ml[k].y * f;
            }
            m = mm;
        }
    bf16* dst = out + (size_t)rows.of(tok) * step.heads * D + (size_t)(kvh * group + hg * HEADS + head) * D + d * 4;
    if (!deep) {
        if (head < group - hg * HEADS && head < HEADS) store_row(dst, acc, l);
        return;
    }
    sums[part][d] = acc;
    if (d == 0) tops[part] = make_float2(m, l);
    __syncthreads();
    if (part || head >= group - hg * HEADS) return;
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) m = fmaxf(m, tops[i].x);
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
        const float f = weight_of(tops[i].x, tops[i].y, m);
        const float4 v = sums[i][d];
        acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
        l += tops[i].y * f;
    }
    store_row(dst, acc, l);
}

// ------------------------------------------------------------------------------------------
// Rows of prompt portions that see a page which is not held, or a position behind their block table.  The portions' keys are read back for
// the prompt kernels, which know no hole among the keys of a row: there such a key is one of zeros, with a score of 0.  This kernel runs
// behind them: a block looks through the pages that its portion sees, and where one is not held (the books of an engine's cache never
// leave that) computes the portion's rows again from the 4-bit pages, a warp a row and query head, a key to eight or sixteen lanes, in 32 bits.
// Nothing is tuned but the look: a call of 2,048 tokens, or of 1,531 behind 9,000, takes 2 us longer with it (55 -> 57, 265 -> 267).
// ------------------------------------------------------------------------------------------
constexpr int UNHELD_THREADS = 256, MAX_PORTIONS = 64;

struct Portion {
    int table_row, position, row0, rows;     // its block-table row, its first token's position, its rows of the step
};
struct Portions {
    int n;
    Portion portion[MAX_PORTIONS];
};

template <int D>
__global__ void __launch_bounds__(UNHELD_THREADS)
unheld_fp4_kernel(const bf16* __restrict__ q, bf16* __restrict__ out, const unsigned char* __restrict__ cache, const Step step,
                  const __grid_constant__ Portions portions) {
    using Unit = Fp4Unit<D>;
    constexpr int LANES = D / 8, AT_ONCE = 32 / LANES;      // lanes of a key, eight features each; keys that a warp takes at a time
    const Portion portion = portions.portion[blockIdx.y];
    const int units_a_page = step.page_size / FP4_TOKENS, lane = threadIdx.x & 31, part = lane % LANES;
    const bool listed = portion.table_row >= 0 && portion.table_row < step.table_rows;
    const int* table = step.block_tables + (size_t)(listed ? portion.table_row : 0) * step.max_blocks;
    auto page_of = [&](int block) { return listed && block < step.max_blocks ? __ldg(table + block) : -1; };
    const int last_block = (portion.position + portion.rows - 1) / step.page_size;
    int missing = 0;
    for (int block = first_visible(portion.position, step.window) / step.page_size + threadIdx.x; block <= last_block && !missing; block += UNHELD_THREADS)
        missing |= (unsigned)page_of(block) >= (unsigned)step.pages;
    if (!__syncthreads_or(missing)) return;

    const int group = step.heads / step.kv_heads;
    const unsigned items = (unsigned)portion.rows * step.heads;
    for (unsigned item = blockIdx.x * (UNHELD_THREADS / 32) + (threadIdx.x >> 5); item < items; item += gridDim.x * (UNHELD_THREADS / 32)) {
        const int i = item / step.heads, head = item - i * step.heads, kvh = head / group;
        const size_t row = portion.row0 + i;
        const int pos = portion.position + i, lo = first_visible(pos, step.window);
        const uint4 raw = *reinterpret_cast<const uint4*>(q + row * step.q_stride + (size_t)head * D + part * 8);
        const __nv_bfloat162* pairs = reinterpret_cast<const __nv_bfloat162*>(&raw);
        float qs[8], largest = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            qs[e] = __bfloat162float(e % 2 ? pairs[e / 2].y : pairs[e / 2].x);
            largest = fmaxf(largest, fabsf(qs[e]));
        }
        const auto [up, down] = powers_of(warp_max(largest));
#pragma unroll
        for (int e = 0; e < 8; ++e) qs[e] *= up;
        const float scale = score_scale(down, step.scale_log2);
        float m = -INFINITY, l = 0.f, acc[8] = {};               // of every AT_ONCE-th key
        for (int unit = lo / FP4_TOKENS, last = min(pos / FP4_TOKENS, step.max_blocks * units_a_page - 1); unit <= last; ++unit) {
            const int block = unit / units_a_page, page = page_of(block);
            if ((unsigned)page >= (unsigned)step.pages) continue;
            const unsigned char* at = cache + (size_t)page * step.page_bytes + (size_t)(kvh * units_a_page + unit - block * units_a_page) * Unit::BYTES;
#pragma unroll 1
            for (int r = lane / LANES; r < FP4_TOKENS; r += AT_ONCE) {
                auto values = [&](int code, int scale_byte, float (&x)[8]) {
                    unsigned two[4];
                    halves_of(*reinterpret_cast<const unsigned*>(at + code), two);
                    const float s = __half2float(__ushort_as_half((unsigned short)(at[scale_byte] << 7)));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two[e]));
                        x[2 * e] = f.x * s;
                        x[2 * e + 1] = f.y * s;
                    }
                };
                float x[8], dot = 0.f;
                values(Unit::k_code(r, part * 4), Unit::k_scale(r, part / 2), x);
#pragma unroll
                for (int e = 0; e < 8; ++e) dot = fmaf(qs[e], x[e], dot);
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
                const int key = unit * FP4_TOKENS + r;
                if (key >= lo && key <= pos) {                   // a hidden key may lie in memory that nothing has written
                    const float score = __fmul_rn(dot, scale), top = fmaxf(m, score);
                    const float corr = m == -INFINITY ? 0.f : exp2f(m - top), p = top == -INFINITY && score == top ? 0.f : exp2f(score - top);
                    values(Unit::v_code(r, part * 4), Unit::v_scale(r, part / 2), x);
                    m = top;
                    l = l * corr + p;
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[e] = acc[e] * corr + p * x[e];
                }
                __syncwarp();
            }
        }
        const float top = warp_max(m), f = weight_of(m, l, top);
        l *= f;
#pragma unroll
        for (int o = LANES; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        uint4 packed;
        __nv_bfloat162* sums = reinterpret_cast<__nv_bfloat162*>(&packed);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            acc[e] *= f;
#pragma unroll
            for (int o = LANES; o < 32; o <<= 1) acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], o);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) sums[e] = __floats2bfloat162_rn(acc[2 * e] * inv, acc[2 * e + 1] * inv);
        if (lane < LANES) *reinterpret_cast<uint4*>(out + (row * step.heads + head) * D + part * 8) = packed;
    }
}

// Lets the decode kernel have its shared memory on the current device, once a device.
template <int D, bool FOUR, bool CLUSTERED> cudaError_t allow_shared() {
    static std::atomic<unsigned long long> allowed{0};
    int device = 0;
    cudaError_t err = cudaGetDevice(&device);
    if (err != cudaSuccess) return err;
    const unsigned long long bit = 1ull << (device & 63);
    if (device < 64 && (allowed.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
    err = cudaFuncSetAttribute(decode_fp4_kernel<D, FOUR, CLUSTERED>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<D, FOUR>::bytes(MAX_TOKENS));
    if (err == cudaSuccess && device < 64) allowed.fetch_or(bit, std::memory_order_relaxed);
    return err;
}

template <int D, bool FOUR>
cudaError_t launch_decode(const bf16* q, bf16* out, const unsigned char* cache, const Step& step, const Rows& rows, int blocks, int cluster,
                          cudaStream_t stream) {
    using Sh = Shape<D, FOUR>;
    const int group = step.heads / step.kv_heads, head_groups = (group + Sh::HEADS - 1) / Sh::HEADS;
    const int pairs = step.tokens * step.kv_heads * head_groups;
    if (cluster) {
        cudaError_t err = allow_shared<D, FOUR, true>();
        if (err != cudaSuccess) return err;
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3(cluster, pairs);
        config.blockDim = dim3(THREADS);
        config.dynamicSmemBytes = Sh::bytes(0);
        config.stream = stream;
        cudaLaunchAttribute attribute[1];
        attribute[0].id = cudaLaunchAttributeClusterDimension;
        attribute[0].val.clusterDim.x = cluster;
        attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
        config.attrs = attribute;
        config.numAttrs = 1;
        return cudaLaunchKernelEx(&config, decode_fp4_kernel<D, FOUR, true>, q, out, cache, step, rows);
    }
    cudaError_t err = allow_shared<D, FOUR, false>();
    if (err != cudaSuccess) return err;
    err = launch_kernel(decode_fp4_kernel<D, FOUR, false>, dim3(blocks), dim3(THREADS), Sh::bytes(step.tokens), stream, q, out, cache, step, rows);
    if (err != cudaSuccess) return err;
    constexpr int GROUPS = MERGE_THREADS / (D / 4);
    const int heads = group < Sh::HEADS ? group : Sh::HEADS;
    const int deep = 4 * pairs < blocks;               // more than four pieces a pair
    return launch_kernel_overlapped(merge_fp4_kernel<D, FOUR>, dim3(pairs, deep ? heads : (heads + GROUPS - 1) / GROUPS), dim3(MERGE_THREADS), 0,
                                    stream, out, step, rows, blocks, deep);
}

template <int D, bool FOUR> int occupancy() {
    int n = 0;
    const size_t smem = Shape<D, FOUR>::bytes(MAX_TOKENS);
    if (allow_shared<D, FOUR, false>() != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, decode_fp4_kernel<D, FOUR, false>, THREADS, smem) != cudaSuccess) return 0;
    return n;
}

// Heads that a block takes of a kv head's group.  Groups of more than eight are cut: sixteen heads in one block (their
// outputs and queries take 96 registers a thread) were slower than reading the pages from the L2 cache for each eight (B200, 16 requests of
// up to 16,384 keys, 32 heads over 2: 39.3 us against 37.9).
int heads_a_block(int group) { return group <= 4 ? 4 : 8; }

}  // namespace

// Blocks of the decode kernel that a multiprocessor holds at once; 0: the device refuses.
MRUN_API int mrun_attn_fp4_occupancy(int head_dim, int group) {
    return head_dim == 64 ? (group <= 4 ? occupancy<64, true>() : occupancy<64, false>())
                          : (group <= 4 ? occupancy<128, true>() : occupancy<128, false>());
}


// One token a row of q, out, positions and token_slot: the first `tokens` rows, or those that `rows` (host memory) names.  scratch:
// 4-byte words: blocks * 2 * (4 or 8 heads) * (head_dim + 2) + tokens + 1, on 16 bytes.  cluster: 0, or the blocks of a
// cluster (1, 2, 4, 8) that takes a pair; `scratch` and `blocks` are not used then.
MRUN_API int mrun_attn_fp4_decode(const void* q, long q_stride, void* out, const void* cache, const int* block_tables, int table_rows,
                                  int max_blocks, const int* token_slot, const int* positions, const int* rows, int tokens, int heads,
                                  int kv_heads, int head_dim, int page_size, long pages, float scale, int window, void* scratch,
                                  int blocks, int cluster, cudaStream_t stream) {
    const char* name = "paged_attention_fp4";
    MRUN_REQUIRE(tokens >= 0 && tokens <= MAX_TOKENS, "%s: %d tokens, a launch takes up to %d", name, tokens, MAX_TOKENS);
    MRUN_REQUIRE(cluster == 0 || cluster == 1 || cluster == 2 || cluster == 4 || cluster == MAX_CLUSTER, "%s: a cluster of %d blocks", name, cluster);
    MRUN_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && (cluster || (blocks > 0 && scratch)) && pages >= 0 && max_blocks >= 0 && table_rows >= 0,
                 "%s: bad sizes", name);
    MRUN_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim=%d: the 4-bit cache takes heads of 64 or 128 features", name, head_dim);
    MRUN_REQUIRE(page_size > 0 && page_size % FP4_TOKENS == 0, "%s: page_size=%d is not a multiple of 16", name, page_size);
    MRUN_REQUIRE((((uintptr_t)q | (uintptr_t)out | (uintptr_t)cache | (uintptr_t)scratch) & 15) == 0 && q_stride % 8 == 0,
                 "%s: rows and pages start on 16 bytes", name);
    const long page_units = page_size / FP4_TOKENS, table_tiles = max_blocks * page_units / UNITS_A_TILE + 1;
    MRUN_REQUIRE(pages < (1L << 31) && page_units * kv_heads * 18 * head_dim < (1L << 31), "%s: pages=%ld of %d tokens and %d kv heads", name,
                 pages, page_size, kv_heads);
    MRUN_REQUIRE(max_blocks * page_units < (1L << 31) && table_tiles * tokens * heads < (1L << 31),
                 "%s: %d tokens of %d heads over block tables of %d pages of %d tokens", name, tokens, heads, max_blocks, page_size);
    MRUN_REQUIRE(scale > 0.f && scale < FLT_MAX, "%s: scale=%g is not a positive number", name, (double)scale);
    if (tokens == 0) return 0;
    const int group = heads / kv_heads, block_heads = heads_a_block(group);
    MRUN_REQUIRE(!cluster || (long)tokens * kv_heads * ((group + block_heads - 1) / block_heads) < 65536,
                 "%s: %d tokens of %d heads are too many for clusters", name, tokens, heads);
    float* part_o = (float*)scratch;
    float2* part_ml = (float2*)(part_o + (size_t)blocks * 2 * block_heads * head_dim);
    Rows selected;
    selected.listed = rows != nullptr;
    if (rows)
        for (int i = 0; i < MAX_TOKENS; ++i) selected.row[i] = i < tokens ? rows[i] : 0;
    const Step step = {block_tables, token_slot, positions, max_blocks, table_rows, tokens, heads, kv_heads, page_size,
                       page_shift_of((int)page_units), window, (int)pages, (unsigned)(page_units * kv_heads * 18 * head_dim), q_stride,
                       scale * 1.4426950408889634f, part_o, part_ml, (int*)(part_ml + (size_t)blocks * 2 * block_heads)};
    auto launch = head_dim == 64 ? (group <= 4 ? launch_decode<64, true> : launch_decode<64, false>)
                                 : (group <= 4 ? launch_decode<128, true> : launch_decode<128, false>);
    MRUN_CHECK_CUDA(launch((const bf16*)q, (bf16*)out, (const unsigned char*)cache, step, selected, blocks, cluster, stream), name);
    MRUN_CHECK_LAUNCH(name);
    return 0;
}

// The rows of `portions` (host memory: int [n, 4], see Portion) that see a page which is not held, or a position behind their block table, again, such
// keys left out; the others stay as they are.  Rows and positions come from `portions` alone.
MRUN_API int mrun_attn_fp4_unheld(const void* q, long q_stride, void* out, const void* cache, const int* block_tables, int table_rows,
                                  int max_blocks, const int* portions, int n, int heads, int kv_heads, int head_dim, int page_size, long pages,
                                  float scale, int window, cudaStream_t stream) {
    const char* name = "paged_attention_fp4";
    MRUN_REQUIRE(n >= 0 && (n == 0 || portions) && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && pages >= 0 && max_blocks >= 0 && table_rows >= 0,
                 "%s: bad sizes", name);
    MRUN_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim=%d: the 4-bit cache takes heads of 64 or 128 features", name, head_dim);
    MRUN_REQUIRE(page_size > 0 && page_size % FP4_TOKENS == 0, "%s: page_size=%d is not a multiple of 16", name, page_size);
    MRUN_REQUIRE((((uintptr_t)q | (uintptr_t)out | (uintptr_t)cache) & 15) == 0 && q_stride % 8 == 0, "%s: rows and pages start on 16 bytes", name);
    const long page_units = page_size / FP4_TOKENS;
    MRUN_REQUIRE(pages < (1L << 31) && page_units * kv_heads * 18 * head_dim < (1L << 31), "%s: pages=%ld of %d tokens and %d kv heads", name,
                 pages, page_size, kv_heads);
    MRUN_REQUIRE(max_blocks * page_units < (1L << 31), "%s: block tables of %d pages of %d tokens", name, max_blocks, page_size);
    MRUN_REQUIRE(scale > 0.f && scale < FLT_MAX, "%s: scale=%g is not a positive number", name, (double)scale);
    Step step = {};
    step.block_tables = block_tables;
    step.max_blocks = max_blocks;
    step.table_rows = table_rows;
    step.heads = heads;
    step.kv_heads = kv_heads;
    step.page_size = page_size;
    step.window = window;
    step.pages = (int)pages;
    step.page_bytes = (unsigned)(page_units * kv_heads * 18 * head_dim);
    step.q_stride = q_stride;
    step.scale_log2 = scale * 1.4426950408889634f;
    for (int first = 0; first < n; first += MAX_PORTIONS) {
        Portions part = {};
        part.n = n - first < MAX_PORTIONS ? n - first : MAX_PORTIONS;
        int most = 1;
        for (int i = 0; i < part.n; ++i) {
            const int* v = portions + 4 * (first + i);
            MRUN_REQUIRE(v[1] >= 0 && v[2] >= 0 && v[3] > 0 && (long)v[1] + v[3] < (1L << 31) && (long)v[3] * heads < (1L << 30),
                         "%s: a portion of %d tokens of %d heads at position %d", name, v[3], heads, v[1]);
            part.portion[i] = Portion{v[0], v[1], v[2], v[3]};
            most = v[3] > most ? v[3] : most;
        }
        // about two blocks a multiprocessor look at the pages; a portion whose rows are computed again has them as well
        const int blocks = 296 / part.n > 1 ? 296 / part.n : 1, wanted = (int)(((long)most * heads + UNHELD_THREADS / 32 - 1) / (UNHELD_THREADS / 32));
        const dim3 grid((unsigned)(blocks < wanted ? blocks : wanted), (unsigned)part.n);
        MRUN_CHECK_CUDA(launch_kernel(head_dim == 64 ? unheld_fp4_kernel<64> : unheld_fp4_kernel<128>, grid, dim3(UNHELD_THREADS), 0, stream,
                                      (const bf16*)q, (bf16*)out, (const unsigned char*)cache, step, part), name);
        MRUN_CHECK_LAUNCH(name);
    }
    return 0;
}
