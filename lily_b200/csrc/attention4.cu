// Decode attention over a paged cache held in four bits (four.cuh): one new token a request, query heads in groups over their kv head.
//
// With x_jf = low_jg + step_jg c_jf (g the group of 64 features that f is in) a key's score and the output are
//   q . k_j = sum_g step_jg (sum_f q_f c_jf) + low_jg sum_f q_f,
//   o_f = sum_j (p_j step_jg) c_jf + sum_j p_j low_jg,
// so codes go into tensor-core products as they are, 0..15, without a conversion.  Keys: four bits of a word, masked, are the half-precision number c 2^-24 (or 16 c 2^-24, which needs no shift either),
// and products are exact; a head's queries are brought to 2^13 .. 2^14 by a power of two for it, so that they stay as they are.  Values: weights times steps are
// half-precision numbers too, steps times a power of two that brings the largest of them to 2^6 .. 2^7 (a warp's own, lowered where a larger one comes; weights are up to 2^8), so that a weight keeps eleven
// bits down to 2^-28 of the largest: with bfloat16's eight the outputs were 1.8e-3 from 64 bits, where their own rounding is 1.6e-3.  Codes are numbers 16 + c there, and 24 is taken off at the end with sums
// of the weights as they were rounded, for low + 8 step is summed in float32 beside it: what the rounding of a weight moves is so c - 8 times it, no more than the value is from its group's middle.  Steps
// meet the sums behind the products (keys) or the weights ahead of them (values).
#include "four.cuh"
#include "mma.cuh"
#include <algorithm>
#include <cuda_fp16.h>
#include <type_traits>

namespace lily {
namespace four {

constexpr float LOG2E = 1.4426950408889634f;

struct DecodeArgs {
    const void* q;                // [requests, nq * d]
    const uint8_t* kv;
    void* out;                    // [requests, nq * d]
    const int* block_table;       // [requests, width]
    int width;
    const int* seq_lens;
    float* part_o;                // [2 blocks, 8, d]: what blocks leave of pairs that they share
    float* part_ml;               // [2 blocks, 8, 2]
    int nq, nkv, d, page_size, pages, longest;
    int page_shift;               // tensor-core kernel: log2 of page_size
    int requests;
    float scale;
};

// A request's places (no more than the caller said there would be).
__device__ __forceinline__ int places_of(const DecodeArgs& a, int req) { return min(max(__ldcg(a.seq_lens + req), 0), a.longest); }
// The page that place `j` of a request lies in (page 0, which is nobody's, where the table names none of the cache).
__device__ __forceinline__ int page_of(const DecodeArgs& a, int req, int j) {
    const int page = a.block_table[(size_t)req * a.width + j / a.page_size];
    return (unsigned)page < (unsigned)a.pages ? page : 0;
}
// ---- bfloat16 on the tensor cores -------------------------------------------------------------------
constexpr int KT = 32;                        // places a tile
constexpr int WARPS = 4, STAGES = 2;          // warps a block, tiles in a warp's ring
constexpr int HEADS = 8;                      // query heads a block: the columns of a product

// A pair's part ends where the warps of its block meet.  Where pairs are many, blocks are one warp, which meets nobody; their many parts would be slow to join where pairs are few, and heads above 128
// have no registers for enough of them.  Measured with 32 query heads of 128 over 8, blocks of four warps (two a multiprocessor) against blocks of one (twelve): 32 rows of 1,024 places 18.3 us
// against 18.7; 64 rows of 1,000 29.9 against 28, 128 of 500 38 against 29, 256 of 130 52 against 30.  (Heads of 256, 64 rows of 1,000: 50 against 59.)
// Blocks of four warps (8 rows of 4,000 places, three a multiprocessor against two): heads of 64 have room for three, 12.9 us against 15.2; heads of 128 have not the registers, 20.6 against 18.8,
// heads of 256 even less, 58 against 30.
constexpr int blocks_a_sm(int d, int warps) { return warps == 1 ? 12 : d == 64 ? 3 : 2; }

template <int D> struct Tile {
    static constexpr int G = D / GROUP, CODES = D / 2;
    static constexpr int KEY_ROW = D == 256 ? CODES + 16 : CODES, VALUE_ROW = CODES + 16;      // padded so that a fragment's reads hit banks of their own
    static constexpr int KEYS = 0, VALUES = KT * KEY_ROW, KEY_HELD = VALUES + KT * VALUE_ROW, VALUE_HELD = KEY_HELD + KT * G * 4, BYTES = VALUE_HELD + KT * G * 4;
};

// Where a warp stands in the row of all tiles: a request, a kv head and a chunk of its query heads (a pair), a tile of the request's places.
struct Place {
    int req, kvh, chunk, tile, tiles, places;
    __device__ __forceinline__ void next_pair(const DecodeArgs& a, int chunks) {
        tile = 0;
        if (++chunk < chunks) return;
        chunk = 0;
        if (++kvh < a.nkv) return;
        kvh = 0;
        for (tiles = 0; tiles == 0 && ++req < a.requests;) {          // (the next request that has places)
            places = places_of(a, req);
            tiles = (places + KT - 1) / KT;
        }
    }
};

// One tile of places into shared memory; what lies behind the request's last place is zeros, or numbers of the page that nobody looks at.
template <int D>
__device__ __forceinline__ void fetch(const DecodeArgs& a, const Place& at, uint32_t dst) {
    using S = Tile<D>;
    constexpr int PIECES = S::CODES / 16, HELD_ROWS = S::G == 3 ? 4 : 4 / S::G, HELD_PIECES = S::G == 3 ? 3 : 1;      // places and pieces of a run of steps
    constexpr int RUNS = KT / HELD_ROWS * HELD_PIECES, STEPS = KT * PIECES / 32;
    const int lane = threadIdx.x & 31, key0 = at.tile * KT, left = at.places - key0, inside = a.page_size - 1;
    const uint32_t rows = (uint32_t)a.page_size * (uint32_t)row_bytes(D);
    auto of_place = [&](int j) {
        const int page = a.block_table[(size_t)at.req * a.width + (j >> a.page_shift)];
        return a.kv + ((size_t)((unsigned)page < (unsigned)a.pages ? page : 0) * a.nkv + at.kvh) * (2 * (size_t)rows);
    };
    if (a.page_size >= KT && left >= KT && 32 % PIECES == 0) {        // the tile lies in one page, its rows one behind the other
        const int slot = key0 & inside;
        const uint8_t *page = of_place(key0), *keys = page + slot * S::CODES + lane * 16, *values = keys + rows;
        const uint32_t to = dst + lane / PIECES * S::KEY_ROW + lane % PIECES * 16, to_v = dst + S::VALUES + lane / PIECES * S::VALUE_ROW + lane % PIECES * 16;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            mma16::cp_async16(to + i * (32 / PIECES) * S::KEY_ROW, keys + i * 512, true);
            mma16::cp_async16(to_v + i * (32 / PIECES) * S::VALUE_ROW, values + i * 512, true);
        }
        if (RUNS == 32 || lane < RUNS) {                              // (RUNS is 8, 16, 24 or 32)
            const uint8_t* held = page + a.page_size * S::CODES + slot * S::G * 4 + lane * 16;
            mma16::cp_async16(dst + S::KEY_HELD + lane * 16, held, true);
            mma16::cp_async16(dst + S::VALUE_HELD + lane * 16, held + rows, true);
        }
        return;
    }
    for (int i = 0; i < STEPS; ++i) {
        const int c = i * 32 + lane, row = c / PIECES, piece = c - row * PIECES, j = min(key0 + row, at.places - 1);
        const uint8_t* p = of_place(j) + (size_t)(j & inside) * S::CODES + piece * 16;
        mma16::cp_async16(dst + S::KEYS + row * S::KEY_ROW + piece * 16, p, row < left);
        mma16::cp_async16(dst + S::VALUES + row * S::VALUE_ROW + piece * 16, p + rows, row < left);
    }
    if (lane < RUNS) {
        const int row = lane / HELD_PIECES * HELD_ROWS, piece = lane % HELD_PIECES, j = min(key0 + row, at.places - 1);
        const uint8_t* p = of_place(j) + (size_t)a.page_size * S::CODES + (size_t)((j & inside) / HELD_ROWS * HELD_ROWS) * S::G * 4 + piece * 16;
        mma16::cp_async16(dst + S::KEY_HELD + lane * 16, p, row < left);
        mma16::cp_async16(dst + S::VALUE_HELD + lane * 16, p + rows, row < left);
    }
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// Codes i of the halves of a word as half-precision numbers 16 + code.  The values' sums are long ones, and tensor cores cut what they add to an accumulator off: what is taken off again at the end is to be
// no more than it must (with 128 + code rows of 1,000 places and more were 2.2e-3 from 64 bits, rows of 100,000 more).
__device__ __forceinline__ uint32_t pair16(uint32_t w, int i) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(i < 2 ? w << (6 - 4 * i) : w >> (4 * i - 6)), "r"(0x03C003C0u), "r"(0x4C004C00u));
    return r;
}
__device__ __forceinline__ uint32_t half_bits(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void mma_half(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int N> __device__ __forceinline__ void words_of(const unsigned char* p, uint32_t (&w)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
            w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(p + 4 * i);
            w[i] = v.x, w[i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
    }
}

// How the work is cut.  Every (request, kv head, chunk of eight query heads) is a pair; its places come in tiles of 32, and all tiles of all pairs, one pair's behind the other's, are
// shared out over the blocks, whatever the lengths: T / B tiles each and one more for the first T % B.  A pair that lies in one block's share is finished there; else each block leaves
// (max, sum, output) of its part in a slot, 2 b for the part that its share begins with and 2 b + 1 for another, and a second kernel joins them.
__device__ __forceinline__ int tiles_of(const DecodeArgs& a, int req) { return (places_of(a, req) + KT - 1) / KT; }
struct Cut {
    int per, more;
    __device__ __forceinline__ Cut(int total, int blocks) : per(total / blocks), more(total - per * blocks) {}
    __device__ __forceinline__ int begins(int b) const { return b * per + min(b, more); }
    __device__ __forceinline__ int owner(int tile) const {
        const int wide = more * (per + 1);
        return tile < wide ? tile / (per + 1) : more + (tile - wide) / per;      // (no tile lies behind the wide shares where the others are empty)
    }
};

// This block's share of the tiles, and where it begins.  Rows without places are zeroed on the way.
template <typename T, int D, int W>
__device__ __forceinline__ void begin_share(const DecodeArgs& a, int pairs, int chunks, Place& at, int& share) {
    const int lane = threadIdx.x & 31;
    auto length = [&](int r) { return r < a.requests ? places_of(a, r) : 0; };
    const int own_length = length(lane);                              // (most steps have no more than 32 rows: one read each)
    int total = (own_length + KT - 1) / KT;
    for (int r = lane + 32; r < a.requests; r += 32) total += tiles_of(a, r);
    total = __reduce_add_sync(0xffffffffu, total);
    const Cut cut(total * pairs, gridDim.x);
    const int first = cut.begins(blockIdx.x);
    share = cut.per + ((int)blockIdx.x < cut.more);
    bool found = share == 0;
    for (int r0 = 0, before = 0; r0 < a.requests; r0 += 32) {
        const int n = r0 ? length(r0 + lane) : own_length, own = (n + KT - 1) / KT * pairs;
        for (unsigned without = __ballot_sync(0xffffffffu, r0 + lane < a.requests && n == 0); without; without &= without - 1) {
            const int r = r0 + __ffs(without) - 1;
            if (r % (int)gridDim.x == (int)blockIdx.x)
                for (int i = threadIdx.x; i < a.nq * D; i += 32 * W) ((T*)a.out)[(size_t)r * a.nq * D + i] = from_float<T>(0.f);
        }
        if (found) continue;
        int run = own;                                                // of the requests up to this lane's
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, run, x);
            if (lane >= x) run += y;
        }
        const unsigned beyond = __ballot_sync(0xffffffffu, before + run > first);
        if (beyond) {
            const int where = __ffs(beyond) - 1;
            at.req = r0 + where;
            at.places = __shfl_sync(0xffffffffu, n, where);
            at.tiles = (at.places + KT - 1) / KT;
            const int in = first - (before + __shfl_sync(0xffffffffu, run - own, where)), pair_no = in / at.tiles;
            at.tile = in - pair_no * at.tiles;
            at.kvh = chunks == 1 ? pair_no : pair_no / chunks;
            at.chunk = pair_no - at.kvh * chunks;
            found = true;
        }
        before += __shfl_sync(0xffffffffu, run, 31);
    }
}

__device__ __forceinline__ void put4(float* to, float4 v) { *reinterpret_cast<float4*>(to) = v; }
__device__ __forceinline__ void put4(__nv_bfloat16* to, float4 v) { *reinterpret_cast<uint2*>(to) = make_uint2(bits(__floats2bfloat162_rn(v.x, v.y)), bits(__floats2bfloat162_rn(v.z, v.w))); }

// The warps' (max in units of log2, sum, output) of a pair's part, in shared memory, together: divided and rounded to the output where the whole pair was here (``alone``), else to
// the part's slot.
template <typename T, int D, int W>
__device__ __forceinline__ void end_part(const DecodeArgs& a, int req, int head0, int heads, bool alone, bool second, const float (*m_s)[HEADS], const float (*l_s)[HEADS], const float* o_s,
                                         int o_warp, int o_head) {
    const size_t part = 2 * (size_t)blockIdx.x + second;
    for (int i = threadIdx.x; i < heads * (D / 4); i += 32 * W) {
        const int h = i / (D / 4), f = 4 * (i - h * (D / 4));
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) m = fmaxf(m, m_s[w][h]);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float by = m_s[w][h] == -INFINITY ? (l_s[w][h] == 0.f ? 0.f : 1.f) : ex2(m_s[w][h] - m);
            const float4 x = *reinterpret_cast<const float4*>(o_s + w * o_warp + h * o_head + f);
            if (by != 0.f) l = fmaf(by, l_s[w][h], l), v.x = fmaf(by, x.x, v.x), v.y = fmaf(by, x.y, v.y), v.z = fmaf(by, x.z, v.z), v.w = fmaf(by, x.w, v.w);
        }
        if (alone) {
            const float by = l == 0.f ? 0.f : 1.f / l;
            put4((T*)a.out + ((size_t)req * a.nq + head0 + h) * D + f, make_float4(v.x * by, v.y * by, v.z * by, v.w * by));
        } else {
            *reinterpret_cast<float4*>(a.part_o + (part * HEADS + h) * D + f) = v;
            if (f == 0) *reinterpret_cast<float2*>(a.part_ml + (part * HEADS + h) * 2) = make_float2(m, l);
        }
    }
}

// Keys on the rows of the products (16 of them), query heads on their eight columns: S^T = K q^T, O^T = V^T P^T.  The warps of a block take the tiles of its share in turn, each through
// a ring of its own that runs on from one pair to the next; they meet where a pair's part ends.
template <int D, int W>
__global__ void __launch_bounds__(32 * W, blocks_a_sm(D, W)) decode_mma_kernel(const DecodeArgs a) {
    using S = Tile<D>;
    constexpr int G = S::G, LD = D + 4;
    extern __shared__ __align__(16) unsigned char ring_s[];
    __shared__ float m_s[W][HEADS], l_s[W][HEADS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = a.nq / a.nkv, chunks = (group + HEADS - 1) / HEADS, pairs = a.nkv * chunks;
    unsigned char* mine = ring_s + warp * STAGES * S::BYTES;
    float* o_s = reinterpret_cast<float*>(ring_s + W * STAGES * S::BYTES);      // [warps][heads][LD]
    const uint32_t ring = mma16::smem_u32(mine);
    pdl_wait();
    pdl_launch_dependents();                                          // (the joining kernel may so read the lengths ahead of its own wait)
    Place at{};
    int share = 0;
    begin_share<__nv_bfloat16, D, W>(a, pairs, chunks, at, share);
    if (share == 0) return;
    // the tile to ask for next, the `asked`-th of the share: this warp's own are `warp` and every fourth behind it
    Place ahead = at;
    int asked = warp, issued = 0;
    ahead.tile += warp;
    auto ask = [&]() {
        if (asked < share) {
            while (ahead.tile >= ahead.tiles) {
                const int over = ahead.tile - ahead.tiles;
                ahead.next_pair(a, chunks);
                ahead.tile = over;
            }
            fetch<D>(a, ahead, ring + issued % STAGES * S::BYTES);
            ++issued;
            asked += W;
            ahead.tile += W;
        }
        mma16::cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) ask();
    int next = warp, used = 0;                                        // this warp's next tile of the share; tiles taken out of the ring
    for (int began = 0; began < share;) {
        const int req = at.req, head0 = at.kvh * group + at.chunk * HEADS, heads = min(HEADS, group - at.chunk * HEADS), ends = min(share, began + at.tiles - at.tile);
        // the queries as the products' second operand, in the order of the keys' words, and their sums: brought by a power of two to 2^13 .. 2^14, a sixteenth of it where codes come as 16 c
        uint32_t q[G][2][4];
        float qs[G][2], scale[2], margin[2];                              // of heads 2 t and 2 t + 1: the sums and the softmax's factor in units of the products; 2^8 of weight as a difference of scores
        {
            uint4 v[G][2];
            float most_q = 0.f, sums[G];
#pragma unroll
            for (int j = 0; j < G; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint4& x = v[j][h];
                    x = make_uint4(0, 0, 0, 0);
                    if (g < heads) x = *reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.q + ((size_t)req * a.nq + head0 + g) * D + 64 * j + 32 * h + 8 * t);
                    if (a.scale < 0.f) x.x ^= 0x80008000u, x.y ^= 0x80008000u, x.z ^= 0x80008000u, x.w ^= 0x80008000u;
                    for (const uint32_t w : {x.x, x.y, x.z, x.w}) most_q = fmaxf(most_q, fmaxf(fabsf(low(w)), fabsf(high(w))));
                }
            most_q = fmaxf(most_q, __shfl_xor_sync(0xffffffffu, most_q, 1));
            most_q = fmaxf(most_q, __shfl_xor_sync(0xffffffffu, most_q, 2));
            const int exponent = (int)(__float_as_uint(most_q) >> 23);    // 2^(exponent - 127) is the largest query's size
            const float by = __uint_as_float((uint32_t)min(max(267 - exponent, 1), 253) << 23), unit = by * 0x1p-24f;      // a product is the sum over queries times codes in units of 2^24 / by
#pragma unroll
            for (int j = 0; j < G; ++j) {
                sums[j] = 0.f;                                            // (of queries times their power, so that large ones' is a number)
#pragma unroll
                for (int h = 0; h < 2; ++h) {                             // features 0 and 4, 1 and 5, 2 and 6, 3 and 7 of the eight
                    const uint4 x = v[j][h];
                    const float less = by * 0.0625f;
                    for (const uint32_t w : {x.x, x.y, x.z, x.w}) sums[j] += low(w) * by + high(w) * by;
                    q[j][h][0] = half_bits(low(x.x) * by, low(x.z) * by);
                    q[j][h][1] = half_bits(high(x.x) * less, high(x.z) * less);
                    q[j][h][2] = half_bits(low(x.y) * by, low(x.w) * by);
                    q[j][h][3] = half_bits(high(x.y) * less, high(x.w) * less);
                }
                sums[j] += __shfl_xor_sync(0xffffffffu, sums[j], 1);
                sums[j] += __shfl_xor_sync(0xffffffffu, sums[j], 2);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float u = __shfl_sync(0xffffffffu, unit, 8 * t + 4 * e);
#pragma unroll
                for (int j = 0; j < G; ++j) qs[j][e] = __shfl_sync(0xffffffffu, sums[j], 8 * t + 4 * e) * 0x1p-24f;
                // (queries from some 2^92 on: two scores that differ at all differ by more than any softmax sees at 2^100 as well, which keeps what it multiplies a number)
                scale[e] = fminf(fabsf(a.scale) * LOG2E / u, 0x1p100f);
                margin[e] = 8.f / scale[e];
            }
        }
        float o[G][4][4], most[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f}, ones[G][4], mids[G][2];      // (scores and their maximum are kept unscaled)
#pragma unroll
        for (int j = 0; j < G; ++j) {
            mids[j][0] = mids[j][1] = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                ones[j][e] = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[j][i][e] = 0.f;
            }
        }
        const uint32_t one[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
        // the largest step's exponent so far, and the power of two for steps: its own is 2^6 (an exponent is one of 0 to 254, a power one of 2^-121 to 2^126)
        uint32_t largest = 7;
        auto power = [](uint32_t exponent) { return __uint_as_float((260u - exponent) << 23); };
        float up = power(largest);
        // Masks only where a request ends, elsewhere they took a select a score and a step (8 rows of 8,192 places 26.0 us, 26.5 with them).  Heads above 128 keep one form: two are more code than short
        // rows fetch in time (heads of 256, 128 rows of 500 58 us, 65 with two).
        auto work = [&](auto whole, const unsigned char* tile, const int left) {
            constexpr bool WHOLE = decltype(whole)::value;
            float s[2][4];                                                // scores of keys g and g + 8, heads 2 t and 2 t + 1
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                const int row = 16 * mt + g;
                uint32_t w0[2 * G], w1[2 * G], h0[G], h1[G];
                words_of<2 * G>(tile + S::KEYS + row * S::KEY_ROW + t * 8 * G, w0);
                words_of<2 * G>(tile + S::KEYS + (row + 8) * S::KEY_ROW + t * 8 * G, w1);
                words_of<G>(tile + S::KEY_HELD + row * 4 * G, h0);
                words_of<G>(tile + S::KEY_HELD + (row + 8) * 4 * G, h1);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[mt][e] = 0.f;
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t x = w0[2 * j + h], y = w1[2 * j + h], x8 = x >> 8, y8 = y >> 8;
                        const uint32_t a0[4] = {x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u}, a1[4] = {x8 & 0x000f000fu, y8 & 0x000f000fu, x8 & 0x00f000f0u, y8 & 0x00f000f0u};
                        mma_half(c, a0, q[j][h][0], q[j][h][1]);
                        mma_half(c, a1, q[j][h][2], q[j][h][3]);
                    }
                    const float s0 = low(h0[j]), s1 = low(h1[j]), b0 = high(h0[j]), b1 = high(h1[j]);
                    s[mt][0] = fmaf(s0, c[0], fmaf(b0, qs[j][0], s[mt][0]));
                    s[mt][1] = fmaf(s0, c[1], fmaf(b0, qs[j][1], s[mt][1]));
                    s[mt][2] = fmaf(s1, c[2], fmaf(b1, qs[j][0], s[mt][2]));
                    s[mt][3] = fmaf(s1, c[3], fmaf(b1, qs[j][1], s[mt][3]));
                }
                if (!WHOLE) {
                    if (row >= left) s[mt][0] = s[mt][1] = -INFINITY;
                    if (row + 8 >= left) s[mt][2] = s[mt][3] = -INFINITY;
                }
            }
            float m0 = fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2])), m1 = fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]));
            // The maximum moves only where a score is 2^8 times its weight ahead (weights of up to 256 are as good as ones of up to 1), which after the first tile is rare.
            if (__any_sync(0xffffffffu, m0 > most[0] + margin[0] || m1 > most[1] + margin[1])) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) {
                    m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, x));
                    m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, x));
                }
                m0 = fmaxf(m0, most[0]);
                m1 = fmaxf(m1, most[1]);
                const float f0 = m0 == most[0] ? 1.f : ex2((most[0] - m0) * scale[0]), f1 = m1 == most[1] ? 1.f : ex2((most[1] - m1) * scale[1]);
                most[0] = m0;
                most[1] = m1;
                sum[0] *= f0;
                sum[1] *= f1;
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    mids[j][0] *= f0;
                    mids[j][1] *= f1;
                    ones[j][0] *= f0;
                    ones[j][1] *= f1;
#pragma unroll
                    for (int n = 0; n < 4; ++n) o[j][n][0] *= f0, o[j][n][1] *= f1, o[j][n][2] *= f0, o[j][n][3] *= f1;
                }
            }
            {
                uint32_t steps[G], e = 0;                                 // of a place a lane
                words_of<G>(tile + S::VALUE_HELD + lane * 4 * G, steps);
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    const uint32_t own = steps[j] >> 7 & 0xffu;
                    if ((WHOLE || lane < left) && own < 255u) e = max(e, own);
                }
                e = __reduce_max_sync(0xffffffffu, e);
                if (e > largest) {                                        // sums so far in units of the new power
                    const float f = __uint_as_float(max(127 + (int)largest - (int)e, 0) << 23);
                    largest = e;
                    up = power(e);
#pragma unroll
                    for (int j = 0; j < G; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            ones[j][i] *= f;
#pragma unroll
                            for (int n = 0; n < 4; ++n) o[j][n][i] *= f;
                        }
                }
            }
            const float z0 = most[0] == -INFINITY ? 0.f : most[0], z1 = most[1] == -INFINITY ? 0.f : most[1];      // (nobody has a score yet)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                const int row = 16 * mt;
                float p[4];
                p[0] = ex2((s[mt][0] - z0) * scale[0]);      // (the difference first: a product of large scores would be off by more than it)
                p[1] = ex2((s[mt][1] - z1) * scale[1]);
                p[2] = ex2((s[mt][2] - z0) * scale[0]);
                p[3] = ex2((s[mt][3] - z1) * scale[1]);
                sum[0] += p[0] + p[2];
                sum[1] += p[1] + p[3];
                uint32_t w[4][G], h0[G], h1[G];
                words_of<G>(tile + S::VALUE_HELD + (row + g) * 4 * G, h0);
                words_of<G>(tile + S::VALUE_HELD + (row + g + 8) * 4 * G, h1);
#pragma unroll
                for (int e = 0; e < 4; ++e) words_of<G>(tile + S::VALUES + (row + 2 * t + (e & 1) + (e >> 1) * 8) * S::VALUE_ROW + g * 4 * G, w[e]);
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    if (!WHOLE) {                                      // (what stands behind the last place may be no number)
                        if (row + g >= left) h0[j] = 0;
                        if (row + g + 8 >= left) h1[j] = 0;
                    }
                    const float s0 = low(h0[j]), s1 = low(h1[j]), mid0 = fmaf(8.f, s0, high(h0[j])), mid1 = fmaf(8.f, s1, high(h1[j]));
                    mids[j][0] = fmaf(p[2], mid1, fmaf(p[0], mid0, mids[j][0]));
                    mids[j][1] = fmaf(p[3], mid1, fmaf(p[1], mid0, mids[j][1]));
                    // weights times steps, rounded to half precision as the second operand asks
                    const float up0 = s0 * up, up1 = s1 * up;
                    const uint32_t b0 = transposed(half_bits(p[0] * up0, p[1] * up0)), b1 = transposed(half_bits(p[2] * up1, p[3] * up1));
                    mma_half(ones[j], one, b0, b1);
                    const uint32_t x0 = __byte_perm(w[0][j], w[1][j], 0x5410), x1 = __byte_perm(w[0][j], w[1][j], 0x7632);
                    const uint32_t y0 = __byte_perm(w[2][j], w[3][j], 0x5410), y1 = __byte_perm(w[2][j], w[3][j], 0x7632);
#pragma unroll
                    for (int n = 0; n < 4; ++n) {                         // features 8 g + 2 n (rows g) and 8 g + 2 n + 1 (rows g + 8) of the group
                        const uint32_t x = n < 2 ? x0 : x1, y = n < 2 ? y0 : y1;
                        const int i0 = 2 * (n & 1);
                        const uint32_t av[4] = {pair16(x, i0), pair16(x, i0 + 1), pair16(y, i0), pair16(y, i0 + 1)};
                        mma_half(o[j][n], av, b0, b1);
                    }
                }
            }
        };
        for (; next < ends; next += W, ++used) {
            ask();
            mma16::cp_async_wait<STAGES - 1>();
            __syncwarp();
            const unsigned char* tile = mine + used % STAGES * S::BYTES;
            const int left = at.places - (at.tile + next - began) * KT;
            if (D <= 128 && left >= KT) work(std::true_type(), tile, left);
            else work(std::false_type(), tile, left);
            __syncwarp();
        }
        // the warps' sums together: finished, where the whole pair was here; else to the part's slot
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
            sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], x);
            sum[1] += __shfl_xor_sync(0xffffffffu, sum[1], x);
#pragma unroll
            for (int j = 0; j < G; ++j) {
                mids[j][0] += __shfl_xor_sync(0xffffffffu, mids[j][0], x);
                mids[j][1] += __shfl_xor_sync(0xffffffffu, mids[j][1], x);
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int h = 2 * t + e;
            if (h >= heads) continue;
            if (g == 0) m_s[warp][h] = most[e] * scale[e], l_s[warp][h] = sum[e];
#pragma unroll
            for (int j = 0; j < G; ++j) {                                 // features 64 j + 8 g + (0..7)
                float4* to = reinterpret_cast<float4*>(o_s + (warp * HEADS + h) * LD + 64 * j + 8 * g);
                auto less = [&](float v) { return fmaf(-24.f, ones[j][e], v); };
                const float down = __uint_as_float((largest - 6u) << 23);      // what `up` undoes
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    to[i] = make_float4(fmaf(less(o[j][2 * i][e]), down, mids[j][e]), fmaf(less(o[j][2 * i][e + 2]), down, mids[j][e]), fmaf(less(o[j][2 * i + 1][e]), down, mids[j][e]),
                                        fmaf(less(o[j][2 * i + 1][e + 2]), down, mids[j][e]));
            }
        }
        __syncthreads();
        end_part<__nv_bfloat16, D, W>(a, req, head0, heads, at.tile == 0 && ends - began == at.tiles, began != 0, m_s, l_s, o_s, HEADS * LD, LD);
        __syncthreads();                                                  // (the next part's sums go where these were)
        began = ends;
        if (began < share) at.next_pair(a, chunks);
    }
}

// The parts of a pair that several blocks have worked on.  A quarter of a block's threads takes every fourth part of a head (SLICES = 4), or every fourth head (SLICES = 1).
// grid (pairs of a request, requests, blocks that a pair's heads are shared out to)
template <typename T, int D, int SLICES>
__global__ void __launch_bounds__(D) join_parts_kernel(const DecodeArgs a, int blocks, int chunk_heads) {
    __shared__ float2 ml_s[SLICES];
    __shared__ float4 o_s[SLICES][D / 4];
    const int req = blockIdx.y, group = a.nq / a.nkv, chunks = (group + chunk_heads - 1) / chunk_heads, pairs = a.nkv * chunks;
    const int kvh = blockIdx.x / chunks, chunk = blockIdx.x - kvh * chunks, head0 = kvh * group + chunk * chunk_heads, heads = min(chunk_heads, group - chunk * chunk_heads);
    pdl_launch_dependents();
    const int tiles = tiles_of(a, req), lane = threadIdx.x & 31;
    int total = 0, before = 0;
    for (int r = lane; r < a.requests; r += 32) {
        const int n = tiles_of(a, r);
        total += n;
        if (r < req) before += n;
    }
    const Cut cut(__reduce_add_sync(0xffffffffu, total) * pairs, blocks);
    const int lo = __reduce_add_sync(0xffffffffu, before) * pairs + (int)blockIdx.x * tiles;
    // the blocks whose shares hold its first and its last tile (those between them have tiles)
    const int b0 = tiles ? cut.owner(lo) : 0, b1 = tiles ? cut.owner(lo + tiles - 1) : 0, behind = tiles && cut.begins(b0) != lo;
    pdl_wait();
    if (b0 == b1) return;
    const int quarter = threadIdx.x / (D / 4), i4 = threadIdx.x % (D / 4);
    const int slice = SLICES == 1 ? 0 : quarter;
    for (int h = SLICES == 1 ? 4 * blockIdx.z + quarter : blockIdx.z; h < heads; h += (SLICES == 1 ? 4 : 1) * gridDim.z) {
        float m = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](const float2 (&ml)[4], const float4 (&v)[4]) {
            const float next = fmaxf(fmaxf(m, fmaxf(ml[0].x, ml[1].x)), fmaxf(ml[2].x, ml[3].x)), was = m == next ? 1.f : ex2(m - next);
            m = next;
            l *= was;
            o.x *= was, o.y *= was, o.z *= was, o.w *= was;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float by = ml[i].x == -INFINITY ? (ml[i].y == 0.f ? 0.f : 1.f) : ex2(ml[i].x - m);
                if (by != 0.f) l = fmaf(by, ml[i].y, l), o.x = fmaf(by, v[i].x, o.x), o.y = fmaf(by, v[i].y, o.y), o.z = fmaf(by, v[i].z, o.z), o.w = fmaf(by, v[i].w, o.w);
            }
        };
        float2 ml[4];
        float4 v[4];
        for (int first = b0 + slice; first <= b1; first += 4 * SLICES) {      // four parts at a time
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int b = min(first + SLICES * i, b1);
                const size_t part = (2 * (size_t)b + (b == b0 ? behind : 0)) * HEADS + h;
                ml[i] = *reinterpret_cast<const float2*>(a.part_ml + part * 2);
                v[i] = *reinterpret_cast<const float4*>(a.part_o + part * D + 4 * i4);
                if (first + SLICES * i > b1) ml[i] = make_float2(-INFINITY, 0.f);
            }
            add(ml, v);
        }
        if constexpr (SLICES > 1) {
            __syncthreads();                                          // (the head before has been read)
            o_s[slice][i4] = o;
            if (i4 == 0) ml_s[slice] = make_float2(m, l);
            __syncthreads();
            if (slice) continue;
#pragma unroll
            for (int i = 0; i < SLICES; ++i) ml[i] = ml_s[i], v[i] = o_s[i][i4];
            m = -INFINITY, l = 0.f;
            o = make_float4(0.f, 0.f, 0.f, 0.f);
            add(ml, v);
        }
        const float by = l == 0.f ? 0.f : 1.f / l;
        put4((T*)a.out + ((size_t)req * a.nq + head0 + h) * D + 4 * i4, make_float4(o.x * by, o.y * by, o.z * by, o.w * by));
    }
}

// ---- float32, and any page, on the CUDA cores ----------------------------------------------------------
// The same cut of the work.  A warp a tile at a time, whose rows its lanes bring to shared memory, a place each: a lane a place for the scores, then a lane a word of eight features of the
// values, D / 8 lanes side by side and what is left of the warp on other places.  Everything is float32: x = lowest + step code in one rounding.  A step has a few tiles a warp at
// most, so it is short loops that count: unrolled ones (the scores' 128 features, 16 places' values) are fetched from memory as they run once (3 rows of up to 2,900 places 20 to 22 us, where these took 18).
template <int D, int HN> struct CoresTile {
    static constexpr int G = D / GROUP, ROW = D / 2 + 16, HELD = 32 * ROW * 2, P = HELD + 32 * 8 * G, BYTES = P + 32 * HN * 4;      // keys' and values' rows, steps, weights
    static constexpr int LD = D + 4, Q = WARPS * BYTES, O = Q + D * HN * 4, ALL = O + WARPS * HN * LD * 4;
};

template <typename T, int D, int HN>
__global__ void __launch_bounds__(32 * WARPS) decode_cores_kernel(const DecodeArgs a) {
    using S = CoresTile<D, HN>;
    constexpr int G = S::G, WORDS = D / 8, ROW = WORDS <= 8 ? 8 : WORDS <= 16 ? 16 : 32, AT_ONCE = 32 / ROW, LD = S::LD;
    extern __shared__ __align__(16) unsigned char cores_s[];
    __shared__ float m_s[WARPS][HEADS], l_s[WARPS][HEADS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = a.nq / a.nkv, chunks = (group + HN - 1) / HN, pairs = a.nkv * chunks;
    unsigned char* mine = cores_s + warp * S::BYTES;
    float (*q_s)[HN] = reinterpret_cast<float (*)[HN]>(cores_s + S::Q);
    float* o_s = reinterpret_cast<float*>(cores_s + S::O);            // [warps][heads][LD]
    float (*p_s)[HN] = reinterpret_cast<float (*)[HN]>(mine + S::P);
    pdl_wait();
    pdl_launch_dependents();
    Place at{};
    int share = 0;
    begin_share<T, D, WARPS>(a, pairs, chunks, at, share);
    const float scale = a.scale * LOG2E;
    const size_t rows = (size_t)a.page_size * row_bytes(D);
    const bool pieces = rows % 16 == 0;                               // (not pages of one or two places)
    for (int began = 0; began < share;) {
        const int req = at.req, head0 = at.kvh * group + at.chunk * HN, heads = min(HN, group - at.chunk * HN), ends = min(share, began + at.tiles - at.tile);
        for (int i = threadIdx.x; i < HN * D; i += 32 * WARPS) {
            const int h = i / D, f = i - h * D;
            q_s[f][h] = h < heads ? to_float(((const T*)a.q)[((size_t)req * a.nq + head0 + h) * D + f]) * scale : 0.f;
        }
        float most[HN], sum[HN], o[HN][8];
#pragma unroll
        for (int h = 0; h < HN; ++h) {
            most[h] = -INFINITY, sum[h] = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[h][e] = 0.f;
        }
        __syncthreads();
        for (int next = began + warp; next < ends; next += WARPS) {
            const int key0 = (at.tile + next - began) * KT, n = min(KT, at.places - key0);
            if (lane < n) {
                const int j = key0 + lane, slot = j % a.page_size;
                const uint8_t* page = a.kv + ((size_t)page_of(a, req, j) * a.nkv + at.kvh) * (2 * rows);
                const uint8_t *codes = page + (size_t)slot * (D / 2), *held = page + (size_t)a.page_size * (D / 2) + (size_t)slot * G * 4;
                unsigned char* to = mine + lane * S::ROW;
#pragma unroll
                for (int kind = 0; kind < 2; ++kind) {
                    if (pieces) {
#pragma unroll
                        for (int i = 0; i < D / 32; ++i) reinterpret_cast<uint4*>(to + kind * 32 * S::ROW)[i] = reinterpret_cast<const uint4*>(codes + kind * rows)[i];
                    } else
                        for (int i = 0; i < WORDS; ++i) reinterpret_cast<uint32_t*>(to + kind * 32 * S::ROW)[i] = reinterpret_cast<const uint32_t*>(codes + kind * rows)[i];
#pragma unroll
                    for (int i = 0; i < G; ++i) reinterpret_cast<uint32_t*>(mine + S::HELD)[(kind * 32 + lane) * G + i] = reinterpret_cast<const uint32_t*>(held + kind * rows)[i];
                }
            }
            __syncwarp();
            float s[HN];
#pragma unroll
            for (int h = 0; h < HN; ++h) s[h] = lane < n ? 0.f : -INFINITY;
            if (lane < n) {
#pragma unroll 1
                for (int at_word = 0; at_word < WORDS; ++at_word) {   // in the order they lie in
                    const int in = at_word % (2 * G), f = 64 * (in >> 1) + 32 * (in & 1) + 8 * (at_word / (2 * G));
                    const uint32_t word = reinterpret_cast<const uint32_t*>(mine + lane * S::ROW)[at_word], hd = reinterpret_cast<const uint32_t*>(mine + S::HELD)[lane * G + (in >> 1)];
                    const float step = low(hd), lowest = high(hd);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float x = fmaf(__uint_as_float((word >> (4 * e) & 15u) | 0x4B000000u) - 8388608.f, step, lowest);
#pragma unroll
                        for (int h = 0; h < HN; ++h) s[h] = fmaf(q_s[f + e][h], x, s[h]);
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < HN; ++h) {
                const float m = fmaxf(most[h], warp_max(s[h])), z = m == -INFINITY ? 0.f : m;
                const float f = most[h] == m ? 1.f : ex2(most[h] - z), p = ex2(s[h] - z);
                most[h] = m;
                sum[h] = fmaf(sum[h], f, p);
#pragma unroll
                for (int e = 0; e < 8; ++e) o[h][e] *= f;
                p_s[lane][h] = p;
            }
            __syncwarp();
            const int l = min(lane % ROW, WORDS - 1);                 // (d = 192: the last lanes follow the one ahead of them and are not looked at)
#pragma unroll 1
            for (int i = lane / ROW; i < n; i += AT_ONCE) {
                const uint32_t word = reinterpret_cast<const uint32_t*>(mine + (32 + i) * S::ROW)[value_word(l, G)], hd = reinterpret_cast<const uint32_t*>(mine + S::HELD)[(32 + i) * G + (l >> 3)];
                const float step = low(hd), lowest = high(hd);
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = fmaf(__uint_as_float((word >> (4 * e) & 15u) | 0x4B000000u) - 8388608.f, step, lowest);
#pragma unroll
                for (int h = 0; h < HN; ++h) {
                    const float p = p_s[i][h];
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[h][e] = fmaf(p, x[e], o[h][e]);
                }
            }
            __syncwarp();
        }
#pragma unroll
        for (int h = 0; h < HN; ++h) {
            sum[h] = warp_sum(sum[h]);
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int x = ROW; x < 32; x <<= 1) o[h][e] += __shfl_xor_sync(0xffffffffu, o[h][e], x);
            if (lane == 0) m_s[warp][h] = most[h], l_s[warp][h] = sum[h];
            if (lane < WORDS) {
                float4* to = reinterpret_cast<float4*>(o_s + (warp * HN + h) * LD + 8 * lane);
                to[0] = make_float4(o[h][0], o[h][1], o[h][2], o[h][3]);
                to[1] = make_float4(o[h][4], o[h][5], o[h][6], o[h][7]);
            }
        }
        __syncthreads();
        end_part<T, D, WARPS>(a, req, head0, heads, at.tile == 0 && ends - began == at.tiles, began != 0, m_s, l_s, o_s, HN * LD, LD);
        __syncthreads();
        began = ends;
        if (began < share) at.next_pair(a, chunks);
    }
}

inline int log2_of(int page_size) {
    int shift = 0;
    while (1 << shift < page_size) ++shift;
    return 1 << shift == page_size ? shift : -1;
}
// The tensor-core kernel takes bfloat16 and pages of a power of two from 16 places on (a run of sixteen bytes of steps lies in one page).
inline bool on_tensor_cores(int page_size, int dtype) { return dtype == kBF16 && page_size >= 16 && log2_of(page_size) >= 0; }

// Query heads of a pair on the CUDA cores.
inline int cores_heads(int group) { return group <= 4 ? 4 : 8; }
// Blocks of the kernel on the CUDA cores that a multiprocessor holds: three by their registers, and by shared memory (228 KB, of which a block takes 1 KB of its own) two where eight heads of 256 features are
// a pair.  With a third more than it holds, shares that are cut evenly would run in two rounds: 8 float32 rows of 2,000 places, 16 query heads of
// 256 over 2, 29.6 us, 40.3 with three.
template <int D> constexpr int cores_a_sm(bool eight) {
    const int room = 228 * 1024, fixed = 1024 + 512;
    return std::min(3, room / ((int)(eight ? CoresTile<D, 8>::ALL : CoresTile<D, 4>::ALL) + fixed));
}
static_assert(cores_a_sm<256>(true) == 2 && cores_a_sm<256>(false) == 3 && cores_a_sm<192>(true) == 3, "");
inline int cores_blocks(int d, int heads) {
    const bool eight = heads == 8;
    return d == 64 ? cores_a_sm<64>(eight) : d == 128 ? cores_a_sm<128>(eight) : d == 192 ? cores_a_sm<192>(eight) : cores_a_sm<256>(eight);
}
// Blocks: as many as are on the device at once, where there is work for them.
struct Plan { bool tensor_cores; int heads, warps, blocks; };
inline Plan plan_of(int requests, int nq, int nkv, int d, int longest, int page_size, int dtype) {
    Plan p{};
    p.tensor_cores = on_tensor_cores(page_size, dtype);
    p.heads = p.tensor_cores ? HEADS : cores_heads(nq / nkv);
    const long long pairs = (long long)requests * nkv * ((nq / nkv + p.heads - 1) / p.heads), tiles = pairs * (((long long)longest + KT - 1) / KT);
    p.warps = p.tensor_cores && d <= 128 && pairs >= 3ll * sm_count() ? 1 : WARPS;      // (at blocks_a_sm)
    // Two tiles a block at least, of four warps, but no two pairs in a block while there are blocks: a pair's end is some 2 us that the next one waits for.  Against a tile a warp: 8 rows of one place
    // 4.6 us for 10.6 (float32 6.9 for 21.1), of 130 8.1 and 8.2, two of 300 6.0 and 7.9, float32 3 rows of 150 to 2,900 10.2 and 15.5 (of 2,000 18.6 and 17.4); a tile a block: 8 rows of 60 6.1 for 4.9.
    // (The lengths that count are the longest there may be.  A captured step is made for rows of thousands of places, so short rows there are cut a tile a block: 8 rows of 60 places 7.0 us, where a call that
    // says 60 takes 4.8; of 1, 130 and 400 places 5.1, 8.8 and 9.5 us, within 0.3 of theirs.  Blocks counted on the device from the rows at hand took 5.8 for the first, and 0.1 to 0.6 us more of all others.)
    const long long wanted = p.warps == 1 ? tiles : max(pairs, (tiles + 1) / 2);
    p.blocks = (int)max(1ll, min((long long)(p.tensor_cores ? blocks_a_sm(d, p.warps) : cores_blocks(d, p.heads)) * sm_count(), wanted));
    return p;
}

}  // namespace four
}  // namespace lily

using namespace lily;

template <int D, int W> static void launch_mma_of(const four::DecodeArgs& a, const four::Plan& plan, cudaStream_t stream) {
    constexpr int bytes = W * (four::STAGES * four::Tile<D>::BYTES + four::HEADS * (D + 4) * 4);
    cudaFuncSetAttribute(four::decode_mma_kernel<D, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    launch_pdl(four::decode_mma_kernel<D, W>, dim3(plan.blocks), dim3(32 * W), bytes, stream, a);
}
template <int D> static void launch_mma(const four::DecodeArgs& a, const four::Plan& plan, cudaStream_t stream) {
    if constexpr (D <= 128)
        if (plan.warps == 1) return launch_mma_of<D, 1>(a, plan, stream);
    launch_mma_of<D, four::WARPS>(a, plan, stream);
}

// float32 of scratch that lily_attention_decode4 needs
LILY_API size_t lily_attention_decode4_floats(int requests, int nq, int nkv, int d, int longest, int page_size, int dtype) {
    if (requests <= 0 || nkv <= 0 || nq <= 0 || nq % nkv || page_size <= 0) return 0;
    return (size_t)2 * four::plan_of(requests, nq, nkv, d, longest, page_size, dtype).blocks * four::HEADS * (d + 2);
}

LILY_API int lily_attention_decode4(const void* q, const void* kv, void* out, const int* block_table, int width, const int* seq_lens, float* scratch, int requests, int longest, int nq,
                                    int nkv, int d, int page_size, int pages, float scale, int dtype, cudaStream_t stream) {
    if (requests == 0) return 0;
    LILY_REQUIRE(d >= four::GROUP && d <= 256 && d % four::GROUP == 0, "attention_decode4: heads of 64, 128, 192 or 256 features, not %d", d);
    LILY_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "attention_decode4: %d query heads over %d kv heads", nq, nkv);
    LILY_REQUIRE(requests > 0 && requests <= 65535 && page_size > 0 && longest >= 0 && longest <= (long long)width * page_size && pages > 0, "attention_decode4: %d requests of up to %d places, %d pages of %d",
                 requests, longest, width, page_size);
    LILY_REQUIRE(longest <= INT32_MAX - 1024 && (long long)page_size * four::row_bytes(d) <= INT32_MAX, "attention_decode4: rows of %d places, pages of %d", longest, page_size);
    LILY_REQUIRE(((uintptr_t)q | (uintptr_t)kv | (uintptr_t)out) % 16 == 0, "attention_decode4: tensors on boundaries of sixteen bytes");
    LILY_REQUIRE(scale != 0.f && scale - scale == 0.f, "attention_decode4: a scale of %g", (double)scale);
    const four::Plan plan = four::plan_of(requests, nq, nkv, d, longest, page_size, dtype);
    const int chunks = (nq / nkv + plan.heads - 1) / plan.heads;
    LILY_REQUIRE((long long)requests * nkv * chunks * ((longest + four::KT - 1) / four::KT) <= INT32_MAX, "attention_decode4: %d requests of up to %d places are too many for one call", requests, longest);
    LILY_REQUIRE(scratch != nullptr && (uintptr_t)scratch % 16 == 0, "attention_decode4: the parts of %d blocks need scratch on a boundary of sixteen bytes", plan.blocks);
    four::DecodeArgs a{};
    a.q = q; a.kv = (const uint8_t*)kv; a.out = out; a.block_table = block_table; a.width = width; a.seq_lens = seq_lens;
    a.requests = requests; a.nq = nq; a.nkv = nkv; a.d = d; a.page_size = page_size; a.pages = pages; a.longest = longest; a.scale = scale;
    a.page_shift = four::log2_of(page_size);
    a.part_o = scratch;
    a.part_ml = scratch + (size_t)2 * plan.blocks * four::HEADS * d;
    const dim3 block(32 * four::WARPS);
    const long long all_pairs = (long long)requests * nkv * chunks;
    // Few pairs have many parts each, which slices of a block join side by side, a block a head: one row of 8,192 places 11.1 us with them and 14.9 without, 4 rows of 4,096 12.4 and 13.1, 16 rows of
    // 2,048 (128 pairs) 18.4 and 18.0, 256 rows of 130 many times more blocks and 85 against 31.
    const bool sliced = 2 * all_pairs <= sm_count();
    const int most_heads = min(plan.heads, nq / nkv);
    const dim3 joins(nkv * chunks, requests, sliced ? most_heads : (most_heads + 3) / 4);
#define JOIN(T, D)                                                                                                                                                 \
    LILY_CHECK_LAUNCH("attention_decode4");                                                                                                                        \
    if (sliced) launch_pdl(four::join_parts_kernel<T, D, 4>, joins, dim3(D), 0, stream, a, plan.blocks, plan.heads);                                               \
    else launch_pdl(four::join_parts_kernel<T, D, 1>, joins, dim3(D), 0, stream, a, plan.blocks, plan.heads)
#define CORES(T, D, HN)                                                                                                                                            \
    do {                                                                                                                                                           \
        constexpr int bytes = four::CoresTile<D, HN>::ALL;                                                                                                         \
        cudaFuncSetAttribute(four::decode_cores_kernel<T, D, HN>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);                                             \
        launch_pdl(four::decode_cores_kernel<T, D, HN>, dim3(plan.blocks), block, bytes, stream, a);                                                               \
    } while (0)
#define DECODE(D)                                                                                                                                                  \
    do {                                                                                                                                                           \
        if (plan.tensor_cores) {                                                                                                                                   \
            launch_mma<D>(a, plan, stream);                                                                                                                        \
            JOIN(__nv_bfloat16, D);                                                                                                                                \
        } else if (dtype == kF32) {                                                                                                                                \
            if (plan.heads == 4) CORES(float, D, 4);                                                                                                               \
            else CORES(float, D, 8);                                                                                                                               \
            JOIN(float, D);                                                                                                                                        \
        } else {                                                                                                                                                   \
            if (plan.heads == 4) CORES(__nv_bfloat16, D, 4);                                                                                                       \
            else CORES(__nv_bfloat16, D, 8);                                                                                                                       \
            JOIN(__nv_bfloat16, D);                                                                                                                                \
        }                                                                                                                                                          \
    } while (0)
    if (d == 64) DECODE(64);
    else if (d == 128) DECODE(128);
    else if (d == 192) DECODE(192);
    else DECODE(256);
#undef DECODE
#undef CORES
#undef JOIN
    LILY_CHECK_LAUNCH("attention_decode4 (join)");
    return 0;
}
