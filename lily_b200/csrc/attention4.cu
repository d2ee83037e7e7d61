// Decode attention over a paged cache held in four bits (four.cuh): one new token a request, query heads in groups over their kv head.
//
// With x_jf = low_jg + step_jg c_jf (g the group of 64 features that f is in) a key's score and the output are
//   q . k_j = sum_g step_jg (sum_f q_f c_jf) + low_jg sum_f q_f,
//   o_f = sum_j (p_j step_jg) c_jf + sum_j p_j low_jg,
// so codes go into tensor-core products as they are, 0..15 as bfloat16 numbers 128 + c, which cost one logical operation a pair and no conversion; steps meet the sums behind the
// products (keys) or the weights ahead of them (values), and the 128 is taken off with sums of the queries and of the weights as they were rounded.
#include "four.cuh"
#include "mma.cuh"

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
    float* part_o;                // [requests, nq, splits, d]
    float* part_ml;               // [requests, nq, splits, 2]
    int splits, nq, nkv, d, page_size, pages, longest;
    float scale;
};

// A request's places (no more than the caller said there would be).
__device__ __forceinline__ int places_of(const DecodeArgs& a, int req) { return min(max(a.seq_lens[req], 0), a.longest); }
// The page that place `j` of a request lies in (page 0, which is nobody's, where the table names none of the cache).
__device__ __forceinline__ int page_of(const DecodeArgs& a, int req, int j) {
    const int page = a.block_table[(size_t)req * a.width + j / a.page_size];
    return (unsigned)page < (unsigned)a.pages ? page : 0;
}
// The places of range `z` of a request: equal shares in steps of `step`.
__device__ __forceinline__ void range_of(const DecodeArgs& a, int req, int z, int step, int& beg, int& end) {
    const int n = places_of(a, req);
    const int per = ((n + a.splits - 1) / a.splits + step - 1) / step * step;
    beg = min(n, z * per);
    end = min(n, beg + per);
}

// What a block found for its range, `heads` of them with (max in units of log2, sum, output not divided yet) in shared memory: to the scratch, or, where it is the only range,
// divided and rounded to the output.
template <typename T>
__device__ __forceinline__ void leave(const DecodeArgs& a, int req, int head0, int heads, const float* m, const float* l, const float* o, int ld) {
    for (int i = threadIdx.x; i < heads * a.d; i += blockDim.x) {
        const int h = i / a.d, f = i - h * a.d;
        const size_t row = (size_t)req * a.nq + head0 + h;
        if (a.splits == 1) ((T*)a.out)[row * a.d + f] = from_float<T>(l[h] == 0.f ? 0.f : o[h * ld + f] / l[h]);
        else {
            const size_t at = row * a.splits + blockIdx.x;
            a.part_o[at * a.d + f] = o[h * ld + f];
            if (f == 0) a.part_ml[2 * at] = m[h], a.part_ml[2 * at + 1] = l[h];
        }
    }
}

// ---- bfloat16 on the tensor cores -------------------------------------------------------------------
constexpr int KT = 64;                        // places a tile
constexpr int WARPS = 4, STAGES = 2;
constexpr int HEADS = 8;                      // query heads a block: the columns of a product

template <int D> struct Tile {
    static constexpr int G = D / GROUP, CODES = D / 2;
    static constexpr int KEY_ROW = D == 256 ? CODES + 16 : CODES, VALUE_ROW = CODES + 16;      // padded so that a fragment's reads hit banks of their own
    static constexpr int KEYS = 0, VALUES = KT * KEY_ROW, KEY_HELD = VALUES + KT * VALUE_ROW, VALUE_HELD = KEY_HELD + KT * G * 4, BYTES = VALUE_HELD + KT * G * 4;
};

// One tile of places from `key0` on into shared memory; what lies behind `end` is zeros, or numbers of the page that nobody looks at.
template <int D>
__device__ __forceinline__ void fetch(const DecodeArgs& a, int req, int kvh, int key0, int end, uint32_t dst) {
    using S = Tile<D>;
    constexpr int PIECES = S::CODES / 16, HELD_ROWS = S::G == 3 ? 4 : 4 / S::G, HELD_PIECES = S::G == 3 ? 3 : 1;      // places and pieces of a run of steps
    const int lane = threadIdx.x & 31;
    const size_t rows = (size_t)a.page_size * row_bytes(D), page_bytes = 2 * rows * a.nkv, head_at = 2 * rows * kvh;
    const bool whole = a.page_size >= KT;
    const int first_page = whole ? page_of(a, req, key0) : 0;
    auto at = [&](int row, int& slot) {           // the page of a row of the tile
        const int j = key0 + row, in = j < end;
        slot = j % a.page_size;
        const int page = whole ? first_page : in ? page_of(a, req, j) : 0;
        return a.kv + page * page_bytes + head_at;
    };
#pragma unroll
    for (int i = 0; i < KT * PIECES / 32; ++i) {
        const int c = i * 32 + lane, row = c / PIECES, piece = c - row * PIECES;
        int slot;
        const uint8_t* page = at(row, slot);
        const uint8_t* p = page + (size_t)slot * S::CODES + piece * 16;
        const bool in = key0 + row < end;
        mma16::cp_async16(dst + S::KEYS + row * S::KEY_ROW + piece * 16, p, in);
        mma16::cp_async16(dst + S::VALUES + row * S::VALUE_ROW + piece * 16, p + rows, in);
    }
    constexpr int RUNS = KT / HELD_ROWS * HELD_PIECES;
    for (int c = lane; c < RUNS; c += 32) {
        const int row = c / HELD_PIECES * HELD_ROWS, piece = c % HELD_PIECES;
        int slot;
        const uint8_t* page = at(row, slot);
        const uint8_t* p = page + (size_t)a.page_size * S::CODES + (size_t)slot * S::G * 4 + piece * 16;
        const bool in = key0 + row < end;
        mma16::cp_async16(dst + S::KEY_HELD + c * 16, p, in);
        mma16::cp_async16(dst + S::VALUE_HELD + c * 16, p + rows, in);
    }
}

__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
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

// Keys on the rows of the products (16 of them), query heads on their eight columns: S^T = K q^T, O^T = V^T P^T.  Each warp walks tiles of its own (every fourth of the block's
// range) through a ring of its own, so that nobody waits for anybody until the range ends.  grid (ranges, kv heads x chunks of eight heads, requests)
template <int D>
__global__ void __launch_bounds__(32 * WARPS, D <= 128 ? 2 : 1) decode_mma_kernel(const DecodeArgs a) {
    using S = Tile<D>;
    constexpr int G = S::G;
    extern __shared__ __align__(16) unsigned char ring_s[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = a.nq / a.nkv, chunks = (group + HEADS - 1) / HEADS, kvh = blockIdx.y / chunks, chunk = blockIdx.y - kvh * chunks, req = blockIdx.z;
    const int head0 = kvh * group + chunk * HEADS, heads = min(HEADS, group - chunk * HEADS);
    pdl_enter_small();
    int beg, end;
    range_of(a, req, blockIdx.x, KT, beg, end);
    const int tiles = (end - beg + KT - 1) / KT;
    unsigned char* mine = ring_s + warp * STAGES * S::BYTES;
    const uint32_t ring = mma16::smem_u32(mine);
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
        const int i = warp + s * WARPS;
        if (i < tiles) fetch<D>(a, req, kvh, beg + i * KT, end, ring + s * S::BYTES);
        mma16::cp_async_commit();
    }
    // the queries as the products' second operand, in the order of the keys' words, and their sums
    uint32_t q[G][2][4];
    float sums[G];
#pragma unroll
    for (int j = 0; j < G; ++j) {
        float sum = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (g < heads) v = *reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.q + ((size_t)req * a.nq + head0 + g) * D + 64 * j + 32 * h + 8 * t);
            sum += low(v.x) + high(v.x) + low(v.y) + high(v.y) + low(v.z) + high(v.z) + low(v.w) + high(v.w);
            q[j][h][0] = __byte_perm(v.x, v.z, 0x5410);               // features 0 and 4, 1 and 5, 2 and 6, 3 and 7 of the eight
            q[j][h][1] = __byte_perm(v.x, v.z, 0x7632);
            q[j][h][2] = __byte_perm(v.y, v.w, 0x5410);
            q[j][h][3] = __byte_perm(v.y, v.w, 0x7632);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sums[j] = sum + __shfl_xor_sync(0xffffffffu, sum, 2);
    }
    float qs[G][2];                                                   // of heads 2 t and 2 t + 1
#pragma unroll
    for (int j = 0; j < G; ++j) qs[j][0] = __shfl_sync(0xffffffffu, sums[j], 8 * t), qs[j][1] = __shfl_sync(0xffffffffu, sums[j], 8 * t + 4);
    const float scale = a.scale * LOG2E;
    float o[G][4][4], most[2] = {-INFINITY, -INFINITY}, total[2] = {0.f, 0.f}, ones[G][4], lows[G][2];
#pragma unroll
    for (int j = 0; j < G; ++j) {
        lows[j][0] = lows[j][1] = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            ones[j][e] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][i][e] = 0.f;
        }
    }
    const uint32_t one[4] = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    int slot = 0;
    for (int i = warp; i < tiles; i += WARPS) {
        {
            const int next = i + (STAGES - 1) * WARPS, to = slot == 0 ? STAGES - 1 : slot - 1;
            if (next < tiles) fetch<D>(a, req, kvh, beg + next * KT, end, ring + to * S::BYTES);
            mma16::cp_async_commit();
        }
        mma16::cp_async_wait<STAGES - 1>();
        __syncwarp();
        const unsigned char* tile = mine + slot * S::BYTES;
        const int left = end - (beg + i * KT);                        // places of the tile that are the request's
        for (int r0 = 0; r0 < KT && r0 < left; r0 += 32) {
            float s[2][4];                                            // scores of keys g and g + 8, heads 2 t and 2 t + 1
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                const int row = r0 + 16 * mt + g;
                uint32_t w0[2 * G], w1[2 * G];
                words_of<2 * G>(tile + S::KEYS + row * S::KEY_ROW + t * 8 * G, w0);
                words_of<2 * G>(tile + S::KEYS + (row + 8) * S::KEY_ROW + t * 8 * G, w1);
                const uint32_t* held0 = reinterpret_cast<const uint32_t*>(tile + S::KEY_HELD) + row * G;
#pragma unroll
                for (int e = 0; e < 4; ++e) s[mt][e] = 0.f;
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t x = w0[2 * j + h], y = w1[2 * j + h];
                        const uint32_t a0[4] = {pair(x, 0), pair(y, 0), pair(x, 1), pair(y, 1)}, a1[4] = {pair(x, 2), pair(y, 2), pair(x, 3), pair(y, 3)};
                        mma16::mma_bf16(c, a0, q[j][h][0], q[j][h][1]);
                        mma16::mma_bf16(c, a1, q[j][h][2], q[j][h][3]);
                    }
                    const uint32_t h0 = held0[j], h1 = held0[8 * G + j];
                    const float s0 = low(h0) * scale, s1 = low(h1) * scale, b0 = fmaf(s0, -128.f, high(h0) * scale), b1 = fmaf(s1, -128.f, high(h1) * scale);
                    s[mt][0] += fmaf(s0, c[0], b0 * qs[j][0]);
                    s[mt][1] += fmaf(s0, c[1], b0 * qs[j][1]);
                    s[mt][2] += fmaf(s1, c[2], b1 * qs[j][0]);
                    s[mt][3] += fmaf(s1, c[3], b1 * qs[j][1]);
                }
                if (row >= left) s[mt][0] = s[mt][1] = -INFINITY;
                if (row + 8 >= left) s[mt][2] = s[mt][3] = -INFINITY;
            }
            float m0 = fmaxf(fmaxf(s[0][0], s[0][2]), fmaxf(s[1][0], s[1][2])), m1 = fmaxf(fmaxf(s[0][1], s[0][3]), fmaxf(s[1][1], s[1][3]));
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) {
                m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, x));
                m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, x));
            }
            if (__any_sync(0xffffffffu, m0 > most[0] || m1 > most[1])) {
                m0 = fmaxf(m0, most[0]);
                m1 = fmaxf(m1, most[1]);
                const float f0 = m0 == most[0] ? 1.f : exp2f(most[0] - m0), f1 = m1 == most[1] ? 1.f : exp2f(most[1] - m1);
                most[0] = m0;
                most[1] = m1;
                total[0] *= f0;
                total[1] *= f1;
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    lows[j][0] *= f0;
                    lows[j][1] *= f1;
                    ones[j][0] *= f0;
                    ones[j][1] *= f1;
                    ones[j][2] *= f0;
                    ones[j][3] *= f1;
#pragma unroll
                    for (int n = 0; n < 4; ++n) o[j][n][0] *= f0, o[j][n][1] *= f1, o[j][n][2] *= f0, o[j][n][3] *= f1;
                }
            }
            const float z0 = most[0] == -INFINITY ? 0.f : most[0], z1 = most[1] == -INFINITY ? 0.f : most[1];      // (nobody has a score yet)
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                const int row = r0 + 16 * mt;
                float p[4];
                p[0] = exp2f(s[mt][0] - z0);
                p[1] = exp2f(s[mt][1] - z1);
                p[2] = exp2f(s[mt][2] - z0);
                p[3] = exp2f(s[mt][3] - z1);
                total[0] += p[0] + p[2];
                total[1] += p[1] + p[3];
                const uint32_t* held0 = reinterpret_cast<const uint32_t*>(tile + S::VALUE_HELD) + (row + g) * G;
                uint32_t w[4][G];
#pragma unroll
                for (int e = 0; e < 4; ++e) words_of<G>(tile + S::VALUES + (row + 2 * t + (e & 1) + (e >> 1) * 8) * S::VALUE_ROW + g * 4 * G, w[e]);
#pragma unroll
                for (int j = 0; j < G; ++j) {
                    const uint32_t h0 = row + g < left ? held0[j] : 0u, h1 = row + g + 8 < left ? held0[8 * G + j] : 0u;      // (what stands behind the last place may be no number)
                    lows[j][0] = fmaf(p[2], high(h1), fmaf(p[0], high(h0), lows[j][0]));
                    lows[j][1] = fmaf(p[3], high(h1), fmaf(p[1], high(h0), lows[j][1]));
                    // weights times steps, rounded to bfloat16 as the second operand asks
                    const uint32_t b0 = transposed(bits(__floats2bfloat162_rn(p[0] * low(h0), p[1] * low(h0))));
                    const uint32_t b1 = transposed(bits(__floats2bfloat162_rn(p[2] * low(h1), p[3] * low(h1))));
                    mma16::mma_bf16(ones[j], one, b0, b1);
                    const uint32_t x0 = __byte_perm(w[0][j], w[1][j], 0x5410), x1 = __byte_perm(w[0][j], w[1][j], 0x7632);
                    const uint32_t y0 = __byte_perm(w[2][j], w[3][j], 0x5410), y1 = __byte_perm(w[2][j], w[3][j], 0x7632);
#pragma unroll
                    for (int n = 0; n < 4; ++n) {                     // features 8 g + 2 n (rows g) and 8 g + 2 n + 1 (rows g + 8) of the group
                        const uint32_t x = n < 2 ? x0 : x1, y = n < 2 ? y0 : y1;
                        const int i0 = 2 * (n & 1);
                        const uint32_t av[4] = {pair(x, i0), pair(x, i0 + 1), pair(y, i0), pair(y, i0 + 1)};
                        mma16::mma_bf16(o[j][n], av, b0, b1);
                    }
                }
            }
        }
        __syncwarp();
        slot = slot == STAGES - 1 ? 0 : slot + 1;
    }
    // the block's warps together: (max, sum, output) of each in shared memory
    mma16::cp_async_wait<0>();
#pragma unroll
    for (int x = 4; x < 32; x <<= 1) {
        total[0] += __shfl_xor_sync(0xffffffffu, total[0], x);
        total[1] += __shfl_xor_sync(0xffffffffu, total[1], x);
#pragma unroll
        for (int j = 0; j < G; ++j) {
            lows[j][0] += __shfl_xor_sync(0xffffffffu, lows[j][0], x);
            lows[j][1] += __shfl_xor_sync(0xffffffffu, lows[j][1], x);
        }
    }
    __syncthreads();
    constexpr int LD = D + 4;
    float* o_s = reinterpret_cast<float*>(ring_s);                    // [warps][heads][LD]
    float* m_s = o_s + WARPS * HEADS * LD;                            // [warps][heads]
    float* l_s = m_s + WARPS * HEADS;
    if (g == 0) {
        m_s[warp * HEADS + 2 * t] = most[0];
        m_s[warp * HEADS + 2 * t + 1] = most[1];
        l_s[warp * HEADS + 2 * t] = total[0];
        l_s[warp * HEADS + 2 * t + 1] = total[1];
    }
#pragma unroll
    for (int j = 0; j < G; ++j)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                o_s[(warp * HEADS + 2 * t + (e & 1)) * LD + 64 * j + 8 * g + 2 * n + (e >> 1)] = fmaf(-128.f, ones[j][e & 1], o[j][n][e] + lows[j][e & 1]);
    __syncthreads();
    float* f_s = l_s + WARPS * HEADS;                                 // [warps][heads]: what each warp's sums count
    if (threadIdx.x < HEADS) {
        const int h = threadIdx.x;
        float m = -INFINITY;
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, m_s[w * HEADS + h]);
        float l = 0.f;
        for (int w = 0; w < WARPS; ++w) {
            const float f = m_s[w * HEADS + h] == -INFINITY ? (l_s[w * HEADS + h] == 0.f ? 0.f : 1.f) : exp2f(m_s[w * HEADS + h] - m);
            f_s[w * HEADS + h] = f;
            l += f * l_s[w * HEADS + h];
        }
        m_s[h] = m;
        l_s[h] = l;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * D; i += 32 * WARPS) {
        const int h = i / D, f = i - h * D;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w)
            if (f_s[w * HEADS + h] != 0.f) v += f_s[w * HEADS + h] * o_s[(w * HEADS + h) * LD + f];
        o_s[h * LD + f] = v;                                          // (read and written by this thread alone)
    }
    __syncthreads();
    leave<__nv_bfloat16>(a, req, head0, heads, m_s, l_s, o_s, LD);
}

// ---- any page, float32 or bfloat16 queries, on the CUDA cores -----------------------------------------
constexpr int SIMT_KT = 32, SIMT_THREADS = 128;

inline size_t simt_floats(int d) { return (size_t)SIMT_KT * (d + 1) + (size_t)SIMT_KT * d + (size_t)2 * HEADS * d + HEADS * SIMT_KT + 3 * HEADS; }

template <typename T>
__global__ void __launch_bounds__(SIMT_THREADS) decode_simt_kernel(const DecodeArgs a) {
    extern __shared__ float sm[];
    const int d = a.d, ld = d + 1, groups = d / GROUP, words = d / 8;
    float* k_s = sm;                                // [places][d + 1]
    float* v_s = k_s + SIMT_KT * ld;                // [places][d]
    float* q_s = v_s + SIMT_KT * d;                 // [heads][d]
    float* o_s = q_s + HEADS * d;                   // [heads][d]
    float* p_s = o_s + HEADS * d;                   // [heads][places]
    float* m_s = p_s + HEADS * SIMT_KT;
    float* l_s = m_s + HEADS;
    float* f_s = l_s + HEADS;
    const int tid = threadIdx.x;
    const int group = a.nq / a.nkv, chunks = (group + HEADS - 1) / HEADS, kvh = blockIdx.y / chunks, chunk = blockIdx.y - kvh * chunks, req = blockIdx.z;
    const int head0 = kvh * group + chunk * HEADS, heads = min(HEADS, group - chunk * HEADS);
    pdl_enter_small();
    int beg, end;
    range_of(a, req, blockIdx.x, SIMT_KT, beg, end);
    const float scale = a.scale * LOG2E;
    for (int i = tid; i < HEADS * d; i += SIMT_THREADS) {
        q_s[i] = i / d < heads ? to_float(((const T*)a.q)[((size_t)req * a.nq + head0) * d + i]) * scale : 0.f;
        o_s[i] = 0.f;
    }
    if (tid < HEADS) m_s[tid] = -INFINITY, l_s[tid] = 0.f;
    const size_t rows = (size_t)a.page_size * row_bytes(d);
    for (int key0 = beg; key0 < end; key0 += SIMT_KT) {
        const int n = min(SIMT_KT, end - key0);
        __syncthreads();
        for (int i = tid; i < n * words * 2; i += SIMT_THREADS) {
            const int value = i >= n * words, x = value ? i - n * words : i, row = x / words, l = x - row * words;
            const int j = key0 + row, slot = j % a.page_size;
            const uint8_t* p = a.kv + (((size_t)page_of(a, req, j) * a.nkv + kvh) * 2 + value) * rows;
            const uint32_t w = reinterpret_cast<const uint32_t*>(p + (size_t)slot * (d / 2))[value ? value_word(l, groups) : key_word(l, groups)];
            const uint32_t h = reinterpret_cast<const uint32_t*>(p + (size_t)a.page_size * (d / 2))[slot * groups + (l >> 3)];
            float* dst = (value ? v_s + row * d : k_s + row * ld) + 8 * l;
#pragma unroll
            for (int e = 0; e < 8; ++e) dst[e] = fmaf((float)(w >> (4 * e) & 15u), low(h), high(h));
        }
        __syncthreads();
        for (int i = tid; i < HEADS * SIMT_KT; i += SIMT_THREADS) {
            const int h = i / SIMT_KT, j = i - h * SIMT_KT;
            float s = -INFINITY;
            if (j < n && h < heads) {
                float s0 = 0.f, s1 = 0.f;
                for (int f = 0; f < d; f += 2) {
                    s0 = fmaf(q_s[h * d + f], k_s[j * ld + f], s0);
                    s1 = fmaf(q_s[h * d + f + 1], k_s[j * ld + f + 1], s1);
                }
                s = s0 + s1;
            }
            p_s[i] = s;
        }
        __syncthreads();
        // a warp two heads, a lane a place
        for (int h = tid >> 5; h < heads; h += SIMT_THREADS / 32) {
            const int lane = tid & 31;
            const float s = p_s[h * SIMT_KT + lane], m = fmaxf(m_s[h], warp_max(s)), z = m == -INFINITY ? 0.f : m;
            const float p = lane < n ? exp2f(s - z) : 0.f, sum = warp_sum(p);
            const float was = m_s[h], f = was == m ? 1.f : exp2f(was - z);
            __syncwarp();
            p_s[h * SIMT_KT + lane] = p;
            if (lane == 0) m_s[h] = m, l_s[h] = l_s[h] * f + sum, f_s[h] = f;
        }
        __syncthreads();
        for (int i = tid; i < heads * d; i += SIMT_THREADS) {
            const int h = i / d, f = i - h * d;
            float v = o_s[i] * f_s[h];
            for (int j = 0; j < n; ++j) v = fmaf(p_s[h * SIMT_KT + j], v_s[j * d + f], v);
            o_s[i] = v;
        }
    }
    __syncthreads();
    leave<T>(a, req, head0, heads, m_s, l_s, o_s, d);
}

// ---- what the ranges of a row left, joined ------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(128) join_kernel(const DecodeArgs a) {
    pdl_enter_small();
    const size_t row = blockIdx.x;                  // request x query head
    const float* ml = a.part_ml + row * a.splits * 2;
    float m = -INFINITY;
    for (int z = 0; z < a.splits; ++z) m = fmaxf(m, ml[2 * z]);
    float l = 0.f;
    for (int z = 0; z < a.splits; ++z) l += ml[2 * z] == -INFINITY ? ml[2 * z + 1] : exp2f(ml[2 * z] - m) * ml[2 * z + 1];
    for (int f = threadIdx.x; f < a.d; f += 128) {
        float v = 0.f;
        for (int z = 0; z < a.splits; ++z) {
            const float w = ml[2 * z] == -INFINITY ? (ml[2 * z + 1] == 0.f ? 0.f : 1.f) : exp2f(ml[2 * z] - m);
            if (w != 0.f) v += w * a.part_o[(row * a.splits + z) * a.d + f];
        }
        ((T*)a.out)[row * a.d + f] = from_float<T>(l == 0.f ? 0.f : v / l);
    }
}

// Ranges a row's places are cut into.
inline int ranges_of(int requests, int nq, int nkv, int d, int longest, int page_size, int dtype) {
    const bool tensor_cores = dtype == kBF16 && page_size % 16 == 0;
    const long long pairs = (long long)requests * nkv * ((nq / nkv + HEADS - 1) / HEADS);
    const int room = (tensor_cores ? (d <= 128 ? 2 : 1) : 3) * sm_count(), step = tensor_cores ? KT * WARPS : SIMT_KT * 2;
    const long long want = pairs > 0 ? room / pairs : 1, most = ((long long)longest + step - 1) / step;
    return (int)max(1ll, min(min(want, most), 256ll));
}

}  // namespace four
}  // namespace lily

using namespace lily;

// float32 of scratch that lily_attention_decode4 needs
LILY_API size_t lily_attention_decode4_floats(int requests, int nq, int nkv, int d, int longest, int page_size, int dtype) {
    if (requests <= 0 || nkv <= 0 || nq <= 0 || nq % nkv || page_size <= 0) return 0;
    const int splits = four::ranges_of(requests, nq, nkv, d, longest, page_size, dtype);
    return splits == 1 ? 0 : (size_t)requests * nq * splits * (d + 2);
}

LILY_API int lily_attention_decode4(const void* q, const void* kv, void* out, const int* block_table, int width, const int* seq_lens, float* scratch, int requests, int longest, int nq,
                                    int nkv, int d, int page_size, int pages, float scale, int dtype, cudaStream_t stream) {
    if (requests == 0) return 0;
    LILY_REQUIRE(d >= four::GROUP && d <= 256 && d % four::GROUP == 0, "attention_decode4: heads of 64, 128, 192 or 256 features, not %d", d);
    LILY_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "attention_decode4: %d query heads over %d kv heads", nq, nkv);
    LILY_REQUIRE(requests > 0 && requests <= 65535 && page_size > 0 && longest >= 0 && longest <= (long long)width * page_size && pages > 0, "attention_decode4: %d requests of up to %d places, %d pages of %d",
                 requests, longest, width, page_size);
    LILY_REQUIRE(longest <= INT32_MAX - 1024, "attention_decode4: rows of %d places", longest);
    LILY_REQUIRE(((uintptr_t)q | (uintptr_t)kv | (uintptr_t)out) % 16 == 0, "attention_decode4: tensors on boundaries of sixteen bytes");
    const int chunks = (nq / nkv + four::HEADS - 1) / four::HEADS;
    LILY_REQUIRE((long long)nkv * chunks <= 65535, "attention_decode4: %d kv heads", nkv);
    four::DecodeArgs a{};
    a.q = q; a.kv = (const uint8_t*)kv; a.out = out; a.block_table = block_table; a.width = width; a.seq_lens = seq_lens;
    a.splits = four::ranges_of(requests, nq, nkv, d, longest, page_size, dtype);
    a.part_o = scratch;
    a.part_ml = scratch + (size_t)requests * nq * a.splits * d;
    a.nq = nq; a.nkv = nkv; a.d = d; a.page_size = page_size; a.pages = pages; a.longest = longest; a.scale = scale;
    LILY_REQUIRE(a.splits == 1 || scratch != nullptr, "attention_decode4: %d ranges need scratch", a.splits);
    const dim3 grid(a.splits, nkv * chunks, requests);
    if (dtype == kBF16 && page_size % 16 == 0) {
#define DECODE(D)                                                                                                                     \
    {                                                                                                                                 \
        constexpr int ring = four::WARPS * four::STAGES * four::Tile<D>::BYTES, join = four::WARPS * four::HEADS * (D + 4 + 3) * 4;   \
        constexpr int bytes = ring > join ? ring : join;                                                                              \
        cudaFuncSetAttribute(four::decode_mma_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);                         \
        launch_pdl(four::decode_mma_kernel<D>, grid, dim3(32 * four::WARPS), bytes, stream, a);                                       \
    }
        if (d == 64) DECODE(64)
        else if (d == 128) DECODE(128)
        else if (d == 192) DECODE(192)
        else DECODE(256)
#undef DECODE
    } else {
        const size_t bytes = four::simt_floats(d) * sizeof(float);
        auto run = [&](auto kernel) {
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
            launch_pdl(kernel, grid, dim3(four::SIMT_THREADS), bytes, stream, a);
        };
        if (dtype == kF32) run(four::decode_simt_kernel<float>);
        else run(four::decode_simt_kernel<__nv_bfloat16>);
    }
    LILY_CHECK_LAUNCH("attention_decode4");
    if (a.splits > 1) {
        if (dtype == kF32) launch_pdl(four::join_kernel<float>, dim3(requests * nq), dim3(128), 0, stream, a);
        else launch_pdl(four::join_kernel<__nv_bfloat16>, dim3(requests * nq), dim3(128), 0, stream, a);
        LILY_CHECK_LAUNCH("attention_decode4 (join)");
    }
    return 0;
}
