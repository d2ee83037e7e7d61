// Products with weights held in four bits: y = x W^T, W_rc = s_rg (code_rc - z_rg), g the group of 32, 64 or 128 columns that c is in (four.cuh says how they lie).
//
// A few tokens are bound by the weights' bytes: a quarter of a bfloat16 matrix's, and a scale a group.  Codes become bfloat16 numbers 128 + code by one logical operation a pair and
// code - z, exactly, by one subtraction; the tensor cores add up a group's products in float32, and its scale multiplies the sum, so no weight is ever rounded.
#include "four.cuh"
#include "mma.cuh"

namespace lily {
namespace four {

struct ProductArgs {
    const void* x;                // [m, k]
    const uint8_t* codes;         // [n / 128, k / 128, 128, 64]
    const __nv_bfloat16* scales;  // [n / 128, groups, 128], groups those of whole tiles of columns
    const uint8_t* zeros;         // the same, or null: 8
    const void* bias;             // [n] or null
    int bias_f32;
    void* out;                    // [m, n]
    int out_f32;
    int m, n, k, tiles;           // tiles of 128 columns
};

__device__ __forceinline__ uint4 weights16(const void* p) {          // weights are read once: not kept in the L1, which the tokens are to stay in
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t minus(uint32_t a, uint32_t b) { return bits(__hsub2(two(a), two(b))); }

constexpr int FEW_WARPS = 8;

// Up to 8 NT tokens: blocks walk tiles of 16 MT rows, their warps an eighth of the columns' tiles each; weights on the rows of the products, tokens on their eight columns.  A warp's weights
// are one stream, from one tile of rows to the next, which it asks for DEPTH steps ahead (the first ones before the kernel ahead has ended); tokens stay in the L1.
// What bounds it: logical operations and subtractions on the codes, of which a pair of codes takes two and a half (8 tokens, 24,576 x 4,096: 16.2 us, 3.2 TB/s of weights, the logic unit 55 % busy).
template <int NT, int PER_GROUP, int MT>                              // PER_GROUP: words of a lane (32 columns each) that share a scale, 1, 2 or 4
__global__ void __launch_bounds__(32 * FEW_WARPS, 2) product_few_kernel(const ProductArgs a, int row_tiles) {
    constexpr int GROUPS = 4 / PER_GROUP, ROWS = 16 * MT, DEPTH = GROUPS == 1 ? 3 : 2;
    __shared__ float sum_s[2][FEW_WARPS][8 * NT][ROWS + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const size_t groups = (size_t)a.tiles * GROUPS;
    const int steps = (a.tiles - warp + FEW_WARPS - 1) / FEW_WARPS;   // of this warp and a tile of rows
    struct Step { uint4 w[MT][2]; unsigned short s[MT][2][GROUPS]; unsigned char z[MT][2][GROUPS]; };
    // what to ask for next
    int ask_tile = blockIdx.x, ask_kt = warp;
    auto ask = [&](Step& c) {
        if (steps == 0 || ask_tile >= row_tiles) return;
        const int row0 = ask_tile * ROWS, in_tile = row0 % 128;
        const size_t tile_row = row0 / 128;
        const uint8_t* p = a.codes + ((tile_row * a.tiles + ask_kt) * 128 + in_tile) * 64 + lane * 16;        // (a lane's sixteen bytes: row g, piece t)
        const size_t held0 = (tile_row * groups + (size_t)ask_kt * GROUPS) * 128 + in_tile + g;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                c.w[mt][e] = weights16(p + (mt * 16 + e * 8) * 64);
#pragma unroll
                for (int i = 0; i < GROUPS; ++i) {
                    const size_t at = held0 + i * 128 + mt * 16 + e * 8;
                    const bool in = ask_kt * 128 + i * (128 / GROUPS) < a.k;             // (what stands behind the last column may be no number)
                    c.s[mt][e][i] = in ? __ldg(reinterpret_cast<const unsigned short*>(a.scales) + at) : 0;
                    c.z[mt][e][i] = a.zeros ? __ldg(a.zeros + at) : 8;
                }
            }
        ask_kt += FEW_WARPS;
        if (ask_kt >= a.tiles) ask_kt = warp, ask_tile += gridDim.x;
    };
    Step ring[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) ask(ring[d]);
    pdl_launch_dependents();
    pdl_wait();
    float total[MT][NT][4];
    auto clear = [&]() {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) total[mt][nt][e] = 0.f;
    };
    clear();
    auto work = [&](const Step& cur, int kt) {
        uint4 xv[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int token = nt * 8 + g, col = kt * 128 + 32 * w + 8 * t;
                xv[nt][w] = make_uint4(0, 0, 0, 0);
                if (token < a.m && col < a.k) xv[nt][w] = *reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.x + (size_t)token * a.k + col);
            }
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) {
            float sum[MT][NT][4];
            uint32_t zero[MT][2];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[mt][nt][e] = 0.f;
#pragma unroll
                for (int e = 0; e < 2; ++e) zero[mt][e] = (0x4300u | cur.z[mt][e][i]) * 0x10001u;
            }
#pragma unroll
            for (int v = 0; v < PER_GROUP; ++v) {
                const int w = i * PER_GROUP + v;
                uint32_t b[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    b[nt][0] = __byte_perm(xv[nt][w].x, xv[nt][w].z, 0x5410);
                    b[nt][1] = __byte_perm(xv[nt][w].x, xv[nt][w].z, 0x7632);
                    b[nt][2] = __byte_perm(xv[nt][w].y, xv[nt][w].w, 0x5410);
                    b[nt][3] = __byte_perm(xv[nt][w].y, xv[nt][w].w, 0x7632);
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const uint32_t p = (&cur.w[mt][0].x)[w], q = (&cur.w[mt][1].x)[w], zp = zero[mt][0], zq = zero[mt][1];
                    const uint32_t a0[4] = {minus(pair(p, 0), zp), minus(pair(q, 0), zq), minus(pair(p, 1), zp), minus(pair(q, 1), zq)};
                    const uint32_t a1[4] = {minus(pair(p, 2), zp), minus(pair(q, 2), zq), minus(pair(p, 3), zp), minus(pair(q, 3), zq)};
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma16::mma_bf16(sum[mt][nt], a0, b[nt][0], b[nt][1]);
                        mma16::mma_bf16(sum[mt][nt], a1, b[nt][2], b[nt][3]);
                    }
                }
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const float s0 = __uint_as_float((uint32_t)cur.s[mt][0][i] << 16), s1 = __uint_as_float((uint32_t)cur.s[mt][1][i] << 16);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    total[mt][nt][0] = fmaf(s0, sum[mt][nt][0], total[mt][nt][0]);
                    total[mt][nt][1] = fmaf(s0, sum[mt][nt][1], total[mt][nt][1]);
                    total[mt][nt][2] = fmaf(s1, sum[mt][nt][2], total[mt][nt][2]);
                    total[mt][nt][3] = fmaf(s1, sum[mt][nt][3], total[mt][nt][3]);
                }
            }
        }
    };
    int tile = blockIdx.x, buffer = 0;
    // the warps' sums of a tile of rows together (one barrier a tile: sums of the next one go to the other buffer)
    auto finish = [&]() {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum_s[buffer][warp][nt * 8 + 2 * t + (e & 1)][mt * 16 + g + (e >> 1) * 8] = total[mt][nt][e];
        __syncthreads();
        for (int i = threadIdx.x; i < 8 * NT * ROWS; i += 32 * FEW_WARPS) {
            const int token = i / ROWS, r = i % ROWS, row = tile * ROWS + r;
            if (token >= a.m || row >= a.n) continue;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < FEW_WARPS; ++w) v += sum_s[buffer][w][token][r];
            if (a.bias) v += a.bias_f32 ? ((const float*)a.bias)[row] : __bfloat162float(((const __nv_bfloat16*)a.bias)[row]);
            const size_t at = (size_t)token * a.n + row;
            if (a.out_f32) ((float*)a.out)[at] = v;
            else ((__nv_bfloat16*)a.out)[at] = __float2bfloat16_rn(v);
        }
        buffer ^= 1;
        tile += gridDim.x;
        clear();
    };
    if (steps == 0) {                                                 // (fewer tiles of columns than warps)
        while (tile < row_tiles) finish();
        return;
    }
    for (int kt = warp; tile < row_tiles;) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            if (tile >= row_tiles) break;
            work(ring[d], kt);
            ask(ring[d]);
            kt += FEW_WARPS;
            if (kt >= a.tiles) {
                kt = warp;
                finish();
            }
        }
    }
}

// Up to eight tokens in float32: a block eight rows, its sixteen warps a sixteenth of the columns' tiles each; a lane eight columns of a row at a time, all products and sums in
// float32, a word's eight of them before their scale.  grid (rows / 8)
// What bounds it is the way to the tokens' numbers, which every warp reads once, so it is warps that count, two blocks a multiprocessor, and registers that are to allow them: three tokens, 2,049 rows of
// 8,192 columns in groups of 32 with zero points 13.4 us (a tenth of its bytes' time), 24.7 in blocks of eight warps that ask three tiles ahead, 14.9 in sixteen that ask two ahead; tokens asked for a
// word ahead 27.5, by the registers that they take.
constexpr int F32_TOKENS = 8, F32_WARPS = 16;
template <int TOKENS>
__global__ void __launch_bounds__(32 * F32_WARPS, 2) product_f32_kernel(const ProductArgs a, int group_shift) {
    __shared__ float sum_s[F32_WARPS][TOKENS][8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int row0 = blockIdx.x * 8, tile_row = row0 / 128;
    const uint8_t* codes = a.codes + ((size_t)tile_row * a.tiles * 128 + row0 % 128) * 64 + lane * 16;
    const size_t held0 = (size_t)tile_row * (a.tiles * 128 >> group_shift) * 128 + row0 % 128 + g;
    uint4 v;                                                          // the next tile's weights
    unsigned short scales[4];
    unsigned char zeros[4];
    auto ask = [&](int kt) {
        if (kt >= a.tiles) return;
        v = weights16(codes + (size_t)kt * 128 * 64);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int col = kt * 128 + 32 * w;
            const size_t at = held0 + (size_t)(col >> group_shift) * 128;
            scales[w] = col < a.k ? __ldg(reinterpret_cast<const unsigned short*>(a.scales) + at) : 0;
            zeros[w] = a.zeros && col < a.k ? __ldg(a.zeros + at) : 8;
        }
    };
    ask(warp);
    pdl_launch_dependents();
    pdl_wait();
    float total[TOKENS];
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) total[i] = 0.f;
    for (int kt = warp; kt < a.tiles; kt += F32_WARPS) {
        uint32_t words[4] = {v.x, v.y, v.z, v.w};
        float s[4], z[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) s[w] = __uint_as_float((uint32_t)scales[w] << 16), z[w] = __uint_as_float(0x4B000000u | zeros[w]);      // (2^23 + zero point)
        ask(kt + F32_WARPS);
#pragma unroll 1
        for (int col = kt * 128 + 8 * t; col < min(a.k, kt * 128 + 128); col += 32) {      // (a short loop: its words in turn)
            float c[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) c[e] = __uint_as_float((words[0] >> (4 * e) & 15u) | 0x4B000000u) - z[0];         // (2^23 + code: exact)
#pragma unroll
            for (int i = 0; i < TOKENS; ++i) {
                if (i >= a.m) break;
                const float4 *p = reinterpret_cast<const float4*>((const float*)a.x + (size_t)i * a.k + col), x0 = p[0], x1 = p[1];
                const float first = fmaf(c[0], x0.x, fmaf(c[1], x0.y, fmaf(c[2], x0.z, c[3] * x0.w))), second = fmaf(c[4], x1.x, fmaf(c[5], x1.y, fmaf(c[6], x1.z, c[7] * x1.w)));
                total[i] = fmaf(s[0], first + second, total[i]);
            }
#pragma unroll
            for (int w = 0; w < 3; ++w) words[w] = words[w + 1], s[w] = s[w + 1], z[w] = z[w + 1];
        }
    }
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) {
        total[i] += __shfl_xor_sync(0xffffffffu, total[i], 1);
        total[i] += __shfl_xor_sync(0xffffffffu, total[i], 2);
        if (t == 0) sum_s[warp][i][g] = total[i];
    }
    __syncthreads();
    if (threadIdx.x < TOKENS * 8) {
        const int i = threadIdx.x / 8, r = threadIdx.x % 8;
        float y = 0.f;
#pragma unroll
        for (int w = 0; w < F32_WARPS; ++w) y += sum_s[w][i][r];
        if (i < a.m && row0 + r < a.n) ((float*)a.out)[(size_t)i * a.n + row0 + r] = y + (a.bias ? ((const float*)a.bias)[row0 + r] : 0.f);
    }
}

// The weights as numbers [n, k] (float32: exact; bfloat16: rounded once).  A warp eight rows of a tile, a lane sixteen bytes of codes, four words of eight.  In bfloat16 code - zero is exact and its product
// with the scale one rounding, of two numbers an operation.  6,144 x 4,096 in bfloat16 10.6 us with the empty kernel behind it, 0.9 of what its bytes take (a word a thread 14.4, number by number besides 16.8).
// grid (tiles of columns / 8, rows / 8 from row0 on)
template <typename T>
__global__ void __launch_bounds__(256) weights_kernel(const ProductArgs a, int group_shift, int row0) {
    pdl_enter_small();
    const int lane = threadIdx.x & 31, t = lane & 3, row = row0 + blockIdx.y * 8 + (lane >> 2), kt = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (kt >= a.tiles || row >= a.n) return;
    const uint4 codes = weights16(a.codes + (((size_t)(row / 128) * a.tiles + kt) * 128 + row % 128) * 64 + t * 16);
    const uint32_t words[4] = {codes.x, codes.y, codes.z, codes.w};
    const size_t held0 = (size_t)(row / 128) * (a.tiles * 128 >> group_shift) * 128 + row % 128;
    __nv_bfloat16 scales[4];
    uint32_t zeros[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int col = kt * 128 + 32 * w;
        const size_t at = held0 + (size_t)(col >> group_shift) * 128;
        scales[w] = col < a.k ? a.scales[at] : __ushort_as_bfloat16(0);
        zeros[w] = a.zeros && col < a.k ? a.zeros[at] : 8u;
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int col = kt * 128 + 32 * w + 8 * t;
        if (col >= a.k) break;
        T* dst = (T*)a.out + (size_t)row * a.k + col;
        if constexpr (sizeof(T) == 2) {
            const uint32_t z = (0x4300u | zeros[w]) * 0x10001u;       // 128 + zero, twice
            const __nv_bfloat162 s = __halves2bfloat162(scales[w], scales[w]);
            uint32_t p[4];                                            // numbers i and i + 4
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = bits(__hmul2(two(minus(pair(words[w], i), z)), s));
            *reinterpret_cast<uint4*>(dst) = make_uint4(__byte_perm(p[0], p[1], 0x5410), __byte_perm(p[2], p[3], 0x5410), __byte_perm(p[0], p[1], 0x7632), __byte_perm(p[2], p[3], 0x7632));
        } else {
            const float s = __bfloat162float(scales[w]), z = __uint_as_float(0x4B000000u | zeros[w]);      // (2^23 + zero)
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (__uint_as_float((words[w] >> (4 * e) & 15u) | 0x4B000000u) - z) * s;
            reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
    }
}

// Nothing.  Kernels that take few rows read their weights' first tiles while the kernel ahead of them may still run; launched the ordinary way behind the numbers, this one begins when
// they are all there.
__global__ void at_rest_kernel() {}

}  // namespace four
}  // namespace lily

using namespace lily;

static bool weights_fit(int n, int k, int group) { return n > 0 && k > 0 && (group == 32 || group == 64 || group == 128) && k % group == 0 && n <= INT32_MAX - 256 && k <= INT32_MAX - 256; }

// Tokens that the kernels for few of them take.
static int few_tokens(int dtype) { return dtype == kBF16 ? 16 : four::F32_TOKENS; }

LILY_API int lily_linear4_few_tokens(int dtype) { return few_tokens(dtype); }

LILY_API int lily_linear4(const void* x, int dtype, const void* codes, const void* scales, const void* zeros, const void* bias, int bias_f32, void* out, int out_f32, int m, int n, int k,
                          int group, cudaStream_t stream) {
    if (m == 0 || n == 0) return 0;
    LILY_REQUIRE(weights_fit(n, k, group), "linear4: a matrix [%d, %d] in groups of %d", n, k, group);
    LILY_REQUIRE(m > 0 && m <= few_tokens(dtype), "linear4: %d tokens", m);
    LILY_REQUIRE(dtype == kBF16 || (out_f32 && (!bias || bias_f32)), "linear4: float32 tokens keep float32");
    LILY_REQUIRE(((uintptr_t)x | (uintptr_t)codes) % 16 == 0, "linear4: tensors on boundaries of sixteen bytes");
    const four::ProductArgs a{x, (const uint8_t*)codes, (const __nv_bfloat16*)scales, (const uint8_t*)zeros, bias, bias_f32, out, out_f32, m, n, k, (k + 127) / 128};
    if (dtype == kF32) {
        const dim3 grid((n + 7) / 8), block(32 * four::F32_WARPS);
        const int shift = group == 32 ? 5 : group == 64 ? 6 : 7;
        if (m == 1) launch_pdl(four::product_f32_kernel<1>, grid, block, 0, stream, a, shift);
        else if (m <= 4) launch_pdl(four::product_f32_kernel<4>, grid, block, 0, stream, a, shift);
        else launch_pdl(four::product_f32_kernel<four::F32_TOKENS>, grid, block, 0, stream, a, shift);
    } else {
        // Up to eight tokens 32 rows a block and turn (24,576 x 4,096 with eight 16.2 us, 18.2 with 16 rows; 6,144 x 4,096 with four 5.9 and 7.2), 16 where that leaves SMs without (4,096 x 4,096 with one
        // token 3.9 us, 5.3 with 32 rows).  From nine on 16, by the registers (12,288 x 4,096 with sixteen 15.0 us, 18.5 with 32; 4,096 x 12,288 14.4 and 26.3; 6,144 x 4,096 9.9 and 9.5).
        const int mt = m > 8 || (n + 31) / 32 <= sm_count() ? 1 : 2, row_tiles = (n + 16 * mt - 1) / (16 * mt);
        const dim3 grid(min(row_tiles, 2 * sm_count())), block(32 * four::FEW_WARPS);
#define FEW_OF(NT, MT)                                                                                               \
    do {                                                                                                             \
        if (group == 128) launch_pdl(four::product_few_kernel<NT, 4, MT>, grid, block, 0, stream, a, row_tiles);     \
        else if (group == 64) launch_pdl(four::product_few_kernel<NT, 2, MT>, grid, block, 0, stream, a, row_tiles); \
        else launch_pdl(four::product_few_kernel<NT, 1, MT>, grid, block, 0, stream, a, row_tiles);                  \
    } while (0)
        if (m > 8) FEW_OF(2, 1);
        else if (mt == 1) FEW_OF(1, 1);
        else FEW_OF(1, 2);
#undef FEW_OF
    }
    LILY_CHECK_LAUNCH("linear4");
    return 0;
}

LILY_API int lily_weights4(const void* codes, const void* scales, const void* zeros, void* out, int dtype, int n, int k, int group, cudaStream_t stream) {
    LILY_REQUIRE(weights_fit(n, k, group), "weights4: a matrix [%d, %d] in groups of %d", n, k, group);
    LILY_REQUIRE(((uintptr_t)out | (uintptr_t)codes) % 16 == 0, "weights4: tensors on boundaries of sixteen bytes");
    const four::ProductArgs a{nullptr, (const uint8_t*)codes, (const __nv_bfloat16*)scales, (const uint8_t*)zeros, nullptr, 0, out, 0, 0, n, k, (k + 127) / 128};
    const int shift = group == 32 ? 5 : group == 64 ? 6 : 7;
    constexpr int MOST = 65535 * 8;                                   // rows of a launch
    for (int row0 = 0; row0 < n; row0 += min(MOST, n - row0)) {
        const dim3 grid((a.tiles + 7) / 8, (min(MOST, n - row0) + 7) / 8);
        if (dtype == kF32) launch_pdl(four::weights_kernel<float>, grid, dim3(256), 0, stream, a, shift, row0);
        else launch_pdl(four::weights_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, a, shift, row0);
        LILY_CHECK_LAUNCH("weights4");
    }
    four::at_rest_kernel<<<1, 32, 0, stream>>>();
    LILY_CHECK_LAUNCH("weights4");
    return 0;
}
