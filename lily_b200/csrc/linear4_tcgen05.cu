// Products with 4-bit weights for more than a few tokens, on tcgen05: Y^T = W X^T, weights on the 128 rows of a tile, up to 256 tokens on its columns.
//
// A block has 128 rows of W and a range of its columns, in steps of 128:
//   warp 0     brings the step's codes (8 KB) and its tokens [tokens, 128] by TMA, its scales and zero points by bulk copies, into a ring of stages;
//   warps 2-9  make the codes bfloat16 numbers, (code - zero) exactly and then its product with the scale, rounded once, and put them into tensor memory as the products' first
//              operand (a thread a row; four warps the even steps, four the odd ones): through shared memory they would be written and read at the bandwidth that bounds the products;
//   warp 1     multiplies: eight 128 x tokens x 16 products a step into one accumulator in tensor memory.
// The blocks of a cluster share out a row tile's columns and add their accumulators up through shared memory, each for its share of the tokens.
// The weights are rounded to bfloat16 because an operand of the tensor cores has one scale for all its columns; their products and sums are float32 throughout.
//
// What bounds it: a step takes a block some 0.5 us, which its eight warps spend on the codes, two blocks a SM side by side (45 tokens, 4,096 x 12,288 in groups of 64 with zero points: 15.6 us, 1.9 TB/s of weights,
// the tensor pipe 15 % busy); through shared memory the weights took 20.8.  Filling and joining take 3 us.
//
// Every wait is bounded: one that runs out leaves its code in a word of the host's memory (lily_linear4_status) and NaN in the outputs of its cluster.  The block then
// waits, a bounded time again, for what it has on its way, copies and products, before it frees its tensor memory and leaves.
#include "four.cuh"
#include "tcgen05.cuh"

#include <atomic>
#include <cooperative_groups.h>
#include <type_traits>

namespace lily {
int* new_host_word();
namespace four {
namespace many {

constexpr int ROWS = 128, STEP = 128;
constexpr int CODES = ROWS * STEP / 2;
constexpr int OPERAND = STEP / 2;                        // columns of tensor memory of a step's weights
constexpr int OPERANDS = 4;                              // at most
constexpr int GROUPS = 2, WORKERS = 4, THREADS = 32 * (2 + GROUPS * WORKERS);      // groups of warps that take steps in turn, a warp a quarter of the rows
constexpr int MOST_TOKENS = 256, MOST_SPLITS = 8;
constexpr int MOST_BYTES = 225 * 1024;                   // of shared memory
constexpr int POLLS = 1 << 17;                           // of up to ten microseconds each: a second before a wait gives up
constexpr int LAST_POLLS = 1 << 16;                      // ... and of the waits of a block that has given up for what it has on its way

struct Args {
    const uint8_t* scales;                               // bytes of bfloat16 numbers
    const uint8_t* zeros;                                // or null: 8
    const void* bias;
    int bias_f32;
    void* out;
    int out_f32;
    int m, n, k, tiles;                                  // tiles of 128 columns
    int tokens;                                          // columns of the accumulator, a multiple of 16
    int stages, splits, operands;
    int columns;                                         // of tensor memory: the accumulator's, then the operands'
    int polls;                                           // how often a wait asks before it gives up
    int* lost;                                           // a word of the host's where it says so: (code << 24 | block)
};

// Asks once, asleep for up to ten microseconds: a warp that polls takes turns away from those that work.
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.b32 %0, 1, 0, p;\n}\n" : "=r"(ok) : "r"(bar), "r"(parity), "r"(10000u) : "memory");
    return ok != 0;
}
struct Waits { volatile int* lost; int* word; int polls; };
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, const Waits& w, int code) {
    bool come = try_wait(bar, parity);
    for (int i = 1; !come && i < w.polls; ++i) {
        if ((i & 15) == 15 && *w.lost) break;
        come = try_wait(bar, parity);
    }
    come = __all_sync(0xffffffffu, come && w.polls > 0);      // (the whole warp goes on, or none of it)
    if (!come && !*w.lost) {
        *w.lost = 1;
        *(volatile int*)w.word = (code << 24) | (int)((blockIdx.x + blockIdx.y * gridDim.x) & 0xFFFFFF);
        __threadfence_system();
    }
    return come;
}
// What is on its way when a block has given up.
__device__ __forceinline__ void last_wait(uint32_t bar, uint32_t parity) {
    for (int i = 0; i < LAST_POLLS && !try_wait(bar, parity); ++i) {}
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// Bytes i of two words of codes 0..15, one code a byte, as a pair of bfloat16 numbers code 2^-133 (the lowest subnormal ones; the bytes above them are the codes' signs, zero).
template <int I>
__device__ __forceinline__ uint32_t tiny_pair(uint32_t even, uint32_t odd) {
    uint32_t r;                                          // (the intrinsic leaves out the selector's bits for signs)
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(even), "r"(odd), "n"(0xC480 + 0x1111 * I));
    return r;
}

// What a stage holds: codes, scales (up to four groups of 128), zero points, tokens (two halves).
__host__ __device__ constexpr int SCALES_AT() { return CODES; }
__host__ __device__ constexpr int ZEROS_AT() { return CODES + 4 * 256; }
__host__ __device__ constexpr int TOKENS_AT() { return CODES + 4 * 256 + 4 * 128 + 512; }       // (a multiple of 1024 for the swizzle)
__host__ __device__ inline int stage_bytes(int tokens) { return TOKENS_AT() + tokens * 256; }

// grid (row tiles x splits, token tiles), cluster (splits)
template <int PER_STEP>                                  // groups of a step: 1, 2 or 4
__global__ void __launch_bounds__(THREADS, 2) product_many_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const Args a) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + (-tc5::smem_u32(smem_raw) & 1023u);      // (an offset, so that it stays an address of shared memory)
    __shared__ __align__(8) uint64_t bars[2 * 8 + 2 * OPERANDS + 1];
    __shared__ uint32_t tmem_s;
    __shared__ int lost_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % a.splits, row_tile = blockIdx.x / a.splits, token0 = blockIdx.y * a.tokens;
    const int kt0 = (int)((long long)a.tiles * rank / a.splits), steps = (int)((long long)a.tiles * (rank + 1) / a.splits) - kt0;
    const int stage = stage_bytes(a.tokens);
    unsigned char* ring = smem;
    const uint32_t full0 = tc5::smem_u32(&bars[0]), empty0 = tc5::smem_u32(&bars[8]), made0 = tc5::smem_u32(&bars[16]), freed0 = tc5::smem_u32(&bars[16 + OPERANDS]),
                   ready = tc5::smem_u32(&bars[16 + 2 * OPERANDS]);
    volatile int* lost = &lost_s;
    const Waits waits{lost, a.lost, a.polls};
    int issued = 0;                                      // warp 0: steps whose copies are on their way or have come
    const uint32_t columns = a.columns;

    if (threadIdx.x == 0) {
        lost_s = 0;
        for (int s = 0; s < a.stages; ++s) {
            tc5::mbar_init(full0 + 8 * s, 1);
            tc5::mbar_init(empty0 + 8 * s, 1);
        }
        for (int s = 0; s < OPERANDS; ++s) {
            tc5::mbar_init(made0 + 8 * s, WORKERS);
            tc5::mbar_init(freed0 + 8 * s, 1);
        }
        tc5::mbar_init(ready, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(tc5::smem_u32(&tmem_s)), "r"(columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    tc5::tc_fence_before();
    __syncthreads();
    tc5::tc_fence_after();
    const uint32_t tmem = tmem_s, operands = tmem + columns - a.operands * OPERAND;
    pdl_launch_dependents();

    if (warp == 0) {
        const uint32_t held = 256u * PER_STEP, bytes = CODES + held + (a.zeros ? held / 2 : 0) + (uint32_t)a.tokens * 256;
        const int codes = (row_tile * a.tiles + kt0) * ROWS;
        const uint8_t* scales = a.scales + ((size_t)row_tile * a.tiles + kt0) * held;
        const uint8_t* zeros = a.zeros ? a.zeros + ((size_t)row_tile * a.tiles + kt0) * (held / 2) : nullptr;
        auto weights = [&](int it, int s) {
            const uint32_t at = tc5::smem_u32(ring + (size_t)s * stage), bar = full0 + 8 * s;
            tc5::mbar_expect_tx(bar, bytes);
            tc5::tma_load_2d(at, &map_w, bar, 0, codes + it * ROWS);
            bulk_copy(at + SCALES_AT(), scales + (size_t)it * held, held, bar);
            if (zeros) bulk_copy(at + ZEROS_AT(), zeros + (size_t)it * (held / 2), held / 2, bar);
        };
        auto tokens = [&](int it, int s) {
            const uint32_t at = tc5::smem_u32(ring + (size_t)s * stage) + TOKENS_AT(), bar = full0 + 8 * s;
            tc5::tma_load_2d(at, &map_x, bar, (kt0 + it) * STEP, token0);
            tc5::tma_load_2d(at + a.tokens * 128, &map_x, bar, (kt0 + it) * STEP + 64, token0);
        };
        // the first stages' weights are nobody's results: on their way before the kernel ahead has ended
        const int early = min(a.stages, steps);
        if (tc5::elect_one())
            for (int it = 0; it < early; ++it) weights(it, it);
        __syncwarp();
        pdl_wait();
        if (tc5::elect_one())
            for (int it = 0; it < early; ++it) tokens(it, it);
        __syncwarp();
        int it = early;
        for (int s = 0, turn = 0; it < steps; ++it) {
            if (!wait(empty0 + 8 * s, turn, waits, 1)) break;
            if (tc5::elect_one()) {
                weights(it, s);
                tokens(it, s);
            }
            __syncwarp();
            if (++s == a.stages) s = 0, turn ^= 1;
        }
        issued = it;
    } else if (warp == 1) {
        // kind::f16, bfloat16 a and b (k-major), float32 d, 128 rows
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(a.tokens >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
        bool ok = true;
        for (int it = 0, s = 0, turn = 0, o = 0, o_turn = 0; it < steps; ++it) {
            ok = wait(full0 + 8 * s, turn, waits, 2) && wait(made0 + 8 * o, o_turn, waits, 3);
            if (!ok) break;
            tc5::tc_fence_after();
            const uint32_t w = operands + o * OPERAND, x = tc5::smem_u32(ring + (size_t)s * stage) + TOKENS_AT();
            if (tc5::elect_one()) {
#pragma unroll
                for (int kk = 0; kk < STEP / 16; ++kk) {
                    const uint64_t db = tc5::desc_k_major(x + (kk / 4) * (a.tokens * 128)) + (uint64_t)((kk % 4) * 2);
                    tc5::umma_ts(tmem, w + kk * 8, db, idesc, (it | kk) != 0 ? 1u : 0u);
                }
                tc5::umma_commit(empty0 + 8 * s);
                tc5::umma_commit(freed0 + 8 * o);
                if (it == steps - 1) tc5::umma_commit(ready);
            }
            __syncwarp();
            if (++s == a.stages) s = 0, turn ^= 1;
            if (++o == a.operands) o = 0, o_turn ^= 1;
        }
        if (!ok) {                                       // products on their way read shared and tensor memory: they end first
            if (tc5::elect_one()) tc5::umma_commit(ready);
            __syncwarp();
            last_wait(ready, 0);
        }
    } else {
        // A thread a row of the step: pieces of sixteen bytes, which the copy has swizzled so that eight threads' lie in all banks, with a word of each 32 columns.
        const int group = (warp - 2) / WORKERS, row = (warp & 3) * 32 + lane;
        const __nv_bfloat162 up = __halves2bfloat162(__ushort_as_bfloat16(0x7F00), __ushort_as_bfloat16(0x7F00));                 // 2^127
        int s = group, turn = 0, o = group, o_turn = 1;  // (there are two stages and two operands at least)
        for (int it = group; it < steps; it += GROUPS) {
            if (!wait(full0 + 8 * s, turn, waits, 4)) break;
            const unsigned char* in = ring + (size_t)s * stage;
            uint4 raw[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) raw[t] = *reinterpret_cast<const uint4*>(in + row * 64 + ((t ^ (row >> 1 & 3)) << 4));
            uint32_t scale[PER_STEP], zero[PER_STEP];
#pragma unroll
            for (int i = 0; i < PER_STEP; ++i) {
                scale[i] = *reinterpret_cast<const unsigned short*>(in + SCALES_AT() + (i * 128 + row) * 2);
                zero[i] = a.zeros ? in[ZEROS_AT() + i * 128 + row] : 8u;
            }
            if (it >= a.operands && !wait(freed0 + 8 * o, o_turn, waits, 5)) break;
            tc5::tc_fence_after();
            const uint32_t to = operands + o * OPERAND + ((uint32_t)((warp & 3) * 32) << 16);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t numbers[32];                    // columns 64 half + (0..63), in pairs
#pragma unroll
                for (int v = 0; v < 2; ++v) {
                    const int w = 2 * half + v, i = w * PER_STEP / 4;
                    // (code - zero) 2^-6 in one operation, exactly; its product with 2^6 scale rounded once
                    const __nv_bfloat162 down = __bfloat162bfloat162(__float2bfloat16_rn((__uint_as_float(0x4B000000u | zero[i]) - 8388608.f) * -0.015625f));
                    float f = __uint_as_float(scale[i] << 16) * 64.f;
                    if ((kt0 + it) * STEP + 32 * w >= a.k) f = 0.f;      // (what stands behind the last column may be no number)
                    const __nv_bfloat162 by = __bfloat162bfloat162(__float2bfloat16_rn(f));
                    auto number = [&](uint32_t tiny) { return bits(__hmul2(__hfma2(two(tiny), up, down), by)); };
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const uint32_t word = w == 0 ? raw[t].x : w == 1 ? raw[t].y : w == 2 ? raw[t].z : raw[t].w;
                        const uint32_t even = word & 0x0F0F0F0Fu, odd = word >> 4 & 0x0F0F0F0Fu;
                        numbers[16 * v + 4 * t] = number(tiny_pair<0>(even, odd));
                        numbers[16 * v + 4 * t + 1] = number(tiny_pair<1>(even, odd));
                        numbers[16 * v + 4 * t + 2] = number(tiny_pair<2>(even, odd));
                        numbers[16 * v + 4 * t + 3] = number(tiny_pair<3>(even, odd));
                    }
                }
                tc5::tmem_st32(to + 32 * half, reinterpret_cast<const float*>(numbers));
            }
            tc5::tmem_wait_st();
            tc5::tc_fence_before();
            __syncwarp();
            if (lane == 0) tc5::mbar_arrive(made0 + 8 * o);
            s += GROUPS;
            while (s >= a.stages) s -= a.stages, turn ^= 1;
            o += GROUPS;
            while (o >= a.operands) o -= a.operands, o_turn ^= 1;
        }
        // the accumulator to shared memory, where the ring was: [tokens][128]
        const bool ok = wait(ready, 0, waits, 6) && !__any_sync(0xffffffffu, *lost);
        tc5::tc_fence_after();
        float* sums = reinterpret_cast<float*>(smem);
        const int quarter = warp & 3, first = (warp - 2) >> 2;      // (a warp reads its quarter of the lanes)
        for (int c = first * 32; ok && c < a.tokens; c += 32 * (GROUPS * WORKERS / 4)) {
            float v[32];
            tc5::tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + c, v);
            tc5::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e)
                if (c + e < a.tokens) sums[(c + e) * ROWS + quarter * 32 + lane] = v[e];
        }
        tc5::tc_fence_before();
    }
    __syncthreads();
    if (warp == 0 && lost_s)                             // (whoever gave up, also behind the loader's last step)
        for (int j = max(0, issued - a.stages); j < issued; ++j) last_wait(full0 + 8 * (j % a.stages), (j / a.stages) & 1);
    if (warp == 1) {
        tc5::tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(columns) : "memory");
    }
    const auto cluster = cooperative_groups::this_cluster();
    if (a.splits > 1) cluster.sync();
    const float* sums = reinterpret_cast<const float*>(smem);
    bool given_up = lost_s;                              // a wait of this block ran out, or of another one of the cluster
    if (a.splits > 1) {
        int theirs = 0;
#pragma unroll
        for (int z = 0; z < MOST_SPLITS; ++z) theirs |= *cluster.map_shared_rank(&lost_s, min(z, a.splits - 1));
        given_up = given_up || theirs;
    }
    // a warp a token, a lane four rows, whose bias it so looks up once, with up to four tokens on their way: 256 tokens, 150 x 128 in 8.8 us, 16.3 with a number a thread and turn
    const int row = row_tile * ROWS + 4 * lane, all = min(a.tokens, a.m - token0);
    const bool whole = a.n % 4 == 0 && row + 4 <= a.n && (uintptr_t)a.out % 16 == 0;
    float bias[4] = {0.f, 0.f, 0.f, 0.f};
    if (a.bias)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (row + e < a.n) bias[e] = a.bias_f32 ? ((const float*)a.bias)[row + e] : __bfloat162float(((const __nv_bfloat16*)a.bias)[row + e]);
    auto put = [&](int token, float4 v) {
        float y[4] = {v.x + bias[0], v.y + bias[1], v.z + bias[2], v.w + bias[3]};
        if (given_up) y[0] = y[1] = y[2] = y[3] = __int_as_float(0x7fffffff);
        const size_t to = (size_t)(token0 + token) * a.n + row;
        if (whole) {
            if (a.out_f32) *reinterpret_cast<float4*>((float*)a.out + to) = make_float4(y[0], y[1], y[2], y[3]);
            else *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + to) = make_uint2(bits(__floats2bfloat162_rn(y[0], y[1])), bits(__floats2bfloat162_rn(y[2], y[3])));
        } else
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (row + e < a.n) {
                    if (a.out_f32) ((float*)a.out)[to + e] = y[e];
                    else ((__nv_bfloat16*)a.out)[to + e] = __float2bfloat16_rn(y[e]);
                }
    };
    auto join = [&](auto parts, auto at_once) {              // of so many blocks, so many tokens on their way
        constexpr int S = decltype(parts)::value, N = decltype(at_once)::value, EVERY = S * (THREADS / 32);
        const float* from[S];
#pragma unroll
        for (int z = 0; z < S; ++z) from[z] = S == 1 ? sums : cluster.map_shared_rank(sums, z);
        for (int t0 = rank + warp * S; t0 < all; t0 += N * EVERY) {
            float4 part[N][S];
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int z = 0; z < S; ++z) part[i][z] = *reinterpret_cast<const float4*>(from[z] + min(t0 + i * EVERY, a.tokens - 1) * ROWS + 4 * lane);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                float4 v = part[i][0];
#pragma unroll
                for (int z = 1; z < S; ++z) v.x += part[i][z].x, v.y += part[i][z].y, v.z += part[i][z].z, v.w += part[i][z].w;
                if (t0 + i * EVERY < all) put(t0 + i * EVERY, v);
            }
        }
    };
    using std::integral_constant;
    if (a.splits == 1) join(integral_constant<int, 1>(), integral_constant<int, 4>());
    else if (a.splits == 2) join(integral_constant<int, 2>(), integral_constant<int, 4>());
    else if (a.splits == 4) join(integral_constant<int, 4>(), integral_constant<int, 2>());
    else join(integral_constant<int, MOST_SPLITS>(), integral_constant<int, 1>());
    if (a.splits > 1) cluster.sync();                    // nobody leaves while its memory is read
}

}  // namespace many
}  // namespace four
}  // namespace lily

using namespace lily;

// The host's word in which the kernel says that a wait ran out; made with the first launch.
static std::atomic<int*> g_lost_word{nullptr};
static int* lost_word() {
    static int* word = [] {
        int* p = new_host_word();
        g_lost_word = p;
        return p;
    }();
    return word;
}

// 0, or (code << 24 | block) of a bounded wait that gave up since the last call; clears it.  `wait`: behind all work of the device; else as far as the host knows (the kernels it has waited for).
LILY_API int lily_linear4_status(int wait) {
    if (wait && cudaDeviceSynchronize() != cudaSuccess) return -1;
    volatile int* word = g_lost_word;
    const int v = word ? *word : 0;
    if (v != 0) *word = 0;
    return v;
}

// polls: how often a wait of the kernel asks before it gives up.
LILY_API int lily_linear4_many_within(const void* x, const void* codes, const void* scales, const void* zeros, const void* bias, int bias_f32, void* out, int out_f32, int m, int n, int k,
                                      int group, int polls, cudaStream_t stream) {
    using namespace four::many;
    if (m == 0 || n == 0) return 0;
    LILY_REQUIRE(n > 0 && k > 0 && (group == 32 || group == 64 || group == 128) && k % group == 0 && n <= INT32_MAX - 256 && k <= INT32_MAX - 256, "linear4: a matrix [%d, %d] in groups of %d", n, k,
                 group);
    LILY_REQUIRE(polls >= 0, "linear4: %d polls", polls);
    LILY_REQUIRE(m > 0 && ((uintptr_t)x | (uintptr_t)codes | (uintptr_t)scales | (uintptr_t)zeros) % 16 == 0, "linear4: tensors on boundaries of sixteen bytes");
    const int token_tiles = (m + MOST_TOKENS - 1) / MOST_TOKENS, row_tiles = (n + ROWS - 1) / ROWS;
    Args a{(const uint8_t*)scales, (const uint8_t*)zeros, bias, bias_f32, out, out_f32, m, n, k, (k + STEP - 1) / STEP};
    a.tokens = ((m + token_tiles - 1) / token_tiles + 15) / 16 * 16;
    a.polls = polls;
    a.lost = lost_word();
    LILY_REQUIRE(a.lost != nullptr, "linear4: no word of the host's memory");
    // columns shared out while there is room for more blocks (two a SM up to 128 tokens), no fewer than two steps a block
    a.splits = 1;
    // (a block a SM: eight parts of the device do not all have room for two clusters of eight, and a second round of them doubles the time: 256 tokens, 2,048 x 2,048 in 11.2 us by four, 21.4 by eight)
    auto places = [&](int splits) { return a.tokens <= 128 ? 2 * sm_count() : splits < 8 ? sm_count() : sm_count() * 3 / 4; };
    while (a.splits < MOST_SPLITS && 2ll * a.splits * row_tiles * token_tiles <= places(2 * a.splits) && a.tiles >= 4 * a.splits) a.splits *= 2;
    // tensor memory: half of it, so that two blocks share an SM, where that holds two operands at least beside the accumulator
    const int accumulator = (a.tokens + 31) / 32 * 32;
    a.columns = accumulator + 2 * OPERAND <= 256 ? 256 : 512;
    a.operands = min(OPERANDS, (a.columns - accumulator) / OPERAND);
    const int stage = stage_bytes(a.tokens), room = (a.columns == 256 ? 112 : 224) * 1024;
    a.stages = min(min(6, room / stage), max(2, (a.tiles + a.splits - 1) / a.splits));
    const int bytes = max(a.stages * stage, a.tokens * ROWS * 4) + 1024;
    LILY_REQUIRE(a.stages >= 2 && (long long)row_tiles * a.tiles <= INT32_MAX / ROWS && token_tiles <= 65535, "linear4: %d tokens, a matrix [%d, %d]", m, n, k);
    tc5::EncodeTiled encode = tc5::encoder();
    LILY_REQUIRE(encode != nullptr, "linear4: no encoder of tensor maps");
    CUtensorMap map;
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)m}, strides[1] = {(cuuint64_t)k * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)a.tokens}, steps[2] = {1, 1};
    const CUresult rc = encode(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(x), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    CUtensorMap map_w;
    const cuuint64_t w_dims[2] = {64, (cuuint64_t)row_tiles * a.tiles * ROWS}, w_strides[1] = {64};
    const cuuint32_t w_box[2] = {64, ROWS};
    const CUresult w_rc = encode(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), w_dims, w_strides, w_box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    LILY_REQUIRE(rc == CUDA_SUCCESS && w_rc == CUDA_SUCCESS, "linear4: tensor map: errors %d, %d", (int)rc, (int)w_rc);
    auto kernel = group == 128 ? product_many_kernel<1> : group == 64 ? product_many_kernel<2> : product_many_kernel<4>;
    // (to one number, whatever the call needs: another thread's launch may lie between)
    LILY_REQUIRE(bytes <= MOST_BYTES && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_BYTES) == cudaSuccess, "linear4: cannot get %d bytes of shared memory", bytes);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(row_tiles * a.splits, token_tiles);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, map, map_w, a);
    LILY_CHECK_LAUNCH("linear4");
    return 0;
}

LILY_API int lily_linear4_many(const void* x, const void* codes, const void* scales, const void* zeros, const void* bias, int bias_f32, void* out, int out_f32, int m, int n, int k, int group,
                               cudaStream_t stream) {
    return lily_linear4_many_within(x, codes, scales, zeros, bias, bias_f32, out, out_f32, m, n, k, group, four::many::POLLS, stream);
}
