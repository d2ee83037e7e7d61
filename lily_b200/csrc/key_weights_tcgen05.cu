// The column sums of the softmax (key_weights.cu says what they are) on the fifth-generation tensor cores: bfloat16, head sizes 64 and
// 128, pages of 8 places and more, up to 128 query heads a kv head.
//
// The query heads of a kv head stand below one another: row t * G + h of a tile is head h of the tile's token t, so one tile of keys serves them all
// and a tile's 128 rows are filled for any number of heads (G * floor(128 / G) of them; TMA brings them as one box).  Two kernels
// of the same build, and a small one between them:
//   rows      S = Q K^T, 128 rows x 256 keys a step, a row a lane of tensor memory: running maximum and sum of each row;
//   (join)    a row's parts become its lse; rows that are none get +inf, which makes their weights zero in what follows;
//   columns   S^T = K Q^T, 128 keys x 256 rows a step, a key a lane: each thread adds up exp2(c s - lse[column]) of its own key, with the lse of the
//             256 columns in shared memory, so no sum crosses lanes.
// Scores are formed twice, since kept they would be 4 bytes for each (row, key) where forming them again is 2 d flops.
// What bounds both is the exponential: 128 x 256 of them take the SM's 16 a cycle 2,048 cycles, the products 1,440.
//
// One block a SM, ten warps: a loader (TMA into two stages of 64 KB), one that issues tcgen05.mma into two accumulators of 256
// columns (all of tensor memory), and two groups of four that read them in turn.  The steps of all (request, kv head, tile) are numbered
// through and every block takes the same number of neighbouring ones, whatever the causal mask leaves of each tile; a tile that
// several blocks share leaves a part in scratch for each, joined in their order (rows: by the join kernel; columns: by the block that
// comes last), so the results do not depend on who is first.
//
// Every wait is bounded: one that runs out sets a status word (lily_key_weights_status), the roles leave their loops and the block frees its
// tensor memory; the weights are then NaN.
#include "common.cuh"
#include "tcgen05.cuh"

namespace lily {
namespace keyw5 {

using namespace tc5;

constexpr int MAX_R = 40;                 // requests a launch
constexpr int AR = 128, BR = 256;         // rows of the standing and of the streamed operand
constexpr int STAGES = 2;
constexpr int THREADS = 320;              // loader, mma, two groups of four warps
constexpr uint32_t SPIN_LIMIT = 1u << 24;
constexpr float LOG2E = 1.4426950408889634f;

__device__ int g_status = 0;              // 0 ok; else (code << 24 | block) of the first wait that gave up

// One request of a launch.
struct Portion {
    int first;                            // row of q of its first heard token
    int heard, place0, prefix, total;     // heard tokens, the place of the first, cached places before and after the portion
    int unit0, step1, per1;               // its first row tile; its first step of the row kernel, steps of one kv head
    int tile0, step2, per2;               // the same of the column kernel (tiles of 128 places)
};

struct Params {
    const int* block_table;
    float* weights;                       // [pages, nkv, page_size]
    float2* parts;                        // rows: [unit + block][group][128] (max, sum)
    float* lse;                           // [units][128]
    int2* info;                           // [units] first block, blocks
    int* done;                            // [tiles] parts that have arrived
    float* sums;                          // columns: [tile + block][group][128]
    int bt_stride, requests, nkv, group, tq, page_size, pages, units, tiles;
    int steps1, quota1, steps2, quota2;   // steps in all and of a block
    float c;                              // scale * log2 e
    Portion p[MAX_R];
};

// Row tiles of a request and kv head (an even number, so that a step of the column kernel has two).
__host__ __device__ inline int row_tiles(const Portion& p, int tq) { return (p.heard + 2 * tq - 1) / (2 * tq) * 2; }
__host__ __device__ inline int key_tiles(const Portion& p) { return (p.total + AR - 1) / AR; }
// Steps of a tile.  Rows: pieces of 256 keys up to the last that its last token sees.  Columns: pieces of two row tiles from the first that sees it.
__host__ __device__ inline int steps1_of(const Portion& p, int tq, int i) {
    if (i * tq >= p.heard) return 0;
    const int end = (i + 1) * tq < p.heard ? (i + 1) * tq : p.heard;
    return (p.place0 + end + BR - 1) / BR;
}
__host__ __device__ inline int first2_of(const Portion& p, int tq, int i) { return i * AR > p.place0 ? (i * AR - p.place0) / (2 * tq) : 0; }
__host__ __device__ inline int steps2_of(const Portion& p, int tq, int i) { return row_tiles(p, tq) / 2 - first2_of(p, tq, i); }

constexpr int a_bytes(int d) { return AR * d * 2; }
constexpr int b_bytes(int d) { return BR * d * 2; }
// shared memory: two standing tiles | stages | lse of the columns (twice 256) | token of each row of a tile | barriers
constexpr int off_b(int d) { return 2 * a_bytes(d); }
constexpr int off_lse(int d) { return off_b(d) + STAGES * b_bytes(d); }
constexpr int off_tok(int d) { return off_lse(d) + 2 * BR * 4; }
constexpr int off_bars(int d) { return off_tok(d) + AR * 4; }
constexpr int NUM_BARS = 4 + 2 * STAGES + 6;
constexpr int off_misc(int d) { return off_bars(d) + 8 * NUM_BARS; }
constexpr int smem_bytes(int d) { return off_misc(d) + 64; }

__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
    for (uint32_t i = 0; i < SPIN_LIMIT; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 1023u) == 1023u && *abort_flag) return false;
    }
    *abort_flag = 1;
    atomicCAS(&g_status, 0, (code << 24) | (int)(blockIdx.x & 0xFFFFFF));
    return false;
}
// The same for a whole warp, whose lanes then agree.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, code));
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void group_sync(int group) { asm volatile("bar.sync %0, 128;\n" ::"r"(group + 1) : "memory"); }

// Where a role stands: tile `i` of (request r, kv head), step `s` of its `n`.
struct Cursor { int r, kvh, i, s, n, unit; };

template <int PASS>
__device__ __forceinline__ int steps_of(const Params& p, int r, int i) { return PASS == 1 ? steps1_of(p.p[r], p.tq, i) : steps2_of(p.p[r], p.tq, i); }
template <int PASS>
__device__ __forceinline__ int tiles_of(const Params& p, int r) { return PASS == 1 ? row_tiles(p.p[r], p.tq) : key_tiles(p.p[r]); }

// On to the next tile that has steps.
template <int PASS>
__device__ __forceinline__ void next_tile(const Params& p, Cursor& c) {
    c.s = 0;
    do {
        ++c.i, ++c.unit;
        if (c.i == tiles_of<PASS>(p, c.r)) {
            c.i = 0;
            if (++c.kvh == p.nkv) {
                c.kvh = 0;
                do ++c.r; while (c.r < p.requests && tiles_of<PASS>(p, c.r) == 0);
            }
        }
        c.n = c.r < p.requests ? steps_of<PASS>(p, c.r, c.i) : 1;
    } while (c.n == 0);
}

// The tile and step of step `g`; all lanes of a warp work it out together.
template <int PASS>
__device__ Cursor find(const Params& p, int g) {
    Cursor c;
    c.r = 0;
    while (c.r + 1 < p.requests && (PASS == 1 ? p.p[c.r + 1].step1 : p.p[c.r + 1].step2) <= g) ++c.r;
    const Portion& q = p.p[c.r];
    int off = g - (PASS == 1 ? q.step1 : q.step2);
    const int per = PASS == 1 ? q.per1 : q.per2, tiles = tiles_of<PASS>(p, c.r), lane = threadIdx.x & 31;
    c.kvh = off / per;
    off -= c.kvh * per;
    c.i = 0;
    for (int i0 = 0; i0 < tiles; i0 += 32) {
        const int i = i0 + lane, n = i < tiles ? steps_of<PASS>(p, c.r, i) : 0;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += u;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, sum > off);
        if (past) {
            const int at = __ffs(past) - 1;
            c.i = i0 + at;
            off -= __shfl_sync(0xffffffffu, sum - n, at);
            break;
        }
        off -= __shfl_sync(0xffffffffu, sum, 31);
    }
    c.s = off;
    c.n = steps_of<PASS>(p, c.r, c.i);
    c.unit = (PASS == 1 ? q.unit0 : q.tile0) + c.kvh * tiles + c.i;
    return c;
}

template <int D, int PASS>
__global__ void __launch_bounds__(THREADS, 1) key_weights_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv,
                                                                    const __grid_constant__ Params p) {
    constexpr int DH = D / 64;
    extern __shared__ __align__(1024) unsigned char smem[];
    float* lse_s = reinterpret_cast<float*>(smem + off_lse(D));       // [2][256]
    int* tok_s = reinterpret_cast<int*>(smem + off_tok(D));           // [128] token of a tile's row
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + off_bars(D));
    uint32_t& tmem_base_s = *reinterpret_cast<uint32_t*>(smem + off_misc(D));
    int& abort_s = *reinterpret_cast<int*>(smem + off_misc(D) + 4);
    int* last_s = reinterpret_cast<int*>(smem + off_misc(D) + 8);     // [2]
    Cursor& start_s = *reinterpret_cast<Cursor*>(smem + off_misc(D) + 16);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem);
    const uint32_t a_smem = base, b_smem = base + off_b(D);
    const uint32_t a_full = smem_u32(bars), a_empty = a_full + 16, b_full = a_empty + 16, b_empty = b_full + 8 * STAGES, s_full = b_empty + 8 * STAGES,
                   s_empty = s_full + 16, l_full = s_empty + 16;
    if (base & 1023u) {                                               // the swizzled tiles need it; never seen, but checked
        if (threadIdx.x == 0) atomicCAS(&g_status, 0, (11 << 24) | (int)(blockIdx.x & 0xFFFFFF));
        return;
    }
    if (threadIdx.x == 0) {
        abort_s = 0;
        for (int s = 0; s < 2; ++s) {
            mbar_init(a_full + 8 * s, 1);
            mbar_init(a_empty + 8 * s, 1);
            mbar_init(s_full + 8 * s, 1);
            mbar_init(s_empty + 8 * s, 128);
            mbar_init(l_full + 8 * s, 1);
        }
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(b_full + 8 * s, 1);
            mbar_init(b_empty + 8 * s, 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (threadIdx.x < AR) tok_s[threadIdx.x] = (int)threadIdx.x < p.group * p.tq ? (int)threadIdx.x / p.group : 1 << 29;
    {
        // rows of a query tile that no box fills are zeros for good
        const int filled = p.group * p.tq, tile_rows = PASS == 1 ? AR : BR;
        unsigned char* q_tiles = smem + (PASS == 1 ? 0 : off_b(D));
        constexpr int tile_size = PASS == 1 ? a_bytes(D) : b_bytes(D);
        const int spare = AR - filled, rows = spare * 2 * DH * (PASS == 1 ? 1 : 2);        // two tiles, halves of 64 columns, two row tiles a stage
        for (int i = threadIdx.x; i < rows * 8; i += THREADS) {
            int x = i >> 3;
            const int row = filled + x % spare;
            x /= spare;
            const int half = x % DH, rest = x / DH, which = rest & 1, second = rest >> 1;
            *reinterpret_cast<uint4*>(q_tiles + which * tile_size + half * tile_rows * 128 + (second * AR + row) * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
    }
    const int steps = PASS == 1 ? p.steps1 : p.steps2, quota = PASS == 1 ? p.quota1 : p.quota2;
    const int g0 = blockIdx.x * quota, mine = min(quota, steps - g0);
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&tmem_base_s)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    if (warp == 0) {
        const Cursor c = find<PASS>(p, g0);
        if (lane == 0) start_s = c;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base_s;
    volatile int* abort_flag = &abort_s;
    Cursor cur = start_s;
    pdl_wait();
    pdl_launch_dependents();

    if (warp == 0) {
        // ---- loader ----
        const int box = min(p.page_size, 64);                        // places a box of the cache
        // the pages of `rows` places from `key` on, a box a lane and step; all lanes stay together
        auto load_keys = [&](uint32_t dst, int rows, int pitch, int r, int kvh, int key, uint32_t bar) {
            const int* table = p.block_table + (size_t)r * p.bt_stride;
            const int boxes = rows / box;
            for (int b0 = 0; b0 < boxes; b0 += 32) {
                const int mine_key = key + (b0 + lane) * box;
                const bool held = b0 + lane < boxes && mine_key < p.p[r].total;
                const int page = held ? table[mine_key / p.page_size] : 0, at = held ? mine_key % p.page_size : 0;
                for (int b = 0; b < min(32, boxes - b0); ++b) {
                    const int pg = __shfl_sync(0xffffffffu, page, b), off = __shfl_sync(0xffffffffu, at, b);
                    if (lane == 0)
#pragma unroll
                        for (int h = 0; h < DH; ++h) tma_load_4d(dst + h * pitch + (b0 + b) * box * 128, &map_kv, bar, h * 64, off, kvh, pg);
                }
            }
        };
        auto load_rows = [&](uint32_t dst, int pitch, int r, int kvh, int tile, uint32_t bar) {
            if (lane == 0)
#pragma unroll
                for (int h = 0; h < DH; ++h) tma_load_3d(dst + h * pitch, &map_q, bar, h * 64, kvh * p.group, p.p[r].first + tile * p.tq);
        };
        const int q_bytes = p.group * p.tq * D * 2;
        bool ok = true;
        int tile = 0, sent_a = 0, sent_b = 0, sent_l = 0;
        for (int k = 0; k < mine && ok; ++k) {
            if (k == 0 || cur.s == 0) {                               // a new standing tile
                ok = warp_wait(a_empty + 8 * (tile & 1), ((tile >> 1) & 1) ^ 1, abort_flag, 1);
                if (!ok) break;
                const uint32_t bar = a_full + 8 * (tile & 1), dst = a_smem + (tile & 1) * a_bytes(D);
                if (lane == 0) mbar_expect_tx(bar, PASS == 1 ? q_bytes : a_bytes(D));
                __syncwarp();
                if (PASS == 1) load_rows(dst, AR * 128, cur.r, cur.kvh, cur.i, bar);
                else load_keys(dst, AR, AR * 128, cur.r, cur.kvh, cur.i * AR, bar);
                ++tile;
                ++sent_a;
            }
            const int st = k % STAGES;
            ok = warp_wait(b_empty + 8 * st, ((k / STAGES) & 1) ^ 1, abort_flag, 2);
            if (!ok) break;
            const uint32_t bar = b_full + 8 * st, dst = b_smem + st * b_bytes(D);
            if (lane == 0) mbar_expect_tx(bar, PASS == 1 ? b_bytes(D) : 2 * q_bytes);
            __syncwarp();
            if (PASS == 1) {
                load_keys(dst, BR, BR * 128, cur.r, cur.kvh, cur.s * BR, bar);
                ++sent_b;
            } else {
                const int t0 = 2 * (first2_of(p.p[cur.r], p.tq, cur.i) + cur.s);
                load_rows(dst, BR * 128, cur.r, cur.kvh, t0, bar);
                load_rows(dst + AR * 128, BR * 128, cur.r, cur.kvh, t0 + 1, bar);
                ++sent_b;
                ok = warp_wait(s_empty + 8 * (k & 1), ((k >> 1) & 1) ^ 1, abort_flag, 3);        // the lse of step k - 2 have been read
                if (!ok) break;
                if (lane == 0) {
                    mbar_expect_tx(l_full + 8 * (k & 1), BR * 4);
                    const int unit = p.p[cur.r].unit0 + cur.kvh * row_tiles(p.p[cur.r], p.tq) + t0;
                    bulk_load(smem_u32(lse_s + (k & 1) * BR), p.lse + (size_t)unit * AR, BR * 4, l_full + 8 * (k & 1));
                }
                ++sent_l;
            }
            if (++cur.s == cur.n) next_tile<PASS>(p, cur);
        }
        if (*abort_flag && lane == 0) {
            // copies already issued still land in this block's shared memory: give each a bounded wait
            for (int j = max(0, sent_a - 2); j < sent_a; ++j)
                for (uint32_t i = 0; i < (1u << 20) && !mbar_try_wait(a_full + 8 * (j & 1), (j >> 1) & 1); ++i) {}
            for (int j = max(0, sent_b - STAGES); j < sent_b; ++j)
                for (uint32_t i = 0; i < (1u << 20) && !mbar_try_wait(b_full + 8 * (j % STAGES), (j / STAGES) & 1); ++i) {}
            for (int j = max(0, sent_l - 2); j < sent_l; ++j)
                for (uint32_t i = 0; i < (1u << 20) && !mbar_try_wait(l_full + 8 * (j & 1), (j >> 1) & 1); ++i) {}
        }
    } else if (warp == 1) {
        // ---- products: accumulator k & 1 = standing tile x streamed tile of step k ----
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BR >> 3) << 17) | ((uint32_t)(AR >> 4) << 24);
        bool ok = true;
        int tile = -1;
        for (int k = 0; k < mine && ok; ++k) {
            const int st = k % STAGES;
            if (k == 0 || cur.s == 0) {
                ++tile;
                ok = warp_wait(a_full + 8 * (tile & 1), (tile >> 1) & 1, abort_flag, 4);
                if (!ok) break;
            }
            ok = warp_wait(b_full + 8 * st, (k / STAGES) & 1, abort_flag, 5) && warp_wait(s_empty + 8 * (k & 1), ((k >> 1) & 1) ^ 1, abort_flag, 6);
            if (!ok) break;
            tc_fence_after();
            const bool last = cur.s + 1 == cur.n || k + 1 == mine;
            if (elect_one()) {
                const uint64_t da = desc_k_major(a_smem + (tile & 1) * a_bytes(D)), db = desc_k_major(b_smem + st * b_bytes(D));
#pragma unroll
                for (int kk = 0; kk < D / 16; ++kk)
                    umma(tmem + (uint32_t)(k & 1) * BR, da + (uint64_t)(((kk >> 2) * AR * 128 + (kk & 3) * 32) >> 4),
                         db + (uint64_t)(((kk >> 2) * BR * 128 + (kk & 3) * 32) >> 4), idesc, kk != 0 ? 1u : 0u);
                umma_commit(b_empty + 8 * st);
                umma_commit(s_full + 8 * (k & 1));
                if (last) umma_commit(a_empty + 8 * (tile & 1));
            }
            __syncwarp();
            if (++cur.s == cur.n) next_tile<PASS>(p, cur);
        }
    } else {
        // ---- two groups of 128 threads, a lane of tensor memory each: group k & 1 takes step k ----
        // (where a wait runs out they go on without it to the ends of the tiles, where they meet, and what they leave is NaN)
        const int which = (warp - 2) >> 2, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t my = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)which * BR;
        const int tok = tok_s[row];
        const float c = p.c;
        float m = -INFINITY, l = 0.f;                                 // rows: running maximum (log2 units) and sum; columns: l is the sum
        bool ok = true;
        int unit_first = g0;                                          // the step at which this block's share of the tile begins
        for (int k = 0; k < mine; ++k) {
            const Portion& q = p.p[cur.r];
            if ((k & 1) == which && ok) {
                ok = warp_wait(s_full + 8 * which, (k >> 1) & 1, abort_flag, 7);
                if (PASS == 2 && ok) ok = warp_wait(l_full + 8 * which, (k >> 1) & 1, abort_flag, 8);
            }
            if (!ok) l = __int_as_float(0x7fffffff);
            if ((k & 1) == which && ok) {
                tc_fence_after();
                if (PASS == 1) {
                    const int key0 = cur.s * BR, first = q.place0 + cur.i * p.tq, own = q.place0 + cur.i * p.tq + tok;      // the last place this row sees
                    const bool masked = key0 + BR - 1 > first;
#pragma unroll 1
                    for (int c0 = 0; c0 < BR; c0 += 64) {
                        float s[64];
                        tmem_ld32(my + (uint32_t)c0, s);
                        tmem_ld32(my + (uint32_t)c0 + 32, s + 32);
                        tmem_wait_ld();
                        if (masked) {
#pragma unroll
                            for (int e = 0; e < 64; ++e) s[e] = key0 + c0 + e <= own ? s[e] : -INFINITY;
                        }
                        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                        for (int e = 4; e < 64; ++e) mx[e & 3] = fmaxf(mx[e & 3], s[e]);
                        const float now = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c), off = now == -INFINITY ? 0.f : now;
                        float sum[4] = {l * ex2(m - off), 0.f, 0.f, 0.f};
                        m = now;
#pragma unroll
                        for (int e = 0; e < 64; ++e) sum[e & 3] += ex2(fmaf(s[e], c, -off));
                        l = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    }
                } else {
                    const int step = first2_of(q, p.tq, cur.i) + cur.s, t0 = step * 2 * p.tq, key = cur.i * AR + row;
                    const bool masked = cur.i * AR + AR - 1 > q.place0 + t0 || t0 + 2 * p.tq > q.heard;
                    const float4* lse4 = reinterpret_cast<const float4*>(lse_s + which * BR);
                    float sum[4] = {l, 0.f, 0.f, 0.f};
#pragma unroll 1
                    for (int c0 = 0; c0 < BR; c0 += 64) {
                        float s[64];
                        tmem_ld32(my + (uint32_t)c0, s);
                        tmem_ld32(my + (uint32_t)c0 + 32, s + 32);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 64; e += 4) {
                            const float4 z = lse4[(c0 + e) >> 2];
                            s[e] = ex2(fmaf(s[e], c, -z.x));
                            s[e + 1] = ex2(fmaf(s[e + 1], c, -z.y));
                            s[e + 2] = ex2(fmaf(s[e + 2], c, -z.z));
                            s[e + 3] = ex2(fmaf(s[e + 3], c, -z.w));
                        }
                        if (masked) {
                            const int t = t0 + (c0 >= AR ? p.tq : 0);
#pragma unroll
                            for (int e = 0; e < 64; ++e) {
                                const int tc = t + tok_s[(c0 & (AR - 1)) + e];
                                s[e] = tc < q.heard && key <= q.place0 + tc ? s[e] : 0.f;
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 64; ++e) sum[e & 3] += s[e];
                    }
                    l = (sum[0] + sum[1]) + (sum[2] + sum[3]);
                }
                tc_fence_before();
                mbar_arrive(s_empty + 8 * which);
            }
            if (cur.s + 1 == cur.n || k + 1 == mine) {
                // the end of this block's share of the tile
                const int at = g0 + k - cur.s, blocks_first = at / quota, blocks = (at + cur.n - 1) / quota - blocks_first + 1;
                const size_t slot = ((size_t)(cur.unit + (int)blockIdx.x) * 2 + which) * AR + row;
                if (PASS == 1) {
                    p.parts[slot] = make_float2(m, l);
                    if (unit_first == at && which == 0 && row == 0) p.info[cur.unit] = make_int2(blocks_first, blocks);
                } else {
                    __stcg(p.sums + slot, l);
                    __threadfence();
                    group_sync(which);
                    if (row == 0) last_s[which] = atomicAdd(p.done + cur.unit, 1) == 2 * blocks - 1;
                    group_sync(which);
                    if (last_s[which]) {
                        __threadfence();
                        float w = 0.f;
                        for (int b = 0; b < 2 * blocks; ++b) w += __ldcg(p.sums + ((size_t)(cur.unit + blocks_first) * 2 + b) * AR + row);
                        const int place = cur.i * AR + row;
                        if (place < q.total) {
                            float* to = p.weights + ((size_t)p.block_table[(size_t)cur.r * p.bt_stride + place / p.page_size] * p.nkv + cur.kvh) * p.page_size +
                                        place % p.page_size;
                            *to = (place < q.prefix ? *to : 0.f) + w;
                        }
                    }
                    group_sync(which);                                // (the word is read before the next tile's)
                }
                m = -INFINITY;
                l = 0.f;
                unit_first = g0 + k + 1;
            }
            if (++cur.s == cur.n) next_tile<PASS>(p, cur);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
    }
}

// A row tile a block: its parts in the order of the blocks that made them, lse = max + log2(sum); +inf for rows that are none.  Also
// clears the column kernel's counters.
__global__ void __launch_bounds__(AR) key_weights_join_kernel(const __grid_constant__ Params p) {
    pdl_enter_small();
    const int unit = blockIdx.x, row = threadIdx.x;
    for (int i = unit * AR + row; i < p.tiles; i += gridDim.x * AR) p.done[i] = 0;
    int r = 0;
    while (r + 1 < p.requests && p.p[r + 1].unit0 <= unit) ++r;
    const Portion& q = p.p[r];
    const int i = (unit - q.unit0) % row_tiles(q, p.tq);
    float lse = INFINITY;
    if (row < p.group * p.tq && i * p.tq + row / p.group < q.heard) {
        const int2 in = p.info[unit];
        const float2* part = p.parts + (size_t)(unit + in.x) * 2 * AR + row;
        float m = -INFINITY, l = 0.f;
        for (int b = 0; b < 2 * in.y; ++b) m = fmaxf(m, part[b * AR].x);
        for (int b = 0; b < 2 * in.y; ++b) {
            const float2 v = part[b * AR];
            if (v.x > -INFINITY || v.y != 0.f) l = fmaf(v.y, exp2f(v.x - m), l);      // (a NaN is no maximum, but makes the sum one)
        }
        lse = m + log2f(l);
    }
    p.lse[(size_t)unit * AR + row] = lse;
}

template <int D>
static int launch(const Params& p, const CUtensorMap& map_q, const CUtensorMap& map_kv, cudaStream_t stream) {
    static bool configured = false;
    if (!configured) {
        cudaError_t e = cudaFuncSetAttribute(key_weights_tc_kernel<D, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(D));
        if (e == cudaSuccess) e = cudaFuncSetAttribute(key_weights_tc_kernel<D, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(D));
        if (e != cudaSuccess) {
            set_error("attention_key_weights: cannot get %d bytes of shared memory: %s", smem_bytes(D), cudaGetErrorString(e));
            return 2;
        }
        configured = true;
    }
    launch_pdl(key_weights_tc_kernel<D, 1>, dim3((p.steps1 + p.quota1 - 1) / p.quota1), dim3(THREADS), (size_t)smem_bytes(D), stream, map_q, map_kv, p);
    launch_pdl(key_weights_join_kernel, dim3(p.units), dim3(AR), 0, stream, p);
    launch_pdl(key_weights_tc_kernel<D, 2>, dim3((p.steps2 + p.quota2 - 1) / p.quota2), dim3(THREADS), (size_t)smem_bytes(D), stream, map_q, map_kv, p);
    return 0;
}

// Fills in what follows from the portions' lengths; the floats of scratch they take.
static size_t plan(Params& p, int requests, const int* prefix, const int* fresh, int observe, int group, int nkv) {
    p.requests = requests;
    p.nkv = nkv;
    p.group = group;
    p.tq = AR / group;
    int first = 0, unit = 0, tile = 0;
    long long s1 = 0, s2 = 0;
    for (int r = 0; r < requests; ++r) {
        Portion& q = p.p[r];
        q.heard = observe > 0 && observe < fresh[r] ? observe : fresh[r];
        q.first = first + fresh[r] - q.heard;
        q.prefix = prefix[r];
        q.total = q.heard > 0 ? prefix[r] + fresh[r] : 0;
        q.place0 = q.total - q.heard;
        q.unit0 = unit;
        q.tile0 = tile;
        q.step1 = (int)s1;
        q.step2 = (int)s2;
        q.per1 = q.per2 = 0;
        const int rows = row_tiles(q, p.tq), keys = key_tiles(q);
        for (int i = 0; i < rows; ++i) q.per1 += steps1_of(q, p.tq, i);
        for (int i = 0; i < keys; ++i) q.per2 += steps2_of(q, p.tq, i);
        s1 += (long long)q.per1 * nkv;
        s2 += (long long)q.per2 * nkv;
        unit += rows * nkv;
        tile += keys * nkv;
        first += fresh[r];
    }
    if (s1 > 0x3fffffff || s2 > 0x3fffffff) return 0;
    const int sms = sm_count();
    p.units = unit;
    p.tiles = tile;
    p.steps1 = (int)s1;
    p.steps2 = (int)s2;
    p.quota1 = s1 > 0 ? (int)((s1 + sms - 1) / sms) : 1;
    p.quota2 = s2 > 0 ? (int)((s2 + sms - 1) / sms) : 1;
    const int b1 = (p.steps1 + p.quota1 - 1) / p.quota1, b2 = (p.steps2 + p.quota2 - 1) / p.quota2;
    // parts | lse | info | counters | sums, each on 16 bytes
    return (size_t)(unit + b1) * 4 * AR + (size_t)unit * AR + (size_t)unit * 2 + ((size_t)tile + 3) / 4 * 4 + (size_t)(tile + b2) * 2 * AR + 16;
}

}  // namespace keyw5
}  // namespace lily

using namespace lily;

// Whether these kernels take the sizes (bfloat16).
LILY_API int lily_key_weights_tc_takes(int nq, int nkv, int d, int page_size, float scale) {
    return (d == 64 || d == 128) && page_size >= 8 && (page_size & (page_size - 1)) == 0 && nkv > 0 && nq % nkv == 0 && nq / nkv >= 1 && nq / nkv <= 128 && scale > 0.f &&
           scale < INFINITY;
}

// Floats of scratch for portions of `fresh` tokens behind `prefix` places (host arrays); 0: nothing to do or too much to number.
LILY_API size_t lily_key_weights_tc_floats(int requests, const int* prefix, const int* fresh, int observe, int nq, int nkv) {
    static thread_local keyw5::Params p;
    size_t most = 0;
    for (int r = 0; r < requests; r += keyw5::MAX_R) {
        const size_t n = keyw5::plan(p, requests - r < keyw5::MAX_R ? requests - r : keyw5::MAX_R, prefix + r, fresh + r, observe, nq / nkv, nkv);
        most = n > most ? n : most;
    }
    return most;
}

// 0, or (code << 24 | block) of the first bounded wait that gave up (synchronises; the word is cleared when read).
LILY_API int lily_key_weights_status() {
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, keyw5::g_status, sizeof(int)) != cudaSuccess) return -1;
    if (v != 0) cudaMemcpyToSymbol(keyw5::g_status, &zero, sizeof(int));
    return v;
}

LILY_API int lily_key_weights_tc(const void* q, int tokens, const void* kv, int pages, float* weights, const int* block_table, int bt_stride, float* scratch,
                                 int requests, const int* prefix, const int* fresh, int observe, int nq, int nkv, int d, int page_size, float scale,
                                 cudaStream_t stream) {
    LILY_REQUIRE(lily_key_weights_tc_takes(nq, nkv, d, page_size, scale), "attention_key_weights: the tcgen05 kernels do not take %d heads over %d of %d, pages of %d", nq, nkv, d, page_size);
    LILY_REQUIRE((((uintptr_t)q | (uintptr_t)kv | (uintptr_t)scratch) & 15) == 0, "attention_key_weights: operands must be 16-byte aligned");
    tc5::EncodeTiled enc = tc5::encoder();
    LILY_REQUIRE(enc != nullptr, "attention_key_weights: the driver does not offer cuTensorMapEncodeTiled");
    const int group = nq / nkv, tq = keyw5::AR / group;
    CUtensorMap map_q, map_kv;
    const cuuint32_t elem[4] = {1, 1, 1, 1};
    {
        const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)nq, (cuuint64_t)tokens}, strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)nq * d * 2};
        const cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)tq};
        const CUresult rc = enc(&map_q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        LILY_REQUIRE(rc == CUDA_SUCCESS, "attention_key_weights: cuTensorMapEncodeTiled (q) failed with %d", (int)rc);
    }
    {
        const cuuint64_t row = (cuuint64_t)d * 2, dims[4] = {(cuuint64_t)d, (cuuint64_t)page_size, (cuuint64_t)2 * nkv, (cuuint64_t)pages};
        const cuuint64_t strides[3] = {row, row * page_size, row * page_size * 2 * nkv};
        const cuuint32_t box[4] = {64, (cuuint32_t)(page_size < 64 ? page_size : 64), 1, 1};
        const CUresult rc = enc(&map_kv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(kv), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
        LILY_REQUIRE(rc == CUDA_SUCCESS, "attention_key_weights: cuTensorMapEncodeTiled (cache) failed with %d", (int)rc);
    }
    keyw5::Params p{};
    int row0 = 0;
    for (int r = 0; r < requests; r += keyw5::MAX_R) {
        const int some = requests - r < keyw5::MAX_R ? requests - r : keyw5::MAX_R;
        const size_t floats = keyw5::plan(p, some, prefix + r, fresh + r, observe, group, nkv);
        LILY_REQUIRE(floats > 0, "attention_key_weights: too many tiles for one call");
        for (int i = 0; i < some; ++i) p.p[i].first += row0;
        if (p.steps1 > 0) {
            p.block_table = block_table + (size_t)r * bt_stride;
            p.weights = weights;
            p.bt_stride = bt_stride;
            p.page_size = page_size;
            p.pages = pages;
            p.c = scale * keyw5::LOG2E;
            const int b1 = (p.steps1 + p.quota1 - 1) / p.quota1;
            float* at = scratch;
            p.parts = reinterpret_cast<float2*>(at);
            at += (size_t)(p.units + b1) * 4 * keyw5::AR;
            p.lse = at;
            at += (size_t)p.units * keyw5::AR;
            p.info = reinterpret_cast<int2*>(at);
            at += (size_t)p.units * 2;
            p.done = reinterpret_cast<int*>(at);
            at += ((size_t)p.tiles + 3) / 4 * 4;
            p.sums = at;
            const int rc = d == 64 ? keyw5::launch<64>(p, map_q, map_kv, stream) : keyw5::launch<128>(p, map_q, map_kv, stream);
            if (rc) return rc;
        }
        for (int i = 0; i < some; ++i) row0 += fresh[r + i];
    }
    LILY_CHECK_LAUNCH("attention_key_weights");
    return 0;
}
