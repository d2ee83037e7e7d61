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
// One block a SM, eighteen warps: a loader (TMA into two stages of 64 KB; it also describes each step once, in a ring that the others read, and
// brings the lse of its columns), one that issues tcgen05.mma into two accumulators of 256 columns (all of tensor memory), and four groups of four that
// read them: two pairs of groups take steps in turn, each group half of a step's columns.  The steps of all (request, kv head, tile) are numbered
// through and every block takes the same number of neighbouring ones, whatever the causal mask leaves of each tile; a tile that
// several blocks share leaves a part in scratch for each, joined in their order (rows: by the join kernel; columns: by the warps that
// come last), so the results do not depend on who is first.
//
// Measured: 2,048 tokens of 32 heads of 128 over 8, 60.4 us (some 7 of them between the kernels; all exponentials on their unit would take 34, the products
// 10); the last 64 of 1,024 tokens behind 15,360 places 36.6.  The CUDA cores of key_weights.cu take 768 for the first, and on the same pages 12.6 for 16 tokens (here 9.5),
// 17.8 for 128 (13.0); they are ahead for 300 tokens of seven heads of 64 over one (14.6, here 17.4), where a dozen tiles leave most SMs idle either way.
//
// Every wait is bounded: one that runs out says so in a word of the host's memory (lily_key_weights_status), the roles leave their loops, what the block
// has on its way is waited for (bounded too), its tensor memory is freed, and what it was to write becomes NaN: the parts of its row tiles, from which all
// that these rows give is NaN, or the weights of its key tiles.  Nothing of it is left to the next call.
#include "common.cuh"
#include "tcgen05.cuh"

#include <atomic>

namespace lily {
int* new_host_word();

namespace keyw5 {

using namespace tc5;

constexpr int MAX_R = 40;                 // requests a launch
constexpr int AR = 128, BR = 256;         // rows of the standing and of the streamed operand
constexpr int STAGES = 2;
constexpr int GROUPS = 4;                 // groups of four warps: two pairs that take steps in turn, each group half of a step's columns
constexpr int COLS = BR / 2;
constexpr int THREADS = 64 + GROUPS * 128;
constexpr float LOG2E = 1.4426950408889634f;

// One request of a launch.
struct Portion {
    int first;                            // row of q of its first heard token
    int heard, place0, prefix, total;     // heard tokens, the place of the first, cached places before and after the portion
    int unit0, step1, per1;               // its first row tile; its first step of the row kernel, steps of one kv head
    int tile0, step2, per2;               // the same of the column kernel (tiles of 128 places)
    int row_steps;                        // pieces of two row tiles
};

struct Params {
    const int* block_table;
    float* weights;                       // [pages, nkv, page_size]
    float2* parts;                        // rows: [unit + block][group][128] (max, sum)
    float* lse;                           // [units][128], negative
    int* done;                            // [tiles][4] parts that have arrived, for each 32 keys
    float* sums;                          // columns: [tile + block][group][128]
    int bt_stride, requests, nkv, group, tq, page_size, pages, units, tiles;
    int steps1, quota1, steps2, quota2;   // steps in all and of a block
    float c;                              // scale * log2 e
    float per_step;                       // 1 / (2 tq)
    int page_shift;
    int polls[2];                         // polls before a wait of the row, the column kernel gives up
    int* lost;                            // a word of the host's where it says so
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
constexpr int LSE = 4;                    // steps whose description (and lse) is held
constexpr int SUMS = 8;                   // tiles whose groups' sums are
// shared memory: two standing tiles | stages | lse of the columns | the groups' sums | descriptions | token of each row of a tile | barriers
constexpr int off_b(int d) { return 2 * a_bytes(d); }
constexpr int off_lse(int d) { return off_b(d) + STAGES * b_bytes(d); }
constexpr int off_sums(int d) { return off_lse(d) + LSE * BR * 4; }
constexpr int off_desc(int d) { return off_sums(d) + SUMS * GROUPS * AR * 4; }
constexpr int off_tok(int d) { return off_desc(d) + LSE * 32; }
constexpr int off_bars(int d) { return off_tok(d) + AR * 4; }
constexpr int NUM_BARS = 4 + 2 * STAGES + 4 + 2 * LSE + SUMS;
constexpr int off_misc(int d) { return off_bars(d) + 8 * NUM_BARS; }
constexpr int smem_bytes(int d) { return off_misc(d) + 128; }

// How the waits of a block end when what they wait for does not come.
struct Waits { volatile int* abort; int* lost; int polls; };
__device__ __forceinline__ void give_up(const Waits& w, int code) {
    *w.abort = 1;
    *(volatile int*)w.lost = (code << 24) | (int)(blockIdx.x & 0xFFFFFF);
    __threadfence_system();
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const Waits& w, int code) {
    for (int i = 0; i < w.polls; ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 1023) == 1023 && *w.abort) return false;
    }
    give_up(w, code);
    return false;
}
// The same for a whole warp, whose lanes then agree.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const Waits& w, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, w, code));
}
__device__ __forceinline__ void mbar_arrive_many(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// One step as the loader describes it to the groups.
//   at        rows: the place of the tile's first token less the step's first key; columns: the tile's first place less that of the step's first token
//   live      columns: heard tokens from the step's first on
//   flags     FIRST, LAST: the first and last step of the tile that this pair of groups takes in this block; EVEN: the pair takes the tile's first step in this
//             block; ALONE: all of the tile's steps are this block's; SINGLE: the tile has one step here; above them the number of such tiles in the block up to this one
//   unit, begin, steps, where (kv head, request), i: the tile
struct Step { int at, live, flags, unit, begin, steps, where, i; };
enum : int { FIRST = 1, LAST = 2, EVEN = 4, ALONE = 8, SINGLE = 16, TILE_SHIFT = 8 };
// Parts that block `b` leaves of a tile: a pair's two groups, or all four where it has two steps or more of it.
__device__ __forceinline__ int parts_of(int begin, int steps, int quota, int b) {
    return min(begin + steps, (b + 1) * quota) - max(begin, b * quota) == 1 ? 2 : 4;
}

// ---- pairs of floats in one register pair (fma.rn.f32x2: two IEEE operations an instruction) ----
typedef unsigned long long Two;
__device__ __forceinline__ Two two(float a, float b) {
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void apart(Two v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ Two add2(Two a, Two b) {
    Two r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
    Two r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

__device__ __forceinline__ Two exp2_of(Two x) {
    float a, b;
    apart(x, a, b);
    return two(ex2(a), ex2(b));
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// The same on the multiply-add unit, for weights (x at most a little above 0, or NaN): x = i + f with |f| <= 1/2, 2^f by the polynomial of degree five whose largest
// relative error is least (fitted by Lawson's iteration: 7.5e-8; 1.6e-7 with its coefficients rounded to float32, the constant term 1 + 2^-23 among them, and
// 2.3e-7 as computed), 2^i by its exponent; below 2^-126.5 it is 0.
__device__ __forceinline__ Two exp2_by_terms(Two x) {
    constexpr float SHIFT = 12582912.f + 127.f;                       // 1.5 * 2^23: the sum's last bits are i + 127
    float a, b;
    apart(x, a, b);
    x = two(max_nan(a, -127.f), max_nan(b, -127.f));
    const Two r = add2(x, two(SHIFT, SHIFT)), f = fma2(add2(r, two(-SHIFT, -SHIFT)), two(-1.f, -1.f), x);
    Two p = fma2(f, two(1.3276472454890609e-3f, 1.3276472454890609e-3f), two(9.675540961325169e-3f, 9.675540961325169e-3f));
    p = fma2(p, f, two(5.550713092088699e-2f, 5.550713092088699e-2f));
    p = fma2(p, f, two(0.24022120237350464f, 0.24022120237350464f));
    p = fma2(p, f, two(0.6931469440460205f, 0.6931469440460205f));
    p = fma2(p, f, two(1.0000001192092896f, 1.0000001192092896f));
    apart(r, a, b);
    return mul2(p, two(__uint_as_float(__float_as_uint(a) << 23), __uint_as_float(__float_as_uint(b) << 23)));
}
// Pair e of sixteen: three of them by terms, the others by the exponentials' unit (2,048 tokens 61.4 us, 8,192 614; none by terms 63.8 and 654, two 61.9 and 621, four 62.2 and 628).
__device__ __forceinline__ Two exp2_of(Two x, int e) { return e % 5 == 2 ? exp2_by_terms(x) : exp2_of(x); }

// Waits for the loads from tensor memory; what they bring is not used ahead of this.
__device__ __forceinline__ void wait_loaded(float (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]),
                   "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]), "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]),
                   "+f"(r[21]), "+f"(r[22]), "+f"(r[23]), "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]),
                   "+f"(r[31])::"memory");
}

// Where a role stands: step `s` of the `n` of tile `i` of (request r, kv head), whose first step `f` is (columns), and the request's lengths.
struct Cursor { int r, kvh, i, s, n, unit, f, tiles, first, heard, place0, prefix, total, unit0; };

__device__ __forceinline__ void of_request(const Params& p, Cursor& c, int tiles) {
    const Portion& q = p.p[c.r];
    c.tiles = tiles;
    c.first = q.first, c.heard = q.heard, c.place0 = q.place0, c.prefix = q.prefix, c.total = q.total, c.unit0 = q.unit0;
}
template <int PASS>
__device__ __forceinline__ int tiles_of(const Params& p, int r) { return PASS == 1 ? row_tiles(p.p[r], p.tq) : key_tiles(p.p[r]); }

// The steps of the cursor's tile (the same as steps1_of and steps2_of; the quotient by float, set right).
template <int PASS>
__device__ __forceinline__ void of_tile(const Params& p, Cursor& c) {
    if (PASS == 1) {
        const int from = c.i * p.tq, end = min(from + p.tq, c.heard);
        c.n = from < c.heard ? (c.place0 + end + BR - 1) / BR : 0;
    } else {
        const int x = c.i * AR - c.place0, d = 2 * p.tq;
        int f = 0;
        if (x > 0) {
            f = (int)((float)x * p.per_step);
            const int rest = x - f * d;
            f += rest >= d ? 1 : rest < 0 ? -1 : 0;
        }
        c.f = f;
        c.n = p.p[c.r].row_steps - f;
    }
}

// On to the next tile that has steps.
template <int PASS>
__device__ __forceinline__ void next_tile(const Params& p, Cursor& c) {
    c.s = 0;
    do {
        ++c.i, ++c.unit;
        if (c.i == c.tiles) {
            c.i = 0;
            if (++c.kvh == p.nkv) {
                c.kvh = 0;
                int tiles = 0;
                do ++c.r; while (c.r < p.requests && (tiles = tiles_of<PASS>(p, c.r)) == 0);
                if (c.r == p.requests) {
                    c.n = 1;
                    return;
                }
                of_request(p, c, tiles);
            }
        }
        of_tile<PASS>(p, c);
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
    of_request(p, c, tiles);
    c.kvh = off / per;
    off -= c.kvh * per;
    c.i = 0;
    for (int i0 = 0; i0 < tiles; i0 += 32) {
        const int i = i0 + lane, n = i < tiles ? (PASS == 1 ? steps1_of(q, p.tq, i) : steps2_of(q, p.tq, i)) : 0;
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
    of_tile<PASS>(p, c);
    c.unit = (PASS == 1 ? q.unit0 : q.tile0) + c.kvh * tiles + c.i;
    return c;
}

// What a block was to write of its `mine` steps from `g0` on, made NaN by all its threads.
template <int PASS>
__device__ __forceinline__ void make_void(const Params& p, int g0, int mine) {
    const float nan = __int_as_float(0x7fffffff);
    Cursor c = find<PASS>(p, g0);
    for (int k = 0; k < mine; k += c.n - c.s, next_tile<PASS>(p, c)) {
        if (PASS == 1)
            for (int i = threadIdx.x; i < GROUPS * AR; i += THREADS) p.parts[(size_t)(c.unit + (int)blockIdx.x) * GROUPS * AR + i] = make_float2(-INFINITY, nan);
        else if (const int place = c.i * AR + (int)threadIdx.x; threadIdx.x < AR && place < c.total)
            p.weights[(((size_t)p.block_table[(size_t)c.r * p.bt_stride + (place >> p.page_shift)] * p.nkv + c.kvh) << p.page_shift) + (place & (p.page_size - 1))] = nan;
    }
}

template <int D, int PASS>
__global__ void __launch_bounds__(THREADS, 1) key_weights_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv,
                                                                    const __grid_constant__ Params p) {
    constexpr int DH = D / 64;
    extern __shared__ __align__(1024) unsigned char smem[];
    float* lse_s = reinterpret_cast<float*>(smem + off_lse(D));       // [LSE][256]
    float* sums_s = reinterpret_cast<float*>(smem + off_sums(D));     // [SUMS][GROUPS][128]
    int* tok_s = reinterpret_cast<int*>(smem + off_tok(D));           // [128] token of a tile's row
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + off_bars(D));
    uint32_t& tmem_base_s = *reinterpret_cast<uint32_t*>(smem + off_misc(D));
    int& abort_s = *reinterpret_cast<int*>(smem + off_misc(D) + 4);
    int4* desc_s = reinterpret_cast<int4*>(smem + off_desc(D));       // [LSE][2]
    Cursor& start_s = *reinterpret_cast<Cursor*>(smem + off_misc(D) + 8);
    static_assert(sizeof(Cursor) <= 56, "");
    int* issued_s = reinterpret_cast<int*>(smem + off_misc(D) + 64);  // what was put on its way: standing tiles, stages, lse, products
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem);
    const uint32_t a_smem = base, b_smem = base + off_b(D);
    const uint32_t a_full = smem_u32(bars), a_empty = a_full + 16, b_full = a_empty + 16, b_empty = b_full + 8 * STAGES, s_full = b_empty + 8 * STAGES,
                   s_empty = s_full + 16, l_full = s_empty + 16, l_empty = l_full + 8 * LSE, sums_full = l_empty + 8 * LSE;
    const int steps = PASS == 1 ? p.steps1 : p.steps2, quota = PASS == 1 ? p.quota1 : p.quota2;
    const int g0 = blockIdx.x * quota, mine = min(quota, steps - g0);
    const Waits waits{&abort_s, p.lost, p.polls[PASS - 1]};
    if (base & 1023u) {                                               // the swizzled tiles need it; never seen, but checked
        if (threadIdx.x == 0) give_up(waits, 11);
        pdl_wait();
        make_void<PASS>(p, g0, mine);
        return;
    }
    if (threadIdx.x == 0) {
        abort_s = 0;
        for (int s = 0; s < 2; ++s) {
            mbar_init(a_full + 8 * s, 1);
            mbar_init(a_empty + 8 * s, 1);
            mbar_init(s_full + 8 * s, 1);
            mbar_init(s_empty + 8 * s, 8);
        }
        for (int s = 0; s < LSE; ++s) {
            mbar_init(l_full + 8 * s, 1);
            mbar_init(l_empty + 8 * s, 8);
        }
        for (int s = 0; s < SUMS; ++s) mbar_init(sums_full + 8 * s, (GROUPS - 1) * 4);
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
    const int group_rows = p.group * p.tq;
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
    Cursor cur = start_s;
    // The column kernel's loader, products and waits begin ahead of the wait for the join kernel: queries and keys were there before the row
    // kernel began.  What reads the lse (the loader, further down) or writes waits.
    if (PASS == 1 || warp >= 2) pdl_wait();
    if (PASS == 1) pdl_launch_dependents();

    if (warp == 0) {
        // ---- loader ----
        // Of a tile of keys lane b has box b (a page, or 64 places of one): it looks its page up a step ahead and asks for it itself.
        const int box = min(p.page_size, 64), mask = p.page_size - 1;
        int page = 0, page_a = 0;
        auto look_up = [&](const Cursor& at, int key, int rows) {
            const int mine_key = key + lane * box;
            return lane * box < rows && mine_key < at.total ? p.block_table[(size_t)at.r * p.bt_stride + (mine_key >> p.page_shift)] : 0;
        };
        auto load_keys = [&](uint32_t dst, int rows, int pitch, int kvh, int key, int pg, uint32_t bar) {
            if (lane * box < rows)
#pragma unroll
                for (int h = 0; h < DH; ++h) tma_load_4d(dst + h * pitch + lane * box * 128, &map_kv, bar, h * 64, (key + lane * box) & mask, kvh, pg);
        };
        auto load_rows = [&](uint32_t dst, int pitch, int kvh, int token, uint32_t bar) {
            if (lane < DH) tma_load_3d(dst + lane * pitch, &map_q, bar, lane * 64, kvh * p.group, token);
        };
        const int q_bytes = group_rows * D * 2;
        bool ok = true;
        int tile = 0, sent_a = 0, sent_b = 0, sent_l = 0, share_k = 0, share_n = 0, alone = 0;      // the tile's first step here, its steps here; tiles that were all this block's
        int rows_in[STAGES], lse_in[LSE];                             // columns: the row tile that a stage, an lse buffer holds (few rows: the same for tile after tile)
        for (int i = 0; i < STAGES; ++i) rows_in[i] = -1;
        for (int i = 0; i < LSE; ++i) lse_in[i] = -1;
        auto look_ahead = [&](bool fresh) {
            if (PASS == 1) page = look_up(cur, cur.s * BR, BR);
            else if (fresh) page_a = look_up(cur, cur.i * AR, AR);
        };
        look_ahead(true);
        for (int k = 0; k < mine && ok; ++k) {
            if (k == 0 || cur.s == 0) {                               // a new standing tile
                ok = warp_wait(a_empty + 8 * (tile & 1), ((tile >> 1) & 1) ^ 1, waits, 1);
                if (!ok) break;
                const uint32_t bar = a_full + 8 * (tile & 1), dst = a_smem + (tile & 1) * a_bytes(D);
                if (lane == 0) mbar_expect_tx(bar, PASS == 1 ? q_bytes : a_bytes(D));
                __syncwarp();
                if (PASS == 1) load_rows(dst, AR * 128, cur.kvh, cur.first + cur.i * p.tq, bar);
                else load_keys(dst, AR, AR * 128, cur.kvh, cur.i * AR, page_a, bar);
                ++tile;
                ++sent_a;
                share_k = k;
                share_n = min(cur.n - cur.s, mine - k);
                alone += share_n == cur.n;
            }
            const int st = k % STAGES;
            ok = warp_wait(b_empty + 8 * st, ((k / STAGES) & 1) ^ 1, waits, 2);
            if (!ok) break;
            const uint32_t bar = b_full + 8 * st, dst = b_smem + st * b_bytes(D);
            const int t0 = PASS == 2 ? 2 * (cur.f + cur.s) : 0, unit = cur.unit0 + cur.kvh * 2 * p.p[cur.r].row_steps + t0;      // columns: the step's row tiles
            bool held = false;
            if (PASS == 2) {
#pragma unroll
                for (int i = 0; i < STAGES; ++i)
                    if (i == st) held = rows_in[i] == unit, rows_in[i] = unit;
            }
            if (lane == 0) {
                if (held) mbar_arrive(bar);
                else mbar_expect_tx(bar, PASS == 1 ? b_bytes(D) : 2 * q_bytes);
            }
            __syncwarp();
            if (PASS == 1) load_keys(dst, BR, BR * 128, cur.kvh, cur.s * BR, page, bar);
            else if (!held) {
                load_rows(dst, BR * 128, cur.kvh, cur.first + t0 * p.tq, bar);
                load_rows(dst + AR * 128, BR * 128, cur.kvh, cur.first + (t0 + 1) * p.tq, bar);
            }
            ++sent_b;
            if (PASS == 2 && k == 0) pdl_wait();
            const int ls = k % LSE, begin = g0 + k - cur.s, j = k - share_k;
            ok = warp_wait(l_empty + 8 * ls, ((k / LSE) & 1) ^ 1, waits, 3);           // step k - LSE has been read
            if (!ok) break;
            held = false;
            if (PASS == 2) {
#pragma unroll
                for (int i = 0; i < LSE; ++i)
                    if (i == ls) held = lse_in[i] == unit, lse_in[i] = unit;
            }
            if (lane == 0) {
                const int at = PASS == 1 ? cur.place0 + cur.i * p.tq - cur.s * BR : cur.i * AR - cur.place0 - t0 * p.tq;
                const int flags = (j < 2 ? FIRST : 0) | (j + 2 >= share_n ? LAST : 0) | (j & 1 ? 0 : EVEN) | (share_n == cur.n ? ALONE : 0) | (share_n == 1 ? SINGLE : 0) |
                                  alone << TILE_SHIFT;
                desc_s[2 * ls] = make_int4(at, cur.heard - t0 * p.tq, flags, cur.unit);
                desc_s[2 * ls + 1] = make_int4(begin, cur.n, cur.kvh | cur.r << 16, cur.i);
                if (PASS == 1 || held) mbar_arrive(l_full + 8 * ls);
                else {
                    mbar_expect_tx(l_full + 8 * ls, BR * 4);
                    bulk_load(smem_u32(lse_s + ls * BR), p.lse + (size_t)unit * AR, BR * 4, l_full + 8 * ls);
                }
            }
            ++sent_l;
            const bool fresh = ++cur.s == cur.n;
            if (fresh) next_tile<PASS>(p, cur);
            if (k + 1 < mine) look_ahead(fresh);
        }
        if (lane == 0) issued_s[0] = sent_a, issued_s[1] = sent_b, issued_s[2] = sent_l;
    } else if (warp == 1) {
        // ---- products: accumulator k & 1 = standing tile x streamed tile of step k ----
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BR >> 3) << 17) | ((uint32_t)(AR >> 4) << 24);
        bool ok = true;
        int tile = -1, k = 0;
        for (; k < mine; ++k) {
            const int st = k % STAGES;
            if (k == 0 || cur.s == 0) {
                ++tile;
                ok = warp_wait(a_full + 8 * (tile & 1), (tile >> 1) & 1, waits, 4);
                if (!ok) break;
            }
            ok = warp_wait(b_full + 8 * st, (k / STAGES) & 1, waits, 5) && warp_wait(s_empty + 8 * (k & 1), ((k >> 1) & 1) ^ 1, waits, 6);
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
        if (lane == 0) issued_s[3] = k;
    } else {
        // ---- groups of 128 threads, a lane of tensor memory each: pair k & 1 takes step k, each of its groups 128 columns ----
        const int which = (warp - 2) >> 2, pair = which >> 1, half = which & 1, quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t my = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(pair * BR + half * COLS);
        const int tok = tok_s[row], tok_first = tok_s[quarter * 32], tok_last = tok_s[quarter * 32 + 31];
        const float c = p.c;
        float m = -INFINITY, l = 0.f;                                 // rows: running maximum (log2 units) and sum; columns: l is the sum
        float* to = nullptr;
        float old = 0.f;
        for (int k = pair; k < mine; k += 2) {
            const int ls = k % LSE;
            if (!warp_wait(l_full + 8 * ls, (k / LSE) & 1, waits, 8)) break;
            const int4 d0 = desc_s[2 * ls], d1 = desc_s[2 * ls + 1];
            const Step st{d0.x, d0.y, d0.z, d0.w, d1.x, d1.y, d1.z, d1.w};
            const bool collects = PASS == 2 && (st.flags & (EVEN | ALONE)) == (EVEN | ALONE) && half == 0;
            if (st.flags & FIRST) {
                m = -INFINITY;
                l = 0.f;
                if (collects) {
                    // where this thread's place has its weight, and what it is: asked for ahead of the tile's steps
                    const int r = st.where >> 16, place = st.i * AR + row;
                    to = nullptr;
                    if (place < p.p[r].total) {
                        to = p.weights + (((size_t)p.block_table[(size_t)r * p.bt_stride + (place >> p.page_shift)] * p.nkv + (st.where & 0xffff)) << p.page_shift) +
                             (place & (p.page_size - 1));
                        old = place < p.p[r].prefix ? *to : 0.f;
                    }
                }
            }
            if (!warp_wait(s_full + 8 * pair, (k >> 1) & 1, waits, 7)) break;
            tc_fence_after();
            // Pieces of 32 columns, which a warp leaves out where no lane sees any of them and masks where not all are seen: rows and keys ascend
            // along lanes and columns, so the first and the last say which it is.
            const int own = st.at + tok - half * COLS;                // rows: the last column this one sees
            const int from = st.at + row - half * p.tq, live = st.live - half * p.tq;      // columns: the row tile's tokens [from, live) see this place
            Two sum[4] = {two(l, 0.f), 0, 0, 0};
#pragma unroll
            for (int c0 = 0; c0 < COLS; c0 += 32) {
                bool some, all;
                if (PASS == 1) some = c0 <= own - tok + tok_last, all = c0 + 31 <= own - tok + tok_first;
                else {
                    const int first = tok_s[c0], last = tok_s[c0 + 31];
                    some = last >= from - lane && first < live;
                    all = first >= from - lane + 31 && last < live;
                }
                float s[32];
                if (some) {
                    tmem_ld32(my + (uint32_t)c0, s);
                    wait_loaded(s);
                }
                if (c0 + 32 == COLS) {                                // the last has come: the accumulator goes back to the products
                    tc_fence_before();
                    warp_arrive(s_empty + 8 * pair);
                }
                if (!some) continue;
                if (PASS == 1) {
                    if (!all) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) s[e] = c0 + e <= own ? s[e] : -INFINITY;
                    }
                    float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                    for (int e = 4; e < 28; e += 8)
#pragma unroll
                        for (int j = 0; j < 4; ++j) mx[j] = max3(mx[j], s[e + 2 * j], s[e + 2 * j + 1]);
                    mx[0] = max3(mx[0], s[28], s[29]);
                    mx[1] = max3(mx[1], s[30], s[31]);
                    const float now = fmaxf(m, fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * c);
                    if (__any_sync(0xffffffffu, now > m)) {
                        const float f = now > m ? ex2(m - now) : 1.f;                 // (0 where m is -inf)
#pragma unroll
                        for (int j = 0; j < 4; ++j) sum[j] = mul2(sum[j], two(f, f));
                        m = now;
                    }
                    const float off = m == -INFINITY ? 0.f : -m;
#pragma unroll
                    for (int e = 0; e < 16; ++e) sum[e & 3] = add2(sum[e & 3], exp2_of(fma2(two(s[2 * e], s[2 * e + 1]), two(c, c), two(off, off)), e));
                } else {
                    const ulonglong2* minus_lse = reinterpret_cast<const ulonglong2*>(lse_s + ls * BR + half * COLS + c0);
                    if (all) {
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const ulonglong2 z = minus_lse[e >> 1];
                            sum[e & 3] = add2(sum[e & 3], exp2_of(fma2(two(s[2 * e], s[2 * e + 1]), two(c, c), z.x), e));
                            sum[(e + 1) & 3] = add2(sum[(e + 1) & 3], exp2_of(fma2(two(s[2 * e + 2], s[2 * e + 3]), two(c, c), z.y), e + 1));
                        }
                    } else {
                        const int low = max(from, 0);
                        const uint32_t seen = max(live - low, 0);
                        const int4* tok4 = reinterpret_cast<const int4*>(tok_s + c0);
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const ulonglong2 z = minus_lse[e >> 1];
                            const int4 t = tok4[e >> 1];
                            float a, b;
                            apart(exp2_of(fma2(two(s[2 * e], s[2 * e + 1]), two(c, c), z.x)), a, b);
                            sum[e & 3] = add2(sum[e & 3], two((uint32_t)(t.x - low) < seen ? a : 0.f, (uint32_t)(t.y - low) < seen ? b : 0.f));
                            apart(exp2_of(fma2(two(s[2 * e + 2], s[2 * e + 3]), two(c, c), z.y)), a, b);
                            sum[(e + 1) & 3] = add2(sum[(e + 1) & 3], two((uint32_t)(t.z - low) < seen ? a : 0.f, (uint32_t)(t.w - low) < seen ? b : 0.f));
                        }
                    }
                }
            }
            float a, b;
            apart(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), a, b);
            l = a + b;
            warp_arrive(l_empty + 8 * ls);
            if (!(st.flags & LAST)) continue;
            // the end of what this pair has of the tile here; its part's number: the pair with the tile's first step comes first
            const int part = (st.flags & EVEN ? 0 : 2) + half;
            const size_t slot = ((size_t)(st.unit + (int)blockIdx.x) * GROUPS + part) * AR + row;
            if (PASS == 1) {
                p.parts[slot] = make_float2(m, l);
            } else if (st.flags & ALONE) {
                // The groups' sums through shared memory, added up by the group that has the tile's first columns; the others go on.  (SUMS tiles of room: a
                // group is at most four tiles ahead of another, whose accumulators the products behind wait for.)
                const int at = (st.flags >> TILE_SHIFT) - 1;
                const uint32_t full = sums_full + 8 * (at % SUMS);
                float* sums = sums_s + (size_t)(at % SUMS) * GROUPS * AR;
                sums[part * AR + row] = l;
                __syncwarp();
                if (part) {
                    // twelve warps' worth of arrivals, of three groups or of one
                    if (lane == 0) mbar_arrive_many(full, st.flags & SINGLE ? 3 : 1);
                } else {
                    if (!warp_wait(full, (at / SUMS) & 1, waits, 9)) break;
                    const int parts = st.flags & SINGLE ? 2 : 4;
                    float w = old;
                    for (int j = 0; j < parts; ++j) w += sums[j * AR + row];
                    if (to) *to = w;
                }
            } else {
                // several blocks: of the warps with these 32 keys the one that comes last joins what all have left in scratch, in their order
                const int b0 = st.begin / quota, b1 = (st.begin + st.steps - 1) / quota;
                int expected = 0;
                for (int b = b0; b <= b1; ++b) expected += parts_of(st.begin, st.steps, quota, b);
                __stcg(p.sums + slot, l);
                __threadfence();
                __syncwarp();
                int before = 0;
                if (lane == 0) before = atomicAdd(p.done + 4 * st.unit + quarter, 1);
                if (__shfl_sync(0xffffffffu, before, 0) == expected - 1) {
                    __threadfence();
                    const int r = st.where >> 16, place = st.i * AR + row;
                    float w = 0.f;
                    for (int b = b0; b <= b1; ++b)
                        for (int j = 0, parts = parts_of(st.begin, st.steps, quota, b); j < parts; ++j)
                            w += __ldcg(p.sums + ((size_t)(st.unit + b) * GROUPS + j) * AR + row);
                    if (place < p.p[r].total) {
                        float* at = p.weights + (((size_t)p.block_table[(size_t)r * p.bt_stride + (place >> p.page_shift)] * p.nkv + (st.where & 0xffff)) << p.page_shift) +
                                    (place & (p.page_size - 1));
                        *at = (place < p.p[r].prefix ? *at : 0.f) + w;
                    }
                }
            }
        }
    }
    if (PASS == 2 && warp < 2) pdl_wait();                            // (a block ends behind the kernels ahead)
    if (PASS == 2) pdl_launch_dependents();
    tc_fence_before();
    __syncthreads();
    if (*waits.abort) {
        // Every role has left.  Copies on their way still land in this block's shared memory and products in its tensor memory: each gets a bounded wait.
        if (threadIdx.x == 0) {
            for (int j = max(0, issued_s[0] - 2); j < issued_s[0]; ++j)
                for (uint32_t i = 0; i < (1u << 20) && !mbar_try_wait(a_full + 8 * (j & 1), (j >> 1) & 1); ++i) {}
            for (int j = max(0, issued_s[1] - STAGES); j < issued_s[1]; ++j)
                for (uint32_t i = 0; i < (1u << 20) && !mbar_try_wait(b_full + 8 * (j % STAGES), (j / STAGES) & 1); ++i) {}
            for (int j = max(0, issued_s[2] - LSE); j < issued_s[2]; ++j)
                for (uint32_t i = 0; i < (1u << 20) && !mbar_try_wait(l_full + 8 * (j % LSE), (j / LSE) & 1); ++i) {}
        }
        if (warp == 1 && issued_s[3] > 0) {
            const int k = issued_s[3] - 1;
            for (uint32_t i = 0; i < (1u << 20) && !mbar_try_wait(s_full + 8 * (k & 1), (k >> 1) & 1); ++i) {}
            __syncwarp();
        }
        make_void<PASS>(p, g0, mine);
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
    }
}

// A row tile a block: its parts joined, lse = max + log2(sum); +inf (its negative is kept) for rows that are none.  Four threads a row, or eight where a tile has
// many blocks' parts, each with one number's part of every (second) block, four of them on their way, joined in the order of the threads.  Also clears the column kernel's counters.
constexpr int JOIN_THREADS = 8 * AR;       // at most
__device__ __forceinline__ void join_part(float& m, float& l, float2 v) {
    if (v.x == -INFINITY && v.y == 0.f) return;                       // no keys (a NaN is no maximum, but makes the sum one)
    const float now = fmaxf(m, v.x);
    l = fmaf(v.y, exp2f(v.x - now), m == -INFINITY && l == 0.f ? 0.f : l * exp2f(m - now));
    m = now;
}
__global__ void __launch_bounds__(JOIN_THREADS) key_weights_join_kernel(const __grid_constant__ Params p) {
    __shared__ float2 part_s[8][AR];
    __shared__ int sum_s[32];
    pdl_enter_small();
    const int unit = blockIdx.x, tid = threadIdx.x, row = tid & (AR - 1), sub = tid / AR, subs = blockDim.x / AR;
    for (int i = unit * blockDim.x + tid; i < 4 * p.tiles; i += gridDim.x * blockDim.x) p.done[i] = 0;
    int r = 0;
    while (r + 1 < p.requests && p.p[r + 1].unit0 <= unit) ++r;
    const Portion& q = p.p[r];
    const int tiles = row_tiles(q, p.tq), i = (unit - q.unit0) % tiles;
    // the tile's steps [begin, begin + steps)
    int ahead = 0;
    for (int j = tid; j < i; j += blockDim.x) ahead += steps1_of(q, p.tq, j);
    ahead = __reduce_add_sync(0xffffffffu, ahead);
    if ((tid & 31) == 0) sum_s[tid >> 5] = ahead;
    __syncthreads();
    const int warps = blockDim.x >> 5, begin = q.step1 + (unit - q.unit0) / tiles * q.per1 + __reduce_add_sync(0xffffffffu, (tid & 31) < warps ? sum_s[tid & 31] : 0), steps = steps1_of(q, p.tq, i);
    const bool live = row < p.group * p.tq && i * p.tq + row / p.group < q.heard;
    float m = -INFINITY, l = 0.f;
    if (live) {
        const int b0 = begin / p.quota1, b1 = (begin + steps - 1) / p.quota1, j = sub & 3;
        const int every = subs >> 2;
        for (int b = b0 + (sub >> 2); b <= b1; b += 4 * every) {
            float2 v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int at = b + u * every;
                v[u] = at <= b1 && j < parts_of(begin, steps, p.quota1, at) ? p.parts[((size_t)(unit + at) * GROUPS + j) * AR + row] : make_float2(-INFINITY, 0.f);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) join_part(m, l, v[u]);
        }
    }
    part_s[sub][row] = make_float2(m, l);
    __syncthreads();
    if (sub) return;
    float lse = -INFINITY;                                            // negative
    if (live) {
        m = -INFINITY, l = 0.f;
        for (int u = 0; u < subs; ++u) join_part(m, l, part_s[u][row]);
        lse = -(m + log2f(l));
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
    int most = 0;                             // steps of a row tile
    for (int r = 0; r < p.requests; ++r) most = p.p[r].heard > 0 && (p.p[r].total + BR - 1) / BR > most ? (p.p[r].total + BR - 1) / BR : most;
    launch_pdl(key_weights_join_kernel, dim3(p.units), dim3(most > 4 * p.quota1 ? JOIN_THREADS : JOIN_THREADS / 2), 0, stream, p);
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
        long long per1 = 0, per2 = 0;
        const int rows = row_tiles(q, p.tq), keys = key_tiles(q);
        q.row_steps = rows / 2;
        for (int i = 0; i < rows; ++i) per1 += steps1_of(q, p.tq, i);
        for (int i = 0; i < keys; ++i) per2 += steps2_of(q, p.tq, i);
        s1 += per1 * nkv;
        s2 += per2 * nkv;
        if (s1 > 0x3fffffff || s2 > 0x3fffffff) return 0;
        q.per1 = (int)per1;
        q.per2 = (int)per2;
        unit += rows * nkv;
        tile += keys * nkv;
        first += fresh[r];
    }
    const int sms = sm_count();
    p.units = unit;
    p.tiles = tile;
    p.steps1 = (int)s1;
    p.steps2 = (int)s2;
    p.quota1 = s1 > 0 ? (int)((s1 + sms - 1) / sms) : 1;
    p.quota2 = s2 > 0 ? (int)((s2 + sms - 1) / sms) : 1;
    const int b1 = (p.steps1 + p.quota1 - 1) / p.quota1, b2 = (p.steps2 + p.quota2 - 1) / p.quota2;
    // parts | lse | counters | sums, each on 16 bytes
    return (size_t)(unit + b1) * 2 * GROUPS * AR + (size_t)unit * AR + (size_t)tile * 4 + (size_t)(tile + b2) * GROUPS * AR + 16;
}

}  // namespace keyw5
}  // namespace lily

using namespace lily;

// Whether these kernels take the sizes (bfloat16).
LILY_API int lily_key_weights_tc_takes(int nq, int nkv, int d, int page_size, float scale) {
    return (d == 64 || d == 128) && page_size >= 8 && (page_size & (page_size - 1)) == 0 && nkv > 0 && nq % nkv == 0 && nq / nkv >= 1 && nq / nkv <= 128 && scale > 0.f &&
           scale < INFINITY;
}

// Floats of scratch for portions of `fresh` tokens behind `prefix` places (host arrays); 0: nothing to do, too much to number, or heads that these kernels do not take.
LILY_API size_t lily_key_weights_tc_floats(int requests, const int* prefix, const int* fresh, int observe, int nq, int nkv) {
    if (nq <= 0 || nkv <= 0 || nq % nkv != 0 || nq / nkv > keyw5::AR) return 0;
    static thread_local keyw5::Params p;
    size_t most = 0;
    for (int r = 0; r < requests; r += keyw5::MAX_R) {
        const size_t n = keyw5::plan(p, requests - r < keyw5::MAX_R ? requests - r : keyw5::MAX_R, prefix + r, fresh + r, observe, nq / nkv, nkv);
        if (n == 0) return 0;
        most = n > most ? n : most;
    }
    return most;
}

// The host's word in which these kernels say that a wait ran out; made with the first launch that may.
static std::atomic<int*> g_lost_word{nullptr};
static int* lost_word() {
    static int* word = [] {
        int* p = new_host_word();
        g_lost_word = p;
        return p;
    }();
    return word;
}

// 0, or (code << 24 | block) of a bounded wait that gave up since the last call; clears it.  `wait`: behind all work of the device; else as far as the host
// knows (the kernels it has waited for).
LILY_API int lily_key_weights_status(int wait) {
    if (wait && cudaDeviceSynchronize() != cudaSuccess) return -1;
    volatile int* word = g_lost_word;
    const int v = word ? *word : 0;
    if (v != 0) *word = 0;
    return v;
}

LILY_API int lily_key_weights_tc(const void* q, int tokens, const void* kv, int pages, float* weights, const int* block_table, int bt_stride, float* scratch,
                                 int requests, const int* prefix, const int* fresh, int observe, int nq, int nkv, int d, int page_size, float scale,
                                 int row_polls, int column_polls, cudaStream_t stream) {
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
    p.polls[0] = row_polls;
    p.polls[1] = column_polls;
    p.lost = lost_word();
    LILY_REQUIRE(p.lost != nullptr, "attention_key_weights: no word of the host's memory");
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
            p.per_step = 1.f / (float)(2 * tq);
            for (p.page_shift = 0; 1 << p.page_shift < page_size;) ++p.page_shift;
            const int b1 = (p.steps1 + p.quota1 - 1) / p.quota1;
            float* at = scratch;
            p.parts = reinterpret_cast<float2*>(at);
            at += (size_t)(p.units + b1) * 2 * keyw5::GROUPS * keyw5::AR;
            p.lse = at;
            at += (size_t)p.units * keyw5::AR;
            p.done = reinterpret_cast<int*>(at);
            at += (size_t)p.tiles * 4;
            p.sums = at;
            const int rc = d == 64 ? keyw5::launch<64>(p, map_q, map_kv, stream) : keyw5::launch<128>(p, map_q, map_kv, stream);
            if (rc) return rc;
        }
        for (int i = 0; i < some; ++i) row0 += fresh[r + i];
    }
    LILY_CHECK_LAUNCH("attention_key_weights");
    return 0;
}
