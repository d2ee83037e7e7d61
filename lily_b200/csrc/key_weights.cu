// What the tokens of a prompt's portion give to every cached key: the column sums of the softmax.
//
// Token t of the n new ones of a request behind p cached places sees the places j <= p + t.  The last `heard` tokens are heard:
//   P_thj = exp(c q_th . k_j - lse_th),  w_gj <- (j < p ? w_gj : 0) + sum over heard t and the heads h of g of P_thj,
// with w float32 [pages, kv_heads, page_size] beside the keys; the weights of the portion's own places are set.
// (bfloat16 heads of 64 and 128 have kernels of their own, key_weights_tcgen05.cu; these are for float32 and every other head size.)
//
// The query heads of a kv head stand below one another, row t * G + h.  Three kernels: tiles of 64 rows x 64 keys of scores with each row's
// (max, sum) over the tile; a row's tiles joined to its lse; the columns, which read the scores back.  On the CUDA cores a score costs
// 2 d = 256 flops, 4 ps at their 72 TFLOP/s, and to keep it and read it again 8 bytes, 1.2 ps of memory and less of L2, so scores are kept
// instead of formed twice; long portions come in runs of rows whose scores fit the scratch, each adding to the weights of the one before.
#include "common.cuh"

#include <cooperative_groups.h>

namespace lily {
namespace keyw {

namespace cg = cooperative_groups;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int TM = 64, TN = 64, KC = 32, LD = KC + 4, THREADS = 256;

constexpr int MAX_R = 48;                 // requests a launch

// One request of a launch, for the heard tokens of this run.
struct Portion {
    int request;                  // row of the block table
    int first, rows;              // row of q of the run's first token; rows
    int place0, last;             // the places of that token and of the run's last
    int prefix, total;            // cached places before and after the portion
    int row_tiles, key_tiles;
    int tile0, rows0, cols0;      // its first tile of scores, tile of rows, tile of keys (of its first kv head)
};

struct Args {
    const void* q;                // [tokens, nq * d]
    const void* kv;               // layer base: [pages, 2, nkv, page_size, d]
    float* weights;               // [pages, nkv, page_size]
    float* scores;                // [tiles][64 rows][64], log2 units; -inf where a row does not see a place
    float2* parts;                // [tiles][64] (max, sum)
    float* lse;                   // [tiles of rows][64]
    const int* block_table;
    int bt_stride, requests, again, nq, nkv, d, page_size, page_shift;      // again: not the first run, which sets the portions' own weights
    float scale;
    Portion p[MAX_R];
};

// The request of tile `at` of a kernel that numbers its tiles by `OFF`, and the tile within it.
template <int Portion::*OFF>
__device__ __forceinline__ const Portion& request_of(const Args& a, int& at) {
    int r = 0;
    while (r + 1 < a.requests && a.p[r + 1].*OFF <= at) ++r;
    at -= a.p[r].*OFF;
    return a.p[r];
}

// Whether a row of the run ahead of row `end` sees a place from `k0` on.  Both the kernel that makes tiles of scores and the one that reads them go by it: a tile
// that it does not name is neither written nor read, whatever the run's last tile of rows is filled to.
__device__ __forceinline__ bool seen(const Portion& p, int end, int k0, int group) { return k0 <= min(p.last, p.place0 + (end - 1) / group); }

__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ float halves(unsigned long long v) {
    float a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
    return a + b;
}
// Four neighbouring numbers of a row from `c` on (zeros behind `d`); VEC: the row is aligned for it and d a multiple of four.
template <typename T, bool VEC>
__device__ __forceinline__ float4 four(const T* row, int c, int d) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (VEC) {
        if (c < d) {
            if constexpr (sizeof(T) == 4) v = *reinterpret_cast<const float4*>(row + c);
            else {
                const uint2 raw = *reinterpret_cast<const uint2*>(row + c);
                const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x)), y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
                v = make_float4(x.x, x.y, y.x, y.y);
            }
        }
    } else {
        if (c < d) v.x = to_float(row[c]);
        if (c + 1 < d) v.y = to_float(row[c + 1]);
        if (c + 2 < d) v.z = to_float(row[c + 2]);
        if (c + 3 < d) v.w = to_float(row[c + 3]);
    }
    return v;
}

// A tile of scores a block (kv heads, row tiles, key tiles of each request, numbered through).  A thread has the 4 x 4 of rows ty + 16 i and keys tx + 16 j, so that the
// rows of both tiles lie in shared memory as they come (36 numbers a row of 32: no two lanes meet in a bank) and products are packed pairs along the
// head; the 32 products of a chunk are added up by themselves, which quarters the error of a long sum of like terms.  The next chunk is on its way
// while one is multiplied.  What bounds it are the reads of shared memory (a warp waits for them 2.6 cycles of 6.7; the multiply-adds' unit is busy 46 % of the
// time): 2,048 tokens of 32 heads of 128 take 666 us, 27 TFLOP/s; 8 x 4 a thread gave 608, and more for few tokens (13.3 us became 14.2).
template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) key_weights_scores_kernel(const __grid_constant__ Args a) {
    __shared__ __align__(16) float q_s[TM][LD], k_s[TN][LD];
    pdl_enter_small();
    int at = blockIdx.x;
    const Portion& sp = request_of<&Portion::tile0>(a, at);
    const int kt = at % sp.key_tiles, rt = at / sp.key_tiles % sp.row_tiles, kvh = at / sp.key_tiles / sp.row_tiles;
    const int group = a.nq / a.nkv, row0 = rt * TM, k0 = kt * TN;
    if (!seen(sp, row0 + TM, k0, group)) return;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int* table = a.block_table + (size_t)sp.request * a.bt_stride;
    // a thread brings columns 4 (tid % 8) of rows tid / 8 and tid / 8 + 32 of either tile
    const T *q_row[2], *k_row[2];
    const int c4 = (tid & 7) * 4;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int r = (tid >> 3) + 32 * u, row = row0 + r, place = k0 + r;
        q_row[u] = row < sp.rows ? (const T*)a.q + ((size_t)(sp.first + row / group) * a.nq + kvh * group + row % group) * a.d : nullptr;
        k_row[u] = place < sp.total ? (const T*)a.kv + ((((size_t)table[place >> a.page_shift] * 2 * a.nkv + kvh) << a.page_shift) + (place & (a.page_size - 1))) * a.d : nullptr;
    }
    float4 q_next[2], k_next[2];
    auto fetch = [&](int c0) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            q_next[u] = q_row[u] ? four<T, VEC>(q_row[u], c0 + c4, a.d) : make_float4(0.f, 0.f, 0.f, 0.f);
            k_next[u] = k_row[u] ? four<T, VEC>(k_row[u], c0 + c4, a.d) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    float s[4][4] = {};
    fetch(0);
    for (int c0 = 0; c0 < a.d; c0 += KC) {
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            *reinterpret_cast<float4*>(&q_s[(tid >> 3) + 32 * u][c4]) = q_next[u];
            *reinterpret_cast<float4*>(&k_s[(tid >> 3) + 32 * u][c4]) = k_next[u];
        }
        __syncthreads();
        if (c0 + KC < a.d) fetch(c0 + KC);
        unsigned long long part[4][4] = {};
#pragma unroll
        for (int c = 0; c < KC; c += 4) {
            ulonglong2 x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[i] = *reinterpret_cast<const ulonglong2*>(&q_s[ty + 16 * i][c]);
                y[i] = *reinterpret_cast<const ulonglong2*>(&k_s[tx + 16 * i][c]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) part[i][j] = fma2(x[i].y, y[j].y, fma2(x[i].x, y[j].x, part[i][j]));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] += halves(part[i][j]);
    }
    const float c = a.scale * LOG2E;
    const size_t tile = blockIdx.x;
    float* to = a.scores + tile * (TM * TN);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty + 16 * i, row = row0 + r, last = row < sp.rows ? sp.place0 + row / group : -1;      // the last place this row sees
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[i][j] = k0 + tx + 16 * j <= last ? s[i][j] * c : -INFINITY;
            to[r * TN + tx + 16 * j] = s[i][j];
            m = fmaxf(m, s[i][j]);
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int j = 0; j < 4; ++j) l += exp2f(s[i][j] - base);
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (tx == 0) a.parts[tile * TM + r] = make_float2(m, l);
    }
}

// A tile of rows a block: the parts of each row joined in their order.  A row whose lse is no number gives NaN to the places it sees and nothing to the others, whose
// scores are -inf: its scores become NaN and -inf here, and its lse 0, so that the columns kernel need not look for it (which took 1.5 us of 32).
__global__ void __launch_bounds__(TM) key_weights_lse_kernel(const __grid_constant__ Args a) {
    pdl_enter_small();
    int at = blockIdx.x;
    const Portion& sp = request_of<&Portion::rows0>(a, at);
    const int rt = at % sp.row_tiles, kvh = at / sp.row_tiles, group = a.nq / a.nkv, row = rt * TM + threadIdx.x;
    // the tiles that were made for this tile of rows
    const int tiles = (sp.place0 + (min((rt + 1) * TM, sp.rows) - 1) / group) / TN + 1;
    const float2* part = a.parts + ((size_t)sp.tile0 + ((size_t)kvh * sp.row_tiles + rt) * sp.key_tiles) * TM + threadIdx.x;
    float m = -INFINITY, l = 0.f;
    for (int t = 0; t < tiles; ++t) m = fmaxf(m, part[(size_t)t * TM].x);
    for (int t = 0; t < tiles; ++t) {
        const float2 v = part[(size_t)t * TM];
        if (v.x > -INFINITY || v.y != 0.f) l = fmaf(v.y, exp2f(v.x - m), l);              // (a NaN is no maximum, but makes the sum one)
    }
    float lse = row < sp.rows ? m + log2f(l) : 0.f;
    if (!(fabsf(lse) < INFINITY)) {
        lse = 0.f;
        float* scores = a.scores + (((size_t)sp.tile0 + ((size_t)kvh * sp.row_tiles + rt) * sp.key_tiles) * TM + threadIdx.x) * TN;
        for (int j = 0; j <= sp.place0 + row / group; ++j) scores[(size_t)(j / TN) * (TM * TN) + j % TN] = __int_as_float(0x7fffffff);
    }
    a.lse[(size_t)blockIdx.x * TM + threadIdx.x] = lse;
}

// grid (tiles of keys, parts): the sums of a tile's columns, four a thread over every 32nd row.  What bounds it is the chain of
// reads: the parts, a cluster of up to four blocks, take turns at the tiles of rows, eight rows a thread on their way, and the first adds up what all have
// found, in their order.
constexpr int COL_THREADS = 512, COL_PARTS = 4;
__global__ void __launch_bounds__(COL_THREADS) key_weights_columns_kernel(const __grid_constant__ Args a) {
    __shared__ __align__(16) float sum_s[32][TN];
    __shared__ float parts_s[COL_PARTS][TN];
    if (gridDim.y > 1) cluster_arrive_started();
    pdl_enter_small();
    int tile_at = blockIdx.x;
    const Portion& sp = request_of<&Portion::cols0>(a, tile_at);
    const int kt = tile_at % sp.key_tiles, kvh = tile_at / sp.key_tiles, group = a.nq / a.nkv, k0 = kt * TN, part = blockIdx.y, parts = gridDim.y;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    // the weights' places, asked for ahead
    float* at = nullptr;
    float sum = 0.f;
    if (part == 0 && tid < TN && k0 + tid < sp.total) {
        const int place = k0 + tid;
        at = a.weights + (((size_t)a.block_table[(size_t)sp.request * a.bt_stride + (place >> a.page_shift)] * a.nkv + kvh) << a.page_shift) + (place & (a.page_size - 1));
        sum = place < sp.prefix || a.again ? *at : 0.f;
    }
    float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
    // the tiles of rows that see any of these places (none where the run ends ahead of them)
    const int tiles = k0 <= sp.last ? sp.row_tiles : 0, first = max(0, k0 - sp.place0) * group / TM;
    for (int t0 = first + part; t0 < tiles; t0 += 4 * parts) {
        float4 s[8];
        float e[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int t = t0 + (u >> 1) * parts, r = ty + 32 * (u & 1);
            s[u] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            e[u] = 0.f;
            if (t < tiles) {
                const size_t rows = (size_t)kvh * sp.row_tiles + t;
                s[u] = reinterpret_cast<const float4*>(a.scores + ((size_t)sp.tile0 + rows * sp.key_tiles + kt) * (TM * TN))[r * (TN / 4) + tx];
                e[u] = a.lse[((size_t)sp.rows0 + rows) * TM + r];
            }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            w.x += exp2f(s[u].x - e[u]);
            w.y += exp2f(s[u].y - e[u]);
            w.z += exp2f(s[u].z - e[u]);
            w.w += exp2f(s[u].w - e[u]);
        }
    }
    *reinterpret_cast<float4*>(&sum_s[ty][4 * tx]) = w;
    __syncthreads();
    if (parts > 1) cluster_wait_started();
    if (tid < TN) {
        float mine = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) mine += sum_s[i][tid];
        if (parts == 1) sum += mine;
        else write_to_block(&parts_s[part][tid], 0, mine);
    }
    if (parts > 1) {
        cg::this_cluster().sync();
        if (tid < TN)
            for (int i = 0; i < parts; ++i) sum += parts_s[i][tid];
    }
    if (at) *at = sum;
}

// The tiles of a launch: heard tokens [from, from + some) of up to MAX_R requests (host lengths).  Requests without such tokens are left out.
struct Tiles { long long scores, rows, keys; };
static Tiles plan(Args& a, int requests, int request0, int token0, const int* prefix, const int* fresh, int observe, int from, int some) {
    Tiles t{};
    const int group = a.nq / a.nkv;
    a.requests = 0;
    for (int r = 0; r < requests; ++r) {
        const int heard = observe > 0 && observe < fresh[r] ? observe : fresh[r], mine = heard - from < some ? heard - from : some;
        if (mine > 0) {
            Portion& p = a.p[a.requests++];
            p.request = request0 + r;
            p.first = token0 + fresh[r] - heard + from;
            p.rows = mine * group;
            p.place0 = prefix[r] + fresh[r] - heard + from;
            p.last = p.place0 + mine - 1;
            p.prefix = prefix[r];
            p.total = prefix[r] + fresh[r];
            p.row_tiles = (p.rows + TM - 1) / TM;
            p.key_tiles = (p.total + TN - 1) / TN;
            p.tile0 = (int)t.scores;
            p.rows0 = (int)t.rows;
            p.cols0 = (int)t.keys;
            t.scores += (long long)a.nkv * p.row_tiles * p.key_tiles;
            t.rows += (long long)a.nkv * p.row_tiles;
            t.keys += (long long)a.nkv * p.key_tiles;
        }
        token0 += fresh[r];
    }
    return t;
}
static size_t floats_of(const Tiles& t) { return (size_t)t.scores * (TM * TN + 2 * TM) + (size_t)t.rows * TM; }

// Heard tokens of a run: as many as keep its scores within about `scores`, a tile of rows at least.
static int run_of(const Args& a, int requests, const int* prefix, const int* fresh, int scores) {
    long long places = 0;
    for (int r = 0; r < requests; ++r) places += prefix[r] + fresh[r] + TN;
    const int group = a.nq / a.nkv, least = (TM + group - 1) / group;
    const long long most = scores / (places * a.nq > 0 ? places * a.nq : 1);
    return most < least ? least : most > 0x7fffff ? 0x7fffff : (int)most;
}

template <typename F>
static int each_run(Args& a, int requests, const int* prefix, const int* fresh, int observe, int scores, F&& use) {
    int token0 = 0;
    for (int r = 0; r < requests; r += MAX_R) {
        const int now = requests - r < MAX_R ? requests - r : MAX_R, some = run_of(a, now, prefix + r, fresh + r, scores);
        int heard = 0, tokens = 0;
        for (int i = r; i < r + now; ++i) {
            const int h = observe > 0 && observe < fresh[i] ? observe : fresh[i];
            heard = h > heard ? h : heard;
            tokens += fresh[i];
        }
        for (int from = 0; from < heard; from += some) {
            const Tiles t = plan(a, now, r, token0, prefix + r, fresh + r, observe, from, some);
            a.again = from > 0;
            if (int rc = use(t)) return rc;
        }
        token0 += tokens;
    }
    return 0;
}

}  // namespace keyw
}  // namespace lily

using namespace lily;

// Floats of scratch for portions of `fresh` tokens behind `prefix` places (host arrays): the scores of a run (about `most_scores` of them), the rows' parts, their lse.
// (0 for heads that do not fit, which the launch refuses)
LILY_API size_t lily_key_weights_floats(int requests, const int* prefix, const int* fresh, int observe, int nq, int nkv, int most_scores) {
    if (nq <= 0 || nkv <= 0 || nq % nkv != 0) return 0;
    static thread_local keyw::Args a;
    a.nq = nq;
    a.nkv = nkv;
    size_t most = 0;
    keyw::each_run(a, requests, prefix, fresh, observe, most_scores, [&](const keyw::Tiles& t) {
        const size_t n = keyw::floats_of(t);
        most = n > most ? n : most;
        return 0;
    });
    return most;
}

LILY_API int lily_key_weights(const void* q, const void* kv, float* weights, const int* block_table, int bt_stride, float* scratch, int requests,
                              const int* prefix, const int* fresh, int observe, int nq, int nkv, int d, int page_size, float scale, int dtype,
                              int most_scores, cudaStream_t stream) {
    LILY_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "attention_key_weights: %d query heads over %d kv heads", nq, nkv);
    LILY_REQUIRE(d >= 1 && page_size > 0 && (page_size & (page_size - 1)) == 0 && observe >= 0, "attention_key_weights: head size %d, pages of %d, the last %d heard", d, page_size,
                 observe);
    LILY_REQUIRE(dtype == kF32 || dtype == kBF16, "attention_key_weights: dtype %d", dtype);
    LILY_REQUIRE(((uintptr_t)scratch & 15) == 0, "attention_key_weights: scratch must be 16-byte aligned");
    keyw::Args a{};
    a.q = q; a.kv = kv; a.weights = weights; a.scores = scratch; a.block_table = block_table; a.bt_stride = bt_stride; a.nq = nq; a.nkv = nkv; a.d = d;
    a.page_size = page_size; a.scale = scale;
    while (1 << a.page_shift < page_size) ++a.page_shift;
    // (reads of four numbers, or of one where rows are not aligned for it: 106 and 115 us for 1,000 tokens of 16 heads of 128)
    const bool vec = d % 4 == 0 && (((uintptr_t)q | (uintptr_t)kv) & 15) == 0;
    const int rc = keyw::each_run(a, requests, prefix, fresh, observe, most_scores, [&](const keyw::Tiles& t) {
        LILY_REQUIRE(t.scores <= 0x7fffffff, "attention_key_weights: %lld tiles", t.scores);
        a.parts = (float2*)(a.scores + (size_t)t.scores * (keyw::TM * keyw::TN));
        a.lse = (float*)(a.parts + (size_t)t.scores * keyw::TM);
        const dim3 grid((unsigned)t.scores);
#define LAUNCH(T, V) launch_pdl(keyw::key_weights_scores_kernel<T, V>, grid, dim3(keyw::THREADS), 0, stream, a)
        if (dtype == kF32) { if (vec) LAUNCH(float, true); else LAUNCH(float, false); }
        else { if (vec) LAUNCH(__nv_bfloat16, true); else LAUNCH(__nv_bfloat16, false); }
#undef LAUNCH
        launch_pdl(keyw::key_weights_lse_kernel, dim3((unsigned)t.rows), dim3(keyw::TM), 0, stream, a);
        // four tiles of rows a block or more (us, float32, 16 heads of 128 over 4, in 1 / 2 / 4 / 8 parts: 1,000 tokens 113 / 102 / 102 / 106, 200 tokens 22 / 19 / 18 / 20,
        // 64 behind 4,000 places 51 / 57 / 66 / 89)
        int tiles = 0;
        for (int r = 0; r < a.requests; ++r) tiles = a.p[r].row_tiles > tiles ? a.p[r].row_tiles : tiles;
        int parts = tiles / 4;
        parts = parts < 1 ? 1 : parts > keyw::COL_PARTS ? keyw::COL_PARTS : parts;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)t.keys, parts);
        cfg.blockDim = dim3(keyw::COL_THREADS);
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = 1;
        attr[1].val.clusterDim.y = parts;
        attr[1].val.clusterDim.z = 1;
        cfg.attrs = pdl_enabled() ? attr : attr + 1;
        cfg.numAttrs = pdl_enabled() ? 2 : 1;
        cudaLaunchKernelEx(&cfg, keyw::key_weights_columns_kernel, a);
        return 0;
    });
    if (rc) return rc;
    LILY_CHECK_LAUNCH("attention_key_weights");
    return 0;
}
