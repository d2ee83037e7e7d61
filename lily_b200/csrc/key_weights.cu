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

namespace lily {
namespace keyw {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int TM = 64, TN = 64, KC = 32, LD = KC + 4, THREADS = 256;

struct Args {
    const void* q;                // [tokens, nq * d]
    const void* kv;               // layer base: [pages, 2, nkv, page_size, d]
    float* weights;               // [pages, nkv, page_size]
    float* scores;                // [requests, nkv, row tiles, key tiles][64][64], log2 units; -inf where a row does not see a place
    float2* parts;                // [requests, nkv, row tiles, key tiles][64] (max, sum)
    float* lse;                   // [requests, nkv, row tiles][64]
    const int* block_table;
    int bt_stride;
    const int* cu_seqlens;        // [requests + 1]
    const int* prefix_lens;       // [requests]
    int observe, from, some;      // heard tokens: the last `observe` (0: all); of those [from, from + some) in this run
    int max_total, nq, nkv, d, page_size, row_tiles, key_tiles;
    float scale;
};

struct Span { int first, rows, place0, prefix, total; };       // first token of the run (row of q), rows, the first one's place, places before and after

__device__ __forceinline__ Span span_of(const Args& a, int req) {
    const int t0 = a.cu_seqlens[req], n = a.cu_seqlens[req + 1] - t0, prefix = a.prefix_lens[req], total = min(prefix + n, a.max_total);
    const int heard = a.observe > 0 ? min(n, a.observe) : n, some = max(0, min(a.some, heard - a.from)), first = n - heard + a.from;
    return {t0 + first, some * (a.nq / a.nkv), prefix + first, prefix, total};
}

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

// grid (key tiles, row tiles, requests * kv heads): a tile of scores.  A thread has the 4 x 4 of rows ty + 16 i and keys tx + 16 j, so that the
// rows of both tiles lie in shared memory as they come (36 numbers a row of 32: no two lanes meet in a bank) and products are packed pairs along the
// head; the 32 products of a chunk are added up by themselves, which quarters the error of a long sum of like terms.  The next chunk is on its way
// while one is multiplied.  What bounds it are the multiply-adds.
template <typename T, bool VEC>
__global__ void __launch_bounds__(THREADS) key_weights_scores_kernel(const Args a) {
    __shared__ __align__(16) float q_s[TM][LD], k_s[TN][LD];
    pdl_enter_small();
    const int req = blockIdx.z / a.nkv, kvh = blockIdx.z % a.nkv, group = a.nq / a.nkv, row0 = blockIdx.y * TM, k0 = blockIdx.x * TN;
    const Span sp = span_of(a, req);
    if (row0 >= sp.rows || k0 > sp.place0 + (min(row0 + TM, sp.rows) - 1) / group) return;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int* table = a.block_table + (size_t)req * a.bt_stride;
    // a thread brings columns 4 (tid % 8) of rows tid / 8 and tid / 8 + 32 of either tile
    const T *q_row[2], *k_row[2];
    const int c4 = (tid & 7) * 4;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int r = (tid >> 3) + 32 * u, row = row0 + r, place = k0 + r;
        q_row[u] = row < sp.rows ? (const T*)a.q + ((size_t)(sp.first + row / group) * a.nq + kvh * group + row % group) * a.d : nullptr;
        k_row[u] = place < sp.total ? (const T*)a.kv + (((size_t)table[place / a.page_size] * 2 * a.nkv + kvh) * a.page_size + place % a.page_size) * a.d : nullptr;
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
    const size_t tile = ((size_t)blockIdx.z * a.row_tiles + blockIdx.y) * a.key_tiles + blockIdx.x;
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

// grid (row tiles, requests * kv heads): a row's tiles joined in their order.
__global__ void __launch_bounds__(TM) key_weights_lse_kernel(const Args a) {
    pdl_enter_small();
    const int req = blockIdx.y / a.nkv, group = a.nq / a.nkv, row = blockIdx.x * TM + threadIdx.x;
    const Span sp = span_of(a, req);
    if (blockIdx.x * TM >= sp.rows) return;
    // the tiles that were made for this tile of rows
    const int tiles = (sp.place0 + (min((int)(blockIdx.x + 1) * TM, sp.rows) - 1) / group) / TN + 1;
    const size_t tile = (size_t)blockIdx.y * a.row_tiles + blockIdx.x;
    const float2* part = a.parts + tile * a.key_tiles * TM + threadIdx.x;
    float m = -INFINITY, l = 0.f;
    for (int t = 0; t < tiles; ++t) m = fmaxf(m, part[(size_t)t * TM].x);
    for (int t = 0; t < tiles; ++t) {
        const float2 v = part[(size_t)t * TM];
        if (v.x > -INFINITY || v.y != 0.f) l = fmaf(v.y, exp2f(v.x - m), l);              // (a NaN is no maximum, but makes the sum one)
    }
    a.lse[tile * TM + threadIdx.x] = row < sp.rows ? m + log2f(l) : 0.f;
}

// grid (key tiles, requests * kv heads): the sums of a tile's columns, four a thread over every sixteenth row.
__global__ void __launch_bounds__(THREADS) key_weights_columns_kernel(const Args a) {
    __shared__ __align__(16) float sum_s[16][TN];
    pdl_enter_small();
    const int req = blockIdx.y / a.nkv, kvh = blockIdx.y % a.nkv, group = a.nq / a.nkv, k0 = blockIdx.x * TN;
    const Span sp = span_of(a, req);
    if (k0 >= sp.total) return;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    // the weights' places, asked for ahead
    float* at = nullptr;
    float sum = 0.f;
    if (tid < TN && k0 + tid < sp.total) {
        const int place = k0 + tid;
        at = a.weights + ((size_t)a.block_table[(size_t)req * a.bt_stride + place / a.page_size] * a.nkv + kvh) * a.page_size + place % a.page_size;
        sum = place < sp.prefix || a.from > 0 ? *at : 0.f;
    }
    float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
    const int first = max(0, k0 - sp.place0) * group / TM;           // the first tile of rows that sees any of these places
    for (int t = first; t * TM < sp.rows; ++t) {
        const size_t tile = (size_t)blockIdx.y * a.row_tiles + t;
        const float4* scores = reinterpret_cast<const float4*>(a.scores + (tile * a.key_tiles + blockIdx.x) * (TM * TN));
        const float* lse = a.lse + tile * TM;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 s = scores[(ty + 16 * i) * (TN / 4) + tx];
            const float e = lse[ty + 16 * i];
            w.x += exp2f(s.x - e);
            w.y += exp2f(s.y - e);
            w.z += exp2f(s.z - e);
            w.w += exp2f(s.w - e);
        }
    }
    *reinterpret_cast<float4*>(&sum_s[ty][4 * tx]) = w;
    __syncthreads();
    if (at) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += sum_s[i][tid];
        *at = sum;
    }
}

// Heard tokens of a run, so that its scores fit about a gigabyte, and the floats of scratch it takes.
struct Runs { int some, row_tiles, key_tiles; size_t tiles, floats; };
static Runs runs_of(int requests, int nq, int nkv, int max_heard, int max_total) {
    Runs r{};
    const int group = nq / nkv;
    r.key_tiles = (max_total + TN - 1) / TN;
    const size_t row_tile = (size_t)requests * nkv * r.key_tiles * TM * TN;          // floats of one tile of rows of every request and head
    const size_t most = (size_t)1 << 28;
    size_t tiles = most / (row_tile ? row_tile : 1);
    if (tiles < 1) tiles = 1;
    const size_t need = ((size_t)max_heard * group + TM - 1) / TM;
    if (tiles >= need) r.some = max_heard;
    else r.some = (int)(tiles * TM / group > 0 ? tiles * TM / group : 1);
    r.row_tiles = (int)(((size_t)r.some * group + TM - 1) / TM);
    r.tiles = (size_t)requests * nkv * r.row_tiles;
    r.floats = r.tiles * r.key_tiles * (TM * TN + 2 * TM) + r.tiles * TM;
    return r;
}

}  // namespace keyw
}  // namespace lily

using namespace lily;

// Floats of scratch: scores, the rows' parts, their lse.
LILY_API size_t lily_key_weights_floats(int requests, int nq, int nkv, int max_heard, int max_total) {
    return requests > 0 && nkv > 0 && max_heard > 0 && max_total > 0 ? keyw::runs_of(requests, nq, nkv, max_heard, max_total).floats : 0;
}

LILY_API int lily_key_weights(const void* q, const void* kv, float* weights, const int* block_table, int bt_stride, const int* cu_seqlens,
                              const int* prefix_lens, float* scratch, int requests, int observe, int max_heard, int max_total, int nq, int nkv,
                              int d, int page_size, float scale, int dtype, cudaStream_t stream) {
    if (requests == 0 || max_total == 0) return 0;
    LILY_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "attention_key_weights: %d query heads over %d kv heads", nq, nkv);
    LILY_REQUIRE(d >= 1 && page_size > 0 && observe >= 0 && max_heard >= 1, "attention_key_weights: head size %d, pages of %d, the last %d heard", d, page_size, observe);
    LILY_REQUIRE((long long)requests * nkv <= 65535, "attention_key_weights: %d requests of %d kv heads", requests, nkv);
    LILY_REQUIRE(dtype == kF32 || dtype == kBF16, "attention_key_weights: dtype %d", dtype);
    const keyw::Runs run = keyw::runs_of(requests, nq, nkv, max_heard, max_total);
    LILY_REQUIRE(run.row_tiles <= 65535, "attention_key_weights: %d tiles of rows", run.row_tiles);
    float* parts = scratch + run.tiles * run.key_tiles * (keyw::TM * keyw::TN);
    keyw::Args a{q, kv, weights, scratch, (float2*)parts, parts + run.tiles * run.key_tiles * 2 * keyw::TM, block_table, bt_stride, cu_seqlens, prefix_lens, observe, 0, run.some,
                 max_total, nq, nkv, d, page_size, run.row_tiles, run.key_tiles, scale};
    const bool vec = d % 4 == 0 && (((uintptr_t)q | (uintptr_t)kv) & 15) == 0;
    for (; a.from < max_heard; a.from += a.some) {
        const dim3 grid(run.key_tiles, run.row_tiles, requests * nkv);
#define LAUNCH(T, V) launch_pdl(keyw::key_weights_scores_kernel<T, V>, grid, dim3(keyw::THREADS), 0, stream, a)
        if (dtype == kF32) { if (vec) LAUNCH(float, true); else LAUNCH(float, false); }
        else { if (vec) LAUNCH(__nv_bfloat16, true); else LAUNCH(__nv_bfloat16, false); }
#undef LAUNCH
        launch_pdl(keyw::key_weights_lse_kernel, dim3(run.row_tiles, requests * nkv), dim3(keyw::TM), 0, stream, a);
        launch_pdl(keyw::key_weights_columns_kernel, dim3(run.key_tiles, requests * nkv), dim3(keyw::THREADS), 0, stream, a);
    }
    LILY_CHECK_LAUNCH("attention_key_weights");
    return 0;
}
