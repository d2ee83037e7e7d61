// What the tokens of a prompt's portion give to every cached key: the column sums of the softmax.
//
// Token t of the n new ones of a request behind p cached places sees the places j <= p + t.  The last `heard` tokens are heard:
//   P_thj = exp(c q_th . k_j - lse_th),  w_gj <- (j < p ? w_gj : 0) + sum over heard t and the heads h of g of P_thj,
// with w float32 [pages, kv_heads, page_size] beside the keys; the weights of the portion's own places are set.
// The sum over rows needs every row's lse first, so there are two kernels: rows (running max and sum over key tiles), then columns.
#include "common.cuh"

namespace lily {
namespace keyw {

constexpr float LOG2E = 1.4426950408889634f;

struct Args {
    const void* q;                // [tokens, nq * d]
    const void* kv;               // layer base: [pages, 2, nkv, page_size, d]
    float* weights;               // [pages, nkv, page_size]
    float* lse;                   // [requests, nq, max_heard], log2 units
    const int* block_table;
    int bt_stride;
    const int* cu_seqlens;        // [requests + 1]
    const int* prefix_lens;       // [requests]
    int observe, max_heard, max_total, nq, nkv, d, page_size;
    float scale;
};

struct Span { int first, heard, prefix, total; };       // first heard token (row of q), heard tokens, cached places before and after

__device__ __forceinline__ Span span_of(const Args& a, int req) {
    const int t0 = a.cu_seqlens[req], n = a.cu_seqlens[req + 1] - t0, prefix = a.prefix_lens[req];
    const int heard = min(a.observe > 0 ? min(n, a.observe) : n, a.max_heard);
    return {t0 + n - heard, heard, prefix, min(prefix + n, a.max_total)};
}

// ---- any head size, float32 or bfloat16, on the CUDA cores: tiles of 64 rows x 64 keys, 4 x 4 a thread -----------
constexpr int TM = 64, TN = 64, KC = 32, THREADS = 256;

// s[i][j] = q(row0 + 4 ty + i) . k(place0 + 4 tx + j) of head `head`; rows and places beyond the ends count as zeros.  The KC products of a
// chunk are added up by themselves first: the error of a long sum of like terms is then a quarter of one added up in a row.
template <typename T>
__device__ __forceinline__ void scores(const Args& a, const Span& sp, int req, int head, int kvh, int row0, int place0,
                                       float (*q_s)[TM + 4], float (*k_s)[TN + 4], float (&s)[4][4]) {
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int* table = a.block_table + (size_t)req * a.bt_stride;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
    for (int c0 = 0; c0 < a.d; c0 += KC) {
        __syncthreads();
        for (int i = tid; i < TM * KC; i += THREADS) {
            const int r = i / KC, c = i % KC, row = row0 + r, place = place0 + r;
            float qv = 0.f, kv = 0.f;
            if (c0 + c < a.d) {
                if (row < sp.heard) qv = to_float(((const T*)a.q)[((size_t)(sp.first + row) * a.nq + head) * a.d + c0 + c]);
                if (place < sp.total)
                    kv = to_float(((const T*)a.kv)[(((size_t)table[place / a.page_size] * 2 * a.nkv + kvh) * a.page_size + place % a.page_size) * a.d + c0 + c]);
            }
            q_s[c][r] = qv;
            k_s[c][r] = kv;
        }
        __syncthreads();
        float part[4][4] = {};
#pragma unroll 8
        for (int c = 0; c < KC; ++c) {
            const float4 qv = *reinterpret_cast<const float4*>(&q_s[c][4 * ty]), kv = *reinterpret_cast<const float4*>(&k_s[c][4 * tx]);
            const float x[4] = {qv.x, qv.y, qv.z, qv.w}, y[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) part[i][j] = fmaf(x[i], y[j], part[i][j]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) s[i][j] += part[i][j];
    }
}

// grid (tiles of heard rows, heads, requests)
template <typename T>
__global__ void __launch_bounds__(THREADS) key_weights_rows_kernel(const Args a) {
    __shared__ __align__(16) float q_s[KC][TM + 4], k_s[KC][TN + 4];
    pdl_enter_small();
    const int req = blockIdx.z, head = blockIdx.y, kvh = head / (a.nq / a.nkv), row0 = blockIdx.x * TM;
    const Span sp = span_of(a, req);
    if (row0 >= sp.heard) return;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int place0 = sp.total - sp.heard;                          // the place of heard row 0
    const float c = a.scale * LOG2E;
    float m[4], l[4], s[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = -INFINITY, l[i] = 0.f;
    const int end = min(sp.total, place0 + row0 + TM);
    for (int k0 = 0; k0 < end; k0 += TN) {
        scores<T>(a, sp, req, head, kvh, row0, k0, q_s, k_s, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int last = place0 + row0 + 4 * ty + i;              // the last place this row sees
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[i][j] = k0 + 4 * tx + j <= last ? s[i][j] * c : -INFINITY;
                mx = fmaxf(mx, s[i][j]);
            }
#pragma unroll
            for (int o = 1; o < 16; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float now = fmaxf(m[i], mx), base = now == -INFINITY ? 0.f : now;
            l[i] *= exp2f(m[i] - base);
            m[i] = now;
#pragma unroll
            for (int j = 0; j < 4; ++j) l[i] += exp2f(s[i][j] - base);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float sum = l[i];
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const int row = row0 + 4 * ty + i;
        if (tx == 0 && row < sp.heard) a.lse[((size_t)req * a.nq + head) * a.max_heard + row] = m[i] + log2f(sum);
    }
}

// grid (tiles of places, kv heads, requests)
template <typename T>
__global__ void __launch_bounds__(THREADS) key_weights_columns_kernel(const Args a) {
    __shared__ __align__(16) float q_s[KC][TM + 4], k_s[KC][TN + 4];
    __shared__ float sum_s[16][TN];
    pdl_enter_small();
    const int req = blockIdx.z, kvh = blockIdx.y, group = a.nq / a.nkv, k0 = blockIdx.x * TN;
    const Span sp = span_of(a, req);
    if (k0 >= sp.total) return;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int place0 = sp.total - sp.heard;
    const float c = a.scale * LOG2E;
    float w[4] = {0.f, 0.f, 0.f, 0.f}, s[4][4];
    const int first = max(0, k0 - place0) / TM * TM;                 // the first tile of rows that sees any of these places
    for (int h = 0; h < group; ++h) {
        const int head = kvh * group + h;
        const float* lse = a.lse + ((size_t)req * a.nq + head) * a.max_heard;
        for (int row0 = first; row0 < sp.heard; row0 += TM) {
            scores<T>(a, sp, req, head, kvh, row0, k0, q_s, k_s, s);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = row0 + 4 * ty + i;
                if (row >= sp.heard) continue;
                const float e = lse[row];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (k0 + 4 * tx + j <= place0 + row) w[j] += exp2f(fmaf(s[i][j], c, -e));
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) sum_s[ty][4 * tx + j] = w[j];
    __syncthreads();
    if (tid < TN && k0 + tid < sp.total) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sum += sum_s[i][tid];
        const int place = k0 + tid;
        float* to = a.weights + ((size_t)a.block_table[(size_t)req * a.bt_stride + place / a.page_size] * a.nkv + kvh) * a.page_size + place % a.page_size;
        *to = (place < sp.prefix ? *to : 0.f) + sum;
    }
}

}  // namespace keyw
}  // namespace lily

using namespace lily;

// Floats of scratch: one lse a heard row and head.
LILY_API size_t lily_key_weights_floats(int requests, int nq, int max_heard) { return (size_t)requests * nq * max_heard; }

LILY_API int lily_key_weights(const void* q, const void* kv, float* weights, const int* block_table, int bt_stride, const int* cu_seqlens,
                              const int* prefix_lens, float* scratch, int requests, int observe, int max_heard, int max_total, int nq, int nkv,
                              int d, int page_size, float scale, int dtype, cudaStream_t stream) {
    if (requests == 0 || max_total == 0) return 0;
    LILY_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "attention_key_weights: %d query heads over %d kv heads", nq, nkv);
    LILY_REQUIRE(d >= 1 && page_size > 0 && observe >= 0 && max_heard >= 1, "attention_key_weights: head size %d, pages of %d, the last %d heard", d, page_size, observe);
    LILY_REQUIRE(requests <= 65535 && nq <= 65535, "attention_key_weights: %d requests, %d heads", requests, nq);
    LILY_REQUIRE(dtype == kF32 || dtype == kBF16, "attention_key_weights: dtype %d", dtype);
    const keyw::Args a{q, kv, weights, scratch, block_table, bt_stride, cu_seqlens, prefix_lens, observe, max_heard, max_total, nq, nkv, d, page_size, scale};
    const dim3 rows((max_heard + keyw::TM - 1) / keyw::TM, nq, requests), columns((max_total + keyw::TN - 1) / keyw::TN, nkv, requests);
    if (dtype == kF32) {
        launch_pdl(keyw::key_weights_rows_kernel<float>, rows, dim3(keyw::THREADS), 0, stream, a);
        launch_pdl(keyw::key_weights_columns_kernel<float>, columns, dim3(keyw::THREADS), 0, stream, a);
    } else {
        launch_pdl(keyw::key_weights_rows_kernel<__nv_bfloat16>, rows, dim3(keyw::THREADS), 0, stream, a);
        launch_pdl(keyw::key_weights_columns_kernel<__nv_bfloat16>, columns, dim3(keyw::THREADS), 0, stream, a);
    }
    LILY_CHECK_LAUNCH("attention_key_weights");
    return 0;
}
