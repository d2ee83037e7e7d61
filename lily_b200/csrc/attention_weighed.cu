// Decode attention over the paged cache that also adds up the weight each cached key is given.
//
// For a request of n cached places (the newest token's own among them) and the query heads h of a kv head g:
//   p_hj = exp(c q_h . k_j - lse_h),  o_h = sum_j p_hj v_j,  w_gj <- (j < n - 1 ? w_gj : 0) + sum_h p_hj,
// with w float32 [pages, kv_heads, page_size] beside the keys: the newest place's weight is set, whatever an earlier owner left there.
// The keys of a request are cut into ranges; a block leaves its scores (in units of log2 e) and its (max, sum, output) in scratch, and a
// second kernel, which knows every range's, writes outputs and weights.
#include "common.cuh"

namespace lily {
namespace weighed {

constexpr float LOG2E = 1.4426950408889634f;

struct DecodeArgs {
    const void* q;                // [requests, nq * d]
    const void* kv;               // layer base: [pages, 2, nkv, page_size, d]
    float* weights;               // [pages, nkv, page_size]
    void* out;                    // [requests, nq * d]
    const int* block_table;       // [requests, bt_stride]
    int bt_stride;
    const int* seq_lens;          // [requests] cached places, this step's among them
    float* scores;                // [requests, nq, score_stride], in units of log2 e
    float* part_o;                // [requests, nq, splits, d]
    float* part_ml;               // [requests, nq, splits, 2]
    int splits, nq, nkv, d, page_size, score_stride;
    float scale;
};

// The places of range `z` of a request: equal shares in steps of 64.
__device__ __forceinline__ void key_range(const DecodeArgs& a, int req, int z, int& beg, int& end) {
    const int n = min(max(a.seq_lens[req], 0), a.score_stride);
    const int per = ((n + a.splits - 1) / a.splits + 63) / 64 * 64;
    beg = min(n, z * per);
    end = min(n, beg + per);
}

// ---- any head size, float32 or bfloat16, on the CUDA cores -----------------------------------------
constexpr int KT = 32;                     // keys a tile
constexpr int RH = 16;                     // query heads a block
constexpr int SIMT_THREADS = 128;

__host__ __device__ inline size_t simt_floats(int d) { return (size_t)2 * KT * (d + 1) + 2 * (size_t)RH * d + RH * KT + 3 * RH; }

template <typename T>
__global__ void __launch_bounds__(SIMT_THREADS) decode_weighed_simt_kernel(const DecodeArgs a) {
    extern __shared__ float sm[];
    const int d = a.d, ld = d + 1;
    float* k_s = sm;                           // [KT][d + 1]
    float* v_s = k_s + KT * ld;
    float* q_s = v_s + KT * ld;                // [RH][d]
    float* o_s = q_s + RH * d;
    float* p_s = o_s + RH * d;                 // [RH][KT]
    float* m_s = p_s + RH * KT;                // [RH] max, sum, factor of this tile
    float* l_s = m_s + RH;
    float* f_s = l_s + RH;
    pdl_enter_small();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = a.nq / a.nkv, chunks = (group + RH - 1) / RH;
    const int req = blockIdx.x, kvh = blockIdx.y / chunks, r0 = blockIdx.y % chunks * RH, rows = min(RH, group - r0), head0 = kvh * group + r0;
    int beg, end;
    key_range(a, req, blockIdx.z, beg, end);
    const T* q = (const T*)a.q + ((size_t)req * a.nq + head0) * d;
    for (int i = tid; i < rows * d; i += SIMT_THREADS) q_s[i] = to_float(q[i]) * (a.scale * LOG2E), o_s[i] = 0.f;
    if (tid < rows) m_s[tid] = -INFINITY, l_s[tid] = 0.f;
    const int* table = a.block_table + (size_t)req * a.bt_stride;
    const size_t head_stride = (size_t)a.page_size * d;
    for (int k0 = beg; k0 < end; k0 += KT) {
        const int n = min(KT, end - k0);
        __syncthreads();
        for (int i = tid; i < n * d; i += SIMT_THREADS) {
            const int r = i / d, col = i % d, place = k0 + r;
            const T* page = (const T*)a.kv + ((size_t)table[place / a.page_size] * 2 * a.nkv + kvh) * head_stride + (size_t)(place % a.page_size) * d + col;
            k_s[r * ld + col] = to_float(page[0]);
            v_s[r * ld + col] = to_float(page[a.nkv * head_stride]);
        }
        __syncthreads();
        for (int h = warp; h < rows; h += SIMT_THREADS / 32) {
            float s = 0.f;
            if (lane < n)
                for (int i = 0; i < d; ++i) s = fmaf(q_s[h * d + i], k_s[lane * ld + i], s);
            if (lane < n) a.scores[((size_t)req * a.nq + head0 + h) * a.score_stride + k0 + lane] = s;
            const float was = m_s[h], now = fmaxf(was, warp_max(lane < n ? s : -INFINITY));
            const float base = now == -INFINITY ? 0.f : now;
            const float p = lane < n ? exp2f(s - base) : 0.f, f = exp2f(was - base);
            const float sum = warp_sum(p);
            p_s[h * KT + lane] = p;
            __syncwarp();
            if (lane == 0) m_s[h] = now, l_s[h] = l_s[h] * f + sum, f_s[h] = f;
        }
        __syncthreads();
        for (int i = tid; i < rows * d; i += SIMT_THREADS) {
            const int h = i / d, col = i % d;
            float o = o_s[i] * f_s[h];
            for (int r = 0; r < n; ++r) o = fmaf(p_s[h * KT + r], v_s[r * ld + col], o);
            o_s[i] = o;
        }
    }
    __syncthreads();
    for (int i = tid; i < rows * d; i += SIMT_THREADS) {
        const size_t at = ((size_t)req * a.nq + head0 + i / d) * a.splits + blockIdx.z;
        a.part_o[at * d + i % d] = o_s[i];
        if (i % d == 0) a.part_ml[at * 2] = m_s[i / d], a.part_ml[at * 2 + 1] = l_s[i / d];
    }
}

// ---- the ranges joined: outputs, then the places' weights ------------------------------------------
constexpr int JOIN_THREADS = 256;
constexpr int JOIN_KEYS = 1024;            // places a block adds up

template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS) decode_weighed_join_kernel(const DecodeArgs a) {
    extern __shared__ float sm[];              // [group] lse (log2 units)
    pdl_enter_small();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = a.nq / a.nkv, req = blockIdx.x, kvh = blockIdx.y, d = a.d;
    const int n = a.seq_lens[req], beg = ((int)blockIdx.z - 1) * JOIN_KEYS;
    if (blockIdx.z > 0 && beg >= n) return;
    for (int h = warp; h < group; h += JOIN_THREADS / 32) {
        const float* ml = a.part_ml + ((size_t)req * a.nq + kvh * group + h) * a.splits * 2;
        float m = -INFINITY, l = 0.f;
        for (int s = lane; s < a.splits; s += 32) m = fmaxf(m, ml[2 * s]);
        m = warp_max(m);
        for (int s = lane; s < a.splits; s += 32) l += ml[2 * s + 1] * exp2f(ml[2 * s] - (m == -INFINITY ? 0.f : m));
        l = warp_sum(l);
        if (lane == 0) sm[h] = m + log2f(l);
    }
    __syncthreads();
    if (blockIdx.z == 0) {
        for (int i = tid; i < group * d; i += JOIN_THREADS) {
            const int h = i / d, col = i % d;
            const size_t at = ((size_t)req * a.nq + kvh * group + h) * a.splits;
            float o = 0.f;
            if (n > 0)
                for (int s = 0; s < a.splits; ++s) {
                    const float m = a.part_ml[(at + s) * 2];
                    if (m == -INFINITY && a.part_ml[(at + s) * 2 + 1] == 0.f) continue;          // a range without keys
                    o = fmaf(a.part_o[(at + s) * d + col], exp2f(m - sm[h]), o);
                }
            ((T*)a.out)[((size_t)req * a.nq + kvh * group + h) * d + col] = from_float<T>(o);
        }
        return;
    }
    const int* table = a.block_table + (size_t)req * a.bt_stride;
    const float* scores = a.scores + ((size_t)req * a.nq + kvh * group) * a.score_stride;
    for (int j = beg + tid; j < min(n, beg + JOIN_KEYS); j += JOIN_THREADS) {
        float* w = a.weights + ((size_t)table[j / a.page_size] * a.nkv + kvh) * a.page_size + j % a.page_size;
        float sum = j < n - 1 ? *w : 0.f;
        for (int h = 0; h < group; ++h) sum += exp2f(scores[(size_t)h * a.score_stride + j] - sm[h]);
        *w = sum;
    }
}

}  // namespace weighed
}  // namespace lily

using namespace lily;

// Floats of scratch: scores, partial outputs, partial (max, sum).
LILY_API size_t lily_attention_decode_weighed_floats(int requests, int nq, int d, int splits, int score_stride) {
    return (size_t)requests * nq * ((size_t)score_stride + (size_t)splits * (d + 2));
}

LILY_API int lily_attention_decode_weighed(const void* q, const void* kv, float* weights, void* out, const int* block_table, int bt_stride,
                                           const int* seq_lens, float* scratch, int requests, int splits, int max_len, int nq, int nkv, int d,
                                           int page_size, float scale, int dtype, cudaStream_t stream) {
    if (requests == 0) return 0;
    LILY_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "attention_decode_weighed: %d query heads over %d kv heads", nq, nkv);
    LILY_REQUIRE(d >= 1 && d <= 256 && page_size > 0 && splits >= 1 && max_len >= 0, "attention_decode_weighed: head size %d (takes up to 256), pages of %d", d, page_size);
    LILY_REQUIRE(dtype == kF32 || dtype == kBF16, "attention_decode_weighed: dtype %d", dtype);
    const int score_stride = (max_len + 3) / 4 * 4, group = nq / nkv;
    weighed::DecodeArgs a{};
    a.q = q; a.kv = kv; a.weights = weights; a.out = out; a.block_table = block_table; a.bt_stride = bt_stride; a.seq_lens = seq_lens;
    a.splits = splits; a.nq = nq; a.nkv = nkv; a.d = d; a.page_size = page_size; a.scale = scale; a.score_stride = score_stride;
    a.scores = scratch;
    a.part_o = a.scores + (size_t)requests * nq * score_stride;
    a.part_ml = a.part_o + (size_t)requests * nq * splits * d;
    const dim3 grid(requests, nkv * ((group + weighed::RH - 1) / weighed::RH), splits);
    const size_t smem = weighed::simt_floats(d) * sizeof(float);
    static bool configured = false;
    if (!configured) {
        const int most = (int)(weighed::simt_floats(256) * sizeof(float));
        cudaError_t e = cudaFuncSetAttribute(weighed::decode_weighed_simt_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(weighed::decode_weighed_simt_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        LILY_REQUIRE(e == cudaSuccess, "attention_decode_weighed: cannot get %d bytes of shared memory: %s", most, cudaGetErrorString(e));
        configured = true;
    }
    const dim3 join(requests, nkv, 1 + (max_len + weighed::JOIN_KEYS - 1) / weighed::JOIN_KEYS);
    if (dtype == kF32) {
        launch_pdl(weighed::decode_weighed_simt_kernel<float>, grid, dim3(weighed::SIMT_THREADS), smem, stream, a);
        launch_pdl(weighed::decode_weighed_join_kernel<float>, join, dim3(weighed::JOIN_THREADS), group * sizeof(float), stream, a);
    } else {
        launch_pdl(weighed::decode_weighed_simt_kernel<__nv_bfloat16>, grid, dim3(weighed::SIMT_THREADS), smem, stream, a);
        launch_pdl(weighed::decode_weighed_join_kernel<__nv_bfloat16>, join, dim3(weighed::JOIN_THREADS), group * sizeof(float), stream, a);
    }
    LILY_CHECK_LAUNCH("attention_decode_weighed");
    return 0;
}
