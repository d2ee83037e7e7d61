// Rotary positions with several axes (time, height, width of a token), fused with the per-head norm ahead of it and the cache write
// behind it, for caches in which a token's place is not its position.
//
// A head x of a token: y = x rsqrt(mean x^2 + eps) g (where there are gains), then for each pair j of the first rd features
//   (y_j, y_(j + rd/2)) <- (y_j c - y_(j + rd/2) s, y_(j + rd/2) c + y_j s),   c, s = tables[position of axis(j)][j],
// the rest as it is; queries go to `q_out`, keys and values to the token's place in its request's pages.  (`qk_norm_rope_write` is the
// case of one axis whose position is also the place.)  The reference's rotation is lily/layers/rotary.py:18-20, 70-87.
//
// A position outside the tables gives NaN (keys and queries that nobody can take for others); a place outside the block table, or in a
// page outside the cache, is not written.
#include "common.cuh"

namespace lily {
namespace axes {

struct Args {
    const void* qkv;                 // [splits][tokens, ld]
    size_t stride;                   // elements between the partial sums
    int splits, ld;
    const void* q_gain;
    const void* k_gain;
    float eps;
    const float* cos_t;              // [table_rows, rd / 2]
    const float* sin_t;
    int table_rows;
    const int* positions;            // [axes, tokens]
    const int* pair_axis;            // [rd / 2]
    int axes, tokens;
    const int* places;               // [tokens]
    const int* token_req;
    const int* block_table;
    int bt_stride;
    void* kv;                        // [pages, 2, nkv, page_size, d]
    int pages;
    void* q_out;                     // [tokens, nq * d]
    int nq, nkv, d, rd, page_size;
};

// Where a head of a token goes: its row of `q_out` or of a page (null: nowhere).
template <typename T>
__device__ __forceinline__ T* target(const Args& a, int n, int head) {
    if (head < a.nq) return (T*)a.q_out + ((size_t)n * a.nq + head) * a.d;
    const int place = a.places[n], at = place / a.page_size;
    if (place < 0 || at >= a.bt_stride) return nullptr;
    const int page = a.block_table[(size_t)a.token_req[n] * a.bt_stride + at];
    if (page < 0 || page >= a.pages) return nullptr;
    return (T*)a.kv + (((size_t)page * 2 * a.nkv + (head - a.nq)) * a.page_size + place % a.page_size) * a.d;
}

// A warp a head, a feature pair a lane and step: any even rotary width, any head size.
template <typename T, typename IN, typename W>
__global__ void __launch_bounds__(128) axes_rope_write_kernel(const Args a) {
    pdl_enter_small();
    const int n = blockIdx.x, head = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (head >= a.nq + 2 * a.nkv) return;
    T* dst = target<T>(a, n, head);
    if (!dst) return;
    const IN* src = (const IN*)a.qkv + (size_t)n * a.ld + (size_t)head * a.d;
    auto in = [&](int i) {
        float v = to_float(src[i]);
        for (int s = 1; s < a.splits; ++s) v += to_float(src[i + s * a.stride]);
        return v;
    };
    if (head >= a.nq + a.nkv) {
        for (int i = lane; i < a.d; i += 32) dst[i] = from_float<T>(in(i));
        return;
    }
    const W* gain = (const W*)(head < a.nq ? a.q_gain : a.k_gain);
    float inv = 1.f;
    if (gain) {
        float ssq = 0.f;
        for (int i = lane; i < a.d; i += 32) {
            const float x = in(i);
            ssq = fmaf(x, x, ssq);
        }
        inv = rsqrtf(warp_sum(ssq) / (float)a.d + a.eps);
    }
    const int half = a.rd / 2;
    for (int j = lane; j < half; j += 32) {
        float x1 = in(j), x2 = in(j + half);
        if (gain) {
            x1 = x1 * inv * to_float(gain[j]);
            x2 = x2 * inv * to_float(gain[j + half]);
        }
        const int axis = a.pair_axis[j];
        const int pos = axis >= 0 && axis < a.axes ? a.positions[(size_t)axis * a.tokens + n] : -1;
        const bool known = pos >= 0 && pos < a.table_rows;
        const float c = known ? a.cos_t[(size_t)pos * half + j] : __int_as_float(0x7fffffff), s = known ? a.sin_t[(size_t)pos * half + j] : c;
        dst[j] = from_float<T>(x1 * c - x2 * s);
        dst[j + half] = from_float<T>(x2 * c + x1 * s);
    }
    for (int i = a.rd + lane; i < a.d; i += 32) dst[i] = from_float<T>(gain ? in(i) * inv * to_float(gain[i]) : in(i));
}

}  // namespace axes
}  // namespace lily

using namespace lily;

LILY_API int lily_axes_rope_write(const void* qkv, int in_dtype, int splits, size_t stride, int ld, const void* q_gain, const void* k_gain,
                                  int gain_dtype, float eps, const float* cos_t, const float* sin_t, int table_rows,
                                  const int* positions, const int* pair_axis, int axes, int tokens, const int* places,
                                  const int* token_req, const int* block_table, int bt_stride, void* kv, int pages, void* q_out,
                                  int act_dtype, int nq, int nkv, int d, int rd, int page_size, cudaStream_t stream) {
    if (tokens == 0) return 0;
    LILY_REQUIRE(d > 0 && rd >= 0 && rd <= d && rd % 2 == 0, "axes_rope_write: rotary_dim %d does not fit head_dim %d", rd, d);
    LILY_REQUIRE(nq >= 0 && nkv >= 0 && nq + nkv > 0 && ld >= (nq + 2 * nkv) * d, "axes_rope_write: rows of %d numbers", ld);
    LILY_REQUIRE((q_gain == nullptr) == (k_gain == nullptr), "axes_rope_write: q and k gains come together");
    LILY_REQUIRE(act_dtype == kF32 || act_dtype == kBF16, "axes_rope_write: dtype %d", act_dtype);
    LILY_REQUIRE(in_dtype == act_dtype || in_dtype == kF32, "axes_rope_write: products are of the cache's dtype or float32");
    LILY_REQUIRE(act_dtype == kBF16 || gain_dtype == kF32 || q_gain == nullptr, "axes_rope_write: float32 heads keep float32 gains");
    LILY_REQUIRE(splits >= 1 && (splits == 1 || in_dtype == kF32), "axes_rope_write: partial sums are float32");
    const axes::Args a{qkv, stride, splits, ld, q_gain, k_gain, eps, cos_t, sin_t, table_rows, positions, pair_axis, axes, tokens, places, token_req,
                       block_table, bt_stride, kv, pages, q_out, nq, nkv, d, rd, page_size};
    const dim3 grid(tokens, (nq + 2 * nkv + 3) / 4);
#define LAUNCH(T, IN, W) launch_pdl(axes::axes_rope_write_kernel<T, IN, W>, grid, dim3(128), 0, stream, a)
    const bool ib = in_dtype == kBF16, gb = gain_dtype == kBF16;
    if (act_dtype == kF32) LAUNCH(float, float, float);
    else if (ib && gb) LAUNCH(__nv_bfloat16, __nv_bfloat16, __nv_bfloat16);
    else if (ib) LAUNCH(__nv_bfloat16, __nv_bfloat16, float);
    else if (gb) LAUNCH(__nv_bfloat16, float, __nv_bfloat16);
    else LAUNCH(__nv_bfloat16, float, float);
#undef LAUNCH
    LILY_CHECK_LAUNCH("axes_rope_write");
    return 0;
}
