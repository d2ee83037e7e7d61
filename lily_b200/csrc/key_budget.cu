// Holding a paged key/value cache to a budget of places: choosing the places each (layer, request, kv head) keeps by the weight that
// attention gave them, and moving what is kept to the front of the pages.
//
// Weights lie beside the keys: float32 [layers, pages, kv_heads, page_size].  Of a request's n places with n > keep, the first `first` and
// the last `recent` are kept, and of those between the (keep - first - recent) heaviest; equal weights: the lower place.  With n <= keep
// all are.  A NaN counts as heavier than everything (nobody knows what it was), -0 as 0.
#include "common.cuh"

namespace lily {
namespace budget {

// A weight as an unsigned number with the same order.
__device__ __forceinline__ uint32_t rank_of(float w) {
    if (w != w) return 0xFFFFFFFFu;
    const uint32_t b = __float_as_uint(w == 0.f ? 0.f : w);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct SelectArgs {
    const float* weights;            // [layers, pages, nkv, page_size]
    const int* block_table;          // [requests, bt_stride]
    const int* lengths;              // [requests]
    int* kept;                       // [layers, requests, nkv, keep]
    int bt_stride, requests, nkv, page_size, pages, keep, first, recent;
};

constexpr int SELECT_THREADS = 512;

// Sums two counts over the block in thread order: `before` what lies ahead of this thread; `total` of the block.
__device__ __forceinline__ void scan2(int a, int b, int& before_a, int& before_b, int& total_a, int& total_b, int2* warp_s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int ia = a, ib = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int ua = __shfl_up_sync(0xffffffffu, ia, o), ub = __shfl_up_sync(0xffffffffu, ib, o);
        if (lane >= o) ia += ua, ib += ub;
    }
    __syncthreads();
    if (lane == 31) warp_s[warp] = make_int2(ia, ib);
    __syncthreads();
    before_a = ia - a, before_b = ib - b, total_a = 0, total_b = 0;
    for (int w = 0; w < warps; ++w) {
        const int2 v = warp_s[w];
        if (w < warp) before_a += v.x, before_b += v.y;
        total_a += v.x, total_b += v.y;
    }
}

// One block a (layer, request, kv head): the rank that the last kept weight has, eight bits a pass over the row, then the kept places in order.
__global__ void __launch_bounds__(SELECT_THREADS) select_keys_kernel(const SelectArgs a) {
    __shared__ int hist[256];
    __shared__ int2 warp_s[SELECT_THREADS / 32];
    __shared__ uint32_t prefix_s;
    __shared__ int need_s;
    pdl_enter_small();
    const int tid = threadIdx.x;
    const int kvh = blockIdx.x % a.nkv, req = blockIdx.x / a.nkv % a.requests, layer = blockIdx.x / a.nkv / a.requests;
    const int n = min(max(a.lengths[req], 0), a.bt_stride * a.page_size);
    int* out = a.kept + (size_t)blockIdx.x * a.keep;
    if (n <= a.keep) {
        for (int i = tid; i < a.keep; i += SELECT_THREADS) out[i] = i < n ? i : -1;
        return;
    }
    const int* table = a.block_table + (size_t)req * a.bt_stride;
    const float* base = a.weights + (size_t)layer * a.pages * a.nkv * a.page_size;
    auto weight = [&](int j) {
        const int page = table[j / a.page_size];
        return page >= 0 && page < a.pages ? rank_of(base[((size_t)page * a.nkv + kvh) * a.page_size + j % a.page_size]) : 0u;
    };
    const int lo = a.first, hi = n - a.recent;                   // the places that compete; more than `need` of them
    int need = a.keep - a.first - a.recent;
    uint32_t prefix = 0;
    if (need > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += SELECT_THREADS) hist[i] = 0;
            __syncthreads();
            for (int j = lo + tid; j < hi; j += SELECT_THREADS) {
                const uint32_t r = weight(j);
                if (shift == 24 || r >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&hist[r >> shift & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int b = 255, above = 0;
                while (above + hist[b] < need) above += hist[b--];
                prefix_s = prefix | (uint32_t)b << shift;
                need_s = need - above;
            }
            __syncthreads();
            prefix = prefix_s;
            need = need_s;
        }
    }
    // now `prefix` is the rank of the last kept weight and `need` how many of that rank are kept, the lowest places first
    int done_kept = 0, done_ties = 0;
    const int wanted = a.keep - a.first - a.recent;
    for (int j0 = 0; j0 < n; j0 += SELECT_THREADS) {
        const int j = j0 + tid;
        int sure = 0, tie = 0;
        if (j < n) {
            if (j < lo || j >= hi) sure = 1;
            else if (wanted > 0) {
                const uint32_t r = weight(j);
                sure = r > prefix;
                tie = r == prefix;
            }
        }
        int bs, bt, ts, tt;
        scan2(sure, tie, bs, bt, ts, tt, warp_s);
        const int ties_before = done_ties + bt;
        const bool mine = sure || (tie && ties_before < need);
        const int at = done_kept + bs + min(ties_before, need);
        if (mine && at < a.keep) out[at] = j;
        done_kept += ts;
        done_ties += tt;
    }
}

struct MoveArgs {
    unsigned char* kv;               // [layers, pages, 2, nkv, page_size, row_bytes]
    float* weights;                  // [layers, pages, nkv, page_size] or null
    const int* block_table;
    const int* to_table;
    const int* kept;                 // [layers, requests, nkv, keep], ascending, -1 behind the last
    int bt_stride, to_stride, requests, nkv, page_size, pages, keep, row_bytes;
};

constexpr int MOVE_THREADS = 256;

// One block a (layer, request, kv head, keys | values | weights) goes through the kept places in order.  In place the target i is at most
// its source and the sources ascend, so nothing that a later tile reads lies where an earlier one writes, and a tile reads all it moves before it writes.
template <typename V>
__global__ void __launch_bounds__(MOVE_THREADS) move_keys_kernel(const MoveArgs a) {
    pdl_enter_small();
    const int kvh = blockIdx.x % a.nkv, req = blockIdx.x / a.nkv % a.requests, layer = blockIdx.x / a.nkv / a.requests, part = blockIdx.y;
    const int* kept = a.kept + (size_t)blockIdx.x * a.keep;
    const int* from = a.block_table + (size_t)req * a.bt_stride;
    const int* to = a.to_table + (size_t)req * a.to_stride;
    const int per = part == 2 ? 1 : a.row_bytes / (int)sizeof(V);          // pieces of a row
    const size_t heads = part == 2 ? a.nkv : 2 * a.nkv, head = part == 2 ? kvh : part * a.nkv + kvh;
    auto offset = [&](const int* table, int width, int place) -> long long {
        if (place < 0 || place / a.page_size >= width) return -1;
        const int page = table[place / a.page_size];
        if (page < 0 || page >= a.pages) return -1;
        return (long long)((((size_t)layer * a.pages + page) * heads + head) * a.page_size + place % a.page_size);
    };
    const int pieces = a.keep * per;
    for (int p0 = 0; p0 < pieces; p0 += MOVE_THREADS) {
        const int p = p0 + threadIdx.x, i = p / per, c = p % per;
        const int place = p < pieces ? kept[i] : -1;
        const long long src = offset(from, a.bt_stride, place), dst = src >= 0 ? offset(to, a.to_stride, i) : -1;
        V v;
        float w;
        if (dst >= 0) {
            if (part == 2) w = a.weights[src];
            else v = reinterpret_cast<const V*>(a.kv)[(size_t)src * per + c];
        }
        __syncthreads();
        if (dst >= 0) {
            if (part == 2) a.weights[dst] = w;
            else reinterpret_cast<V*>(a.kv)[(size_t)dst * per + c] = v;
        }
    }
}

}  // namespace budget
}  // namespace lily

using namespace lily;

LILY_API int lily_select_keys(const float* weights, const int* block_table, int bt_stride, const int* lengths, int* kept, int layers, int pages,
                              int requests, int nkv, int page_size, int keep, int first, int recent, cudaStream_t stream) {
    const long long rows = (long long)layers * requests * nkv;
    if (rows == 0 || keep == 0) return 0;
    LILY_REQUIRE(keep > 0 && first >= 0 && recent >= 0 && (long long)first + recent <= keep, "select_keys: the first %d and the last %d do not fit %d places",
                 first, recent, keep);
    LILY_REQUIRE(page_size > 0 && bt_stride > 0 && rows <= 0x7fffffff && (long long)bt_stride * page_size <= 0x7fffffff, "select_keys: %lld rows, tables of %d pages", rows, bt_stride);
    const budget::SelectArgs a{weights, block_table, lengths, kept, bt_stride, requests, nkv, page_size, pages, keep, first, recent};
    launch_pdl(budget::select_keys_kernel, dim3((unsigned)rows), dim3(budget::SELECT_THREADS), 0, stream, a);
    LILY_CHECK_LAUNCH("select_keys");
    return 0;
}

LILY_API int lily_move_keys(void* kv, float* weights, const int* block_table, int bt_stride, const int* to_table, int to_stride, const int* kept,
                            int layers, int pages, int requests, int nkv, int page_size, int row_bytes, int keep, cudaStream_t stream) {
    const long long rows = (long long)layers * requests * nkv;
    if (rows == 0 || keep == 0) return 0;
    LILY_REQUIRE(page_size > 0 && bt_stride > 0 && to_stride > 0 && rows <= 0x7fffffff && row_bytes > 0 && row_bytes % 2 == 0, "move_keys: %lld rows of %d bytes", rows, row_bytes);
    const budget::MoveArgs a{(unsigned char*)kv, weights, block_table, to_table, kept, bt_stride, to_stride, requests, nkv, page_size, pages, keep, row_bytes};
    const dim3 grid((unsigned)rows, weights ? 3 : 2);
    LILY_REQUIRE((long long)keep * row_bytes <= 0x7fffffff, "move_keys: %d places of %d bytes", keep, row_bytes);
    if (row_bytes % 16 == 0 && (uintptr_t)kv % 16 == 0) launch_pdl(budget::move_keys_kernel<uint4>, grid, dim3(budget::MOVE_THREADS), 0, stream, a);
    else if (row_bytes % 4 == 0 && (uintptr_t)kv % 4 == 0) launch_pdl(budget::move_keys_kernel<uint32_t>, grid, dim3(budget::MOVE_THREADS), 0, stream, a);
    else launch_pdl(budget::move_keys_kernel<uint16_t>, grid, dim3(budget::MOVE_THREADS), 0, stream, a);
    LILY_CHECK_LAUNCH("move_keys");
    return 0;
}
