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
    int bt_stride, requests, nkv, page_size, page_shift, pages, max_length, keep, first, recent;
};

constexpr int SELECT_MOST = 1024;          // threads of a block at most
constexpr int SELECT_HELD = 48 * 1024;     // places whose ranks a block holds in shared memory; of longer rows they are worked out again a pass

// One block a (layer, request, kv head); a warp has a stretch of the row.  The weights are read once, as ranks that a thread keeps in REGS registers
// (0: rows of more than eight places a thread, in shared memory), and are asked for before the row's length has arrived.  The rank that the last kept weight has comes
// out eight bits a pass (a histogram of the competing ranks that share the bits found so far, in shared memory; lanes that meet in a counter are added
// up by the hardware), until a bin has no more than 32, which every warp then ranks by itself.  Then every warp counts what it
// keeps of its stretch and writes it behind what the warps ahead keep.  What bounds it is the chain of reads and passes, not the bytes: 6.2 us for 64 rows of 4,096,
// 10.4 for 384 of up to 3,500 (12.9 with 48 registers, where an SM holds two of these blocks).
template <int REGS>
__global__ void __maxnreg__(40) select_keys_kernel(const SelectArgs a) {
    constexpr int P = REGS ? REGS : 4;
    extern __shared__ uint32_t rank_s[];                             // [min(max_length, SELECT_HELD)] without registers
    __shared__ __align__(16) int hists[4][256];
    __shared__ int2 warp_s[32];
    __shared__ uint32_t prefix_s, few_s[32];
    __shared__ int need_s, bin_s, few;
    pdl_enter_small();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, threads = blockDim.x, warps = threads >> 5;
    const int kvh = blockIdx.x % a.nkv, req = blockIdx.x / a.nkv % a.requests, layer = blockIdx.x / a.nkv / a.requests;
    const int* table = a.block_table + (size_t)req * a.bt_stride;
    const float* base = a.weights + ((size_t)layer * a.pages * a.nkv + kvh) * a.page_size;
    const size_t page_stride = (size_t)a.nkv * a.page_size;
    const int length = a.lengths[req];
    float w[P];
    uint32_t mine[P];
    auto ask = [&](int j0, int step) {                               // the weights of P places; one without a page counts as the lightest
        int page[P];
#pragma unroll
        for (int u = 0; u < P; ++u) page[u] = j0 + u * step < a.max_length ? table[(j0 + u * step) >> a.page_shift] : -1;
#pragma unroll
        for (int u = 0; u < P; ++u)
            w[u] = page[u] >= 0 && page[u] < a.pages ? base[page[u] * page_stride + ((j0 + u * step) & (a.page_size - 1))] : -INFINITY;
    };
    if (REGS) ask(warp * (32 * P) + lane, 32);
    for (int i = tid; i < 1024; i += threads) hists[0][i] = 0;
    if (tid == 0) few = 0;
    const int n = min(max(length, 0), a.max_length);
    int* out = a.kept + (size_t)blockIdx.x * a.keep;
    if (n <= a.keep) {
        for (int i = tid; i < a.keep; i += threads) out[i] = i < n ? i : -1;
        return;
    }
    const int wanted = a.keep - a.first - a.recent, lo = a.first, hi = n - a.recent;      // more than `wanted` places compete, [lo, hi)
    const bool held = REGS || n <= SELECT_HELD;
    const int per = REGS ? 32 * P : (n + threads - 1) / threads * 32, beg = warp * per, end = min(n, beg + per);      // this warp's stretch
    if (REGS) {
#pragma unroll
        for (int u = 0; u < P; ++u)
            if (beg + 32 * u < end) mine[u] = rank_of(w[u]);
    } else if (held) {
        for (int j0 = beg + lane; j0 < end; j0 += 32 * P) {
            ask(j0, 32);
#pragma unroll
            for (int u = 0; u < P; ++u)
                if (j0 + 32 * u < end) rank_s[j0 + 32 * u] = rank_of(w[u]);
        }
        __syncwarp();
    }
    // f(place, rank) for this thread's places that compete
    auto each = [&](auto f) {
        if (REGS) {
#pragma unroll
            for (int u = 0; u < P; ++u) {
                const int j = beg + 32 * u + lane;
                if (beg + 32 * u < end && j >= lo && j < hi) f(mine[u]);
            }
        } else
            for (int j = beg + lane; j < end; j += 32) {
                if (j < lo || j >= hi) continue;
                if (held) f(rank_s[j]);
                else {
                    const int page = table[j >> a.page_shift];
                    f(page >= 0 && page < a.pages ? rank_of(base[page * page_stride + (j & (a.page_size - 1))]) : rank_of(-INFINITY));
                }
            }
    };
    uint32_t prefix = 0;
    int need = wanted;
    __syncthreads();
    if (wanted > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            int* hist = hists[shift >> 3];
            each([&](uint32_t r) {
                if (shift == 24 || r >> ((shift + 8) & 31) == prefix >> ((shift + 8) & 31)) atomicAdd(&hist[r >> shift & 255u], 1);
            });
            __syncthreads();
            if (warp == 0) {
                // eight bins a lane, the highest with the first: the bin in which the count from above reaches what is needed
                const int top = 248 - 8 * lane;
                const int4 u = *reinterpret_cast<const int4*>(hist + top + 4), v = *reinterpret_cast<const int4*>(hist + top);
                const int c[8] = {u.w, u.z, u.y, u.x, v.w, v.z, v.y, v.x};
                int sum = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += c[i];
                int upto = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int t = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += t;
                }
                int above = upto - sum;
                if (above < need && need <= upto) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (above < need && need <= above + c[i]) {
                            // all of a bin: whatever its ranks are beyond these bits, they are above the bin below it
                            const bool whole = need == above + c[i];
                            prefix_s = (prefix | (uint32_t)(top + 7 - i) << shift) - (whole ? 1u : 0u);
                            need_s = whole ? 0 : need - above;
                            bin_s = c[i];
                            break;
                        }
                        above += c[i];
                    }
                }
            }
            __syncthreads();
            prefix = prefix_s;
            need = need_s;
            const int rest = bin_s;
            if (need == 0) break;
            if (shift > 0 && rest <= 32) {
                each([&](uint32_t r) {
                    if (r >> shift == prefix >> shift) few_s[atomicAdd(&few, 1)] = r;
                });
                __syncthreads();
                // the one of these with fewer than `need` above it and `need` or more up to it
                const uint32_t r = few_s[lane];
                int above = 0, upto = 0;
                for (int i = 0; i < rest; ++i) {
                    const uint32_t other = few_s[i];
                    above += other > r;
                    upto += other >= r;
                }
                const uint32_t last = __ballot_sync(0xffffffffu, lane < rest && above < need && need <= upto);
                prefix = __shfl_sync(0xffffffffu, r, __ffs(last) - 1);
                need -= __shfl_sync(0xffffffffu, above, __ffs(last) - 1);
                break;
            }
        }
    }
    // now `prefix` is the rank of the last kept weight and `need` how many of that rank are kept, the lowest places first (none: what is above it is kept)
    auto kinds = [&](int j0, uint32_t r, uint32_t& sure, uint32_t& tie) {
        const int j = j0 + lane;
        const bool in = j < end, fixed = j < lo || j >= hi;
        sure = __ballot_sync(0xffffffffu, in && (fixed || (wanted > 0 && r > prefix)));
        tie = __ballot_sync(0xffffffffu, in && !fixed && wanted > 0 && r == prefix);
    };
    auto rank = [&](int j) {
        if (j >= end) return 0u;
        if (held) return rank_s[j];
        const int page = table[j >> a.page_shift];
        return page >= 0 && page < a.pages ? rank_of(base[page * page_stride + (j & (a.page_size - 1))]) : rank_of(-INFINITY);
    };
    int sures = 0, ties = 0;
    uint32_t sure[P], tie[P];
    if (REGS) {
#pragma unroll
        for (int u = 0; u < P; ++u) {
            if (beg + 32 * u >= end) break;
            kinds(beg + 32 * u, mine[u], sure[u], tie[u]);
            sures += __popc(sure[u]);
            ties += __popc(tie[u]);
        }
    } else
        for (int j0 = beg; j0 < end; j0 += 32) {
            kinds(j0, rank(j0 + lane), sure[0], tie[0]);
            sures += __popc(sure[0]);
            ties += __popc(tie[0]);
        }
    if (lane == 0) warp_s[warp] = make_int2(sures, ties);
    __syncthreads();
    const int2 before = lane < warps && lane < warp ? warp_s[lane] : make_int2(0, 0);
    int at_sure = __reduce_add_sync(0xffffffffu, before.x), at_tie = __reduce_add_sync(0xffffffffu, before.y);
    const uint32_t ahead = (1u << lane) - 1u;
    auto put = [&](int j0, uint32_t s, uint32_t t) {
        const int tb = at_tie + __popc(t & ahead);
        const bool kept = (s >> lane & 1u) || ((t >> lane & 1u) && tb < need);
        const int at = at_sure + __popc(s & ahead) + min(tb, need);
        if (kept && at < a.keep) out[at] = j0 + lane;
        at_sure += __popc(s);
        at_tie += __popc(t);
    };
    if (REGS) {
#pragma unroll
        for (int u = 0; u < P; ++u) {
            if (beg + 32 * u >= end) break;
            put(beg + 32 * u, sure[u], tie[u]);
        }
    } else
        for (int j0 = beg; j0 < end; j0 += 32) {
            kinds(j0, rank(j0 + lane), sure[0], tie[0]);
            put(j0, sure[0], tie[0]);
        }
}

struct MoveArgs {
    unsigned char* kv;               // [layers, pages, 2, nkv, page_size, row_bytes]
    float* weights;                  // [layers, pages, nkv, page_size] or null
    const int* block_table;
    const int* to_table;
    const int* kept;                 // [layers, requests, nkv, keep], ascending, -1 behind the last
    int bt_stride, to_stride, requests, nkv, page_size, page_shift, pages, keep, row_bytes;
    int block_rows;                  // rows a block moves at a time
};

constexpr int MOVE_THREADS = 256, MOVE_AHEAD = 8;        // pieces a thread has on their way
constexpr int MOVE_CLUSTER = 8, MOVE_ROWS = 128;         // rows a block moves at most

// A block moves the keys, values and weights of some rows of one (layer, request, kv head): the rows' places and pages are looked up once, by a
// thread a row, then every thread has eight pieces on their way.  Into other pages every block works for itself.  In place (IN_PLACE) the
// eight blocks of a cluster go through the list together, a round of eight blocks' rows at a time: all read before any writes, for which the cluster's barrier
// is enough, since the target i is at most its source and the sources ascend, so nothing that a later round reads lies where an earlier
// one writes.  What bounds it are the bytes where there are enough (384 lists of 512 rows of 2 x 256 bytes: 34.4 us, 5.9 TB/s; in place 37), else the chain place, page, row (64
// lists of 1,024: 13.7; in place 15.8).
template <typename V, bool IN_PLACE>
__global__ void __launch_bounds__(MOVE_THREADS) move_keys_kernel(const MoveArgs a) {
    __shared__ long long src_s[MOVE_ROWS], dst_s[MOVE_ROWS];         // rows of the cache; -1: not moved
    // (no launch_dependents: the kernel behind may read keys ahead of its wait)
    pdl_wait();
    const int tid = threadIdx.x, list = blockIdx.y;
    const int kvh = list % a.nkv, req = list / a.nkv % a.requests, layer = list / a.nkv / a.requests;
    const int* kept = a.kept + (size_t)list * a.keep;
    const int* from = a.block_table + (size_t)req * a.bt_stride;
    const int* to = a.to_table + (size_t)req * a.to_stride;
    const int per = a.row_bytes / (int)sizeof(V), both = 2 * per;          // pieces of a key, of key and value
    const long long to_value = (long long)a.nkv * a.page_size;             // rows from a key to its value
    const int rounds = IN_PLACE ? (a.keep + gridDim.x * a.block_rows - 1) / (gridDim.x * a.block_rows) : 1;
    for (int round = 0; round < rounds; ++round) {
        const int row0 = (round * gridDim.x + blockIdx.x) * a.block_rows;
        float w = 0.f;
        long long w_to = -1;
        if (tid < a.block_rows) {
            const int i = row0 + tid, place = i < a.keep ? kept[i] : -1, at = place >> a.page_shift, to_at = i >> a.page_shift;
            long long src = -1, dst = -1;
            // (a row that stays where it is need not move)
            if (place >= 0 && at < a.bt_stride && to_at < a.to_stride && !(IN_PLACE && place == i)) {
                const int page = from[at], to_page = to[to_at];
                if (page >= 0 && page < a.pages && to_page >= 0 && to_page < a.pages) {
                    const size_t r = (size_t)layer * a.pages + page, t = (size_t)layer * a.pages + to_page;
                    const int off = place & (a.page_size - 1), to_off = i & (a.page_size - 1);
                    src = (long long)(((r * 2 * a.nkv + kvh) << a.page_shift) + off);
                    dst = (long long)(((t * 2 * a.nkv + kvh) << a.page_shift) + to_off);
                    if (a.weights) {
                        w = a.weights[((r * a.nkv + kvh) << a.page_shift) + off];
                        w_to = (long long)(((t * a.nkv + kvh) << a.page_shift) + to_off);
                    }
                }
            }
            src_s[tid] = src;
            dst_s[tid] = dst;
        }
        __syncthreads();
        V v[MOVE_AHEAD];
        long long dst[MOVE_AHEAD];
#pragma unroll
        for (int u = 0; u < MOVE_AHEAD; ++u) {
            const int p = tid + u * MOVE_THREADS, i = p / both, in = p - i * both;
            dst[u] = -1;
            if (i < a.block_rows && src_s[i] >= 0) {
                const long long more = in < per ? (long long)in : to_value * per + (in - per);
                dst[u] = dst_s[i] * per + more;
                v[u] = reinterpret_cast<const V*>(a.kv)[src_s[i] * per + more];
            }
        }
        if (IN_PLACE) asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
#pragma unroll
        for (int u = 0; u < MOVE_AHEAD; ++u)
            if (dst[u] >= 0) reinterpret_cast<V*>(a.kv)[dst[u]] = v[u];
        if (w_to >= 0) a.weights[w_to] = w;
        if (IN_PLACE) __syncthreads();                                     // the rows have been read before the next round's are put there
    }
}

template <typename V>
static void launch_move(MoveArgs a, long long rows, bool in_place, cudaStream_t stream) {
    const int most = MOVE_THREADS * MOVE_AHEAD / (2 * (a.row_bytes / (int)sizeof(V)));
    a.block_rows = most < MOVE_ROWS ? most : MOVE_ROWS;
    const unsigned blocks = (unsigned)((a.keep + a.block_rows - 1) / a.block_rows);
    if (!in_place) {
        launch_pdl(move_keys_kernel<V, false>, dim3(blocks, (unsigned)rows), dim3(MOVE_THREADS), 0, stream, a);
        return;
    }
    const unsigned cluster = blocks < (unsigned)MOVE_CLUSTER ? blocks : MOVE_CLUSTER;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster, (unsigned)rows);
    cfg.blockDim = dim3(MOVE_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, move_keys_kernel<V, true>, a);
}

}  // namespace budget
}  // namespace lily

using namespace lily;

LILY_API int lily_select_keys(const float* weights, const int* block_table, int bt_stride, const int* lengths, int* kept, int layers, int pages,
                              int requests, int nkv, int page_size, int max_length, int keep, int first, int recent, cudaStream_t stream) {
    const long long rows = (long long)layers * requests * nkv;
    if (rows == 0 || keep == 0) return 0;
    LILY_REQUIRE(keep > 0 && first >= 0 && recent >= 0 && (long long)first + recent <= keep, "select_keys: the first %d and the last %d do not fit %d places",
                 first, recent, keep);
    LILY_REQUIRE(page_size > 0 && (page_size & (page_size - 1)) == 0, "select_keys: page_size %d is not a power of two", page_size);
    LILY_REQUIRE(bt_stride > 0 && max_length >= 0 && max_length <= (long long)bt_stride * page_size && rows <= 0x7fffffff, "select_keys: %lld rows of up to %d places, tables of %d pages",
                 rows, max_length, bt_stride);
    budget::SelectArgs a{weights, block_table, lengths, kept, bt_stride, requests, nkv, page_size, 0, pages, max_length, keep, first, recent};
    while (1 << a.page_shift < page_size) ++a.page_shift;
    static bool configured = false;
    if (!configured) {
        const cudaError_t e = cudaFuncSetAttribute(budget::select_keys_kernel<0>, cudaFuncAttributeMaxDynamicSharedMemorySize, budget::SELECT_HELD * 4);
        LILY_REQUIRE(e == cudaSuccess, "select_keys: cannot get %d bytes of shared memory: %s", budget::SELECT_HELD * 4, cudaGetErrorString(e));
        configured = true;
    }
    // Four places a thread, more where the rows would not all run at once (2,048 threads a SM).  Measured, us, at 128 / 256 / 512 / 1,024 threads: 64 rows of 4,096 places 21 / 13
    // / 6.0 / 6.6, 384 of 3,000 26 / 19 / 12 / 17, 2,304 of 1,152 25 / 24 / 28 / 73, 8 of 1,152 8.1 / 4.2 / 3.8 / 5.3.  Ranks in registers / in shared memory: 6.6 / 8.8, 12.1 / 15.1, 25 / 25, 3.8 / 5.1.
    int threads = 128;
    while (threads < budget::SELECT_MOST && threads * 4 < max_length && rows * threads * 2 <= 2048LL * sm_count()) threads *= 2;
    const size_t smem = (size_t)(max_length < budget::SELECT_HELD ? max_length : budget::SELECT_HELD) * 4;
    if (max_length <= 4 * threads) launch_pdl(budget::select_keys_kernel<4>, dim3((unsigned)rows), dim3(threads), 0, stream, a);
    else if (max_length <= 8 * threads) launch_pdl(budget::select_keys_kernel<8>, dim3((unsigned)rows), dim3(threads), 0, stream, a);
    else launch_pdl(budget::select_keys_kernel<0>, dim3((unsigned)rows), dim3(threads), smem, stream, a);
    LILY_CHECK_LAUNCH("select_keys");
    return 0;
}

LILY_API int lily_move_keys(void* kv, float* weights, const int* block_table, int bt_stride, const int* to_table, int to_stride, const int* kept,
                            int layers, int pages, int requests, int nkv, int page_size, int row_bytes, int keep, int in_place, cudaStream_t stream) {
    const long long rows = (long long)layers * requests * nkv;
    if (rows == 0 || keep == 0) return 0;
    LILY_REQUIRE(page_size > 0 && (page_size & (page_size - 1)) == 0, "move_keys: page_size %d is not a power of two", page_size);
    LILY_REQUIRE(bt_stride > 0 && to_stride > 0 && row_bytes > 0 && row_bytes % 2 == 0 && (long long)keep * row_bytes <= 0x7fff0000, "move_keys: %d places of %d bytes", keep, row_bytes);
    const int vec = row_bytes % 16 == 0 && (uintptr_t)kv % 16 == 0 ? 16 : row_bytes % 4 == 0 && (uintptr_t)kv % 4 == 0 ? 4 : 2;
    LILY_REQUIRE(row_bytes / vec <= budget::MOVE_THREADS * budget::MOVE_AHEAD / 2, "move_keys: rows of %d bytes in pieces of %d", row_bytes, vec);
    for (long long at = 0; at < rows;) {
        // (a grid has 65,535 lists at most: whole layers of them)
        const long long layer_rows = (long long)requests * nkv, some = layer_rows > 65535 ? 0 : 65535 / layer_rows < layers ? 65535 / layer_rows : layers;
        LILY_REQUIRE(some > 0, "move_keys: %d requests of %d kv heads", requests, nkv);
        const long long first_layer = at / layer_rows, now = first_layer + some <= layers ? some : layers - first_layer;
        budget::MoveArgs a{(unsigned char*)kv + (size_t)first_layer * pages * 2 * nkv * page_size * row_bytes,
                           weights ? weights + (size_t)first_layer * pages * nkv * page_size : nullptr, block_table, to_table,
                           kept + (size_t)at * keep, bt_stride, to_stride, requests, nkv, page_size, 0, pages, keep, row_bytes, 0};
        while (1 << a.page_shift < page_size) ++a.page_shift;
        const long long lists = now * layer_rows;
        if (vec == 16) budget::launch_move<uint4>(a, lists, in_place, stream);
        else if (vec == 4) budget::launch_move<uint32_t>(a, lists, in_place, stream);
        else budget::launch_move<uint16_t>(a, lists, in_place, stream);
        at += lists;
    }
    LILY_CHECK_LAUNCH("move_keys");
    return 0;
}
