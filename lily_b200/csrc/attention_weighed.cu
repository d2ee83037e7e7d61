// Decode attention over the paged cache that also adds up the weight each cached key is given.
//
// For a request of n cached places (the newest token's own among them) and the query heads h of a kv head g:
//   p_hj = exp(c q_h . k_j - lse_h),  o_h = sum_j p_hj v_j,  w_gj <- (j < n - 1 ? w_gj : 0) + sum_h p_hj,
// with w float32 [pages, kv_heads, page_size] beside the keys: the newest place's weight is set, whatever an earlier owner left there.
// The keys of a request are cut into ranges of a block each.  A key's weight needs the row's (max, sum) over all ranges, so scores are kept in scratch (in
// units of log2 e) and read again when that is known: from the blocks of a cluster, or by a second kernel that joins what the ranges left.
#include "attention_args.cuh"
#include "common.cuh"
#include "tcgen05.cuh"

#include <cooperative_groups.h>

#include <atomic>

namespace lily {
bool attention_decode_f32_takes(const AttnArgs& a);
int attention_decode_f32_weighed(const AttnArgs& a, int requests, cudaStream_t stream);
int* decode_lost_word();

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
    int splits, nq, nkv, d, page_size, score_stride, max_len;
    float scale;
    int pages;                    // pages of the layer
    int longest_first;            // tensor-core kernel: blocks go to the rows in the order of their lengths
    int tile_polls;               // tensor-core kernel: polls before a wait for a tile gives up
    int* lost;                    // tensor-core kernel: a word of the host's where it says so
};

// A request's places (no more than the caller said there would be).
__device__ __forceinline__ int places_of(const DecodeArgs& a, int req) { return min(max(a.seq_lens[req], 0), a.max_len); }

// The places of range `z` of a request: equal shares in steps of 64.
__device__ __forceinline__ void key_range(const DecodeArgs& a, int req, int z, int& beg, int& end) {
    const int n = places_of(a, req);
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
constexpr int JOIN_KEYS = 4 * JOIN_THREADS;      // places a block adds up

template <typename T>
__global__ void __launch_bounds__(JOIN_THREADS) decode_weighed_join_kernel(const DecodeArgs a) {
    extern __shared__ float sm[];              // [group] lse (log2 units)
    pdl_enter_small();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = a.nq / a.nkv, req = blockIdx.x, kvh = blockIdx.y, d = a.d;
    const int n = places_of(a, req), beg = ((int)blockIdx.z - 1) * JOIN_KEYS;
    if (blockIdx.z > 0 && beg >= n) return;
    for (int h = warp; h < group; h += JOIN_THREADS / 32) {
        const float* ml = a.part_ml + ((size_t)req * a.nq + kvh * group + h) * a.splits * 2;
        float m = -INFINITY, l = 0.f;
        for (int s = lane; s < a.splits; s += 32) {
            const float ms = ml[2 * s], ls = ml[2 * s + 1], mn = fmaxf(m, ms), base = mn == -INFINITY ? 0.f : mn;
            l = fmaf(ls, exp2f(ms - base), l * exp2f(m - base));
            m = mn;
        }
        const float most = warp_max(m);
        l = warp_sum(l * exp2f(m - (most == -INFINITY ? 0.f : most)));
        if (lane == 0) sm[h] = most + log2f(l);
    }
    __syncthreads();
    if (blockIdx.z == 0) {
        const bool vec = (d & 3) == 0;
        const int step = vec ? 4 : 1;
        for (int i = tid * step; i < group * d; i += JOIN_THREADS * step) {
            const int h = i / d, col = i % d;
            const size_t row = (size_t)req * a.nq + kvh * group + h, at = row * a.splits;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            if (n > 0) {
#pragma unroll 8
                for (int s = 0; s < a.splits; ++s) {
                    const float m = a.part_ml[(at + s) * 2], l = a.part_ml[(at + s) * 2 + 1];
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    const float* part = a.part_o + (at + s) * d + col;
                    if (vec) v = *reinterpret_cast<const float4*>(part);
                    else v.x = *part;
                    if (m == -INFINITY && l == 0.f) continue;          // a range without keys
                    const float f = exp2f(m - sm[h]);
                    o.x = fmaf(v.x, f, o.x), o.y = fmaf(v.y, f, o.y), o.z = fmaf(v.z, f, o.z), o.w = fmaf(v.w, f, o.w);
                }
            }
            T* to = (T*)a.out + row * d + col;
            to[0] = from_float<T>(o.x);
            if (vec) to[1] = from_float<T>(o.y), to[2] = from_float<T>(o.z), to[3] = from_float<T>(o.w);
        }
        return;
    }
    // four neighbouring places a thread where they lie in one page
    const int* table = a.block_table + (size_t)req * a.bt_stride;
    const float* scores = a.scores + ((size_t)req * a.nq + kvh * group) * a.score_stride;
    const int end = min(n, beg + JOIN_KEYS);
    auto weights_at = [&](int j) { return a.weights + ((size_t)table[j / a.page_size] * a.nkv + kvh) * a.page_size + j % a.page_size; };
    if ((a.page_size & 3) == 0 && ((uintptr_t)a.weights & 15) == 0) {
        const int j = beg + 4 * tid;
        if (j >= end) return;
        float* at = weights_at(j);
        float4 w = *reinterpret_cast<const float4*>(at);
        w = make_float4(j == n - 1 ? 0.f : w.x, j + 1 == n - 1 ? 0.f : w.y, j + 2 == n - 1 ? 0.f : w.z, j + 3 == n - 1 ? 0.f : w.w);
#pragma unroll 4
        for (int h = 0; h < group; ++h) {
            const float4 t = *reinterpret_cast<const float4*>(scores + (size_t)h * a.score_stride + j);
            w.x += exp2f(t.x - sm[h]);
            w.y += exp2f(t.y - sm[h]);
            w.z += exp2f(t.z - sm[h]);
            w.w += exp2f(t.w - sm[h]);
        }
        if (j + 4 <= n) *reinterpret_cast<float4*>(at) = w;
        else {
            at[0] = w.x;
            if (j + 1 < n) at[1] = w.y;
            if (j + 2 < n) at[2] = w.z;
        }
        return;
    }
    for (int j = beg + tid; j < end; j += JOIN_THREADS) {
        float* w = weights_at(j);
        float sum = j < n - 1 ? *w : 0.f;
        for (int h = 0; h < group; ++h) sum += exp2f(scores[(size_t)h * a.score_stride + j] - sm[h]);
        *w = sum;
    }
}

// ---- bfloat16, head sizes 64 and 128, on the tensor cores (mma.sync m16n8k16) ----------------------
//
// A block has the up to 16 query heads of a kv head as its rows and walks its range of keys in tiles of 64, of which each of four warps
// takes 16 with a (max, sum, output) of its own, merged in the order of the warps at the end.  Tiles come by TMA where a page is a whole number
// of them (halves of 64 columns in the hardware's 128-byte swizzle), else piece by piece with cp.async.  Scores leave for scratch as
// they are formed (16 bytes a key and kv head of four query heads beside its 512 bytes of key and value; they stay in L2) and come back when the
// row's lse is known:  alone (one range), from the other blocks of a thread-block cluster (each sends every other its share of the sums and its
// rows' (max, sum) through distributed shared memory), or in the join kernel behind.  What bounds it are the bytes, and the ends of blocks, when nothing of their own
// is on the way: eight rows of 4,096 keys, 32 heads over 8, 29.1 us (134 MB: 4.7 TB/s), 64 rows of 250 to 1,750 48.2; without the weights' phase 26.9 and 43.2, without the
// scores' writes besides 25.0 and 40.2.
namespace cg = cooperative_groups;

constexpr int BN = 64, THREADS = 128, MAX_CLUSTER = 16, POLLS = 1 << 22;
__host__ __device__ constexpr int stages_of(int d) { return d == 64 ? 4 : 2; }          // 64 KB of tiles a block, three blocks a SM

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Shared memory: [1024-byte aligned] key tiles, value tiles, queries; behind them, in a cluster, what the other blocks send.
__host__ __device__ constexpr size_t tiles_bytes(int d) { return 1024 + 2 * (size_t)stages_of(d) * BN * d * 2 + 16 * (size_t)d * 2; }
// Output sums a block of a cluster of `splits` blocks finishes: its share of rows x d.
__host__ __device__ constexpr int cluster_share(int rows, int d, int splits) { return ((rows * d + splits - 1) / splits + 3) / 4 * 4; }
constexpr size_t recv_bytes(int rows, int d, int splits) { return ((size_t)splits * cluster_share(rows, d, splits) + (size_t)splits * 32) * sizeof(float); }

template <int D, bool CLUSTER, bool TMA>
__global__ void __launch_bounds__(THREADS, 3) decode_weighed_mma_kernel(const DecodeArgs a, const int page_shift, const __grid_constant__ CUtensorMap map_kv) {
    constexpr int CH = D / 8, KSTEPS = D / 16, TILE = BN * D * 2, STAGES = stages_of(D);
    extern __shared__ __align__(128) unsigned char smem_raw[];
    unsigned char* k_s = reinterpret_cast<unsigned char*>(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* v_s = k_s + STAGES * TILE;
    unsigned char* q_s = v_s + STAGES * TILE;                       // [16][D]
    __shared__ __align__(8) uint64_t full_s[STAGES];
    __shared__ int lost_s, row_s;
    __shared__ float lse_s[16];
    // the 16-byte piece `ch` of row `r` of a tile: halves of 64 columns, rows of 128 bytes, pieces exchanged by row
    auto piece = [](int r, int ch) { return (uint32_t)((ch >> 3) * (BN * 128) + r * 128 + (((ch ^ r) & 7) << 4)); };
    auto q_piece = [](int r, int ch) { return (uint32_t)(r * (D * 2) + ((((ch ^ r) & 7) | (ch & ~7)) << 4)); };
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
    if (CLUSTER) cluster_arrive_started();
    const uint32_t full0 = smem_u32(full_s);
    if (TMA && tid == 0) {
        lost_s = 0;
#pragma unroll
        for (int st = 0; st < STAGES; ++st) tc5::mbar_init(full0 + 8 * st, 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    pdl_enter_small();
    int bx = blockIdx.x, by = blockIdx.y, bz = blockIdx.z;
    if (a.longest_first) {
        // the blocks of the row that is next by length: its kv heads and ranges side by side
        int* len_s = reinterpret_cast<int*>(q_s);                   // the queries come there later
        const int rows = gridDim.x, part = CLUSTER ? gridDim.y : gridDim.y * gridDim.z;
        const int at = blockIdx.x + gridDim.x * (blockIdx.y + (CLUSTER ? 0 : gridDim.y * blockIdx.z)), want = at / part;
        const int mine = tid < rows ? a.seq_lens[tid] : 0;
        len_s[tid] = mine;
        __syncthreads();
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < rows; ++j) {
            const int other = len_s[j];
            rank += other > mine || (other == mine && j < tid);
        }
        if (tid < rows && rank == want) row_s = tid;
        __syncthreads();
        bx = row_s;
        by = CLUSTER ? at % part : at % part / gridDim.z;
        bz = CLUSTER ? blockIdx.z : at % part % gridDim.z;
    }
    const int group = a.nq / a.nkv, chunks = (group + 15) / 16, req = bx, kvh = by / chunks, r0 = by % chunks * 16;
    const int nrows = min(16, group - r0), head0 = kvh * group + r0;
    int kbeg, kend;
    key_range(a, req, bz, kbeg, kend);
    const int ntiles = (kend - kbeg + BN - 1) / BN;
    const int* table = a.block_table + (size_t)req * a.bt_stride;
    const size_t head_stride = (size_t)a.page_size * D, page_stride = 2 * (size_t)a.nkv * head_stride;
    const __nv_bfloat16* kv_head = (const __nv_bfloat16*)a.kv + (size_t)kvh * head_stride;
    const int page_mask = (1 << page_shift) - 1;
    auto load_tile = [&](int t) {                                   // piece by piece
        const int kb = kbeg + t * BN;
        unsigned char *kd = k_s + t % STAGES * TILE, *vd = v_s + t % STAGES * TILE;
#pragma unroll
        for (int i = tid; i < BN * CH; i += THREADS) {
            const int r = i / CH, ch = i % CH, place = kb + r;
            const bool ok = place < kend;
            const __nv_bfloat16* src = kv_head + (size_t)(ok ? table[place >> page_shift] : 0) * page_stride + (((ok ? place : 0) & page_mask) * D + ch * 8);
            cp_async16(smem_u32(kd + piece(r, ch)), src, ok);
            cp_async16(smem_u32(vd + piece(r, ch)), src + (size_t)a.nkv * head_stride, ok);
        }
    };
    auto ask_tile = [&](int t) {                                    // one thread: a tile lies in one page
        const int kb = kbeg + t * BN, st = t % STAGES, page = table[kb >> page_shift], off = kb & page_mask;
        const uint32_t bar = full0 + 8 * st, kd = smem_u32(k_s + st * TILE), vd = smem_u32(v_s + st * TILE);
        tc5::mbar_expect_tx(bar, 2 * TILE);
#pragma unroll
        for (int h = 0; h < D / 64; ++h) tc5::tma_load_4d(kd + h * (BN * 128), &map_kv, bar, h * 64, off, kvh, page);
#pragma unroll
        for (int h = 0; h < D / 64; ++h) tc5::tma_load_4d(vd + h * (BN * 128), &map_kv, bar, h * 64, off, a.nkv + kvh, page);
    };
    int asked = min(STAGES, ntiles);                                // tiles that were asked for (by the first thread)
    if (TMA) {
        if (tid == 0) {
            asm volatile("fence.proxy.async;\n" ::: "memory");      // the kernel ahead wrote keys by threads
            for (int t = 0; t < asked; ++t) ask_tile(t);
        }
    } else {
#pragma unroll
        for (int t = 0; t < STAGES - 1; ++t) {
            if (t < ntiles) load_tile(t);
            cp_async_commit();
        }
    }
    for (int i = tid; i < 16 * CH; i += THREADS) {
        const int r = i / CH, ch = i % CH;
        *reinterpret_cast<uint4*>(q_s + q_piece(r, ch)) =
            r < nrows ? *reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.q + ((size_t)req * a.nq + head0 + r) * D + ch * 8) : make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    uint32_t qf[KSTEPS][4];
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk)
        ldmatrix_x4(smem_u32(q_s + q_piece(lane & 15, kk * 2 + (lane >> 4))), qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3]);
    float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;      // rows g and g + 8
    float o[D / 8][4];
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    const float sl2 = a.scale * LOG2E;
    float* sc_lo = a.scores + ((size_t)req * a.nq + head0 + g) * a.score_stride;
    float* sc_hi = sc_lo + (size_t)8 * a.score_stride;

    for (int t = 0; t < ntiles; ++t) {
        const int buf = t % STAGES, kb = kbeg + t * BN, key0 = warp * 16;
        unsigned char *kt = k_s + buf * TILE, *vt = v_s + buf * TILE;
        if (TMA) {
            int left = a.tile_polls;
            while (left > 0 && !tc5::mbar_try_wait(full0 + 8 * buf, (t / STAGES) & 1))
                if ((--left & 1023) == 0 && *(volatile int*)&lost_s) left = 0;
            if (left == 0) {
                lost_s = 1;
                if (lane == 0) {
                    *(volatile int*)a.lost = 1 + (bx & 0x7fff);
                    __threadfence_system();
                }
            }
            if (kb + BN > kend) {                                   // values beyond the range are cleared: a weight of zero meets no infinity
                for (int i = tid; i < BN * CH; i += THREADS)
                    if (kb + i / CH >= kend) *reinterpret_cast<uint4*>(vt + piece(i / CH, i % CH)) = make_uint4(0, 0, 0, 0);
                __syncthreads();
            }
        } else {
            cp_async_wait<STAGES - 2>();
            __syncthreads();                                        // tile t has landed; tile t - 1's readers are done
            if (t + STAGES - 1 < ntiles) load_tile(t + STAGES - 1);
            cp_async_commit();
        }
        float s[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
            uint32_t b0, b1, b2, b3;
            ldmatrix_x4(smem_u32(kt + piece(key0 + (lane & 7) + ((lane >> 4) << 3), kk * 2 + ((lane >> 3) & 1))), b0, b1, b2, b3);
            mma_bf16(s[0], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], b0, b1);
            mma_bf16(s[1], qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3], b2, b3);
        }
        float mx_lo = -INFINITY, mx_hi = -INFINITY;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int place = kb + key0 + j * 8 + 2 * c;
#pragma unroll
            for (int e = 0; e < 4; ++e) s[j][e] = place + (e & 1) < kend ? s[j][e] * sl2 : -INFINITY;
            if (place < kend) {                                     // (an odd end's neighbour lies in the row's rounding)
                if (g < nrows) *reinterpret_cast<float2*>(sc_lo + place) = make_float2(s[j][0], s[j][1]);
                if (g + 8 < nrows) *reinterpret_cast<float2*>(sc_hi + place) = make_float2(s[j][2], s[j][3]);
            }
            mx_lo = fmaxf(mx_lo, fmaxf(s[j][0], s[j][1]));
            mx_hi = fmaxf(mx_hi, fmaxf(s[j][2], s[j][3]));
        }
        mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, 1));
        mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, 2));
        mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, 1));
        mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, 2));
        const float mn_lo = fmaxf(m_lo, mx_lo), mn_hi = fmaxf(m_hi, mx_hi);
        const float base_lo = mn_lo == -INFINITY ? 0.f : mn_lo, base_hi = mn_hi == -INFINITY ? 0.f : mn_hi;
        const float al_lo = exp2f(m_lo - base_lo), al_hi = exp2f(m_hi - base_hi);
        m_lo = mn_lo;
        m_hi = mn_hi;
        l_lo *= al_lo;                                              // a thread's own share of the sum
        l_hi *= al_hi;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            s[j][0] = exp2f(s[j][0] - base_lo);
            s[j][1] = exp2f(s[j][1] - base_lo);
            s[j][2] = exp2f(s[j][2] - base_hi);
            s[j][3] = exp2f(s[j][3] - base_hi);
            l_lo += s[j][0] + s[j][1];
            l_hi += s[j][2] + s[j][3];
        }
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
            o[j][0] *= al_lo;
            o[j][1] *= al_lo;
            o[j][2] *= al_hi;
            o[j][3] *= al_hi;
        }
        // the weights are rounded to bfloat16 for the product with the values, as in the other attention kernels of this precision (in two halves 1 to 4 % slower; what the
        // outputs are from 64 bits, 1.5e-3 of them at some hundred places and 2.0e-3 at four, is mostly their own rounding, 1.7e-3 where the weights keep 32 bits)
        const uint32_t a0 = tc5::pack2(s[0][0], s[0][1]), a1 = tc5::pack2(s[0][2], s[0][3]), a2 = tc5::pack2(s[1][0], s[1][1]), a3 = tc5::pack2(s[1][2], s[1][3]);
#pragma unroll
        for (int jp = 0; jp < D / 16; ++jp) {
            uint32_t b0, b1, b2, b3;
            ldmatrix_x4_trans(smem_u32(vt + piece(key0 + (lane & 7) + (((lane >> 3) & 1) << 3), jp * 2 + (lane >> 4))), b0, b1, b2, b3);
            mma_bf16(o[2 * jp], a0, a1, a2, a3, b0, b1);
            mma_bf16(o[2 * jp + 1], a0, a1, a2, a3, b2, b3);
        }
        if (TMA && t + STAGES < ntiles) {
            __syncthreads();                                        // every warp is done with this buffer
            if (tid == 0 && !*(volatile int*)&lost_s) {
                ask_tile(t + STAGES);
                asked = t + STAGES + 1;
            }
        }
    }
    l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 1);
    l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 2);
    l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 1);
    l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 2);
    __syncthreads();                                                // every warp is done with the tiles
    if (TMA && lost_s) {
        if (tid == 0)                                               // the last copy into each buffer lands before it is used for something else
            for (int t = max(0, asked - STAGES); t < asked; ++t)
                for (int left = POLLS; left > 0 && !tc5::mbar_try_wait(full0 + 8 * (t % STAGES), (t / STAGES) & 1); --left) {}
        l_lo = l_hi = __int_as_float(0x7fffffff);
        __syncthreads();
    }

    // The weights of this thread's first four places and their scores are asked for here, ahead of the joining.
    const float* scores = a.scores + ((size_t)req * a.nq + head0) * a.score_stride;
    const int newest = places_of(a, req) - 1;
    auto weights_at = [&](int j) { return a.weights + (((size_t)table[j >> page_shift] * a.nkv + kvh) << page_shift) + (j & page_mask); };
    float* first_at = nullptr;
    float4 first_w = make_float4(0.f, 0.f, 0.f, 0.f), first_s[4] = {first_w, first_w, first_w, first_w};
    if ((CLUSTER || a.splits == 1) && kbeg + 4 * tid < kend) {
        first_at = weights_at(kbeg + 4 * tid);
        first_w = *reinterpret_cast<const float4*>(first_at);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r < nrows) first_s[r] = *reinterpret_cast<const float4*>(scores + (size_t)r * a.score_stride + kbeg + 4 * tid);
    }

    // ---- the four warps' results joined --------------------------------------------------------------
    float* mo = reinterpret_cast<float*>(k_s);                      // [4 warps][16 rows][D]
    float* mml = mo + 4 * 16 * D;                                   // [4 warps][16 rows][2]
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
        const int col = j * 8 + 2 * c;
        if (g < nrows) *reinterpret_cast<float2*>(mo + (warp * 16 + g) * D + col) = make_float2(o[j][0], o[j][1]);
        if (g + 8 < nrows) *reinterpret_cast<float2*>(mo + (warp * 16 + g + 8) * D + col) = make_float2(o[j][2], o[j][3]);
    }
    if (c == 0) {
        *reinterpret_cast<float2*>(mml + (warp * 16 + g) * 2) = make_float2(m_lo, l_lo);
        *reinterpret_cast<float2*>(mml + (warp * 16 + g + 8) * 2) = make_float2(m_hi, l_hi);
    }
    cg::cluster_group cluster = cg::this_cluster();
    const int splits = a.splits, share = cluster_share(min(16, group), D, splits);
    float* recv_o = reinterpret_cast<float*>(smem_raw + tiles_bytes(D));        // [splits][share]
    float* recv_ml = recv_o + (size_t)splits * share;                            // [splits][16][2]
    __syncthreads();
    if (CLUSTER) cluster_wait_started();
    for (int i4 = tid; i4 < nrows * (D / 4); i4 += THREADS) {
        const int r = i4 / (D / 4), col = (i4 % (D / 4)) * 4, i = r * D + col;
        float mx = -INFINITY, den = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) mx = fmaxf(mx, mml[(w * 16 + r) * 2]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float2 ml = *reinterpret_cast<const float2*>(mml + (w * 16 + r) * 2);
            if (ml.x == -INFINITY && ml.y == 0.f) continue;         // no keys (a NaN is no maximum, but makes the sum one)
            const float f = exp2f(ml.x - mx);
            const float4 v = *reinterpret_cast<const float4*>(mo + (w * 16 + r) * D + col);
            acc.x = fmaf(v.x, f, acc.x), acc.y = fmaf(v.y, f, acc.y), acc.z = fmaf(v.z, f, acc.z), acc.w = fmaf(v.w, f, acc.w);
            den = fmaf(ml.y, f, den);
        }
        if (CLUSTER) {
            const int owner = i / share;
            write_to_block(reinterpret_cast<float4*>(recv_o + bz * share + (i - owner * share)), owner, acc);
            if (col / 4 < splits)                                   // group p of four columns tells block p the row's (max, sum)
                write_to_block(reinterpret_cast<float2*>(recv_ml + (bz * 16 + r) * 2), col / 4, make_float2(mx, den));
        } else if (splits > 1) {
            const size_t at = ((size_t)req * a.nq + head0 + r) * splits + bz;
            *reinterpret_cast<float4*>(a.part_o + at * D + col) = acc;
            if (col == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(mx, den);
        } else {
            const float inv = den == 0.f ? 0.f : 1.f / den;
            *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + ((size_t)req * a.nq + head0 + r) * D + col) =
                make_uint2(tc5::pack2(acc.x * inv, acc.y * inv), tc5::pack2(acc.z * inv, acc.w * inv));
            if (col == 0) lse_s[r] = mx + log2f(den);
        }
    }
    if (!CLUSTER && splits > 1) return;
    if (CLUSTER) {
        cluster.sync();                                             // every block's sums have arrived; nobody is written to after this
        if (tid < nrows) {
            float mx = -INFINITY, den = 0.f;
            for (int sp = 0; sp < splits; ++sp) mx = fmaxf(mx, recv_ml[(sp * 16 + tid) * 2]);
            for (int sp = 0; sp < splits; ++sp) {
                const float2 ml = *reinterpret_cast<const float2*>(recv_ml + (sp * 16 + tid) * 2);
                if (ml.x > -INFINITY || ml.y != 0.f) den = fmaf(ml.y, exp2f(ml.x - mx), den);
            }
            lse_s[tid] = mx + log2f(den);
        }
    }
    __syncthreads();
    if (CLUSTER)
        for (int slot = tid * 4; slot < share; slot += THREADS * 4) {
            const int i = bz * share + slot;
            if (i >= nrows * D) break;
            const int r = i / D, col = i % D;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int sp = 0; sp < splits; ++sp) {                   // in the order of the ranges, whichever block joins them
                const float2 ml = *reinterpret_cast<const float2*>(recv_ml + (sp * 16 + r) * 2);
                if (ml.x == -INFINITY && ml.y == 0.f) continue;
                const float f = exp2f(ml.x - lse_s[r]);
                const float4 v = *reinterpret_cast<const float4*>(recv_o + sp * share + slot);
                acc.x = fmaf(v.x, f, acc.x), acc.y = fmaf(v.y, f, acc.y), acc.z = fmaf(v.z, f, acc.z), acc.w = fmaf(v.w, f, acc.w);
            }
            *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + ((size_t)req * a.nq + head0 + r) * D + col) =
                make_uint2(tc5::pack2(acc.x, acc.y), tc5::pack2(acc.z, acc.w));
        }
    // ---- what the places of this range were given: four neighbouring places a thread, which lie in one page ------------
    for (int j = kbeg + 4 * tid, turn = 0; j < kend; j += 4 * THREADS, ++turn) {
        float* at = first_at;
        float4 w = first_w;
        if (turn > 0) {
            at = weights_at(j);
            w = *reinterpret_cast<const float4*>(at);
        }
        // the newest place is set
        w = make_float4(j == newest ? 0.f : w.x, j + 1 == newest ? 0.f : w.y, j + 2 == newest ? 0.f : w.z, j + 3 == newest ? 0.f : w.w);
        for (int r = 0; r < nrows; ++r) {
            const float4 t = turn == 0 && r < 4 ? (r == 0 ? first_s[0] : r == 1 ? first_s[1] : r == 2 ? first_s[2] : first_s[3])
                                                : *reinterpret_cast<const float4*>(scores + (size_t)r * a.score_stride + j);
            const float lse = lse_s[r];
            w.x += exp2f(t.x - lse);
            w.y += exp2f(t.y - lse);
            w.z += exp2f(t.z - lse);
            w.w += exp2f(t.w - lse);
        }
        if (j + 4 <= kend) *reinterpret_cast<float4*>(at) = w;
        else {
            at[0] = w.x;
            if (j + 1 < kend) at[1] = w.y;
            if (j + 2 < kend) at[2] = w.z;
        }
    }
}

// What any of the kernel's blocks may ask for.
template <int D, bool CLUSTER>
constexpr size_t most_smem() {
    size_t most = 0;
    for (int splits = 2; CLUSTER && splits <= MAX_CLUSTER; ++splits) most = recv_bytes(16, D, splits) > most ? recv_bytes(16, D, splits) : most;
    return tiles_bytes(D) + most;
}
// Raises the kernel's limit of dynamic shared memory, once and to that: threads that launch other sizes at the same time set the same limit.
template <int D, bool CLUSTER, bool TMA>
static bool allow_smem() {
    static std::atomic<bool> allowed{false};
    if (!allowed) {
        if (cudaFuncSetAttribute(decode_weighed_mma_kernel<D, CLUSTER, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most_smem<D, CLUSTER>()) != cudaSuccess ||
            (CLUSTER && cudaFuncSetAttribute(decode_weighed_mma_kernel<D, CLUSTER, TMA>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)) {
            cudaGetLastError();
            return false;
        }
        allowed = true;
    }
    return true;
}

template <int D, bool TMA>
static int launch_mma(DecodeArgs a, int requests, bool cluster, int page_shift, const CUtensorMap& map, cudaStream_t stream) {
    const int group = a.nq / a.nkv, rows = group < 16 ? group : 16;
    const dim3 grid(requests, a.nkv * ((group + 15) / 16), a.splits);
    const long blocks = (long)grid.x * grid.y * grid.z, places = 3L * sm_count();
    a.longest_first = grid.x > 1 && grid.x <= THREADS && blocks > places && blocks <= (cluster ? 3 : 2) * places;
    if (cluster) {
        const size_t smem = tiles_bytes(D) + recv_bytes(rows, D, a.splits);
        if (!allow_smem<D, true, TMA>()) {
            set_error("attention_decode_weighed: cannot get %zu bytes of shared memory in clusters", smem);
            return 2;
        }
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = grid;
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 1;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = a.splits;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = pdl_enabled() ? 2 : 1;
        cudaLaunchKernelEx(&cfg, decode_weighed_mma_kernel<D, true, TMA>, a, page_shift, map);
        return 0;
    }
    const size_t smem = tiles_bytes(D);
    if (!allow_smem<D, false, TMA>()) {
        set_error("attention_decode_weighed: cannot get %zu bytes of shared memory", smem);
        return 2;
    }
    launch_pdl(decode_weighed_mma_kernel<D, false, TMA>, grid, dim3(THREADS), smem, stream, a, page_shift, map);
    return 0;
}

// How many clusters of `splits` blocks the device holds at once (0: such a cluster cannot be placed).
template <int D>
static int cluster_room(int rows, int splits) {
    static int known[17][MAX_CLUSTER + 1] = {};                     // 0 not asked, -1 none, else the count
    int& k = known[rows][splits];
    if (k == 0) {
        const size_t smem = tiles_bytes(D) + recv_bytes(rows, D, splits);
        int clusters = 0;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(1, 1, splits);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 1;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = splits;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const bool ok = allow_smem<D, true, true>() && cudaOccupancyMaxActiveClusters(&clusters, decode_weighed_mma_kernel<D, true, true>, &cfg) == cudaSuccess && clusters > 0;
        if (!ok) cudaGetLastError();
        k = ok ? clusters : -1;
    }
    return k > 0 ? k : 0;
}

struct Plan { int splits; bool mma, cluster; };

// How the keys are cut; a function of the sizes alone.
// Which kernel takes a call, and how many ranges.  Measured, us, bfloat16 heads of 128, 32 over 8 where not said:
//   tensor cores / CUDA cores: eight rows of 4,096 keys 29 / 428 (heads of 64: 16 / 232), one of 900, 16 over 4, 6.3 / 57; float32, the kernel that cuts a row over
//   warps / the tiles: three rows 15 / 69 at best, 32 of 2,000 114 / 1,656.  Tiles by TMA / piece by piece: 29.4 / 30.9, heads of 64 15.5 / 17.7.
//   clusters as long as they fit at once, the longest first: one row of 4,096 in 16 blocks 10.4, 8 11.3, 4 18, in 16 ranges with the second kernel 11.9; eight rows in 4 or 6
//   29.2, 8 34.6, 16 43.7, 16 ranges 31.9; four of 2,000 in 8 10.6, 4 13.7;
//   a wave of ranges from 16,384 keys on where it has a quarter more blocks: one row of 16,384 48 ranges 20, a cluster of 16 24; of 65,536 57 and 83.
//   rows that would not all run at once go by length where they differ: 64 of 250 to 1,750 keys 54.6 / 58.9 as they come.
static Plan plan_of(int requests, int nq, int nkv, int d, int max_len, int page_size, int dtype) {
    const int group = nq / nkv, sms = sm_count();
    const bool mma = dtype == kBF16 && (d == 64 || d == 128) && page_size >= 4 && (page_size & (page_size - 1)) == 0;
    if (dtype == kF32 && group <= 8 && d % 4 == 0 && d <= 256) {
        // the kernel that cuts a row's keys over the warps of a block: a wave of blocks, none under 64 keys (three rows of up to 2,900 keys, 16 heads
        // over 4: 6 ranges 20.2 us, 12, a wave, 15.1, 24 17.3; 32 rows of 2,000 over 8: 1 range 114, 2 and 4 121)
        const long pairs = (long)requests * nkv, most = (max_len + 63) / 64;
        long s = sms / pairs;
        s = s < most ? s : most;
        return {(int)(s < 1 ? 1 : s > 64 ? 64 : s), false, false};
    }
    if (!mma) {
        const long pairs = (long)requests * nkv * ((group + RH - 1) / RH);
        long s = (3L * sms + pairs - 1) / pairs, most = (max_len + 127) / 128;
        s = s < most ? s : most;
        return {(int)(s < 1 ? 1 : s > 64 ? 64 : s), false, false};
    }
    const int chunks = (group + 15) / 16, rows = group < 16 ? group : 16;
    const long pairs = (long)requests * nkv * chunks, places = 3L * sms;
    const int limit = (max_len + 127) / 128;
    if (limit <= 1) return {chunks > 1 ? 2 : 1, true, false};       // (heads in several blocks are joined behind them)
    long full = places / pairs;
    full = full > 64 ? 64 : full;
    if (chunks == 1)
        for (int s = limit < MAX_CLUSTER ? limit : MAX_CLUSTER; s >= 2; --s) {
            const int room = d == 64 ? cluster_room<64>(rows, s) : cluster_room<128>(rows, s);
            if (10 * pairs > (s <= 8 ? 10 : 9) * (long)room) continue;
            const int wave = (int)(full < (max_len + 511) / 512 ? full : (max_len + 511) / 512);
            if (wave * 4 >= s * 5 && max_len >= 16384) return {wave, true, false};
            return {s, true, true};
        }
    // A little more pairs than places, long rows: the second wave would run nearly empty, so two blocks share a pair, longest first.  Measured, us,
    // one / two, 512 pairs of 128 on 444 places: 4,096 keys each 223 / 191, 100 to 8,000 199 / 166, 1,000 60 / 60, 250 to 1,750 54 / 58, 250 to 500 23 / 30;
    // 800 pairs of 4,096 279 / 280.
    if (chunks == 1 && max_len >= 4096 && pairs > places && 4 * pairs <= 5 * places && (d == 64 ? cluster_room<64>(rows, 2) : cluster_room<128>(rows, 2)) > 0)
        return {2, true, true};
    // more pairs than clusters: just enough ranges to take every place, none under 768 keys
    long s = (places + pairs - 1) / pairs, most = max_len / 768;
    s = s < most ? s : most;
    if (chunks > 1 && s < 2) s = 2;
    return {(int)(s < 1 ? 1 : s > 64 ? 64 : s), true, false};
}

}  // namespace weighed
}  // namespace lily

using namespace lily;

// The ranges a call with these sizes cuts its keys into, and the floats of scratch it needs: scores, partial outputs, partial (max, sum).
LILY_API size_t lily_attention_decode_weighed_floats(int requests, int nq, int nkv, int d, int max_len, int page_size, int dtype) {
    if (requests <= 0 || nkv <= 0 || nq < nkv || max_len < 0 || page_size <= 0) return 0;
    const weighed::Plan p = weighed::plan_of(requests, nq, nkv, d, max_len, page_size, dtype);
    const bool parts = !p.mma || (p.splits > 1 && !p.cluster);
    return (size_t)requests * nq * (((size_t)max_len + 3) / 4 * 4 + (parts ? (size_t)p.splits * (d + 2) : 0));
}

LILY_API int lily_attention_decode_weighed(const void* q, const void* kv, float* weights, void* out, const int* block_table, int bt_stride,
                                           const int* seq_lens, float* scratch, int requests, int max_len, int nq, int nkv, int d,
                                           int page_size, int pages, float scale, int dtype, int polls, cudaStream_t stream) {
    if (requests == 0) return 0;
    LILY_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0, "attention_decode_weighed: %d query heads over %d kv heads", nq, nkv);
    LILY_REQUIRE(d >= 1 && d <= 256 && page_size > 0 && max_len >= 0, "attention_decode_weighed: head size %d (takes up to 256), pages of %d", d, page_size);
    LILY_REQUIRE(dtype == kF32 || dtype == kBF16, "attention_decode_weighed: dtype %d", dtype);
    LILY_REQUIRE(((uintptr_t)scratch & 15) == 0, "attention_decode_weighed: scratch must be 16-byte aligned");
    const int score_stride = (max_len + 3) / 4 * 4, group = nq / nkv;
    const weighed::Plan plan = weighed::plan_of(requests, nq, nkv, d, max_len, page_size, dtype);
    weighed::DecodeArgs a{};
    a.q = q; a.kv = kv; a.weights = weights; a.out = out; a.block_table = block_table; a.bt_stride = bt_stride; a.seq_lens = seq_lens;
    a.splits = plan.splits; a.nq = nq; a.nkv = nkv; a.d = d; a.page_size = page_size; a.scale = scale; a.score_stride = score_stride; a.max_len = max_len; a.pages = pages;
    a.scores = scratch;
    a.part_o = a.scores + (size_t)requests * nq * score_stride;
    a.part_ml = a.part_o + (size_t)requests * nq * plan.splits * d;
    const dim3 join(requests, nkv, 1 + (max_len + weighed::JOIN_KEYS - 1) / weighed::JOIN_KEYS);
    if (plan.mma) {
        LILY_REQUIRE((((uintptr_t)q | (uintptr_t)kv | (uintptr_t)out | (uintptr_t)scratch | (uintptr_t)weights) & 15) == 0, "attention_decode_weighed: operands must be 16-byte aligned");
        LILY_REQUIRE(nkv * ((group + 15) / 16) <= 65535, "attention_decode_weighed: %d kv heads", nkv);
        int shift = 0;
        while ((1 << shift) < page_size) ++shift;
        CUtensorMap map{};
        const bool tma = page_size % weighed::BN == 0 && tc5::encoder() != nullptr;
        if (tma) {
            a.tile_polls = polls;
            a.lost = decode_lost_word();
            LILY_REQUIRE(a.lost != nullptr, "attention_decode_weighed: no word of the host's memory");
            const cuuint64_t row = (cuuint64_t)d * 2;
            const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)page_size, (cuuint64_t)2 * nkv, (cuuint64_t)pages};
            const cuuint64_t strides[3] = {row, row * page_size, row * page_size * 2 * nkv};
            const cuuint32_t box[4] = {64, weighed::BN, 1, 1}, elem[4] = {1, 1, 1, 1};
            const CUresult rc = tc5::encoder()(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(kv), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
            LILY_REQUIRE(rc == CUDA_SUCCESS, "attention_decode_weighed: cuTensorMapEncodeTiled failed with %d (%d pages of %d)", (int)rc, pages, page_size);
        }
        int rc;
        if (d == 64) rc = tma ? weighed::launch_mma<64, true>(a, requests, plan.cluster, shift, map, stream) : weighed::launch_mma<64, false>(a, requests, plan.cluster, shift, map, stream);
        else rc = tma ? weighed::launch_mma<128, true>(a, requests, plan.cluster, shift, map, stream) : weighed::launch_mma<128, false>(a, requests, plan.cluster, shift, map, stream);
        if (rc) return rc;
        if (plan.splits > 1 && !plan.cluster)
            launch_pdl(weighed::decode_weighed_join_kernel<__nv_bfloat16>, join, dim3(weighed::JOIN_THREADS), group * sizeof(float), stream, a);
        LILY_CHECK_LAUNCH("attention_decode_weighed");
        return 0;
    }
    if (dtype == kF32) {
        AttnArgs f{};
        f.q = q; f.kv = kv; f.out = out; f.block_table = block_table; f.bt_stride = bt_stride; f.seq_lens = seq_lens; f.part_o = a.part_o; f.part_ml = a.part_ml;
        f.splits = plan.splits; f.nq = nq; f.nkv = nkv; f.d = d; f.dv = d; f.page_size = page_size; f.scale = scale;
        f.scores = a.scores; f.score_stride = score_stride; f.max_len = max_len;
        if (attention_decode_f32_takes(f)) {
            if (int rc = attention_decode_f32_weighed(f, requests, stream)) return rc;
            launch_pdl(weighed::decode_weighed_join_kernel<float>, join, dim3(weighed::JOIN_THREADS), group * sizeof(float), stream, a);
            LILY_CHECK_LAUNCH("attention_decode_weighed");
            return 0;
        }
    }
    const dim3 grid(requests, nkv * ((group + weighed::RH - 1) / weighed::RH), plan.splits);
    const size_t smem = weighed::simt_floats(d) * sizeof(float);
    static bool configured = false;
    if (!configured) {
        const int most = (int)(weighed::simt_floats(256) * sizeof(float));
        cudaError_t e = cudaFuncSetAttribute(weighed::decode_weighed_simt_kernel<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(weighed::decode_weighed_simt_kernel<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
        LILY_REQUIRE(e == cudaSuccess, "attention_decode_weighed: cannot get %d bytes of shared memory: %s", most, cudaGetErrorString(e));
        configured = true;
    }
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
