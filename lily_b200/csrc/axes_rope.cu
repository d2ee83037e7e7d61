// Rotary positions with several axes (time, height, width of a token), fused with the per-head norm ahead of it and the cache write
// behind it, for caches in which a token's place is not its position.
//
// A head x of a token: y = x rsqrt(mean x^2 + eps) g (where there are gains), then for each pair j of the first rd features
//   (y_j, y_(j + rd/2)) <- (y_j c - y_(j + rd/2) s, y_(j + rd/2) c + y_j s),   c, s = tables[position of axis(j)][j],
// the rest as it is; queries go to `q_out`, keys and values to the token's place in its request's pages.  (`qk_norm_rope_write` is the
// case of one axis whose position is also the place.)  The reference's rotation is lily/layers/rotary.py:18-20, 70-87.
//
// A position outside the tables gives NaN (keys and queries that nobody can take for others); a place or a request outside the block table, or
// a page outside the cache, is not written.
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
    const int* block_table;          // [requests, bt_stride]
    int requests, bt_stride;
    void* kv;                        // [pages, 2, nkv, page_size, d]
    int pages;
    void* q_out;                     // [tokens, nq * d]
    int nq, nkv, d, rd, page_size;
    int page_shift;                  // log2 of page_size, or -1
};

// Where a head of a token goes: its row of `q_out` or of a page (null: nowhere).
template <typename T>
__device__ __forceinline__ T* target(const Args& a, int n, int head, int place, int req) {
    if (head < a.nq) return (T*)a.q_out + ((size_t)n * a.nq + head) * a.d;
    // (the quotient, a page that is not a power of two, is some thirty instructions in the chain)
    const int at = a.page_shift >= 0 ? place >> a.page_shift : place / a.page_size;
    const bool in = place >= 0 && at < a.bt_stride && (unsigned)req < (unsigned)a.requests;
    const int page = in ? a.block_table[(size_t)req * a.bt_stride + at] : -1;
    if ((unsigned)page >= (unsigned)a.pages) return nullptr;
    return (T*)a.kv + (((size_t)page * 2 * a.nkv + (head - a.nq)) * a.page_size + (place - at * a.page_size)) * a.d;
}

// A warp a head, a feature pair a lane and step: any even rotary width, any head size, any alignment.
template <typename T, typename IN, typename W>
__global__ void __launch_bounds__(128) axes_rope_write_kernel(const Args a) {
    pdl_enter_small();
    const int n = blockIdx.x, head = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (head >= a.nq + 2 * a.nkv) return;
    T* dst = target<T>(a, n, head, head < a.nq ? 0 : a.places[n], head < a.nq ? 0 : a.token_req[n]);
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

// Sixteen bytes of activations an access (N = 8 bfloat16 or 4 float32 numbers) and G = d / (2 N) threads a head (a power of two, at most a
// warp), each with two pieces: of the rotated features N neighbouring ones and their partners rd / 2 further, of the rest two neighbouring pieces.  So the
// rotation needs no exchange and the norm log2(G) shuffles.  The positions of up to four axes are read
// beside the axes of a thread's pairs, not behind them.  What bounds it is the chain of reads (axis and positions, tables, result), for few tokens
// and for many, which small blocks of short-lived threads hide best: 2,048 tokens of 32 + 2 x 8 heads of 128 in bfloat16, with gains, take 13.7 us (51 MB: 3.7 TB/s; a
// plain copy of as many bytes 9.3; with the places read behind the tables 15.1), eight tokens out of four planes of partial sums 3.2.  (For many tokens the
// chain does not explain it all: 8,192 take 4.1 times as long as 2,048, and each warp looks up what its token's other warps have looked up.)
constexpr int WIDE_THREADS = 128, AHEAD = 4;

// Numbers in pairs (mul and fma.rn.f32x2: two IEEE operations an instruction).
typedef unsigned long long Two;
__device__ __forceinline__ Two two(float a, float b) {
    Two r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 apart(Two v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
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
__device__ __forceinline__ Two two_of(uint32_t bf16_pair) { return two(__uint_as_float(bf16_pair << 16), __uint_as_float(bf16_pair & 0xffff0000u)); }

// Sixteen bytes as pairs.
template <typename T, int N>
__device__ __forceinline__ void unpack(const uint4 raw, Two (&v)[N / 2]) {
    if constexpr (sizeof(T) == 2) v[0] = two_of(raw.x), v[1] = two_of(raw.y), v[2] = two_of(raw.z), v[3] = two_of(raw.w);
    else v[0] = two(__uint_as_float(raw.x), __uint_as_float(raw.y)), v[1] = two(__uint_as_float(raw.z), __uint_as_float(raw.w));
}
// N numbers of the product (the planes added up).
template <typename IN, int N>
__device__ __forceinline__ void load_piece(const Args& a, const IN* src, Two (&v)[N / 2]) {
    if constexpr (sizeof(IN) == 2) unpack<IN, N>(*reinterpret_cast<const uint4*>(src), v);
    else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) v[i] = 0;
        for (int s0 = 0; s0 < a.splits; s0 += AHEAD) {
            ulonglong2 t[AHEAD][N / 4];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
#pragma unroll
                for (int i = 0; i < N / 4; ++i)
                    t[u][i] = s0 + u < a.splits ? *reinterpret_cast<const ulonglong2*>(src + (size_t)(s0 + u) * a.stride + 4 * i) : make_ulonglong2(0, 0);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)                          // in the order of the planes
#pragma unroll
                for (int i = 0; i < N / 4; ++i) v[2 * i] = add2(v[2 * i], t[u][i].x), v[2 * i + 1] = add2(v[2 * i + 1], t[u][i].y);
        }
    }
}
// N gains (16-byte aligned).
template <typename W, int N>
__device__ __forceinline__ void load_gain(const W* g, Two (&v)[N / 2]) {
    if constexpr (sizeof(W) == 2 && N == 8) unpack<W, N>(*reinterpret_cast<const uint4*>(g), v);
    else if constexpr (sizeof(W) == 4) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const ulonglong2 t = *reinterpret_cast<const ulonglong2*>(g + 4 * i);
            v[2 * i] = t.x;
            v[2 * i + 1] = t.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) v[i] = two(to_float(g[2 * i]), to_float(g[2 * i + 1]));
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_piece(T* dst, const Two (&v)[N / 2]) {
    if constexpr (sizeof(T) == 2) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = apart(v[i]);
            const __nv_bfloat162 two = __floats2bfloat162_rn(f.x, f.y);
            w[i] = *reinterpret_cast<const uint32_t*>(&two);
        }
        *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    } else *reinterpret_cast<ulonglong2*>(dst) = make_ulonglong2(v[0], v[1]);
}

// The tables' numbers of N pairs from `j` on, for the lanes of a warp that `need` them (of one token, `mine`: shared memory of the warp's, room for
// two rows of the tables).  Where each lane's pairs share an axis they are 16-byte reads; else the warp brings each pair of the token once, side by side, and
// hands them round through shared memory (axes in turn, 2,048 tokens: 15.2 us; a read a pair and thread took 20.7).
template <int N>
__device__ __forceinline__ void load_turn(const Args& a, int n, int j, bool need, float* mine, Two (&c)[N / 2], Two (&s)[N / 2]) {
    const int half = a.rd / 2;
    int pos[4], axis = -1;
#pragma unroll
    for (int k = 0; k < 4; ++k) pos[k] = k < a.axes ? a.positions[(size_t)k * a.tokens + n] : -1;
    bool alike = true;
    if (need) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const int4 t = *reinterpret_cast<const int4*>(a.pair_axis + j + i);
            if (i == 0) axis = t.x;
            alike = alike && t.x == axis && t.y == axis && t.z == axis && t.w == axis;
        }
    }
    auto position = [&](int ax) {
        int at = ax == 0 ? pos[0] : ax == 1 ? pos[1] : ax == 2 ? pos[2] : ax == 3 ? pos[3] : -1;
        if (ax >= 4 && ax < a.axes) at = a.positions[(size_t)ax * a.tokens + n];
        return at < a.table_rows ? at : -1;
    };
    const float nan = __int_as_float(0x7fffffff);
    if (__all_sync(0xffffffffu, alike)) {
        if (!need) return;
        const int at = position(axis);
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            ulonglong2 x = make_ulonglong2(two(nan, nan), two(nan, nan)), y = x;
            if (at >= 0) {
                x = *reinterpret_cast<const ulonglong2*>(a.cos_t + (size_t)at * half + j + 4 * i);
                y = *reinterpret_cast<const ulonglong2*>(a.sin_t + (size_t)at * half + j + 4 * i);
            }
            c[2 * i] = x.x, c[2 * i + 1] = x.y, s[2 * i] = y.x, s[2 * i + 1] = y.y;
        }
        return;
    }
    for (int p = threadIdx.x & 31; p < half; p += 32) {
        const int at = position(a.pair_axis[p]);
        mine[p] = at >= 0 ? a.cos_t[(size_t)at * half + p] : nan;
        mine[half + p] = at >= 0 ? a.sin_t[(size_t)at * half + p] : nan;
    }
    __syncwarp();
    if (!need) return;
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const ulonglong2 x = *reinterpret_cast<const ulonglong2*>(mine + j + 4 * i), y = *reinterpret_cast<const ulonglong2*>(mine + half + j + 4 * i);
        c[2 * i] = x.x, c[2 * i + 1] = x.y, s[2 * i] = y.x, s[2 * i + 1] = y.y;
    }
}

// grid (tokens, blocks of a token's heads)
template <typename T, typename IN, typename W>
__global__ void __launch_bounds__(WIDE_THREADS, 8) axes_rope_write_wide_kernel(const Args a, const int group_shift) {
    constexpr int N = 16 / sizeof(T);
    extern __shared__ __align__(16) float turns_s[];                 // [warps][rd]
    pdl_enter_small();
    const int n = blockIdx.x, tid = threadIdx.x, half = a.rd / 2, group = 1 << group_shift;
    const int most = a.nq + 2 * a.nkv - 1, asked = (blockIdx.y * WIDE_THREADS + tid) >> group_shift, t = tid & (group - 1);
    if ((blockIdx.y * WIDE_THREADS + (tid & ~31)) >> group_shift > most) return;
    const int head = min(asked, most);                               // (a warp's threads behind the last head follow it and write nothing)
    const bool value = head >= a.nq + a.nkv;
    // this thread's two pieces
    const bool turned = t * N < half;
    const int i0 = turned ? t * N : a.rd + 2 * (t * N - half), i1 = turned ? i0 + half : i0 + N;
    Two x[N / 2], y[N / 2], c[N / 2], s[N / 2];
    const IN* src = (const IN*)a.qkv + (size_t)n * a.ld + (size_t)head * a.d;
    uint4 raw_x, raw_y;                                              // (unpacked when they are used: fewer registers, more blocks)
    if constexpr (sizeof(IN) == 2) raw_x = *reinterpret_cast<const uint4*>(src + i0), raw_y = *reinterpret_cast<const uint4*>(src + i1);
    else {
        load_piece<IN, N>(a, src + i0, x);
        load_piece<IN, N>(a, src + i1, y);
    }
    const W* gain = value ? nullptr : (const W*)(head < a.nq ? a.q_gain : a.k_gain);
    uint4 raw_gx, raw_gy;
    if constexpr (sizeof(W) == 2 && N == 8)
        if (gain) raw_gx = *reinterpret_cast<const uint4*>(gain + i0), raw_gy = *reinterpret_cast<const uint4*>(gain + i1);
    const bool cached = head >= a.nq;
    const int place = cached ? a.places[n] : 0, req = cached ? a.token_req[n] : 0;      // asked for beside the positions, not behind the tables
    load_turn<N>(a, n, i0, !value && turned, turns_s + (tid >> 5) * a.rd, c, s);
    T* dst = asked > most ? nullptr : target<T>(a, n, head, place, req);
    if constexpr (sizeof(IN) == 2) {
        unpack<IN, N>(raw_x, x);
        unpack<IN, N>(raw_y, y);
    }
    if (!value) {
        if (gain) {
            Two gx[N / 2], gy[N / 2], squares = 0;
            if constexpr (sizeof(W) == 2 && N == 8) {
                unpack<W, N>(raw_gx, gx);
                unpack<W, N>(raw_gy, gy);
            } else {
                load_gain<W, N>(gain + i0, gx);
                load_gain<W, N>(gain + i1, gy);
            }
#pragma unroll
            for (int i = 0; i < N / 2; ++i) squares = fma2(x[i], x[i], fma2(y[i], y[i], squares));
            const float2 both = apart(squares);
            float ssq = both.x + both.y;
            const uint32_t mine = group == 32 ? 0xffffffffu : ((1u << group) - 1u) << (tid & 31 & ~(group - 1));
            for (int o = group >> 1; o > 0; o >>= 1) ssq += __shfl_xor_sync(mine, ssq, o);
            const float inv = rsqrtf(ssq / (float)a.d + a.eps);
            const Two inv2 = two(inv, inv);
#pragma unroll
            for (int i = 0; i < N / 2; ++i) x[i] = mul2(mul2(x[i], inv2), gx[i]), y[i] = mul2(mul2(y[i], inv2), gy[i]);
        }
        if (turned) {
            const Two minus = two(-1.f, -1.f);
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                const Two was = x[i];
                x[i] = fma2(mul2(y[i], s[i]), minus, mul2(was, c[i]));
                y[i] = fma2(was, s[i], mul2(y[i], c[i]));
            }
        }
    }
    if (!dst) return;
    store_piece<T, N>(dst + i0, x);
    store_piece<T, N>(dst + i1, y);
}

}  // namespace axes
}  // namespace lily

using namespace lily;

LILY_API int lily_axes_rope_write(const void* qkv, int in_dtype, int splits, size_t stride, int ld, const void* q_gain, const void* k_gain,
                                  int gain_dtype, float eps, const float* cos_t, const float* sin_t, int table_rows,
                                  const int* positions, const int* pair_axis, int axes, int tokens, const int* places,
                                  const int* token_req, const int* block_table, int requests, int bt_stride, void* kv, int pages, void* q_out,
                                  int act_dtype, int nq, int nkv, int d, int rd, int page_size, cudaStream_t stream) {
    if (tokens == 0) return 0;
    LILY_REQUIRE(d > 0 && rd >= 0 && rd <= d && rd % 2 == 0, "axes_rope_write: rotary_dim %d does not fit head_dim %d", rd, d);
    LILY_REQUIRE(page_size > 0, "axes_rope_write: pages of %d places", page_size);
    LILY_REQUIRE(nq >= 0 && nkv >= 0 && nq + nkv > 0 && ld >= (nq + 2 * nkv) * d, "axes_rope_write: rows of %d numbers", ld);
    LILY_REQUIRE((q_gain == nullptr) == (k_gain == nullptr), "axes_rope_write: q and k gains come together");
    LILY_REQUIRE(act_dtype == kF32 || act_dtype == kBF16, "axes_rope_write: dtype %d", act_dtype);
    LILY_REQUIRE(in_dtype == act_dtype || in_dtype == kF32, "axes_rope_write: products are of the cache's dtype or float32");
    LILY_REQUIRE(act_dtype == kBF16 || gain_dtype == kF32 || q_gain == nullptr, "axes_rope_write: float32 heads keep float32 gains");
    LILY_REQUIRE(splits >= 1 && (splits == 1 || in_dtype == kF32), "axes_rope_write: partial sums are float32");
    int page_shift = -1;
    if ((page_size & (page_size - 1)) == 0)
        for (page_shift = 0; 1 << page_shift < page_size;) ++page_shift;
    const axes::Args a{qkv, stride, splits, ld, q_gain, k_gain, eps, cos_t, sin_t, table_rows, positions, pair_axis, axes, tokens, places, token_req,
                       block_table, requests, bt_stride, kv, pages, q_out, nq, nkv, d, rd, page_size, page_shift};
    const int bytes = act_dtype == kBF16 ? 2 : 4, piece = 16 / bytes, group = d / (2 * piece);
    int shift = 0;
    while (1 << shift < group) ++shift;
    const uintptr_t where = (uintptr_t)qkv | (uintptr_t)kv | (uintptr_t)q_out | (uintptr_t)q_gain | (uintptr_t)k_gain |
                            (uintptr_t)cos_t | (uintptr_t)sin_t | (uintptr_t)pair_axis;
    // Whole pieces of 16 bytes on every side; else, and for heads that are no power of two of pieces, a warp a head.  Measured, us, in pieces / a warp a
    // head, on the same operands, other ones each call: 2,048 tokens of 48 heads of 128 in bfloat16 with gains 13.7 / 38.7 (axes in turn 15.9 / 38.1), without 11.4 / 38.7 (13.6 / 37.9),
    // 8,192 tokens with gains 54.8 / 153, eight tokens 2.4 / 3.4, from four planes 3.2 / 5.4; float32 without gains, 1,000 tokens of 24 heads of 128 with half of each turned
    // 8.1 / 10.0, of 64 5.1 / 7.2.
    const bool wide = d % (2 * piece) == 0 && 1 << shift == group && group <= 32 && rd % (2 * piece) == 0 && ld % piece == 0 &&
                      (in_dtype == act_dtype || ld % 4 == 0) && (size_t)stride % 4 == 0 && where % 16 == 0;
    const dim3 grid = wide ? dim3(tokens, (unsigned)((((nq + 2 * nkv) << shift) + axes::WIDE_THREADS - 1) / axes::WIDE_THREADS)) : dim3(tokens, (nq + 2 * nkv + 3) / 4);
#define LAUNCH(T, IN, W)                                                                                                        \
    do {                                                                                                                        \
        if (wide) launch_pdl(axes::axes_rope_write_wide_kernel<T, IN, W>, grid, dim3(axes::WIDE_THREADS), axes::WIDE_THREADS / 32 * rd * sizeof(float), stream, a, shift); \
        else launch_pdl(axes::axes_rope_write_kernel<T, IN, W>, grid, dim3(128), 0, stream, a);                                 \
    } while (0)
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
