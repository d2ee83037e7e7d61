// A paged cache held in four bits (four.cuh says how it lies): what writes it and what reads it as numbers again.
//
// Writing: a head x of a token, y = x r g with r = (mean x^2 + eps)^(-1/2) where there are gains, the first rd features turned by halves
//   (y_j, y_(j + rd/2)) <- (y_j c - y_(j + rd/2) s, y_(j + rd/2) c + y_j s),   c, s = tables[position][j],
// queries to their row of `q_out`; of keys and values each group of 64 features becomes
//   step = bf16((max - min) / 15), lowest = bf16(min), code = min(15, max(0, rint((y - lowest) / step)))
// at the place `position` of the token's request.  A group that holds what is not finite, or whose spread is not, has NaN for both and reads as NaN.
//
// A number next to the border of two codes is a whole step off where its last bit falls the other way, so a token's codes are made a function of its numbers
// alone: the sum of squares is taken in 64 bits (squares of float32 numbers are exact there, and no order of adding them up shows in the root's 24 bits), and every other
// operation is one IEEE operation, none contracted.  The same token gets the same codes in a prompt, alone, and from a statement in plain operations.
#include "attention_args.cuh"
#include "four.cuh"

#include <cuda_fp16.h>

namespace lily {
namespace four {

struct WriteArgs {
    const void* qkv;                 // [tokens, (nq + 2 nkv) d]
    int ld;
    const void* q_gain;
    const void* k_gain;
    double eps, by_d;                // 1 / d
    const float* cos_t;              // [table_rows, rd / 2]
    const float* sin_t;
    int table_rows;
    const int* positions;            // [tokens]
    const int* token_req;
    const int* block_table;          // [requests, bt_stride]
    int requests, bt_stride;
    uint8_t* kv;
    int pages;
    void* q_out;                     // [tokens, nq * d]
    int nq, nkv, d, rd, page_size, tokens;
};

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&v)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    v[0] = low(raw.x), v[1] = high(raw.x), v[2] = low(raw.y), v[3] = high(raw.y);
    v[4] = low(raw.z), v[5] = high(raw.z), v[6] = low(raw.w), v[7] = high(raw.w);
}
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
    *reinterpret_cast<uint4*>(p) = make_uint4(bits(__floats2bfloat162_rn(v[0], v[1])), bits(__floats2bfloat162_rn(v[2], v[3])), bits(__floats2bfloat162_rn(v[4], v[5])),
                                              bits(__floats2bfloat162_rn(v[6], v[7])));
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}

// Half-precision numbers where bfloat16 ones would lie.
__device__ __forceinline__ void store_halves(void* p, const float (&v)[8], float by) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(v[2 * i] * by, v[2 * i + 1] * by);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

constexpr int WRITE_WARPS = 4;

// Eight codes min(15, max(0, rint((y - lowest) / step))) as a word.  The quotient by the step's reciprocal is within 2 10^-6 of the rounded one (two roundings of numbers up to 15 or so), so where no
// code is that near to the border of two it gives the same; else, and where the reciprocal is not a number, they are divided.
__device__ __forceinline__ uint32_t codes_of(const float (&y)[8], float lowest, float step) {
    const float by = __frcp_rn(step);
    uint32_t word = 0;
    bool near = !(step > 1e-30f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float t = fminf(fmaxf(__fmul_rn(__fsub_rn(y[i], lowest), by), 0.f), 15.f), whole = t + 12582912.f;      // 1.5 2^23: the sum's last bits are the nearest whole number
        near = near || fabsf(t - (whole - 12582912.f)) > 0.49999f;
        word |= (__float_as_uint(whole) & 15u) << (4 * i);
    }
    if (near) {
        word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) word |= (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(y[i], lowest), step)), 0.f), 15.f) << (4 * i);
    }
    return word;
}

// A thread eight features, d / 8 threads a head, 32 / (d / 8) heads a warp.  grid (blocks of a token's heads, tokens)
template <typename T, typename W, typename Q, bool WHOLE_PIECES>
__global__ void __launch_bounds__(32 * WRITE_WARPS) write_kernel(const WriteArgs a) {
    __shared__ __align__(16) float turn_s[WRITE_WARPS][256];
    pdl_enter_small();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, words = a.d / 8, per_warp = 32 / words;
    const int mine = min(lane / words, per_warp - 1), l = lane - mine * words;                 // (d = 192: lanes 24 to 31 have no word)
    const int n = blockIdx.y, asked = (blockIdx.x * WRITE_WARPS + warp) * per_warp + mine, most = a.nq + 2 * a.nkv;
    const bool in = asked < most && l < words;
    const int head = min(asked, most - 1), f = min(l, words - 1) * 8;
    const int kind = head < a.nq ? 0 : head < a.nq + a.nkv ? 1 : 2;
    float y[8];
    load8((const T*)a.qkv + (size_t)n * a.ld + (size_t)head * a.d + f, y);
    const W* gain = kind == 2 ? nullptr : (const W*)(kind ? a.k_gain : a.q_gain);
    const int pos = a.positions[n], req = kind ? a.token_req[n] : 0, half = a.rd / 2;
    const bool known = pos >= 0 && pos < a.table_rows, turned = kind != 2 && f < a.rd;
    const float *ct = a.cos_t + (size_t)(known ? pos : 0) * half, *st = a.sin_t + (size_t)(known ? pos : 0) * half;
    float c[8], sn[8], g[8];                             // asked for ahead of the sums
    if (WHOLE_PIECES && turned) {
        load8(ct + (f < half ? f : f - half), c);
        load8(st + (f < half ? f : f - half), sn);
    }
    if (gain) load8(gain + f, g);
    if (__any_sync(0xffffffffu, gain != nullptr)) {
        double squares = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) squares = fma((double)y[i], (double)y[i], squares);
        if (l >= words) squares = 0.0;
        // (a head of 192 features over 24 of 32 lanes: the others bring nothing)
        for (int o = words == 24 ? 16 : words >> 1; o > 0; o >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, o);
        if (gain) {
            const float r = (float)rsqrt(fma(squares, a.by_d, a.eps));
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = __fmul_rn(__fmul_rn(y[i], r), g[i]);
        }
    }
    float* row = turn_s[warp] + mine * a.d;
    if (l < words) store8(row + f, y);
    __syncwarp();
    if (turned) {
        const float nan = __int_as_float(0x7fffffff);
        if (WHOLE_PIECES) {                              // half a multiple of eight: a thread's features are of one half
            float other[8];
            load8(row + (f < half ? f + half : f - half), other);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float first = __fmul_rn(y[i], c[i]), second = __fmul_rn(other[i], sn[i]);
                y[i] = !known ? nan : f < half ? __fsub_rn(first, second) : __fadd_rn(first, second);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int e = f + i, j = e < half ? e : e - half;
                if (e >= a.rd) continue;
                const float first = __fmul_rn(y[i], ct[j]), second = __fmul_rn(row[e < half ? e + half : j], st[j]);
                y[i] = !known ? nan : e < half ? __fsub_rn(first, second) : __fadd_rn(first, second);
            }
        }
    }
    if (kind == 0 && in) store8((Q*)a.q_out + ((size_t)n * a.nq + head) * a.d + f, y);
    if (__all_sync(0xffffffffu, kind == 0)) return;
    // eight neighbouring lanes hold a group of 64 features
    float most_v = y[0], least = y[0];
    bool fine = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        most_v = fmaxf(most_v, y[i]);
        least = fminf(least, y[i]);
        fine = fine && isfinite(y[i]);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        most_v = fmaxf(most_v, __shfl_xor_sync(0xffffffffu, most_v, o));
        least = fminf(least, __shfl_xor_sync(0xffffffffu, least, o));
    }
    fine = (__ballot_sync(0xffffffffu, fine) >> (lane & 24) & 0xffu) == 0xffu;
    const __nv_bfloat16 step_b = __float2bfloat16_rn(__fmul_rn(__fsub_rn(most_v, least), (float)(1.0 / 15.0))), low_b = __float2bfloat16_rn(least);
    const float step = __bfloat162float(step_b), lowest = __bfloat162float(low_b);
    fine = fine && isfinite(step) && isfinite(lowest);
    if (kind == 0 || !in) return;
    const int at = pos >= 0 ? pos / a.page_size : -1;
    if (at < 0 || at >= a.bt_stride || (unsigned)req >= (unsigned)a.requests) return;
    const int page = a.block_table[(size_t)req * a.bt_stride + at];
    if ((unsigned)page >= (unsigned)a.pages) return;
    const uint32_t word = fine && step > 0.f ? codes_of(y, lowest, step) : 0u;
    const int groups = a.d / GROUP, slot = pos - at * a.page_size;
    uint8_t* rows = a.kv + (((size_t)page * a.nkv + (head - a.nq - (kind == 2 ? a.nkv : 0))) * 2 + (kind == 2)) * ((size_t)a.page_size * row_bytes(a.d));
    reinterpret_cast<uint32_t*>(rows + (size_t)slot * (a.d / 2))[kind == 1 ? key_word(l, groups) : value_word(l, groups)] = word;
    if ((l & 7) == 0) {
        const __nv_bfloat16 nan = __float2bfloat16_rn(__int_as_float(0x7fffffff));
        reinterpret_cast<uint32_t*>(rows + (size_t)a.page_size * (a.d / 2))[slot * groups + (l >> 3)] =
            bits(fine ? __halves2bfloat162(step_b, low_b) : __halves2bfloat162(nan, nan));
    }
}

// The same where all features are turned and heads are 64, 128 or 256 features: a thread a word and its partners', d / 16 threads a head, which so needs no exchange but for sums and extremes, and half as
// much work that is not its numbers'.  1,500 tokens of 32 heads over 8 of 128, with the pages as numbers behind: 16.8 us, 23.6 by the kernel above (8 tokens 5.5 and 5.8); what bounds it is instructions,
// 0.58 a cycle and scheduler, over blocks of one token.  grid (blocks of a token's heads, tokens)
template <typename T, typename W, typename Q, int D>
__global__ void __launch_bounds__(32 * WRITE_WARPS) write_turned_kernel(const WriteArgs a, const int page_shift) {
    constexpr int THREADS = D / 16, HALF = D / 2, G = D / GROUP;
    pdl_enter_small();
    const int n = blockIdx.y, t = threadIdx.x % THREADS, asked = blockIdx.x * (32 * WRITE_WARPS / THREADS) + threadIdx.x / THREADS, most = a.nq + 2 * a.nkv, lane = threadIdx.x & 31;
    const bool in = asked < most;
    const int head = min(asked, most - 1), kind = head < a.nq ? 0 : head < a.nq + a.nkv ? 1 : 2;
    const T* src = (const T*)a.qkv + (size_t)n * a.ld + (size_t)head * D + t * 8;
    float x[8], y[8], c[8], s[8];
    load8(src, x);
    load8(src + HALF, y);
    const int pos = a.positions[n], req = kind ? a.token_req[n] : 0;
    const bool known = pos >= 0 && pos < a.table_rows;
    if (kind != 2) {
        load8(a.cos_t + (size_t)(known ? pos : 0) * HALF + t * 8, c);
        load8(a.sin_t + (size_t)(known ? pos : 0) * HALF + t * 8, s);
    }
    const W* gain = kind == 2 ? nullptr : (const W*)(kind ? a.k_gain : a.q_gain);
    if (__any_sync(0xffffffffu, gain != nullptr)) {
        float gx[8], gy[8];
        if (gain) load8(gain + t * 8, gx), load8(gain + HALF + t * 8, gy);
        double squares = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) squares = fma((double)y[i], (double)y[i], fma((double)x[i], (double)x[i], squares));
#pragma unroll
        for (int o = THREADS / 2; o > 0; o >>= 1) squares += __shfl_xor_sync(0xffffffffu, squares, o);
        if (gain) {
            const float r = (float)rsqrt(fma(squares, 1.0 / D, a.eps));
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], r), gx[i]), y[i] = __fmul_rn(__fmul_rn(y[i], r), gy[i]);
        }
    }
    if (kind != 2) {
        const float nan = __int_as_float(0x7fffffff);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float was = x[i];
            x[i] = known ? __fsub_rn(__fmul_rn(was, c[i]), __fmul_rn(y[i], s[i])) : nan;
            y[i] = known ? __fadd_rn(__fmul_rn(y[i], c[i]), __fmul_rn(was, s[i])) : nan;
        }
    }
    if (kind == 0 && in) {
        Q* to = (Q*)a.q_out + ((size_t)n * a.nq + head) * D + t * 8;
        store8(to, x);
        store8(to + HALF, y);
    }
    if (__all_sync(0xffffffffu, kind == 0)) return;
    // extremes of the groups of 64 features: eight threads' words, or (64 features a head) both words of four
    float most_x = x[0], least_x = x[0], most_y = y[0], least_y = y[0];
    bool fine_x = true, fine_y = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        most_x = fmaxf(most_x, x[i]), least_x = fminf(least_x, x[i]), most_y = fmaxf(most_y, y[i]), least_y = fminf(least_y, y[i]);
        fine_x = fine_x && isfinite(x[i]), fine_y = fine_y && isfinite(y[i]);
    }
    if (D == 64) {
        most_x = most_y = fmaxf(most_x, most_y), least_x = least_y = fminf(least_x, least_y);
        fine_x = fine_y = fine_x && fine_y;
    }
    constexpr int SPAN = D == 64 ? 4 : 8;
#pragma unroll
    for (int o = SPAN / 2; o > 0; o >>= 1) {
        most_x = fmaxf(most_x, __shfl_xor_sync(0xffffffffu, most_x, o)), least_x = fminf(least_x, __shfl_xor_sync(0xffffffffu, least_x, o));
        if (D != 64) most_y = fmaxf(most_y, __shfl_xor_sync(0xffffffffu, most_y, o)), least_y = fminf(least_y, __shfl_xor_sync(0xffffffffu, least_y, o));
    }
    if (D == 64) most_y = most_x, least_y = least_x;
    constexpr uint32_t ALL = (1u << SPAN) - 1;
    fine_x = (__ballot_sync(0xffffffffu, fine_x) >> (lane & ~(SPAN - 1)) & ALL) == ALL;
    fine_y = D == 64 ? fine_x : (__ballot_sync(0xffffffffu, fine_y) >> (lane & ~(SPAN - 1)) & ALL) == ALL;
    if (kind == 0 || !in) return;
    const int at = pos < 0 ? -1 : page_shift >= 0 ? pos >> page_shift : pos / a.page_size;
    if (at < 0 || at >= a.bt_stride || (unsigned)req >= (unsigned)a.requests) return;
    const int page = a.block_table[(size_t)req * a.bt_stride + at];
    if ((unsigned)page >= (unsigned)a.pages) return;
    const int slot = pos - at * a.page_size;
    uint8_t* rows = a.kv + (((size_t)page * a.nkv + (head - a.nq - (kind == 2 ? a.nkv : 0))) * 2 + (kind == 2)) * ((size_t)a.page_size * row_bytes(D));
    uint32_t* words = reinterpret_cast<uint32_t*>(rows + (size_t)slot * (D / 2));
    uint32_t* held = reinterpret_cast<uint32_t*>(rows + (size_t)a.page_size * (D / 2)) + slot * G;
    auto put = [&](const float (&v)[8], int l, float most_v, float least, bool fine, bool says) {
        const __nv_bfloat16 step_b = __float2bfloat16_rn(__fmul_rn(__fsub_rn(most_v, least), (float)(1.0 / 15.0))), low_b = __float2bfloat16_rn(least), nan = __float2bfloat16_rn(__int_as_float(0x7fffffff));
        const float step = __bfloat162float(step_b), lowest = __bfloat162float(low_b);
        fine = fine && isfinite(step) && isfinite(lowest);
        words[kind == 1 ? key_word(l, G) : value_word(l, G)] = fine && step > 0.f ? codes_of(v, lowest, step) : 0u;
        if (says) held[l >> 3] = bits(fine ? __halves2bfloat162(step_b, low_b) : __halves2bfloat162(nan, nan));
    };
    put(x, t, most_x, least_x, fine_x, (t & 7) == 0);
    put(y, t + THREADS, most_y, least_y, fine_y, D != 64 && (t & 7) == 0);
}

// Pages as numbers, lowest + step code in one rounding: of every page that a block table names to [requests, width, 2, nkv, page_size, d] (``compact`` false), or of the pages
// that portions of prompts see, one request's behind the other's, [pages, 2, nkv, page_size, d], with a block table of them and zeros behind a request's last place.
// Eight threads a place and kind, each with the words that lie side by side, one a group.  ``spans`` [2 (keys, values), requests, nkv]: half-precision numbers times powers of two (attention_args.cuh).
// grid (pages, requests, kv heads x 2)
template <typename T, int G, bool HALVES>
__global__ void __launch_bounds__(256) values_kernel(const uint8_t* __restrict__ kv, int pages, const int* __restrict__ block_table, int width, T* __restrict__ out, int nkv, int page_size,
                                                     const int* __restrict__ cu, const int* __restrict__ prefix, int* __restrict__ table_out, int table_width, int most_pages, const unsigned* __restrict__ spans) {
    constexpr int D = G * GROUP;
    __shared__ int sum_s[8];
    pdl_enter_small();
    const int r = blockIdx.y, at = blockIdx.x, head = blockIdx.z >> 1, value = blockIdx.z & 1;
    int page = at < width ? block_table[(size_t)r * width + at] : 0;
    size_t to = (size_t)r * width + at;
    int places = page_size;
    if (cu) {
        // pages of the requests ahead of this one
        auto places_of = [&](int i) { return cu[i + 1] > cu[i] ? prefix[i] + cu[i + 1] - cu[i] : 0; };
        const int total = places_of(r);
        if (at >= (total + page_size - 1) / page_size) return;
        places = min(page_size, total - at * page_size);
        int before = 0;
        if (r > 0) {
            for (int i = threadIdx.x; i < r; i += 256) before += (places_of(i) + page_size - 1) / page_size;
            before = __reduce_add_sync(0xffffffffu, before);
            if ((threadIdx.x & 31) == 0) sum_s[threadIdx.x >> 5] = before;
            __syncthreads();
            before = 0;
            for (int w = 0; w < 8; ++w) before += sum_s[w];
        }
        to = (size_t)before + at;
        if (to >= (size_t)most_pages || at >= table_width) return;
        if (threadIdx.x == 0 && blockIdx.z == 0) table_out[(size_t)r * table_width + at] = (int)to;
    }
    if ((unsigned)page >= (unsigned)pages) page = 0;
    const uint8_t* rows = kv + (((size_t)page * nkv + head) * 2 + value) * ((size_t)page_size * row_bytes(D));
    const uint32_t *words = reinterpret_cast<const uint32_t*>(rows), *held = reinterpret_cast<const uint32_t*>(rows + (size_t)page_size * (D / 2));
    T* dst = out + ((to * 2 + value) * nkv + head) * ((size_t)page_size * D);
    const int i8 = threadIdx.x & 7;
    const float by = HALVES ? span_multiplier(spans[((size_t)value * gridDim.y + r) * nkv + head]) : 1.f;
#pragma unroll 2
    for (int slot = threadIdx.x >> 3; slot < page_size; slot += 32) {
        uint32_t w[G], h[G];
#pragma unroll
        for (int e = 0; e < G; ++e) w[e] = words[(size_t)slot * (D / 8) + i8 * G + e], h[e] = held[slot * G + e];
#pragma unroll
        for (int e = 0; e < G; ++e) {
            const int in = (i8 & 1) * G + e;              // a key's words of lane column i8 / 2: (j, h) one behind the other
            const int l = value ? 8 * e + i8 : 8 * (in >> 1) + 4 * (in & 1) + (i8 >> 1), j = l >> 3;
            const uint32_t of = G == 1 ? h[0] : G == 2 ? (j ? h[1] : h[0]) : G == 3 ? (j == 0 ? h[0] : j == 1 ? h[1] : h[G - 1]) : (j < 2 ? (j ? h[1] : h[0]) : (j == 2 ? h[2 % G] : h[G - 1]));
            float v[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] = slot < places ? fmaf(__uint_as_float((w[e] >> (4 * c) & 15u) | 0x4B000000u) - 8388608.f, low(of), high(of)) : 0.f;
            if (HALVES) store_halves(dst + (size_t)slot * D + l * 8, v, by);
            else store8(dst + (size_t)slot * D + l * 8, v);
        }
    }
}

// What portions attend with in half precision (attention_args.cuh).  blocks [0, query_blocks): queries, times the power of two of their token and head, eight numbers a thread and d / 8 threads a head;
// the others, a block a (page, request) and a warp a kv head and kind at a time: a bound of the keys' or values' magnitudes from their steps and lowest values (lowest + 15 step, or lowest), as bits that
// are compared as whole numbers.  What is no number counts for nothing.
__global__ void __launch_bounds__(256) halves_kernel(const __nv_bfloat16* __restrict__ q, size_t heads, __nv_bfloat16* __restrict__ out, float* __restrict__ units, int query_blocks,
                                                     const uint8_t* __restrict__ kv, int pages, const int* __restrict__ block_table, int width, int nkv, int d, int page_size,
                                                     const int* __restrict__ cu, const int* __restrict__ prefix, int requests, int most, unsigned* __restrict__ spans) {
    pdl_enter_small();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float m = 0.f;
    auto take = [&](float v) {
        v = fabsf(v);
        if (v <= 3e38f) m = fmaxf(m, v);
    };
    if ((int)blockIdx.x < query_blocks) {
        const int words = d / 8, per_warp = 32 / words, mine = lane / words, l = lane - mine * words;      // (d = 192: lanes 24 to 31 have no word)
        const size_t head = ((size_t)blockIdx.x * 8 + warp) * per_warp + mine;
        const bool in = mine < per_warp && head < heads;
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (in) raw = *reinterpret_cast<const uint4*>(q + head * d + l * 8);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[2 * i] = low(w[i]), v[2 * i + 1] = high(w[i]);
        uint32_t most_w = 0;                                          // magnitudes as whole numbers, two at a time; those of infinities and of what is no number are the largest
#pragma unroll
        for (int i = 0; i < 4; ++i) most_w = __vmaxu2(most_w, w[i] & 0x7fff7fffu);
        m = __uint_as_float(max(most_w & 0xffffu, most_w >> 16) << 16);
        if (!(m <= 3e38f)) {
            m = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) take(v[i]);
        }
        for (int o = words == 24 ? 16 : words >> 1; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (!in) return;
        store_halves(out + head * d + l * 8, v, span_multiplier(__float_as_uint(m)));
        if (l == 0) units[head] = span_unit(__float_as_uint(m));
        return;
    }
    const int r = ((int)blockIdx.x - query_blocks) / most, at = ((int)blockIdx.x - query_blocks) % most, groups = d / GROUP;
    const int total = cu[r + 1] > cu[r] ? prefix[r] + cu[r + 1] - cu[r] : 0, places = min(page_size, total - at * page_size);
    if (places <= 0) return;
    int page = at < width ? block_table[(size_t)r * width + at] : 0;
    if ((unsigned)page >= (unsigned)pages) page = 0;
    const size_t rows = (size_t)page_size * row_bytes(d);
    for (int which = warp; which < 2 * nkv; which += 8) {            // (head, kind)
        const uint32_t* held = reinterpret_cast<const uint32_t*>(kv + ((size_t)page * nkv * 2 + which) * rows + (size_t)page_size * (d / 2));
        m = 0.f;
#pragma unroll 4
        for (int i = lane; i < places * groups; i += 32) {
            const uint32_t h = held[i];
            take(high(h)), take(fmaf(15.f, low(h), high(h)));
        }
        const unsigned bits = __reduce_max_sync(0xffffffffu, __float_as_uint(m));
        if (lane == 0 && bits) atomicMax(spans + ((size_t)(which & 1) * requests + r) * nkv + (which >> 1), bits);
    }
}

// Zeros to the spans and the block table, and the portions' tiles, which come with the launch: a copy of them would have 2,048 tokens wait 6 us.  (A kernel and not a memset, which the one behind it waits for
// in full: portions of 2,048 tokens 70.5 us in a graph, 74.2 with a memset.)
constexpr int MOST_TILES = 480;
struct Tiles { int n, of[2 * MOST_TILES]; };
__global__ void __launch_bounds__(256) zero_kernel(unsigned* __restrict__ words, int n, int* __restrict__ tiles_out, const __grid_constant__ Tiles tiles) {
    pdl_enter_small();
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) words[i] = 0u;
    if (i < 2 * tiles.n) tiles_out[i] = tiles.of[i];
}

constexpr int F32_TO_BF16 = 2;               // a dtype of heads: float32 ones, whose queries leave as bfloat16

inline bool head_fits(int d) { return d >= GROUP && d <= 256 && d % GROUP == 0; }

}  // namespace four
}  // namespace lily

using namespace lily;

LILY_API int lily_qk_norm_rope_write4(const void* qkv, int dtype, int ld, const void* q_gain, const void* k_gain, int gain_dtype, double eps, const float* cos_t, const float* sin_t,
                                      int table_rows, const int* positions, int tokens, const int* token_req, const int* block_table, int requests, int bt_stride, void* kv, int pages,
                                      void* q_out, int nq, int nkv, int d, int rd, int page_size, cudaStream_t stream) {
    if (tokens == 0) return 0;
    LILY_REQUIRE(four::head_fits(d), "qk_norm_rope_write4: heads of 64, 128, 192 or 256 features, not %d", d);
    LILY_REQUIRE(rd >= 0 && rd <= d && rd % 2 == 0 && (rd == 0 || (cos_t && sin_t && table_rows > 0)), "qk_norm_rope_write4: rotary_dim %d does not fit head_dim %d, or tables of %d positions", rd, d, table_rows);
    LILY_REQUIRE(page_size > 0 && tokens > 0 && tokens <= 65535 * 32, "qk_norm_rope_write4: %d tokens, pages of %d places", tokens, page_size);
    LILY_REQUIRE(nq >= 0 && nkv >= 0 && nq + nkv > 0 && ld >= (nq + 2 * nkv) * d, "qk_norm_rope_write4: rows of %d numbers", ld);
    LILY_REQUIRE((q_gain == nullptr) == (k_gain == nullptr), "qk_norm_rope_write4: q and k gains come together");
    LILY_REQUIRE(dtype == kF32 || dtype == kBF16 || dtype == four::F32_TO_BF16, "qk_norm_rope_write4: dtype %d", dtype);
    LILY_REQUIRE(dtype != kF32 || gain_dtype == kF32 || !q_gain, "qk_norm_rope_write4: float32 heads keep float32 gains");
    const uintptr_t where = (uintptr_t)qkv | (uintptr_t)kv | (uintptr_t)q_out | (uintptr_t)q_gain | (uintptr_t)k_gain | (uintptr_t)cos_t | (uintptr_t)sin_t;
    LILY_REQUIRE(where % 16 == 0 && ld % 8 == 0, "qk_norm_rope_write4: tensors on boundaries of sixteen bytes");
    const int per_block = four::WRITE_WARPS * (32 / (d / 8));
    const bool pieces = rd % 16 == 0;
    int shift = 0;
    while (1 << shift < page_size) ++shift;
    if (1 << shift != page_size) shift = -1;
    for (int t0 = 0; t0 < tokens; t0 += 65535) {
        const int n = min(65535, tokens - t0), item = dtype == kBF16 ? 2 : 4, q_item = dtype == kF32 ? 4 : 2;
        const four::WriteArgs a{(const char*)qkv + (size_t)t0 * ld * item, ld, q_gain, k_gain, eps, 1.0 / d, cos_t, sin_t, table_rows, positions + t0, token_req + t0, block_table, requests, bt_stride,
                                (uint8_t*)kv, pages, (char*)q_out + (size_t)t0 * nq * d * q_item, nq, nkv, d, rd, page_size, n};
        const dim3 grid((nq + 2 * nkv + per_block - 1) / per_block, n), turned((nq + 2 * nkv + 2 * per_block - 1) / (2 * per_block), n);
#define TURNED(T, W, Q, D) launch_pdl(four::write_turned_kernel<T, W, Q, D>, turned, dim3(32 * four::WRITE_WARPS), 0, stream, a, shift)
#define LAUNCH(T, W, Q)                                                                                                           \
    do {                                                                                                                          \
        if (rd == d && d == 64) TURNED(T, W, Q, 64);                                                                                  \
        else if (rd == d && d == 128) TURNED(T, W, Q, 128);                                                                           \
        else if (rd == d && d == 256) TURNED(T, W, Q, 256);                                                                           \
        else if (pieces) launch_pdl(four::write_kernel<T, W, Q, true>, grid, dim3(32 * four::WRITE_WARPS), 0, stream, a);                  \
        else launch_pdl(four::write_kernel<T, W, Q, false>, grid, dim3(32 * four::WRITE_WARPS), 0, stream, a);                        \
    } while (0)
        if (dtype == kF32) LAUNCH(float, float, float);
        else if (dtype == four::F32_TO_BF16 && gain_dtype == kBF16) LAUNCH(float, __nv_bfloat16, __nv_bfloat16);
        else if (dtype == four::F32_TO_BF16) LAUNCH(float, float, __nv_bfloat16);
        else if (gain_dtype == kBF16) LAUNCH(__nv_bfloat16, __nv_bfloat16, __nv_bfloat16);
        else LAUNCH(__nv_bfloat16, float, __nv_bfloat16);
#undef LAUNCH
#undef TURNED
        LILY_CHECK_LAUNCH("qk_norm_rope_write4");
    }
    return 0;
}

// spans: null, or the largest magnitudes of keys and values, for numbers in half precision (lily_halves4).  cu, prefix, table_out: null, or of a step's portions (offsets of their tokens, tokens cached ahead of them, a block
// table [requests, table_width] of the pages written, of which there is room for `most_pages`).
LILY_API int lily_cache4_values(const void* kv, int pages, const int* block_table, int requests, int width, void* out, int dtype, int nkv, int d, int page_size, const int* cu,
                                const int* prefix, int* table_out, int table_width, int most_pages, const unsigned* spans, cudaStream_t stream) {
    if (requests == 0 || width == 0) return 0;
    LILY_REQUIRE(four::head_fits(d), "cache4_values: heads of 64, 128, 192 or 256 features, not %d", d);
    LILY_REQUIRE(page_size > 0 && nkv > 0 && nkv <= 32767 && requests > 0 && requests <= 65535 && width > 0, "cache4_values: %d requests, %d kv heads, pages of %d places", requests, nkv, page_size);
    LILY_REQUIRE(((uintptr_t)kv | (uintptr_t)out) % 16 == 0, "cache4_values: tensors on boundaries of sixteen bytes");
    const dim3 grid(cu ? table_width : width, requests, 2 * nkv);
    if (grid.x == 0) return 0;
#define VALUES(T, G, HALVES) \
    launch_pdl(four::values_kernel<T, G, HALVES>, grid, dim3(256), 0, stream, (const uint8_t*)kv, pages, block_table, width, (T*)out, nkv, page_size, cu, prefix, table_out, table_width, most_pages, spans)
#define VALUES_OF(T, HALVES)                 \
    do {                                     \
        if (d == 64) VALUES(T, 1, HALVES);   \
        else if (d == 128) VALUES(T, 2, HALVES); \
        else if (d == 192) VALUES(T, 3, HALVES); \
        else VALUES(T, 4, HALVES);           \
    } while (0)
    LILY_REQUIRE(!spans || dtype == kBF16, "cache4_values: numbers in half precision lie where bfloat16 ones would");
    if (dtype == kF32) VALUES_OF(float, false);
    else if (spans) VALUES_OF(__nv_bfloat16, true);
    else VALUES_OF(__nv_bfloat16, false);
#undef VALUES_OF
#undef VALUES
    LILY_CHECK_LAUNCH("cache4_values");
    return 0;
}

// What portions attend with in half precision (attention_args.cuh): the largest magnitudes of keys and values to `spans` [2, requests, nkv] (`zeroed` bytes from there on are set to zero first), the queries times powers
// of two to `out`, what undoes them to `units` [tokens, nq].  tiles: up to lily_halves4_tiles() of the portions' tiles, numbers of the host (requests, then offsets), which go to `tiles_out`.
LILY_API int lily_halves4_tiles() { return four::MOST_TILES; }
LILY_API int lily_halves4(const void* q, int tokens, int nq, const void* kv, int pages, const int* block_table, int requests, int width, int nkv, int d, int page_size, const int* cu, const int* prefix,
                          int most_pages, unsigned* spans, size_t zeroed, const int* tiles, int tile_count, int* tiles_out, void* out, float* units, cudaStream_t stream) {
    if (tokens == 0 || requests == 0) return 0;
    LILY_REQUIRE(four::head_fits(d) && page_size > 0 && nkv > 0 && nq > 0 && most_pages > 0 && (long long)requests * most_pages <= INT32_MAX / 2, "halves4: %d requests of up to %d pages", requests, most_pages);
    LILY_REQUIRE(((uintptr_t)q | (uintptr_t)out | (uintptr_t)kv) % 16 == 0, "halves4: tensors on boundaries of sixteen bytes");
    const size_t heads = (size_t)tokens * nq, a_block = 8 * (32 / (d / 8)), query_blocks = (heads + a_block - 1) / a_block;
    LILY_REQUIRE(query_blocks <= INT32_MAX / 2, "halves4: %d tokens", tokens);
    LILY_REQUIRE(zeroed >= (size_t)2 * requests * nkv * sizeof(unsigned) && zeroed % 4 == 0 && zeroed <= INT32_MAX, "halves4: %zu bytes of spans and tables", zeroed);
    LILY_REQUIRE(tile_count >= 0 && tile_count <= four::MOST_TILES && (tile_count == 0 || (tiles && tiles_out)), "halves4: %d tiles", tile_count);
    four::Tiles with;
    with.n = tile_count;
    for (int i = 0; i < 2 * tile_count; ++i) with.of[i] = tiles[i];
    launch_pdl(four::zero_kernel, dim3((unsigned)((max((int)(zeroed / 4), 2 * tile_count) + 255) / 256)), dim3(256), 0, stream, spans, (int)(zeroed / 4), tiles_out, with);
    LILY_CHECK_LAUNCH("halves4");
    launch_pdl(four::halves_kernel, dim3((unsigned)query_blocks + requests * most_pages), dim3(256), 0, stream, (const __nv_bfloat16*)q, heads, (__nv_bfloat16*)out, units, (int)query_blocks,
               (const uint8_t*)kv, pages, block_table, width, nkv, d, page_size, cu, prefix, requests, most_pages, spans);
    LILY_CHECK_LAUNCH("halves4");
    return 0;
}
