// A K/V cache in pages of 8-bit codes: rows are quantised as they are written, and read back as values.
//
// A row is one token of one K/V head: D codes of one byte that share a scale, kept in fp32.
//   e4m3   scale = 2^e with the smallest e for which max|x| <= 448 * 2^e: dividing by it is exact, so a code is x rounded
//          once, to four significant bits
//   int8   scale = max|x| * (1/127) in fp32, code = x / scale rounded to the nearest integer (IEEE division, ties to even)
// The scale is 2^-126 at least, so that it and its reciprocal are normal numbers.  A row with an infinity or a NaN in it
// gets the scale NaN and zero codes: it reads back as NaN and makes NaN of the attention rows that see it, of no others.
// 32-bit scales cost 4 bytes a row beside 64 to 256 of codes; powers of two would fit a byte, the int8 scales would not.
//
// Pages: k, v [pages, kv_heads, page_size, D] bytes, scales [pages, kv_heads, page_size].  The page table [batch, table_len]
// says where token `pos` of a sequence lies: entry pos / page_size, place pos % page_size.  An entry outside [0, pages), or
// a position beyond the table, is never followed: the row is left out and KV_ERR_PAGE reported, in a word of its own, since a
// report in the word for waits that ran out would stop what is queued behind, and the sequences that are not concerned.
//
// Both kernels' bound: HBM.  A lane holds eight elements, so a row is D / 8 lanes side by side and every access is 16
// (values) or 8 (codes) contiguous bytes a lane; K and V of KV_MOVE_STEPS rows are requested before the first is worked on.  A CTA
// stays inside one head of one sequence, so that only it divides, and loads that hang on a page come behind those that do not: a
// prompt of 8 x 8 x 4096 rows, d 128, fp16 to e4m3 (201 MB) 56 -> 41 us to write, 35 to read.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "api_internal.h"
#include "ptx.cuh"

namespace txb {

enum : int { KV_E4M3 = 0, KV_INT8 = 1 };

struct KvPages {
    uint8_t *k, *v;
    float *ks, *vs;
    const int32_t *table;     // [batch, table_len]
    int64_t table_len;
    int pages, Hkv, page_shift;

    // Row index (in units of D codes, or of one scale) of token `pos` of sequence b and head h; -1 where there is none
    __device__ __forceinline__ int64_t row(int b, int h, int64_t pos) const
    {
        const int64_t entry = pos >> page_shift;
        const int page = pos >= 0 && entry < table_len ? __ldg(table + (int64_t)b * table_len + entry) : -1;
        const int64_t r = ((((int64_t)page * Hkv + h) << page_shift)) + (pos & ((1 << page_shift) - 1));
        return page >= 0 && page < pages ? r : -1;
    }
};

struct KvMoveParams {
    KvPages pages;
    void *k, *v;              // [batch, Hkv, tokens, D], fp16 or fp32: what is written, or where the values go
    const int32_t *start;     // optional [batch]: position of the call's token 0 (none: 0)
    const int32_t *counts;    // optional [batch]: how many of the call's tokens there are (none: all)
    const int32_t *pick;      // write only, optional [batch, tokens]: token t is row pick[b, t] of k and v
    int ctas;                 // CTAs that share a head of a sequence
    int tokens, src_tokens;   // src_tokens: rows a head of k and v has
    int *page_status;
};

// Eight values of a lane as they are in memory, and as floats
template <typename T>
struct KvRaw8 {
    uint4 u[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T *p)
    {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) u[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
    }
    __device__ __forceinline__ void floats(float *x) const
    {
        if constexpr (sizeof(T) == 2) {
            const uint32_t w[4] = {u[0].x, u[0].y, u[0].z, u[0].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                x[2 * i] = f.x; x[2 * i + 1] = f.y;
            }
        } else {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
                x[4 * i] = __uint_as_float(u[i].x); x[4 * i + 1] = __uint_as_float(u[i].y);
                x[4 * i + 2] = __uint_as_float(u[i].z); x[4 * i + 3] = __uint_as_float(u[i].w);
            }
        }
    }
};
__device__ __forceinline__ void kv_store8(__half *p, const float *x)
{
    __stcs(reinterpret_cast<uint4 *>(p), make_uint4(ptx::pack_half2(x[0], x[1]), ptx::pack_half2(x[2], x[3]),
                                                    ptx::pack_half2(x[4], x[5]), ptx::pack_half2(x[6], x[7])));
}
__device__ __forceinline__ void kv_store8(float *p, const float *x)
{
#pragma unroll
    for (int i = 0; i < 2; ++i) __stcs(reinterpret_cast<float4 *>(p) + i, make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]));
}

// Scale of a row whose largest magnitude has the bits `top` (a positive float's bits are ordered as the float is)
template <int FMT>
__device__ __forceinline__ float kv_scale(uint32_t top)
{
    if (top >= 0x7f800000u) return __int_as_float(0x7fc00000);
    if constexpr (FMT == KV_E4M3) {
        // 448 = 1.75 * 2^8
        const int e = (int)(top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
        return __int_as_float(max(e, 1) << 23);
    } else {
        return fmaxf(__uint_as_float(top) * (1.f / 127.f), 1.17549435e-38f);
    }
}

// Eight codes of eight values; zero for a row without a finite scale
template <int FMT>
__device__ __forceinline__ uint2 kv_codes8(const float *x, float scale)
{
    uint2 w = make_uint2(0u, 0u);
    if (!(scale < INFINITY)) return w;
    uint32_t *out = &w.x;
    if constexpr (FMT == KV_E4M3) {
        const float inv = __int_as_float((254 << 23) - __float_as_int(scale));      // 2^-e, exactly
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const __nv_fp8x2_storage_t a = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i] * inv, x[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
            const __nv_fp8x2_storage_t b = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * i + 2] * inv, x[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
            out[i] = (uint32_t)a | (uint32_t)b << 16;
        }
    } else {
        // Products with the reciprocal are within 2^-22 of the quotients relatively, 2^-15 absolutely: where one is further
        // than that from the middle of two codes, both round the same way.  Elsewhere the division decides (with eight divisions
        // a lane the prompt above took 66 us to write, so 52).  2^23 + 2^22 added to a number leaves its nearest
        // integer in the low bits.
        const float inv = __frcp_rn(scale);
        constexpr float kMagic = 12582912.f;
        uint32_t n[8];
        bool close = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float q = x[i] * inv, r = q + kMagic;
            close |= fabsf(q - (r - kMagic)) > 0.4999f;
            n[i] = __float_as_uint(r);
        }
        if (close)
#pragma unroll
            for (int i = 0; i < 8; ++i) n[i] = __float_as_uint(__fdiv_rn(x[i], scale) + kMagic);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            out[i] = __byte_perm(__byte_perm(n[4 * i], n[4 * i + 1], 0x0040), __byte_perm(n[4 * i + 2], n[4 * i + 3], 0x0040), 0x5410);
    }
    return w;
}

// Two codes (the low 16 bits) as an fp16 pair: both formats' values are fp16 numbers
__device__ __forceinline__ uint32_t kv_e4m3x2_half2(uint32_t two)
{
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(two));
    return r;
}
__device__ __forceinline__ uint32_t kv_e4m3x2_half2_hi(uint32_t two)
{
    uint32_t r;
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(two));
    return r;
}
// Bytes 0, 1 (sel 0x4140) or 2, 3 (sel 0x4342) of four int8 codes whose sign bits are flipped: 0x64uu is the fp16 number
// 1024 + u, and u = code + 128
template <int SEL>
__device__ __forceinline__ uint32_t kv_int8x2_half2(uint32_t flipped)
{
    const uint32_t biased = __byte_perm(flipped, 0x64646464u, SEL);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&biased), __half2half2(__ushort_as_half((unsigned short)0x6480)));
    return *reinterpret_cast<const uint32_t *>(&r);
}
// Four codes as two fp16 pairs, in order
template <int FMT>
__device__ __forceinline__ void kv_halves(uint32_t w, uint32_t &lo, uint32_t &hi)
{
    if constexpr (FMT == KV_E4M3) {
        lo = kv_e4m3x2_half2(w);
        hi = kv_e4m3x2_half2_hi(w);
    } else {
        const uint32_t f = w ^ 0x80808080u;
        lo = kv_int8x2_half2<0x4140>(f);
        hi = kv_int8x2_half2<0x4342>(f);
    }
}
template <int FMT>
__device__ __forceinline__ void kv_values4(uint32_t w, float scale, float *x)
{
    uint32_t h[2];
    kv_halves<FMT>(w, h[0], h[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[i]));
        x[2 * i] = f.x * scale; x[2 * i + 1] = f.y * scale;
    }
}

constexpr int KV_MOVE_THREADS = 256, KV_MOVE_STEPS = 2;

// The head of a sequence a CTA works on, and the tokens of one of its lanes: t0, t0 + step, ...
template <int D>
struct KvMoveItem {
    static constexpr int STEP = KV_MOVE_THREADS / (D / 8), PER_CTA = STEP * KV_MOVE_STEPS;
    int64_t bh, start;
    int b, h, t0, count;
    __device__ __forceinline__ KvMoveItem(const KvMoveParams &p)
    {
        const int bh_ = (int)(blockIdx.x / (unsigned)p.ctas);
        bh = bh_;
        b = bh_ / p.pages.Hkv;
        h = bh_ - b * p.pages.Hkv;
        t0 = (int)(blockIdx.x - (unsigned)bh_ * p.ctas) * PER_CTA + (int)threadIdx.x / (D / 8);
        count = p.counts ? min(__ldg(p.counts + b), p.tokens) : p.tokens;
        start = p.start ? __ldg(p.start + b) : 0;
    }
};

template <typename T, int FMT, int D>
__global__ void __launch_bounds__(KV_MOVE_THREADS) kv_write_kernel(const KvMoveParams p)
{
    constexpr int LPR = D / 8, STEPS = KV_MOVE_STEPS;
    const int gl = threadIdx.x % LPR;
    const KvMoveItem<D> item(p);
    KvRaw8<T> raw[STEPS][2];
    int64_t to[STEPS];
    bool wanted[STEPS];
    // all loads first: what depends on one of them comes behind the last
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int t = item.t0 + s * item.STEP;
        wanted[s] = t < item.count;
        int from = wanted[s] ? t : -1;
        if (p.pick && wanted[s]) from = __ldg(p.pick + (int64_t)item.b * p.tokens + t);
        const bool there = from >= 0 && from < p.src_tokens;
        if (there) {
            const int64_t at = (item.bh * p.src_tokens + from) * D + gl * 8;
            raw[s][0].load(static_cast<const T *>(p.k) + at);
            raw[s][1].load(static_cast<const T *>(p.v) + at);
        }
        to[s] = there ? p.pages.row(item.b, item.h, item.start + t) : -1;
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        if (wanted[s] && to[s] < 0 && gl == 0) ptx::report(p.page_status, KV_ERR_PAGE);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            float x[8];
            uint32_t top = 0;
            raw[s][kv].floats(x);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
#pragma unroll
            for (int w = LPR / 2; w > 0; w >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, w));
            if (to[s] < 0) continue;
            const float scale = kv_scale<FMT>(top);
            uint8_t *codes = kv ? p.pages.v : p.pages.k;
            float *scales = kv ? p.pages.vs : p.pages.ks;
            *reinterpret_cast<uint2 *>(codes + to[s] * D + gl * 8) = kv_codes8<FMT>(x, scale);
            if (gl == 0) scales[to[s]] = scale;
        }
    }
}

// Rows beyond a sequence's count are left as they were.
template <typename T, int FMT, int D>
__global__ void __launch_bounds__(KV_MOVE_THREADS) kv_read_kernel(const KvMoveParams p)
{
    constexpr int LPR = D / 8, STEPS = KV_MOVE_STEPS;
    const int gl = threadIdx.x % LPR;
    const KvMoveItem<D> item(p);
    uint2 c[STEPS][2];
    float scale[STEPS][2];
    bool ok[STEPS];
    int64_t rows[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int t = item.t0 + s * item.STEP;
        rows[s] = t < item.count ? p.pages.row(item.b, item.h, item.start + t) : -1;
        ok[s] = false;
        if (t < item.count && rows[s] < 0 && gl == 0) ptx::report(p.page_status, KV_ERR_PAGE);
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int64_t from = rows[s];
        if (from < 0) continue;
        ok[s] = true;
        c[s][0] = __ldcs(reinterpret_cast<const uint2 *>(p.pages.k + from * D + gl * 8));
        c[s][1] = __ldcs(reinterpret_cast<const uint2 *>(p.pages.v + from * D + gl * 8));
        scale[s][0] = __ldg(p.pages.ks + from);
        scale[s][1] = __ldg(p.pages.vs + from);
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        if (!ok[s]) continue;
        const int64_t at = (item.bh * p.tokens + item.t0 + s * item.STEP) * D + gl * 8;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            float x[8];
            kv_values4<FMT>(c[s][kv].x, scale[s][kv], x);
            kv_values4<FMT>(c[s][kv].y, scale[s][kv], x + 4);
            kv_store8(static_cast<T *>(kv ? p.v : p.k) + at, x);
        }
    }
}

}  // namespace txb
