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
// a position beyond the table, is never followed: the row is left out and the failure word says KV_ERR_PAGE.
//
// Both kernels' bound: HBM.  A lane holds eight elements, so a row is D / 8 lanes side by side and every access is 16
// (values) or 8 (codes) contiguous bytes a lane; K and V of two rows are requested before the first is worked on.
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
        if (pos < 0 || entry >= table_len) return -1;
        const int page = __ldg(table + (int64_t)b * table_len + entry);
        if (page < 0 || page >= pages) return -1;
        return ((((int64_t)page * Hkv + h) << page_shift)) + (pos & ((1 << page_shift) - 1));
    }
};

struct KvMoveParams {
    KvPages pages;
    void *k, *v;              // [batch, Hkv, tokens, D], fp16 or fp32: what is written, or where the values go
    const int32_t *start;     // optional [batch]: position of the call's token 0 (none: 0)
    const int32_t *counts;    // optional [batch]: how many of the call's tokens there are (none: all)
    const int32_t *pick;      // write only, optional [batch, tokens]: token t is row pick[b, t] of k and v
    int64_t rows;             // batch * Hkv * tokens
    int tokens, src_tokens;   // src_tokens: rows a head of k and v has
    int *status;
};

// Eight values of a lane, whatever their type
__device__ __forceinline__ void kv_load8(const __half *p, float *x)
{
    const uint4 u = __ldcs(reinterpret_cast<const uint4 *>(p));
    const __half2 *h = reinterpret_cast<const __half2 *>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h[i]);
        x[2 * i] = f.x; x[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void kv_load8(const float *p, float *x)
{
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float4 f = __ldcs(reinterpret_cast<const float4 *>(p) + i);
        x[4 * i] = f.x; x[4 * i + 1] = f.y; x[4 * i + 2] = f.z; x[4 * i + 3] = f.w;
    }
}
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

// Four codes of four values; zero for a row without a finite scale
template <int FMT>
__device__ __forceinline__ uint32_t kv_codes4(const float *x, float scale)
{
    if (!(scale < INFINITY)) return 0u;
    if constexpr (FMT == KV_E4M3) {
        const float inv = __int_as_float((254 << 23) - __float_as_int(scale));      // 2^-e, exactly
        const __nv_fp8x2_storage_t a = __nv_cvt_float2_to_fp8x2(make_float2(x[0] * inv, x[1] * inv), __NV_SATFINITE, __NV_E4M3);
        const __nv_fp8x2_storage_t b = __nv_cvt_float2_to_fp8x2(make_float2(x[2] * inv, x[3] * inv), __NV_SATFINITE, __NV_E4M3);
        return (uint32_t)a | (uint32_t)b << 16;
    } else {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= ((uint32_t)max(-127, min(127, __float2int_rn(__fdiv_rn(x[i], scale)))) & 255u) << (8 * i);
        return w;
    }
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

// The call's row number n as (b, h, t), and whether the call has such a token
struct KvMoveRow {
    int b, h, t;
    bool ok;
};
__device__ __forceinline__ KvMoveRow kv_move_row(const KvMoveParams &p, int64_t n)
{
    KvMoveRow r;
    r.ok = n < p.rows;
    const int64_t m = r.ok ? n : 0, bh = m / p.tokens;
    r.t = (int)(m - bh * p.tokens);
    r.b = (int)(bh / p.pages.Hkv);
    r.h = (int)(bh - (int64_t)r.b * p.pages.Hkv);
    if (p.counts && r.t >= __ldg(p.counts + r.b)) r.ok = false;
    return r;
}

template <typename T, int FMT, int D>
__global__ void __launch_bounds__(KV_MOVE_THREADS) kv_write_kernel(const KvMoveParams p)
{
    constexpr int LPR = D / 8, RPW = 32 / LPR, STEPS = KV_MOVE_STEPS;
    const int lane = threadIdx.x & 31, gl = lane % LPR;
    const int64_t n0 = ((int64_t)blockIdx.x * (KV_MOVE_THREADS / 32) + (threadIdx.x >> 5)) * (RPW * STEPS) + lane / LPR;
    float x[STEPS][2][8];
    int64_t to[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const KvMoveRow r = kv_move_row(p, n0 + s * RPW);
        to[s] = -1;
        if (!r.ok) continue;
        int from = r.t;
        if (p.pick) from = __ldg(p.pick + (int64_t)r.b * p.tokens + r.t);
        to[s] = p.pages.row(r.b, r.h, (int64_t)(p.start ? __ldg(p.start + r.b) : 0) + r.t);
        if (to[s] < 0 || from < 0 || from >= p.src_tokens) {
            to[s] = -1;
            if (gl == 0) ptx::report(p.status, KV_ERR_PAGE);
            continue;
        }
        const int64_t at = (((int64_t)r.b * p.pages.Hkv + r.h) * p.src_tokens + from) * D + gl * 8;
        kv_load8(static_cast<const T *>(p.k) + at, x[s][0]);
        kv_load8(static_cast<const T *>(p.v) + at, x[s][1]);
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            uint32_t top = 0;
            if (to[s] >= 0)
#pragma unroll
                for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[s][kv][i]) & 0x7fffffffu);
#pragma unroll
            for (int w = LPR / 2; w > 0; w >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, w));
            if (to[s] < 0) continue;
            const float scale = kv_scale<FMT>(top);
            uint8_t *codes = kv ? p.pages.v : p.pages.k;
            float *scales = kv ? p.pages.vs : p.pages.ks;
            *reinterpret_cast<uint2 *>(codes + to[s] * D + gl * 8) =
                make_uint2(kv_codes4<FMT>(x[s][kv], scale), kv_codes4<FMT>(x[s][kv] + 4, scale));
            if (gl == 0) scales[to[s]] = scale;
        }
    }
}

// Rows beyond a sequence's count are left as they were.
template <typename T, int FMT, int D>
__global__ void __launch_bounds__(KV_MOVE_THREADS) kv_read_kernel(const KvMoveParams p)
{
    constexpr int LPR = D / 8, RPW = 32 / LPR, STEPS = KV_MOVE_STEPS;
    const int lane = threadIdx.x & 31, gl = lane % LPR;
    const int64_t n0 = ((int64_t)blockIdx.x * (KV_MOVE_THREADS / 32) + (threadIdx.x >> 5)) * (RPW * STEPS) + lane / LPR;
    uint2 c[STEPS][2];
    float scale[STEPS][2];
    bool ok[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const KvMoveRow r = kv_move_row(p, n0 + s * RPW);
        ok[s] = false;
        if (!r.ok) continue;
        const int64_t from = p.pages.row(r.b, r.h, (int64_t)(p.start ? __ldg(p.start + r.b) : 0) + r.t);
        if (from < 0) {
            if (gl == 0) ptx::report(p.status, KV_ERR_PAGE);
            continue;
        }
        ok[s] = true;
        c[s][0] = __ldcs(reinterpret_cast<const uint2 *>(p.pages.k + from * D + gl * 8));
        c[s][1] = __ldcs(reinterpret_cast<const uint2 *>(p.pages.v + from * D + gl * 8));
        scale[s][0] = __ldg(p.pages.ks + from);
        scale[s][1] = __ldg(p.pages.vs + from);
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        if (!ok[s]) continue;
        const int64_t at = (n0 + s * RPW) * D + gl * 8;
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
