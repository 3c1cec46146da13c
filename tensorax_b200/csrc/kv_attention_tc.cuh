// Attention over the paged 8-bit cache for many query rows per K/V head -- trees of drafted tokens with shared heads -- on the
// fifth-generation tensor cores.  Same operator as kv_attention.cuh, which takes the calls of few rows; fp16 queries, d = 64, 128.
//
// Bound: the tensor pipe and the softmax's exponentials, as in sdpa_tc_pair_kernel, whose softmax, issue order and tensor-memory
// layout (P over S) this kernel has.  mma.sync, which the other kernel uses, does a third of tcgen05's work at best (549 TFLOP/s
// measured); at 256 rows a head it took 341 us where this kernel takes 96 us (B8 Hkv8, 8192 keys in the window, d 128: 717 TFLOP/s).
//
// One CTA: two 128-row query tiles of one (batch, K/V head) and a share of the keys in tiles of 128; CTAs of a cluster share the
// keys and add their results in rank order.
//   warp 0        owns tensor memory and issues the MMAs, QK0 PV0 QK1 PV1
//   warps 1-7     converters: they copy codes to shared memory a tile ahead, sixteen keys a unit (asynchronous copies that the
//                 copying lane itself reads back: no barrier), turn them into fp16 and store them in the swizzled layout that
//                 the MMAs read, two stages of K and of V (with one stage the conversion stood between QK and the next QK:
//                 195 us; three converter warps instead of seven: 162)
//   warps 8-15    softmax of query tiles 0 and 1, thread = row = tensor-memory lane
// Scales: key j's codes are multiplied by ks_j / kref, value j's by vs_j / vref, where kref is the power of two at or above the
// largest ks of the tile and vref the same of vs over the tiles so far.  Both quotients are at most 1, kref joins the softmax
// scale, and O is rescaled when vref grows.  e4m3 scales are powers of two: the products are exact down to fp16's smallest
// numbers, 2^-24 against 224 in the tile's largest row; int8 products are rounded to fp16 once (2^-11), as a cache in fp16 is.
// A row whose scale is not finite gets NaN keys and zero values: only the rows that see it are touched, by their maximum, which
// keeps a NaN that the polynomial exponential would drop, and their sum.
// Every mbarrier wait is bounded.
#pragma once
#include "kv_attention.cuh"
#include "sdpa_tc.cuh"
#include "window.cuh"

namespace txb {

enum : int { KV_TC_ERR_MMA = 55, KV_TC_ERR_CONVERT = 56, KV_TC_ERR_SOFTMAX = 57 };

template <int FMT_, int D_, int POLY_>
struct KvTcCfg {
    static constexpr int FMT = FMT_, D = D_, POLY = POLY_;
    static constexpr int BM = 128, BN = 128, MR = 2 * BM, THREADS = 512, CONVERTERS = 7;
    // 256 * 72 + 256 * 184 = 65536 = 512 * 128
    static constexpr int REGS_LIGHT = 72, REGS_SOFTMAX = 184;
    static constexpr int KP = D / 64, UNITS = BN / 16;                     // 128-byte panels of a row; sixteens of keys in a tile
    static constexpr uint32_t Q_TILE = BM * D * 2, KV_TILE = BN * D * 2, PANEL = BN * 128;
    static constexpr uint32_t OFF_Q = 0, OFF_K = 2 * Q_TILE, OFF_V = OFF_K + 2 * KV_TILE;
    static constexpr uint32_t OFF_CODES = OFF_V + 2 * KV_TILE;             // [16 units: sixteens of K, then of V][16 * D]
    static constexpr uint32_t UNIT = 16 * D;
    static constexpr uint32_t OFF_ML = OFF_CODES + 16 * UNIT;         // float2 [MR]: max, sum
    static constexpr uint32_t OFF_FACTORS = OFF_ML + MR * 8;               // float2 [4]: kref, vref of tile j & 3
    // k_ready[2] k_free[2] v_ready[2] v_free[2] s_full[2] p_full[2] pv_done[2] factors[4]
    static constexpr uint32_t OFF_BAR = OFF_FACTORS + 4 * 8;
    static constexpr int N_BARS = 18;
    static constexpr uint32_t OFF_TMEM = OFF_BAR + N_BARS * 8, OFF_ABORT = OFF_TMEM + 4;
    static constexpr uint32_t SMEM = ((OFF_ABORT + 8 + 127) / 128) * 128;
    static constexpr uint32_t COL_S0 = 0, COL_S1 = BN, COL_O0 = 2 * BN, COL_O1 = 2 * BN + D, TMEM_COLS = 512;
    static constexpr int MAX_SPLITS = 8;
    static_assert(D == 64 || D == 128, "head dims");
    static_assert(MR * D * 4 <= OFF_CODES, "the staged result lies over the operand tiles");
    static_assert(SMEM <= 232448, "more than the 227 KB a CTA may have");
};

__device__ __forceinline__ void kv_copy16(uint32_t dst, const void *src, bool there)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
// Smallest power of two at or above the positive float with the bits `top` (2^-126 at least), as bits
__device__ __forceinline__ uint32_t kv_pow2_above(uint32_t top) { return min(max((top + 0x7fffffu) & 0x7f800000u, 1u << 23), 253u << 23); }

// v where `bits` has the bit, else -inf: a test and a select, no branch
__device__ __forceinline__ uint32_t kv_keep_if_bit(uint32_t v, uint32_t bits, uint32_t bit)
{
    uint32_t r;
    asm("{\n\t.reg .pred p;\n\t.reg .b32 t;\n\tand.b32 t, %2, %3;\n\tsetp.ne.u32 p, t, 0;\n\tselp.b32 %0, %1, 0xff800000, p;\n\t}"
        : "=r"(r) : "r"(v), "r"(bits), "r"(bit));
    return r;
}

// What a lane keeps of a factor f (at most 1, or NaN) for kv_scaled16, and sixteen codes times it as fp16
template <int FMT>
__device__ __forceinline__ uint32_t kv_factor(float f)
{
    if constexpr (FMT == KV_E4M3) return ptx::pack_half2(f, f);
    else return __float_as_uint(f);
}
template <int FMT>
__device__ __forceinline__ void kv_scaled16(const uint4 &codes, uint32_t factor, uint4 *out)
{
    const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t h[2];
        kv_halves<FMT>(w[i], h[0], h[1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            if constexpr (FMT == KV_E4M3) {
                const __half2 x = __hmul2(*reinterpret_cast<const __half2 *>(&h[e]), *reinterpret_cast<const __half2 *>(&factor));
                r[2 * i + e] = *reinterpret_cast<const uint32_t *>(&x);
            } else {
                const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&h[e]));
                const float2 y = __fmul2_rn(x, make_float2(__uint_as_float(factor), __uint_as_float(factor)));
                r[2 * i + e] = ptx::pack_half2(y.x, y.y);
            }
        }
    }
    out[0] = make_uint4(r[0], r[1], r[2], r[3]);
    out[1] = make_uint4(r[4], r[5], r[6], r[7]);
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 1)
kv_attention_tc_kernel(const __grid_constant__ KvAttnParams p)
{
    constexpr int D = Cfg::D, BM = Cfg::BM, BN = Cfg::BN, FMT = Cfg::FMT, MR = Cfg::MR;
    namespace cg = cooperative_groups;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sbase = ptx::smem_u32(smem);
    const uint32_t q_s = sbase + Cfg::OFF_Q, k_s = sbase + Cfg::OFF_K, v_s = sbase + Cfg::OFF_V;
    const uint32_t bar0 = sbase + Cfg::OFF_BAR;
    const uint32_t k_ready = bar0, k_free = bar0 + 16, v_ready = bar0 + 32, v_free = bar0 + 48;           // of stage j & 1
    const uint32_t s_full = bar0 + 64, p_full = bar0 + 80, pv_done = bar0 + 96, factors_full = bar0 + 112;
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(smem + Cfg::OFF_TMEM);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + Cfg::OFF_ABORT), *bad = abort_flag + 1;
    float2 *ml = reinterpret_cast<float2 *>(smem + Cfg::OFF_ML);
    volatile float *factors = reinterpret_cast<volatile float *>(smem + Cfg::OFF_FACTORS);
    cg::cluster_group cluster = cg::this_cluster();
    const int split = (int)cluster.block_rank(), splits = (int)cluster.num_blocks();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    ptx::grid_wait();            // as in kv_attention_kernel
    // work item and keys, numbered as in kv_attention_kernel
    const int item = (int)blockIdx.x / splits;
    const int kvh = item / p.row_parts, row0 = (item % p.row_parts) * MR;
    const int b = kvh / p.pages.Hkv, h = kvh - b * p.pages.Hkv;
    const int rows = p.group * p.tokens;
    bool beyond = false;
    const int len = kv_length(p, b, beyond);
    const int nodes = min(kv_nodes_asked(p, b), len);
    const int ctx = len - nodes;
    int first = 0, s_end = 0;
    if (p.window > 0) {
        first = max(0, ctx - p.window + 1) & ~15;
        s_end = min((min(p.sinks, first) + 15) & ~15, first);
    }
    const int skip = first - s_end, n_vis = len - skip;
    const int all_see = p.window > 0 ? ctx + nodes - p.window : 0;
    const int share = ((n_vis + splits - 1) / splits + BN - 1) / BN * BN;
    const int c_from = min(split * share, n_vis), c_to = min(c_from + share, n_vis);
    const int n_tiles = (c_to - c_from + BN - 1) / BN;
    const bool live1 = row0 + BM < rows;
    const int n1 = live1 ? n_tiles : 0;

    if (tid == 0) {
        *bad = beyond ? 1 : 0;
        if (beyond) ptx::report(p.page_status, KV_ERR_PAGE);
        *abort_flag = 0;
        for (int t = 0; t < 2; ++t) {
            ptx::mbar_init(k_ready + 8 * t, Cfg::CONVERTERS);     // one arrival per converter warp
            ptx::mbar_init(v_ready + 8 * t, Cfg::CONVERTERS);
            ptx::mbar_init(k_free + 8 * t, 1);
            ptx::mbar_init(v_free + 8 * t, 1);
            ptx::mbar_init(s_full + 8 * t, 1);
            ptx::mbar_init(p_full + 8 * t, 4);                    // one arrival per softmax warp of the tile
            ptx::mbar_init(pv_done + 8 * t, 1);
        }
        for (int i = 0; i < 4; ++i) ptx::mbar_init(factors_full + 8 * i, 1);
        ptx::fence_mbar_init();
        if (sbase & 1023u) {
            *abort_flag = 1;
            ptx::report(p.status, TC_ERR_ALIGN);
        }
        if (*reinterpret_cast<volatile int *>(p.status) != 0) *abort_flag = 1;
    }
    if (warp == 0) {
        ptx::tmem_alloc(ptx::smem_u32(const_cast<uint32_t *>(tmem_slot)), Cfg::TMEM_COLS);
        ptx::tmem_relinquish();
    }
    // Q: rows of this part are one run of memory; rows behind the last are zero
    constexpr int Q_LOADS = MR * (D / 8) / Cfg::THREADS;
    static_assert(MR * (D / 8) % Cfg::THREADS == 0, "whole turns");
    uint4 q_in[Q_LOADS];
#pragma unroll
    for (int n = 0; n < Q_LOADS; ++n) {
        const int i = n * Cfg::THREADS + tid, r = i / (D / 8), c = i % (D / 8);
        q_in[n] = make_uint4(0u, 0u, 0u, 0u);
        if (row0 + r < rows) q_in[n] = reinterpret_cast<const uint4 *>(static_cast<const __half *>(p.q) + ((int64_t)kvh * rows + row0 + r) * D)[c];
    }
#pragma unroll
    for (int n = 0; n < Q_LOADS; ++n) {
        const int i = n * Cfg::THREADS + tid, r = i / (D / 8), c = i % (D / 8);
        ptx::st_shared_v4(q_s + (r / BM) * Cfg::Q_TILE + (c >> 3) * (BM * 128) + (r % BM) * 128 + (((c & 7) ^ (r & 7)) << 4), q_in[n].x, q_in[n].y,
                          q_in[n].z, q_in[n].w);
    }
    ptx::fence_proxy_async_smem();
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    const bool run = *abort_flag == 0 && n_tiles > 0;

    if (warp < 8) {
    ptx::setmaxnreg_dec<Cfg::REGS_LIGHT>();
    if (warp == 0) {
        // ------------------------------------------------------------ MMA issuer (see sdpa_tc_pair_kernel)
        if (run) {
            const bool leader = ptx::elect_one();
            constexpr uint32_t idesc_qk = ptx::idesc_f16(BM, BN, false), idesc_pv = ptx::idesc_f16(BM, D, true);
            constexpr uint32_t desc_hi = ptx::smem_desc_sw128_hi(1024);
            const uint32_t q_lo = ptx::smem_desc_sw128_lo(q_s, 16), k_lo = ptx::smem_desc_sw128_lo(k_s, 16);
            const uint32_t v_lo = ptx::smem_desc_sw128_lo(v_s, Cfg::PANEL);
            bool ok = true;
            auto issue_qk = [&](int t, int j) -> bool {
                if (!ptx::mbar_wait(k_ready + 8 * (j & 1), (uint32_t)(j >> 1) & 1u, abort_flag)) return false;
                ptx::tc_fence_after_sync();
                const uint32_t qt_lo = q_lo + (uint32_t)t * (Cfg::Q_TILE >> 4), kt_lo = k_lo + (uint32_t)(j & 1) * (Cfg::KV_TILE >> 4), t_s = tmem + (t ? Cfg::COL_S1 : Cfg::COL_S0);
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t qa = ((kk >> 2) * (BM * 128) + (kk & 3) * 32) >> 4, kb = ((kk >> 2) * Cfg::PANEL + (kk & 3) * 32) >> 4;
                        ptx::mma_ss(t_s, ptx::make_desc(qt_lo + qa, desc_hi), ptx::make_desc(kt_lo + kb, desc_hi), idesc_qk, kk > 0);
                    }
                    ptx::mma_commit(s_full + 8 * t);
                    if (t == 1 || !live1) ptx::mma_commit(k_free + 8 * (j & 1));
                }
                __syncwarp();
                return true;
            };
            auto issue_pv = [&](int t, int j) -> bool {
                if (!ptx::mbar_wait(v_ready + 8 * (j & 1), (uint32_t)(j >> 1) & 1u, abort_flag)) return false;
                if (!ptx::mbar_wait(p_full + 8 * t, (uint32_t)j & 1u, abort_flag)) return false;
                ptx::tc_fence_after_sync();
                const uint32_t vt_lo = v_lo + (uint32_t)(j & 1) * (Cfg::KV_TILE >> 4);
                const uint32_t t_o = tmem + (t ? Cfg::COL_O1 : Cfg::COL_O0), t_p = tmem + (t ? Cfg::COL_S1 : Cfg::COL_S0);
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < BN / 16; ++kk)
                        ptx::mma_ts(t_o, t_p + kk * 8, ptx::make_desc(vt_lo + kk * ((16 * 128) >> 4), desc_hi), idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
                    ptx::mma_commit(pv_done + 8 * t);
                    if (t == 1 || !live1) ptx::mma_commit(v_free + 8 * (j & 1));
                }
                __syncwarp();
                return true;
            };
            ok = issue_qk(0, 0);
            if (ok && live1) ok = issue_qk(1, 0);
            for (int j = 0; j < n_tiles && ok; ++j) {
                ok = issue_pv(0, j);
                if (ok && j + 1 < n_tiles) ok = issue_qk(0, j + 1);
                if (ok && live1) ok = issue_pv(1, j);
                if (ok && live1 && j + 1 < n_tiles) ok = issue_qk(1, j + 1);
            }
            if (!ok && leader) { *abort_flag = 1; ptx::report(p.status, KV_TC_ERR_MMA); }
        }
    } else if (run) {
        // ------------------------------------------------------------ converters
        const int w = warp - 1;
        constexpr int PASSES = D / 32;                            // 16-byte chunks of a unit per lane
        // Eight lanes side by side store four chunks of a panel for two rows: every bank once.  A lane's rows of a unit are
        // r0, r0 + STEP, ...; the chunk of sixteen fp16 numbers is two of 16 bytes, side by side but for the swizzle.
        constexpr int STEP = 16 / PASSES;
        const int c4 = lane & 3, r0 = (D == 128 ? (lane >> 4) * 2 : (lane >> 3) * 2) + ((lane >> 2) & 1);
        const int chunk = (D == 128 ? (lane >> 3 & 1) * 4 : 0) + c4;
        const uint32_t at0 = (chunk >> 2) * Cfg::PANEL + r0 * 128 + (((uint32_t)c4 * 2 ^ (uint32_t)(r0 & 7)) << 4);
        // Units 0 to 7 are the sixteens of K, 8 to 15 of V; the warp's are w, w + 7 and w + 14.
        constexpr int W = Cfg::CONVERTERS, MINE = (2 * Cfg::UNITS + W - 1) / W;
        uint8_t *codes = smem + Cfg::OFF_CODES + lane * 16;

        int page = -1;                                            // lane g: of the g-th sixteen of the tile looked up last
        // (any number may stand in a page table: whether a lane has a sixteen is not to be told from its page)
        auto wanted = [&](int j) { return j < n_tiles && lane < Cfg::UNITS && c_from + j * BN + lane * 16 < c_to; };
        auto look_up = [&](int j) {
            const int c = c_from + j * BN + lane * 16, pos = c < s_end ? c : c + skip;
            page = -1;
            if (wanted(j) && (pos >> p.pages.page_shift) < p.pages.table_len)
                page = __ldg(p.pages.table + (int64_t)b * p.pages.table_len + (pos >> p.pages.page_shift));
        };
        // first row of the tile's g-th sixteen (rows of a cache are 31-bit numbers), or -1: from the pages looked up last
        auto first_row = [&](int j) -> int {
            const int c = c_from + j * BN + lane * 16, pos = c < s_end ? c : c + skip;
            if (!wanted(j)) return -1;
            if (page < 0 || page >= p.pages.pages) { *bad = 1; ptx::report(p.page_status, KV_ERR_PAGE); return -1; }
            return ((page * p.pages.Hkv + h) << p.pages.page_shift) + (pos & ((1 << p.pages.page_shift) - 1));
        };
        float kc[4], vc[4];                                       // scales of keys lane, lane + 32, ... of a tile
        int mine = -1;                                        // lane g: first row of the g-th sixteen of the tile asked for
        auto turn = [&](int j) { mine = first_row(j); look_up(j + 1); };      // rows of tile j, pages of the one behind it
        auto ask = [&](int j) {                                   // scales of that tile
            const int left = c_to - (c_from + j * BN);            // keys that the tile has
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int row = __shfl_sync(0xffffffffu, mine, 2 * e + (lane >> 4));
                const bool there = row >= 0 && e * 32 + lane < left;
                kc[e] = there ? __ldg(p.pages.ks + row + (lane & 15)) : 0.f;
                vc[e] = there ? __ldg(p.pages.vs + row + (lane & 15)) : 0.f;
            }
        };
        auto request = [&](int j, int u) {                        // codes of unit u of tile j, the tile asked for last
            const int g = u % Cfg::UNITS, left = c_to - (c_from + j * BN) - g * 16;
            const int row = __shfl_sync(0xffffffffu, mine, g);
            if (u < 2 * Cfg::UNITS && j < n_tiles) {
                const uint32_t dst = ptx::smem_u32(codes + u * Cfg::UNIT);
                const uint8_t *from = (u < Cfg::UNITS ? p.pages.k : p.pages.v) + (row >= 0 ? (int64_t)(row + r0) * D + chunk * 16 : 0);
                if (row >= 0 && left >= 16) {
#pragma unroll
                    for (int i = 0; i < PASSES; ++i) ptx::cp_async16(dst + i * 512, from + i * STEP * D);
                } else {                                          // zeros behind the last key
#pragma unroll
                    for (int i = 0; i < PASSES; ++i) {
                        const bool there = row >= 0 && r0 + i * STEP < left;
                        kv_copy16(dst + i * 512, from + (there ? i * STEP * D : 0), there);
                    }
                }
            }
            kv_copy_commit();
        };
        bool ok = true;
        uint32_t vref = 1u << 23;
        look_up(0);
        turn(0);
        ask(0);
        for (int n = 0; n < MINE; ++n) request(0, w + W * n);
        for (int j = 0; j < n_tiles && ok; ++j) {
            float kf[4], vf[4];
            uint32_t factor[MINE], ktop = 0, vtop = 0;            // the lane's of the units, as key lane of the 32 that hold the unit
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                kf[e] = kc[e]; vf[e] = vc[e];
                if (kf[e] < INFINITY && vf[e] < INFINITY) { ktop = max(ktop, __float_as_uint(kf[e])); vtop = max(vtop, __float_as_uint(vf[e])); }
            }
            const uint32_t kref = kv_pow2_above(__reduce_max_sync(0xffffffffu, ktop));
            vref = max(vref, kv_pow2_above(__reduce_max_sync(0xffffffffu, vtop)));
            if (w == 0 && lane == 0) {
                factors[2 * (j & 3)] = __uint_as_float(kref);
                factors[2 * (j & 3) + 1] = __uint_as_float(vref);
                ptx::mbar_arrive(factors_full + 8 * (j & 3));
            }
            const float k_inv = __uint_as_float((254u << 23) - kref), v_inv = __uint_as_float((254u << 23) - vref);
#pragma unroll
            for (int n = 0; n < MINE; ++n) {
                const int u = w + W * n, g = u % Cfg::UNITS, e = g >> 1;
                const bool of_k = u < Cfg::UNITS;
                const float kq = e < 2 ? (e == 0 ? kf[0] : kf[1]) : (e == 2 ? kf[2] : kf[3]), vq = e < 2 ? (e == 0 ? vf[0] : vf[1]) : (e == 2 ? vf[2] : vf[3]);
                const bool ok_key = kq < INFINITY && vq < INFINITY;
                factor[n] = kv_factor<FMT>(of_k ? (ok_key ? kq * k_inv : __int_as_float(0x7fc00000)) : (ok_key ? vq * v_inv : 0.f));
            }
            turn(j + 1);
            bool k_done = false;
#pragma unroll
            for (int n = 0; n < MINE && ok; ++n) {
                const int u = w + W * n, g = u % Cfg::UNITS;
                const bool of_k = u < Cfg::UNITS;
                if (!of_k && !k_done) {                           // the K stage is this warp's no more
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(k_ready + 8 * (j & 1));
                    k_done = true;
                }
                kv_copy_wait<MINE - 1>();                         // the unit's codes, as far as this lane copied them
                uint4 x[PASSES];
#pragma unroll
                for (int i = 0; i < PASSES; ++i) x[i] = *reinterpret_cast<const uint4 *>(codes + min(u, 15) * Cfg::UNIT + i * 512);
                request(j + 1, u);
                if (n == 0) ask(j + 1);                           // (in front of the units: 103 us for 98)
                if (j > 1) ok = ptx::mbar_wait((of_k ? k_free : v_free) + 8 * (j & 1), (uint32_t)((j >> 1) - 1) & 1u, abort_flag);
                if (ok && u < 2 * Cfg::UNITS) {
                    uint8_t *dst = smem + (of_k ? Cfg::OFF_K : Cfg::OFF_V) + (j & 1) * Cfg::KV_TILE + g * 2048;
#pragma unroll
                    for (int i = 0; i < PASSES; ++i) {
                        // four rows further the swizzle's third bit changes, eight rows further nothing does
                        const uint32_t at = (at0 ^ (STEP == 4 && (i & 1) ? 64u : 0u)) + i * STEP * 128;
                        uint4 out[2];
                        kv_scaled16<FMT>(x[i], __shfl_sync(0xffffffffu, factor[n], (g & 1) * 16 + r0 + i * STEP), out);
                        *reinterpret_cast<uint4 *>(dst + at) = out[0];
                        *reinterpret_cast<uint4 *>(dst + (at ^ 16u)) = out[1];
                    }
                }
            }
            if (!ok) break;
            ptx::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (!k_done) ptx::mbar_arrive(k_ready + 8 * (j & 1));
                ptx::mbar_arrive(v_ready + 8 * (j & 1));
            }
        }
        if (!ok && lane == 0) { *abort_flag = 1; ptx::report(p.status, KV_TC_ERR_CONVERT); }
        kv_copy_wait<0>();
    }
    } else {
        ptx::setmaxnreg_inc<Cfg::REGS_SOFTMAX>();
        // ------------------------------------------------------------ softmax (see sdpa_tc_pair_kernel)
        const int t = (warp - 8) >> 2, quarter = warp & 3, r = quarter * 32 + lane;
        const int row = row0 + t * BM + r, nt = t ? n1 : n_tiles;
        const uint32_t lane_base = (uint32_t)(quarter * 32) << 16;
        const uint32_t t_s = tmem + lane_base + (t ? Cfg::COL_S1 : Cfg::COL_S0), t_o = tmem + lane_base + (t ? Cfg::COL_O1 : Cfg::COL_O0);
        const int node = min(row, rows - 1) % p.tokens;
        uint64_t word = p.tree ? p.tree[(int64_t)b * p.tokens + node] : ~0ull >> (63 - node);
        const int low = p.window > 0 ? ctx + max(__popcll(word), 1) - p.window : 0;
        if (nodes < 64) word &= (1ull << nodes) - 1;
        float m_used = -1.0e30f, l = 0.f, vref = 1.f;             // a finite stand-in for "no key seen yet"
        bool ok = run && nt > 0;
        for (int j = 0; j < nt && ok; ++j) {
            const int c0 = c_from + j * BN;
            ok = ptx::mbar_wait(factors_full + 8 * (j & 3), (uint32_t)(j >> 2) & 1u, abort_flag);
            if (!ok) break;
            const float kref = factors[2 * (j & 3)], vnew = factors[2 * (j & 3) + 1];
            ok = ptx::mbar_wait(s_full + 8 * t, (uint32_t)j & 1u, abort_flag);
            if (!ok) break;
            ptx::tc_fence_after_sync();
            uint32_t sv[BN];
            ptx::tmem_ld_cols<BN>(t_s, sv);
            ptx::tmem_wait_ld();
            ptx::reg_fence_cols<BN>(sv);
            const int key0 = c0 < s_end ? c0 : c0 + skip, key1 = c0 + BN - 1 < s_end ? c0 + BN - 1 : c0 + BN - 1 + skip;
            if (key1 >= ctx || (key0 < all_see && key1 >= p.sinks)) {
                // What the row sees of the tile's columns, as bits.  [0, a) are sinks' sixteens, [a, z) the window's part of the
                // context, then come nodes, node 0 at column `base`.  (Column by column in the loop this took 24 us a tile.)
                const int base = ctx - skip - c0, a = min(max(s_end - c0, 0), BN), z = min(max(base, 0), BN);
#pragma unroll
                for (int w = 0; w < BN / 32; ++w) {
                    auto below = [&](int n) { return n <= 32 * w ? 0u : n >= 32 * w + 32 ? ~0u : (1u << (n - 32 * w)) - 1u; };
                    const uint32_t front = below(a) & (below(p.sinks - c0) | ~below(low - c0));
                    const uint32_t behind = below(z) & ~below(a) & (below(p.sinks - skip - c0) | ~below(low - skip - c0));
                    const int n0 = 32 * w - base;                 // the node of column 32 w
                    const uint32_t nodes_seen = n0 >= 64 || n0 <= -32 ? 0u : n0 >= 0 ? (uint32_t)(word >> n0) : (uint32_t)word << -n0;
                    const uint32_t seen = front | behind | nodes_seen;
#pragma unroll
                    for (int i = 0; i < 32; ++i) sv[32 * w + i] = kv_keep_if_bit(sv[32 * w + i], seen, 1u << i);
                }
            }
            // not 0, however small the factor: -inf * 0 would make a NaN of a key that is not seen
            const float scale = fmaxf(p.scale_log2 * kref, 1.17549435e-38f);
            float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
            for (int i = 0; i < BN; i += 8) {
                mx0 = ptx::max3_nan(mx0, __uint_as_float(sv[i]), __uint_as_float(sv[i + 1]));
                mx1 = ptx::max3_nan(mx1, __uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3]));
                mx2 = ptx::max3_nan(mx2, __uint_as_float(sv[i + 4]), __uint_as_float(sv[i + 5]));
                mx3 = ptx::max3_nan(mx3, __uint_as_float(sv[i + 6]), __uint_as_float(sv[i + 7]));
            }
            const float mx = ptx::max3_nan(ptx::max3_nan(mx0, mx1, mx2), mx3, mx3);
            const float m_new = fmaxf(m_used, mx * scale);
            const float m_next = (m_new > m_used + kLazyRescaleLog2) ? m_new : m_used;
            const float alpha = ptx::ex2_approx(m_used - m_next);
            const float alpha_o = j > 0 ? alpha * (vref * __uint_as_float((254u << 23) - __float_as_uint(vnew))) : 1.f;   // powers of two
            m_used = m_next;
            vref = vnew;
            const float2 scale2 = make_float2(scale, scale), negm2 = make_float2(-m_next, -m_next);
            float2 sum_a = make_float2(0.f, 0.f), sum_b = make_float2(0.f, 0.f);
            uint32_t pk[BN / 2];
#pragma unroll
            for (int i = 0; i < BN; i += 4) {
                const float2 xa = __ffma2_rn(make_float2(__uint_as_float(sv[i]), __uint_as_float(sv[i + 1])), scale2, negm2);
                const float2 xb = __ffma2_rn(make_float2(__uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3])), scale2, negm2);
                const int e0 = i & 15;
                const bool poly_a = (Cfg::POLY >> e0) & 1, poly_b = (Cfg::POLY >> (e0 + 2)) & 1;
                const float2 ea = poly_a ? ptx::ex2_poly2(xa) : make_float2(ptx::ex2_approx(xa.x), ptx::ex2_approx(xa.y));
                const float2 eb = poly_b ? ptx::ex2_poly2(xb) : make_float2(ptx::ex2_approx(xb.x), ptx::ex2_approx(xb.y));
                sum_a = __fadd2_rn(sum_a, ea);
                sum_b = __fadd2_rn(sum_b, eb);
                pk[i / 2] = ptx::pack_half2(ea.x, ea.y);
                pk[i / 2 + 1] = ptx::pack_half2(eb.x, eb.y);
            }
            l = l * alpha + ((sum_a.x + sum_a.y) + (sum_b.x + sum_b.y));
            // a score of NaN or +inf makes the row NaN; the polynomial exponential alone would drop it
            if (!(mx < INFINITY)) l = __int_as_float(0x7fc00000);
            if (j > 0) {
                ok = ptx::mbar_wait(pv_done + 8 * t, (uint32_t)(j - 1) & 1u, abort_flag);
                if (!ok) break;
                ptx::tc_fence_after_sync();
                if (__any_sync(0xffffffffu, alpha_o != 1.0f)) {
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c) {
                        uint32_t o[16];
                        ptx::tmem_ld16(t_o + c * 16, o);
                        ptx::tmem_wait_ld();
                        ptx::reg_fence16(o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha_o);
                        ptx::tmem_st16(t_o + c * 16, o);
                    }
                }
            }
            ptx::tmem_st_cols<BN / 2>(t_s, pk);
            ptx::tmem_wait_st();
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(p_full + 8 * t);
        }
        if (ok) {
            ok = ptx::mbar_wait(pv_done + 8 * t, (uint32_t)(nt - 1) & 1u, abort_flag);
            ptx::tc_fence_after_sync();
        }
        if (run && nt > 0 && !ok) { *abort_flag = 1; ptx::report(p.status, KV_TC_ERR_SOFTMAX); }
        // the row's max and sum: a row without a key has neither (the polynomial's 2^(-inf) is not quite 0).  A sum that is NaN stays:
        // the row sees a key that is not finite, here perhaps that alone.
        if (m_used == -1.0e30f && l == l) l = 0.f;
        ml[t * BM + r] = make_float2(m_used, l);
        // both tiles' MMAs are done before the operands make room for the result
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const bool none = !ok || l == 0.f;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            ptx::tmem_ld32(t_o + c * 32, o);
            ptx::tmem_wait_ld();
            ptx::reg_fence32(o);
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                float4 v = make_float4(__uint_as_float(o[i]) * vref, __uint_as_float(o[i + 1]) * vref, __uint_as_float(o[i + 2]) * vref,
                                       __uint_as_float(o[i + 3]) * vref);
                if (none) v = make_float4(0.f, 0.f, 0.f, 0.f);
                const int quad = c * 8 + i / 4;
                *reinterpret_cast<float4 *>(smem + (t * BM + r) * D * 4 + ((quad ^ (r & 7)) << 4)) = v;
            }
        }
    }
    // ------------------------------------------------------------ result: CTAs of the cluster, in rank order
    ptx::tc_fence_before_sync();
    if (splits > 1) cluster.sync();
    else __syncthreads();
    if (*abort_flag)
        for (int i = 0; i < 64; ++i) __nanosleep(2000);           // let copies in flight land
    // Each CTA takes an equal share of the rows.  First what every CTA's part of a row is worth, then the rows, four of a warp
    // under way at once (element by element, weights and all, this took 40 us).
    if (warp >= 8) {
        constexpr int QUADS = D / 4, S = Cfg::MAX_SPLITS, RPW = 32 / QUADS > 0 ? 32 / QUADS : 1;    // rows a warp takes side by side
        float *worth = reinterpret_cast<float *>(smem + Cfg::OFF_CODES);         // [row of the share][CTA]
        const int row_share = (MR + splits - 1) / splits, r_first = split * row_share, mine = min(row_share, MR - r_first);
        if (tid - 256 < mine) {
            const int r = r_first + tid - 256;
            float2 s[S];
            float mn = -1.0e30f, sum = 0.f;
            int failed = 0;
#pragma unroll
            for (int c = 0; c < S; ++c)
                if (c < splits) {
                    s[c] = *cluster.map_shared_rank(ml + r, c);
                    failed |= *cluster.map_shared_rank(const_cast<int *>(abort_flag), c) | *cluster.map_shared_rank(const_cast<int *>(bad), c);
                    mn = fmaxf(mn, s[c].x);
                }
#pragma unroll
            for (int c = 0; c < S; ++c)
                if (c < splits) { s[c].x = ptx::ex2_approx(s[c].x - mn); sum += s[c].y * s[c].x; }
            const float f = failed ? __int_as_float(0x7fc00000) : 1.f / sum;         // no visible key: 0 * inf = NaN
#pragma unroll
            for (int c = 0; c < S; ++c)
                if (c < splits) worth[(tid - 256) * S + c] = s[c].x * f;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        constexpr int U = 4;
        const int asked = kv_nodes_asked(p, b);
        for (int first_r = (warp - 8) * RPW; first_r < mine; first_r += 8 * RPW * U) {
            float4 acc[U];
#pragma unroll
            for (int u = 0; u < U; ++u) acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
            for (int c = 0; c < splits; ++c) {
                float4 v[U];
                float f[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int rl = min(first_r + u * 8 * RPW + lane / QUADS, mine - 1), r = r_first + rl;
                    v[u] = *cluster.map_shared_rank(reinterpret_cast<const float4 *>(smem + r * D * 4 + (((lane % QUADS) ^ (r & 7)) << 4)), c);
                    f[u] = worth[rl * S + c];
                }
#pragma unroll
                for (int u = 0; u < U; ++u) { acc[u].x += v[u].x * f[u]; acc[u].y += v[u].y * f[u]; acc[u].z += v[u].z * f[u]; acc[u].w += v[u].w * f[u]; }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int rl = first_r + u * 8 * RPW + lane / QUADS, row_o = row0 + r_first + rl;
                if (rl >= mine || row_o >= rows || row_o % p.tokens >= asked) continue;
                if (row_o % p.tokens >= nodes) acc[u].x = acc[u].y = acc[u].z = acc[u].w = __int_as_float(0x7fc00000);
                const int64_t to = ((int64_t)kvh * rows + row_o) * D + (lane % QUADS) * 4;
                if (p.out_f16)
                    *reinterpret_cast<uint2 *>(static_cast<__half *>(p.out) + to) = make_uint2(ptx::pack_half2(acc[u].x, acc[u].y), ptx::pack_half2(acc[u].z, acc[u].w));
                else
                    *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + to) = acc[u];
            }
        }
    }
    if (warp == 0) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem, Cfg::TMEM_COLS);
    }
    if (splits > 1) cluster.sync();                               // nobody leaves while its shared memory is read
}

}  // namespace txb
