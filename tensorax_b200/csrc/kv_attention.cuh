// Attention of a few tokens per sequence -- one, a chain, or a tree of drafted ones -- over the paged 8-bit cache.
//
// Sequence b holds len_b keys, of which the last n_b are this call's own tokens (its nodes, at most 64); ctx = len_b - n_b.
// Node t sees key j of the context iff j > ctx + depth(t) - window or j < sinks (all of it without a window), and node u iff
// bit u of its word is set; depth(t) is the number of other bits in the word.  With codes k8, v8 and scales ks, vs:
//     s_tj = (q_t . k8_j) * ks_j / sqrt(D)        O_t = sum_j p_tj * vs_j * v8_j / sum_j p_tj,   p_tj = 2^(s_tj log2e - m_t)
// so a key's scale is applied to its score and a value's to its weight, and the codes go to the matrix unit as fp16, which
// holds every code of both formats exactly.  Weights times scales have to fit fp16: they are divided by a running power
// of two at least as large as every vs so far (`ref`; O is rescaled when it grows).
//
// Bound: HBM, the cache read once for all query rows of its head.  The rows of one (batch, K/V head) -- nodes times query
// heads that share it -- are cut into parts of MR; the visible keys of a part are cut over the CTAs of a cluster, stages of
// KT keys come in through a ring of asynchronous copies (16 bytes each, so pages of any size from 16 tokens on), and inside a
// CTA RB warps side by side hold 16 rows each while KS warps behind one another take KW keys of every stage.
//   S = Q K^T    mma m16n8k16, fp16 operands, fp32 sums.  The order of the 16 elements of a step is free as long as Q and K
//                agree: a lane takes 16 consecutive codes of its key (one 16-byte load) as its share of four steps.
//   O += P V     the columns' order is free too: a lane takes 16 consecutive columns of four keys, and the pairs of keys that
//                an operand register wants come out of byte permutes; P stays in the registers it was computed in.
// Stages are laid out so that both loads touch every bank once (kv_k_at, kv_v_at).  Warps' and CTAs' partial results are
// added in a fixed order: the same bits on every run.
//
// fp32 queries: Q (scaled by a power of two per row) and P are carried as two fp16 numbers each, and the products of a
// stage are added to O in fp32 instead of in the matrix unit, whose sums are cut off rather than rounded.
#pragma once
#include <cfloat>
#include <cooperative_groups.h>

#include "kv_cache.cuh"

namespace txb {

struct KvAttnParams {
    KvPages pages;
    const void *q;             // [batch, Hq, tokens, D]
    void *out;                 // the same, fp32 or fp16 (out_f16); rows of nodes that a sequence does not have stay as they were
    const int32_t *kv_lens;    // [batch]: keys of each sequence, this call's nodes among them
    const int32_t *q_lens;     // optional [batch]: nodes of each sequence (none: all)
    const uint64_t *tree;      // optional [batch, tokens]: what a node sees of the nodes (none: node t sees 0 .. t)
    int *status;
    int tokens, group;         // group = Hq / Hkv
    int row_parts;             // CTAs (per split) that share the rows of a head, MR each
    int window, sinks;         // window 0: no window
    int out_f16;
    float scale_log2;          // log2(e) / sqrt(D)
};

// Byte offsets of 16-byte chunk c of row r in a stage's K and V tile
template <int D>
__device__ __forceinline__ uint32_t kv_k_at(int r, int c)
{
    // read: chunk t (+ 4 i) of rows n, n + 1 by eight lanes
    if constexpr (D == 64) return (uint32_t)(r * 64 + c * 16);
    else return (uint32_t)(r * D + ((c & ~7) | ((c & 7) ^ ((r & 1) << 2))) * 16);
}
template <int D>
__device__ __forceinline__ uint32_t kv_v_at(int r, int c)
{
    // read: chunks n, n + 1 of rows 0, 2, 4, 6 (1, 3, 5, 7) by eight lanes; at D = 64 halves of two chunks by sixteen
    if constexpr (D == 64) return (uint32_t)((r >> 1) * 128 + ((((r & 1) << 2) | c) ^ (((r >> 1) & 3) << 1)) * 16);
    else return (uint32_t)(r * D + ((c & ~7) | ((c & 7) ^ (r & 7))) * 16);
}

template <typename TQ_, int FMT_, int D_, int RB_, int KS_, int KW_, int NS_, int CTAS_PER_SM_>
struct KvAttnCfg {
    using TQ = TQ_;
    static constexpr int FMT = FMT_, D = D_, RB = RB_, KS = KS_, KW = KW_, NS = NS_, CTAS_PER_SM = CTAS_PER_SM_;
    static constexpr bool F32 = sizeof(TQ_) == 4;
    static constexpr bool Q_IN_REGS = !F32 && D <= 128;
    static constexpr int MR = 16 * RB, KT = KS * KW, THREADS = 32 * RB * KS;
    static constexpr int CPR = D / 16;                                    // 16-byte chunks of a row
    static constexpr uint32_t TILE = KT * D, STAGE = 2 * TILE + KT * 8;   // K, V, their scales
    static constexpr uint32_t RING = NS * STAGE;
    static constexpr uint32_t MERGE = RB * KS * 16 * D * 4;               // partial O of every warp, over the drained ring
    static constexpr uint32_t OFF_Q = RING > MERGE ? RING : MERGE;
    static constexpr uint32_t Q_BYTES = Q_IN_REGS ? 0 : MR * D * 2 * (F32 ? 2 : 1);   // operand order, hi (and lo)
    static constexpr uint32_t OFF_ML = OFF_Q + Q_BYTES;                   // float2 [RB * KS][16]: max, sum; then [MR]: the CTA's
    static constexpr uint32_t OFF_FLAG = OFF_ML + (RB * KS * 16 + MR) * 8;
    static constexpr uint32_t SMEM = OFF_FLAG + 16;
    static constexpr int MAX_SPLITS = 16;
    static_assert(D == 64 || D == 128 || D == 256, "head dims");
    static_assert(KW % 16 == 0 && KW <= 32 && THREADS % CPR == 0 && KT % (THREADS / CPR) == 0, "copy and step shapes");
    static_assert(SMEM <= 232448 && (CTAS_PER_SM * (SMEM + 1024) <= 233472), "shared memory of an SM");
};

__device__ __forceinline__ void kv_mma(float *c, const uint32_t *a, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 or 4 bytes, or as many zeros
__device__ __forceinline__ void kv_copy16(uint32_t dst, const void *src, bool there)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void kv_copy4(uint32_t dst, const void *src, bool there)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void kv_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void kv_copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Bytes 0 (1, 2, 3) of a and of b as an fp16 pair, for the four bytes at once
template <int FMT>
__device__ __forceinline__ void kv_pairs(uint32_t a, uint32_t b, uint32_t *out)
{
    uint32_t lo = __byte_perm(a, b, 0x5140), hi = __byte_perm(a, b, 0x7362);
    kv_halves<FMT>(lo, out[0], out[1]);
    kv_halves<FMT>(hi, out[2], out[3]);
}

// Weights are kept at 2^kKvShift times what they are: the row's largest then leaves fp16 smaller ones room below (2^-30 of
// it) and room above for a maximum that has grown by less than 2^kKvLazy since the last rescale.
constexpr float kKvShift = 6.f, kKvLazy = 8.f;

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, Cfg::CTAS_PER_SM)
kv_attention_kernel(const __grid_constant__ KvAttnParams p)
{
    using TQ = typename Cfg::TQ;
    constexpr int D = Cfg::D, RB = Cfg::RB, KS = Cfg::KS, KW = Cfg::KW, KT = Cfg::KT, NS = Cfg::NS, FMT = Cfg::FMT;
    constexpr int CPR = Cfg::CPR, NT = KW / 8, KSTEPS = D / 16, OT = D / 8;
    constexpr bool F32 = Cfg::F32;
    namespace cg = cooperative_groups;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sbase = ptx::smem_u32(smem);
    volatile int *bad = reinterpret_cast<volatile int *>(smem + Cfg::OFF_FLAG);
    float2 *ml = reinterpret_cast<float2 *>(smem + Cfg::OFF_ML);
    cg::cluster_group cluster = cg::this_cluster();
    const int split = (int)cluster.block_rank(), splits = (int)cluster.num_blocks();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rb = warp / KS, ks = warp % KS;
    const int n = lane >> 2, t4 = lane & 3;                       // row / column and quarter of the operand layouts

    const int item = (int)blockIdx.x / splits;
    const int kvh = item / p.row_parts, row0 = (item % p.row_parts) * Cfg::MR;    // b * Hkv + h, first row of this part
    const int b = kvh / p.pages.Hkv, h = kvh - b * p.pages.Hkv;
    const int rows = p.group * p.tokens;
    const int len = max(__ldg(p.kv_lens + b), 0);
    const int nodes = min(p.q_lens ? min(max(__ldg(p.q_lens + b), 0), p.tokens) : p.tokens, len);
    const int ctx = len - nodes;
    // Visible keys as one range of numbers: the sinks in front of the window, then the keys from the window of the shallowest
    // node on.  Number c stands for key c, or c + skip behind the sinks.
    int first = 0, s_end = 0;
    if (p.window > 0) {
        first = max(0, ctx - p.window + 1);
        s_end = min(p.sinks, first);
    }
    const int skip = first - s_end, n_vis = len - skip;
    // keys of the context from here on are in every node's window
    const int all_see = p.window > 0 ? ctx + nodes - p.window : 0;
    const int share = ((n_vis + splits - 1) / splits + KT - 1) / KT * KT;
    const int c_from = min(split * share, n_vis), c_to = min(c_from + share, n_vis);
    const int n_stages = (c_to - c_from + KT - 1) / KT;

    if (tid == 0) *bad = *reinterpret_cast<volatile int *>(p.status) != 0 ? 1 : 0;
    __syncthreads();

    // ------------------------------------------------------------ stages of keys
    // Threads side by side copy the chunks of a row; a row's page is looked up a stage ahead of its copy.
    constexpr int RPP = Cfg::THREADS / CPR, PASSES = KT / RPP;    // rows a pass
    const int my_chunk = tid % CPR, my_row = tid / CPR;
    int64_t at[PASSES];
    auto look_up = [&](int j) {
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int c = c_from + j * KT + my_row + i * RPP;
            at[i] = -1;
            if (j < n_stages && c < c_to) {
                at[i] = p.pages.row(b, h, c < s_end ? c : c + skip);
                if (at[i] < 0) { *bad = 1; ptx::report(p.status, KV_ERR_PAGE); }
            }
        }
    };
    auto load = [&](int j) {
        const uint32_t k_s = sbase + (uint32_t)(j % NS) * Cfg::STAGE, v_s = k_s + Cfg::TILE, sc_s = v_s + Cfg::TILE;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
            const int r = my_row + i * RPP;
            const bool there = at[i] >= 0;
            const int64_t from = there ? at[i] : 0;
            kv_copy16(k_s + kv_k_at<D>(r, my_chunk), p.pages.k + from * D + my_chunk * 16, there);
            kv_copy16(v_s + kv_v_at<D>(r, my_chunk), p.pages.v + from * D + my_chunk * 16, there);
            if (my_chunk == 0) kv_copy4(sc_s + r * 4, p.pages.ks + from, there);
            if (my_chunk == 1) kv_copy4(sc_s + KT * 4 + r * 4, p.pages.vs + from, there);
        }
    };
    look_up(0);
#pragma unroll
    for (int j = 0; j < NS - 1; ++j) {
        if (j < n_stages) load(j);
        kv_copy_commit();
        look_up(j + 1);
    }

    // ------------------------------------------------------------ queries
    // This lane's rows of the 16-row block: n and n + 8.  A row beyond the last repeats it and is never written.
    uint32_t qr[Cfg::Q_IN_REGS ? KSTEPS : 1][4];
    float rowf[2] = {p.scale_log2, p.scale_log2};                 // what a product of the row is multiplied by
    uint64_t word[2];
    int low[2];                                                   // the row's window starts here
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = min(row0 + rb * 16 + n + 8 * i, rows - 1), t = row % p.tokens;
        word[i] = p.tree ? __ldg(p.tree + (int64_t)b * p.tokens + t) : ~0ull >> (63 - t);
        low[i] = p.window > 0 ? ctx + max(__popcll(word[i]), 1) - p.window : 0;
        const TQ *q = static_cast<const TQ *>(p.q) + ((int64_t)kvh * rows + row) * D;
        if constexpr (!F32) {
            // elements 16 (t4 + 4 c) + 4 s + {0, 1} and + {2, 3} are this lane's share of step 4 c + s
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint4 u = __ldg(reinterpret_cast<const uint4 *>(q + 16 * (t4 + 4 * c)) + half);
                    if constexpr (Cfg::Q_IN_REGS) {
                        qr[4 * c + 2 * half][i] = u.x; qr[4 * c + 2 * half][2 + i] = u.y;
                        qr[4 * c + 2 * half + 1][i] = u.z; qr[4 * c + 2 * half + 1][2 + i] = u.w;
                    } else if (ks == 0) {
                        uint32_t *dst = reinterpret_cast<uint32_t *>(smem + Cfg::OFF_Q) + ((rb * KSTEPS + 4 * c + 2 * half) * 32 + lane) * 4;
                        dst[i] = u.x; dst[2 + i] = u.y;
                        dst[128 + i] = u.z; dst[128 + 2 + i] = u.w;
                    }
                }
        } else {
            // the row's power of two brings its largest element to [2^12, 2^13)
            uint32_t top = 0;
            float x[D / 4];
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float4 f = __ldg(reinterpret_cast<const float4 *>(q + 16 * (t4 + 4 * c)) + e);
                    x[16 * c + 4 * e] = f.x; x[16 * c + 4 * e + 1] = f.y; x[16 * c + 4 * e + 2] = f.z; x[16 * c + 4 * e + 3] = f.w;
                }
#pragma unroll
            for (int e = 0; e < D / 4; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e2 = min(max((int)(top >> 23), 14), 254) - 12;               // exponent of 2^-12 times the row's largest
            const float up = __int_as_float((254 - e2) << 23);
            rowf[i] = p.scale_log2 * __int_as_float(e2 << 23);
            if (ks == 0) {
                uint32_t *dst = reinterpret_cast<uint32_t *>(smem + Cfg::OFF_Q) + (rb * KSTEPS * 32 + lane) * 4;
                constexpr int LO = RB * KSTEPS * 32 * 4;
#pragma unroll
                for (int s = 0; s < KSTEPS; ++s)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float a = x[4 * s + 2 * half] * up, c = x[4 * s + 2 * half + 1] * up;
                        const __half ah = __float2half_rn(a), ch = __float2half_rn(c);
                        dst[s * 128 + 2 * half + i] = ptx::pack_half2(__half2float(ah), __half2float(ch));
                        dst[LO + s * 128 + 2 * half + i] = ptx::pack_half2(a - __half2float(ah), c - __half2float(ch));
                    }
            }
        }
    }

    // ------------------------------------------------------------ the keys of this CTA
    float o[OT][4];
#pragma unroll
    for (int i = 0; i < OT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
    float m[2] = {-FLT_MAX, -FLT_MAX}, l[2] = {0.f, 0.f};
    uint32_t ref = 1u << 23;                                      // bits of the power of two that weights are divided by
    float inv_ref = __int_as_float(253 << 23);

    for (int j = 0; j < n_stages; ++j) {
        kv_copy_wait<NS - 2>();
        __syncthreads();                                          // stage j has landed, stage j - 1 is read
        if (j + NS - 1 < n_stages) load(j + NS - 1);
        kv_copy_commit();
        look_up(j + NS);

        const uint8_t *k_s = smem + (uint32_t)(j % NS) * Cfg::STAGE, *v_s = k_s + Cfg::TILE;
        const float *ksc = reinterpret_cast<const float *>(v_s + Cfg::TILE) + ks * KW, *vsc = ksc + KT;
        const int c0 = c_from + j * KT + ks * KW;                 // number of the warp's first key
        if (c0 >= c_to) continue;
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[nt][e] = 0.f;
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                const uint4 kw = *reinterpret_cast<const uint4 *>(k_s + kv_k_at<D>(ks * KW + nt * 8 + n, t4 + 4 * c));
                const uint32_t w[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t b0, b1;
                    kv_halves<FMT>(w[e], b0, b1);
                    if constexpr (Cfg::Q_IN_REGS) {
                        kv_mma(s[nt], qr[4 * c + e], b0, b1);
                    } else {
                        const uint4 a = *(reinterpret_cast<const uint4 *>(smem + Cfg::OFF_Q) + (rb * KSTEPS + 4 * c + e) * 32 + lane);
                        const uint32_t aw[4] = {a.x, a.y, a.z, a.w};
                        kv_mma(s[nt], aw, b0, b1);
                        if constexpr (F32) {
                            const uint4 al = *(reinterpret_cast<const uint4 *>(smem + Cfg::OFF_Q) + ((RB + rb) * KSTEPS + 4 * c + e) * 32 + lane);
                            const uint32_t alw[4] = {al.x, al.y, al.z, al.w};
                            kv_mma(s[nt], alw, b0, b1);
                        }
                    }
                }
            }
        }
        // scores in units of log2, masks
        const int key0 = c0 < s_end ? c0 : c0 + skip, key1 = c0 + KW - 1 < s_end ? c0 + KW - 1 : c0 + KW - 1 + skip;
        const bool need_mask = key1 >= ctx || (key0 < all_see && key1 >= s_end);
        float mx[2] = {-FLT_MAX, -FLT_MAX};
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float2 f = *reinterpret_cast<const float2 *>(ksc + nt * 8 + 2 * t4);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                s[nt][2 * i] *= f.x * rowf[i];
                s[nt][2 * i + 1] *= f.y * rowf[i];
            }
            if (need_mask) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int c = c0 + nt * 8 + 2 * t4 + e, key = c < s_end ? c : c + skip;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const bool sees = key < ctx ? (key >= low[i] || key < p.sinks) : (c < c_to && (word[i] >> (key - ctx) & 1));
                        if (!sees) s[nt][2 * i + e] = -INFINITY;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) mx[i] = fmaxf(mx[i], fmaxf(s[nt][2 * i], s[nt][2 * i + 1]));
        }
        // the largest scale of the step's values; one that is not finite counts for the rows that see it only
        float my_vs = lane < KW ? vsc[lane] : 0.f;
        if (!(my_vs < INFINITY)) my_vs = 0.f;
        const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(my_vs));
        float alpha[2];
        bool rescale = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
            const float next = mx[i] > m[i] + kKvLazy ? mx[i] : m[i];
            alpha[i] = ptx::ex2_approx(m[i] - next);
            rescale |= next != m[i];
            m[i] = next;
            l[i] *= alpha[i];
        }
        if (top > ref) {
            const uint32_t next = min((top + 0x7fffffu) & 0x7f800000u, 253u << 23);
            const float f = __uint_as_float(ref) * __uint_as_float((254u << 23) - next);      // powers of two
            ref = next;
            inv_ref = __uint_as_float((254u << 23) - next);
            alpha[0] *= f; alpha[1] *= f;
            rescale = true;
        }
        if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
            for (int i = 0; i < OT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][e] *= alpha[e >> 1];
        }
        // weights, as operands of the second product
        uint32_t pa[KW / 16][4], pl[F32 ? KW / 16 : 1][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float2 f = *reinterpret_cast<const float2 *>(vsc + nt * 8 + 2 * t4);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float w0 = ptx::ex2_approx(s[nt][2 * i] - m[i] + kKvShift), w1 = ptx::ex2_approx(s[nt][2 * i + 1] - m[i] + kKvShift);
                l[i] += w0 + w1;
                float x0 = w0 * (f.x * inv_ref), x1 = w1 * (f.y * inv_ref);
                if (need_mask) {                                  // 0 times a scale that is not finite
                    if (s[nt][2 * i] == -INFINITY) x0 = 0.f;
                    if (s[nt][2 * i + 1] == -INFINITY) x1 = 0.f;
                }
                const uint32_t hi = ptx::pack_half2(x0, x1);
                pa[nt >> 1][(nt & 1) * 2 + i] = hi;
                if constexpr (F32) {
                    const float2 g = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                    pl[nt >> 1][(nt & 1) * 2 + i] = ptx::pack_half2(x0 - g.x, x1 - g.y);
                }
            }
        }
        // O += P V, four columns' tiles of a word at a time
#pragma unroll
        for (int c = 0; c < (D + 127) / 128; ++c) {
            constexpr int WORDS = D == 64 ? 2 : 4;
            uint32_t v[KW / 16][4][WORDS];
#pragma unroll
            for (int kk = 0; kk < KW / 16; ++kk)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = ks * KW + kk * 16 + 2 * t4 + (r & 1) + (r >> 1) * 8;
                    if constexpr (D == 64) {
                        const uint2 u = *reinterpret_cast<const uint2 *>(v_s + kv_v_at<D>(row, n >> 1) + (n & 1) * 8);
                        v[kk][r][0] = u.x; v[kk][r][1] = u.y;
                    } else {
                        const uint4 u = *reinterpret_cast<const uint4 *>(v_s + kv_v_at<D>(row, n + 8 * c));
                        v[kk][r][0] = u.x; v[kk][r][1] = u.y; v[kk][r][2] = u.z; v[kk][r][3] = u.w;
                    }
                }
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
                float part[F32 ? 4 : 1][4];
                if constexpr (F32)
#pragma unroll
                    for (int e = 0; e < 16; ++e) part[e >> 2][e & 3] = 0.f;
#pragma unroll
                for (int kk = 0; kk < KW / 16; ++kk) {
                    uint32_t b0[4], b1[4];
                    kv_pairs<FMT>(v[kk][0][w], v[kk][1][w], b0);
                    kv_pairs<FMT>(v[kk][2][w], v[kk][3][w], b1);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float *acc = F32 ? part[F32 ? e : 0] : o[c * 16 + w * 4 + e];
                        kv_mma(acc, pa[kk], b0[e], b1[e]);
                        if constexpr (F32) kv_mma(acc, pl[kk], b0[e], b1[e]);
                    }
                }
                if constexpr (F32)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[c * 16 + w * 4 + (e >> 2)][e & 3] += part[e >> 2][e & 3];
            }
        }
    }

    // ------------------------------------------------------------ partial results
    // Column 2 t4 (+ 1) of tile 16 c + i is element 128 c + 16 (2 t4 (+ 1)) + i: sixteen (at D = 64 eight) in a row.
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    kv_copy_wait<0>();
    __syncthreads();                                              // the ring is drained
    float *part = reinterpret_cast<float *>(smem);                // [RB * KS][16][D]
    {
        constexpr int RUN = D == 64 ? 8 : 16;
        const float unit = __uint_as_float(ref);
        float *mine = part + warp * 16 * D;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (t4 == 0) ml[warp * 16 + n + 8 * i] = make_float2(m[i], l[i]);
#pragma unroll
            for (int c = 0; c < (D + 127) / 128; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int x = 0; x < RUN; x += 4) {
                        const int ot = c * 16 + x;
                        *reinterpret_cast<float4 *>(mine + (n + 8 * i) * D + 128 * c + RUN * (2 * t4 + e) + x) =
                            make_float4(o[ot][2 * i + e] * unit, o[ot + 1][2 * i + e] * unit, o[ot + 2][2 * i + e] * unit, o[ot + 3][2 * i + e] * unit);
                    }
        }
    }
    __syncthreads();
    // Warps of the CTA: number `i` of MR x D / 4 float4s over the KS warps of its rows, into the first one's place
    constexpr int QUADS = D / 4;
    auto write = [&](int r, int quad, float4 v, float sum) {
        const int row = row0 + r;
        if (row >= rows || row % p.tokens >= nodes) return;
        const float f = *bad ? __int_as_float(0x7fc00000) : 1.f / sum;               // no visible key: 0 * inf = NaN
        v.x *= f; v.y *= f; v.z *= f; v.w *= f;
        const int64_t to = ((int64_t)kvh * rows + row) * D + quad * 4;
        if (p.out_f16)
            *reinterpret_cast<uint2 *>(static_cast<__half *>(p.out) + to) = make_uint2(ptx::pack_half2(v.x, v.y), ptx::pack_half2(v.z, v.w));
        else
            *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + to) = v;
    };
    auto add = [](float4 &a, const float4 &x, float f) { a.x += x.x * f; a.y += x.y * f; a.z += x.z * f; a.w += x.w * f; };
    for (int i = tid; i < Cfg::MR * QUADS; i += Cfg::THREADS) {
        const int r = i / QUADS, quad = i % QUADS, w0 = (r >> 4) * KS, rr = r & 15;
        float mn = -FLT_MAX, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < KS; ++w) mn = fmaxf(mn, ml[(w0 + w) * 16 + rr].x);
#pragma unroll
        for (int w = 0; w < KS; ++w) {
            const float2 s = ml[(w0 + w) * 16 + rr];
            const float f = ptx::ex2_approx(s.x - mn);
            add(acc, *reinterpret_cast<const float4 *>(part + ((w0 + w) * 16 + rr) * D + quad * 4), f);
            sum += s.y * f;
        }
        if (splits == 1) write(r, quad, acc, sum);
        else {
            *reinterpret_cast<float4 *>(part + (w0 * 16 + rr) * D + quad * 4) = acc;
        }
    }
    if (splits == 1) return;
    __syncthreads();
    float2 *cta_ml = ml + RB * KS * 16;                           // [MR], behind the warps' own
    for (int r = tid; r < Cfg::MR; r += Cfg::THREADS) {
        const int w0 = (r >> 4) * KS, rr = r & 15;
        float mn = -FLT_MAX, sum = 0.f;
#pragma unroll
        for (int w = 0; w < KS; ++w) mn = fmaxf(mn, ml[(w0 + w) * 16 + rr].x);
#pragma unroll
        for (int w = 0; w < KS; ++w) sum += ml[(w0 + w) * 16 + rr].y * ptx::ex2_approx(ml[(w0 + w) * 16 + rr].x - mn);
        cta_ml[r] = make_float2(mn, *bad ? __int_as_float(0x7fc00000) : sum);
    }
    cluster.sync();
    for (int i = split * Cfg::THREADS + tid; i < Cfg::MR * QUADS; i += splits * Cfg::THREADS) {
        const int r = i / QUADS, quad = i % QUADS;
        const float *at_part = part + ((r >> 4) * KS * 16 + (r & 15)) * D + quad * 4;
        constexpr int S = Cfg::MAX_SPLITS;
        float2 s[S];
        float4 v[S];
        float mn = -FLT_MAX, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        // all remote loads first: they take as long as one
#pragma unroll
        for (int c = 0; c < S; ++c)
            if (c < splits) {
                s[c] = *cluster.map_shared_rank(cta_ml + r, c);
                v[c] = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(at_part, c));
                mn = fmaxf(mn, s[c].x);
            }
#pragma unroll
        for (int c = 0; c < S; ++c)
            if (c < splits) {
                const float f = ptx::ex2_approx(s[c].x - mn);
                add(acc, v[c], f);
                sum += s[c].y * f;
            }
        write(r, quad, acc, sum);
    }
    cluster.sync();                                               // nobody leaves while its shared memory is read
}

}  // namespace txb
