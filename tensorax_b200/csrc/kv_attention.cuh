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
// heads that share it -- are cut into parts of 8 NR; the visible keys of a part are cut over the CTAs of a cluster and the
// warps of a CTA.  A warp is on its own until its keys are done: it looks pages up and brings KW keys a step through a ring
// of its own (sixteen keys a copy: a page holds whole sixteens, and they are one run of bytes in it).  With one ring for the CTA,
// filled by all threads 16 bytes each, copying took 220 of 650 instructions per warp and sixteen keys; filled by one warp, that
// warp's issue of the copies held up the others.
//   S^T = K Q^T    mma m16n8k16, fp16 operands, fp32 sums: sixteen keys by eight rows, so that a decoding step of up to eight
//                  rows a head fills its tiles, and a key's codes are converted once for all of the warp's rows.  The order of
//                  the 16 elements of a step is free as long as K and Q agree: a lane takes 16 consecutive codes of its key
//                  (one 16-byte load) as its share of four steps.
//   O^T += V^T P^T the same shape; the order of the columns is free: a lane takes 16 consecutive columns of four keys, and the
//                  pairs of keys that an operand register wants come out of byte permutes.  P^T changes from the layout of
//                  results to that of operands by a transposing register move.
// The copies swizzle their 128-byte lines, and which key is a product's row n is chosen so that both loads touch every bank once
// (kv_key).  Warps' and CTAs' partial results are added in a fixed order: the same bits on every run.  Waits are bounded.
//
// fp32 queries: Q (scaled by a power of two per row) and P are carried as two fp16 numbers each, and the products of a
// stage are added to O in fp32 instead of in the matrix unit, whose sums are cut off rather than rounded.
//
// The same kernel takes decoding steps of the windowed attention over plain fp16 keys (KV_PLAIN): B8 Hq32 Hkv8 d128, window 2048,
// four sinks, 16.9 us, 27.7 by the kernel of sdpa_decode.cuh, whose products are fp32 FMAs.  Weights are two numbers each there, as
// that kernel's are fp32; over the cache fp16 queries have one (2^-11, below the codes' own rounding of 2^-4 or 1/254).
#pragma once
#include <cfloat>
#include <cooperative_groups.h>

#include "kv_cache.cuh"
#include "kv_lens.cuh"

namespace txb {

// Not a cache's format: K and V as they are, [B, Hkv, Sk, D] fp16, the rows of a window (window.cuh) at its keys.  A page is a
// head's keys, and there are no scales; sixteen keys at the end of one head may be the next one's (masked, V's zeroed).
constexpr int KV_PLAIN = 2;

struct KvAttnParams {
    KvPages pages;
    const void *q;             // [batch, Hq, tokens, D]
    void *out;                 // the same, fp32 or fp16 (out_f16); rows from q_lens on stay as they were
    const int32_t *kv_lens;    // [batch]: keys of each sequence, this call's nodes among them
    const int32_t *q_lens;     // optional [batch]: nodes of each sequence (none: all)
    const uint64_t *tree;      // optional [batch, tokens]: what a node sees of the nodes (none: node t sees 0 .. t)
    int *status, *page_status; // waits that ran out; pages that do not exist (no part of plain keys)
    int most_keys;             // what a page table can hold
    int tokens, group;         // group = Hq / Hkv
    int row_parts;             // CTAs (per split) that share the rows of a head, MR each
    int window, sinks;         // window 0: no window
    int out_f16;
    float scale_log2;          // log2(e) / sqrt(D)
};

struct KvPlainParams : KvAttnParams {
    KvLens lens;
    int Sk, align_end;
};

enum : int { KV_ERR_ROWS = 54 };

// Byte offset of 16-byte chunk c of key r, B bytes long, in a stage's K or V tile: 128-byte lines, their chunks swizzled by the copy
template <int B>
__device__ __forceinline__ uint32_t kv_at(int r, int c)
{
    const int at = r * (B / 16) + c, line = at >> 3;
    return (uint32_t)(line * 128 + (((at & 7) ^ (line & 7)) << 4));
}
// Which of eight keys is row n of the products, as 3 bits each.  K is read by eight lanes at a time, chunks t (+ 4 i) of rows
// 2 t', 2 t' + 1: the two keys must lie in different halves of their lines.  V by eight lanes, chunks n, n + 1 of rows 0, 2, 4, 6
// or 1, 3, 5, 7 (at 64 bytes by sixteen, halves of two chunks): four keys whose swizzles take these to different quarters.
template <int B>
__device__ __forceinline__ int kv_key(int n)
{
    constexpr int order[3][8] = {{0, 3, 4, 7, 1, 2, 5, 6}, {0, 5, 2, 7, 4, 1, 6, 3}, {0, 6, 1, 7, 2, 4, 3, 5}};
    constexpr int w = B == 64 ? 0 : B == 128 ? 1 : 2;
    constexpr uint32_t bits = order[w][0] | order[w][1] << 3 | order[w][2] << 6 | order[w][3] << 9 | order[w][4] << 12 |
                              order[w][5] << 15 | order[w][6] << 18 | order[w][7] << 21;
    return bits >> (3 * n) & 7;
}

template <typename TQ_, int FMT_, int D_, int NR_, int WARPS_, int KW_, int NS_, int CTAS_PER_SM_>
struct KvAttnCfg {
    using TQ = TQ_;
    static constexpr int FMT = FMT_, D = D_, NR = NR_, WARPS = WARPS_, KW = KW_, NS = NS_, CTAS_PER_SM = CTAS_PER_SM_;
    static constexpr bool F32 = sizeof(TQ_) == 4, PLAIN = FMT == KV_PLAIN, P2 = F32 || PLAIN;
    using Params = std::conditional_t<PLAIN, KvPlainParams, KvAttnParams>;
    static constexpr int ROW = PLAIN ? 2 * D : D;                         // bytes of a key
    static constexpr bool Q_IN_REGS = !F32 && D * NR <= 256;
    static constexpr int MR = 8 * NR, THREADS = 32 * WARPS, KT = WARPS * KW;
    static constexpr uint32_t TILE = KW * ROW, STAGE = 2 * TILE;            // K, V of a step of one warp
    static constexpr uint32_t OFF_SCALES = WARPS * NS * STAGE;            // [WARPS][NS][K, V][KW]
    static constexpr uint32_t RING = OFF_SCALES + (PLAIN ? 0 : WARPS * NS * KW * 8);
    static constexpr uint32_t MERGE = WARPS * MR * D * 4;                 // partial O of every warp, over the drained rings
    static constexpr uint32_t OFF_Q = RING > MERGE ? RING : MERGE;
    static constexpr uint32_t Q_BYTES = Q_IN_REGS ? 0 : MR * D * 2 * (F32 ? 2 : 1);   // operand order, hi (and lo)
    static constexpr uint32_t OFF_WORDS = OFF_Q + Q_BYTES;                // uint64 [MR]: what a row sees of the nodes
    static constexpr uint32_t OFF_LOW = OFF_WORDS + MR * 8;               // int [MR]: where its window starts
    static constexpr uint32_t OFF_ML = OFF_LOW + MR * 4;                  // float2 [WARPS][MR]: max, sum; then [MR]: the CTA's
    static constexpr uint32_t OFF_BAR = OFF_ML + (WARPS + 1) * MR * 8;    // full [WARPS][NS]
    static constexpr uint32_t OFF_FLAG = OFF_BAR + WARPS * NS * 8;
    static constexpr uint32_t SMEM = OFF_FLAG + 16;
    static constexpr int MAX_SPLITS = 16;
    static_assert(D == 64 || D == 128 || D == 256, "head dims");
    static_assert(!PLAIN || (!F32 && D <= 128), "plain keys: fp16, up to 256 bytes");
    static_assert(KW == 16 || KW == 32, "step shapes");
    static_assert(SMEM <= 232448 && (CTAS_PER_SM * (SMEM + 1024) <= 233472), "shared memory of an SM");
};

__device__ __forceinline__ void kv_mma(float *c, const uint32_t *a, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void kv_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void kv_copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// 8 x 8 fp16 numbers, a row's pair 2 t, 2 t + 1 in lane 4 row + t: the transpose in the same places
__device__ __forceinline__ uint32_t kv_transpose(uint32_t x)
{
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
// Bytes 0 (1, 2, 3) of a and of b as an fp16 pair, for the four bytes at once
template <int FMT>
__device__ __forceinline__ void kv_pairs(uint32_t a, uint32_t b, uint32_t *out)
{
    uint32_t lo = __byte_perm(a, b, 0x5140), hi = __byte_perm(a, b, 0x7362);
    kv_halves<FMT>(lo, out[0], out[1]);
    kv_halves<FMT>(hi, out[2], out[3]);
}

// Keys of sequence b.  More than its page table can hold is an error, and not walked.
__device__ __forceinline__ int kv_length(const KvAttnParams &p, int b, bool &beyond)
{
    const int len = p.kv_lens[b];
    beyond = len > p.most_keys;
    return max(0, min(len, p.most_keys));
}

// Nodes whose rows are written; those that the sequence has no key for get NaN.
__device__ __forceinline__ int kv_nodes_asked(const KvAttnParams &p, int b) { return p.q_lens ? min(max(p.q_lens[b], 0), p.tokens) : p.tokens; }

// Weights are kept at 2^kKvShift times what they are: the row's largest then leaves fp16 smaller ones room below (2^-30 of
// it) and room above for a maximum that has grown by less than 2^kKvLazy since the last rescale.
constexpr float kKvShift = 6.f, kKvLazy = 8.f;

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, Cfg::CTAS_PER_SM)
kv_attention_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const __grid_constant__ typename Cfg::Params p)
{
    using TQ = typename Cfg::TQ;
    constexpr int D = Cfg::D, ROW = Cfg::ROW, NR = Cfg::NR, KW = Cfg::KW, KT = Cfg::KT, NS = Cfg::NS, FMT = Cfg::FMT, MR = Cfg::MR;
    constexpr int NG = KW / 16, KSTEPS = D / 16, OT = D / 16;
    constexpr bool F32 = Cfg::F32, PLAIN = Cfg::PLAIN, P2 = Cfg::P2;
    namespace cg = cooperative_groups;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sbase = ptx::smem_u32(smem);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + Cfg::OFF_FLAG), *bad = abort_flag + 1;
    float2 *ml = reinterpret_cast<float2 *>(smem + Cfg::OFF_ML);
    uint64_t *words = reinterpret_cast<uint64_t *>(smem + Cfg::OFF_WORDS);
    int *lows = reinterpret_cast<int *>(smem + Cfg::OFF_LOW);
    cg::cluster_group cluster = cg::this_cluster();
    const int split = (int)cluster.block_rank(), splits = (int)cluster.num_blocks();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = lane >> 2, t4 = lane & 3;                       // row / column and quarter of the operand layouts

    if (tid == 0) {
        *bad = 0;
        *abort_flag = 0;
        for (int i = 0; i < Cfg::WARPS * NS; ++i) ptx::mbar_init(sbase + Cfg::OFF_BAR + 8 * i, 1);
        ptx::fence_mbar_init();
    }
    // What is in front of this launch in the stream may still run up to here; the loads whose address does not come from one
    // behind it are plain, since __ldg's may be moved across (a step of 13 tokens over 1500 keys, alone on the chip, again and again: 14.3 us without, 13.0 us).
    ptx::grid_wait();
    const int item = (int)blockIdx.x / splits;
    const int kvh = item / p.row_parts, row0 = (item % p.row_parts) * MR;    // b * Hkv + h, first row of this part
    const int b = kvh / p.pages.Hkv, h = kvh - b * p.pages.Hkv;
    const int rows = p.group * p.tokens;
    int len, nodes, ctx;                                          // keys of the sequence, nodes among them, position of the first
    if constexpr (PLAIN) {
        len = p.lens.limit(b, p.Sk);
        nodes = p.tokens;
        ctx = p.align_end ? len - p.tokens : 0;
        len = max(0, min(len, ctx + p.tokens));
    } else {
        bool beyond;
        len = kv_length(p, b, beyond);
        if (beyond && tid == 0) { *bad = 1; ptx::report(p.page_status, KV_ERR_PAGE); }
        nodes = min(kv_nodes_asked(p, b), len);
        ctx = len - nodes;
    }
    // Visible keys as one range of numbers: the sinks in front of the window, then the keys from the window of the shallowest
    // node on, both in whole sixteens.  Number c stands for key c, or c + skip behind the sinks.
    int first = 0, s_end = 0;
    if (p.window > 0) {
        first = max(0, ctx - p.window + 1) & ~15;
        s_end = min((min(p.sinks, first) + 15) & ~15, first);
    }
    const int skip = first - s_end, n_vis = len - skip;
    // keys of the context from here on are in every node's window
    const int all_see = p.window > 0 ? ctx + nodes - p.window : 0;
    const int share = ((n_vis + splits - 1) / splits + KT - 1) / KT * KT;
    const int c_from = min(split * share, n_vis), c_to = min(c_from + share, n_vis);

    if (tid == 0 && *reinterpret_cast<volatile int *>(p.status) != 0) *abort_flag = 1;
    for (int r = tid; r < MR; r += Cfg::THREADS) {           // a row beyond the last repeats it and is never written
        const int t = min(row0 + r, rows - 1) % p.tokens;
        if constexpr (PLAIN) { lows[r] = ctx + t + 1 - p.window; continue; }
        const uint64_t word = p.tree ? p.tree[(int64_t)b * p.tokens + t] : ~0ull >> (63 - t);
        words[r] = word;
        lows[r] = p.window > 0 ? ctx + max(__popcll(word), 1) - p.window : 0;
    }
    __syncthreads();
    const bool run = *abort_flag == 0;
    float *part = reinterpret_cast<float *>(smem);                // [WARPS][MR][D], once the ring is drained
    float2 *cta_ml = ml + Cfg::WARPS * MR;                        // [MR], behind the warps' own

    // ------------------------------------------------------------ steps of keys
    // The warp's keys: KW of every KT of the CTA's.  Lane i looks up the page of sixteen of them, a step ahead of the copy.
    const int n_steps = max(0, (c_to - c_from - warp * KW + KT - 1) / KT);
    const uint32_t full = sbase + Cfg::OFF_BAR + warp * NS * 8, ring = sbase + warp * NS * Cfg::STAGE;
    const uint32_t ring_sc = sbase + Cfg::OFF_SCALES + warp * NS * KW * 8;
    bool ok = run;
    int page = -1;
    auto position = [&](int j) {
        const int c = c_from + j * KT + warp * KW + lane * 16;
        return c >= c_to || lane >= NG ? -1 : c < s_end ? c : c + skip;
    };
    auto look_up = [&](int j) {
        if constexpr (PLAIN) return;
        const int pos = j < n_steps ? position(j) : -1;
        page = -1;
        if (pos >= 0 && (pos >> p.pages.page_shift) < p.pages.table_len)
            page = __ldg(p.pages.table + (int64_t)b * p.pages.table_len + (pos >> p.pages.page_shift));
    };
    auto request = [&](int j) {                                   // step j, into the place that the warp is done with
        const int slot = j % NS, pos = position(j);
        const bool there = pos >= 0 && (PLAIN || (page >= 0 && page < p.pages.pages));
        int64_t row;
        if constexpr (PLAIN) row = (int64_t)kvh * p.Sk + pos;
        else row = ((((int64_t)page * p.pages.Hkv + h) << p.pages.page_shift)) + (pos & ((1 << p.pages.page_shift) - 1));
        if (!there && pos >= 0) { *bad = 1; ptx::report(p.page_status, KV_ERR_PAGE); }
        look_up(j + 1);
        const uint32_t n_there = NG == 1 ? (there ? 1 : 0) : __popc(__ballot_sync(0xffffffffu, there));
        if (lane == 0) ptx::mbar_arrive_expect_tx(full + 8 * slot, n_there * (16 * 2 * ROW));
        if (NG > 1) __syncwarp();
        if (there) {
            const uint32_t k_s = ring + slot * Cfg::STAGE + lane * 16 * ROW;
            const int line = (int)(row * ROW / 128);
            ptx::tma_load_3d(k_s, &tm_k, full + 8 * slot, 0, line, 0);
            ptx::tma_load_3d(k_s + Cfg::TILE, &tm_v, full + 8 * slot, 0, line, 0);
        }
        if constexpr (PLAIN) return;
        // a scale a lane: bulk copies of 64 bytes cost the copy engine as much as the codes'
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int64_t r = __shfl_sync(0xffffffffu, there ? row : -1, g);
            if (r >= 0) ptx::cp_async4(ring_sc + slot * KW * 8 + (lane >> 4) * KW * 4 + g * 64 + (lane & 15) * 4, (lane < 16 ? p.pages.ks : p.pages.vs) + r + (lane & 15));
        }
    };
    if (run) {
        look_up(0);
#pragma unroll
        for (int j = 0; j < NS - 1; ++j) {
            if (j < n_steps) request(j);
            kv_copy_commit();
        }
    }

    // ------------------------------------------------------------ queries
    // As operands: rows n + 8 r.  Elements 16 (t4 + 4 c) + 4 e + {0, 1} and + {2, 3} of a row are this lane's share
    // of step 4 c + e.
    uint2 qr[Cfg::Q_IN_REGS ? KSTEPS : 1][NR];
    uint2 *q_s = reinterpret_cast<uint2 *>(smem + Cfg::OFF_Q);    // [hi, lo][step][NR][lane]
    constexpr int Q_LO = KSTEPS * NR * 32;
    float *rowf_s = reinterpret_cast<float *>(ml);                // fp32: what a row's products are multiplied by, until the loop
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const int row = min(row0 + 8 * r + n, rows - 1);
        const TQ *q = static_cast<const TQ *>(p.q) + ((int64_t)kvh * rows + row) * D;
        if constexpr (PLAIN) {
            // a lane's chunk is eight elements here, its share of two steps
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                const uint4 u = *reinterpret_cast<const uint4 *>(q + 8 * (t4 + 4 * c));
                qr[2 * c][r] = make_uint2(u.x, u.y);
                qr[2 * c + 1][r] = make_uint2(u.z, u.w);
            }
        } else if constexpr (!F32) {
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint4 u = reinterpret_cast<const uint4 *>(q + 16 * (t4 + 4 * c))[half];
                    const int step = 4 * c + 2 * half;
                    if constexpr (Cfg::Q_IN_REGS) {
                        qr[step][r] = make_uint2(u.x, u.y);
                        qr[step + 1][r] = make_uint2(u.z, u.w);
                    } else if (warp == 0) {
                        q_s[(step * NR + r) * 32 + lane] = make_uint2(u.x, u.y);
                        q_s[((step + 1) * NR + r) * 32 + lane] = make_uint2(u.z, u.w);
                    }
                }
        } else if (warp == 0) {
            // the row's power of two brings its largest element to [2^12, 2^13)
            uint32_t top = 0;
            float x[D / 4];
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float4 f = reinterpret_cast<const float4 *>(q + 16 * (t4 + 4 * c))[e];
                    x[16 * c + 4 * e] = f.x; x[16 * c + 4 * e + 1] = f.y; x[16 * c + 4 * e + 2] = f.z; x[16 * c + 4 * e + 3] = f.w;
                }
#pragma unroll
            for (int e = 0; e < D / 4; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e2 = min(max((int)(top >> 23), 14), 254) - 12;               // exponent of 2^-12 times the row's largest
            const float up = __int_as_float((254 - e2) << 23);
            if (t4 == 0) rowf_s[8 * r + n] = p.scale_log2 * __int_as_float(e2 << 23);
#pragma unroll
            for (int step = 0; step < KSTEPS; ++step) {
                uint32_t hi[2], lo[2];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float a = x[4 * step + 2 * half] * up, c = x[4 * step + 2 * half + 1] * up;
                    const __half ah = __float2half_rn(a), ch = __float2half_rn(c);
                    hi[half] = ptx::pack_half2(__half2float(ah), __half2float(ch));
                    lo[half] = ptx::pack_half2(a - __half2float(ah), c - __half2float(ch));
                }
                q_s[(step * NR + r) * 32 + lane] = make_uint2(hi[0], hi[1]);
                q_s[Q_LO + (step * NR + r) * 32 + lane] = make_uint2(lo[0], lo[1]);
            }
        }
    }
    // this lane's rows from here on, as columns of the products: 8 r + 2 t4 + i
    float rowf[F32 ? NR : 1][2];
    if constexpr (F32 || !Cfg::Q_IN_REGS) __syncthreads();
    if constexpr (F32) {
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int i = 0; i < 2; ++i) rowf[r][i] = rowf_s[8 * r + 2 * t4 + i];
    }

    // ------------------------------------------------------------ the keys of this CTA
    float o[OT][NR][4];
#pragma unroll
    for (int i = 0; i < OT * NR * 4; ++i) o[i / (NR * 4)][i / 4 % NR][i % 4] = 0.f;
    float m[NR][2], l[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i) { m[r][i] = -FLT_MAX; l[r][i] = 0.f; }
    uint32_t ref = PLAIN ? 127u << 23 : 1u << 23;                 // bits of the power of two that weights are divided by
    float inv_ref = __int_as_float(PLAIN ? 127 << 23 : 253 << 23);

    const int key_n = kv_key<ROW>(n), key_t[2] = {kv_key<ROW>(2 * t4), kv_key<ROW>(2 * t4 + 1)};    // K's row and V's of this lane
    auto step = [&](int j) {
        const uint8_t *k_s = smem + (warp * NS + j % NS) * Cfg::STAGE, *v_s = k_s + Cfg::TILE;
        const float *ksc = reinterpret_cast<const float *>(smem + Cfg::OFF_SCALES + (warp * NS + j % NS) * KW * 8), *vsc = ksc + KW;
        const int c0 = c_from + j * KT + warp * KW;               // number of the step's first key
        const int key0 = c0 < s_end ? c0 : c0 + skip, key1 = c0 + KW - 1 < s_end ? c0 + KW - 1 : c0 + KW - 1 + skip;
        auto clear = [&](int i) {                                 // chunk i of V's stage
            *reinterpret_cast<uint4 *>(const_cast<uint8_t *>(v_s) + kv_at<ROW>(i / (ROW / 16), i % (ROW / 16))) = make_uint4(0u, 0u, 0u, 0u);
        };
        if (PLAIN && key0 < ctx + 1 - p.window && key1 >= p.sinks) {
            // between the sinks and the first row's window: keys that no row sees may hold anything, NaN too (codes are finite)
            for (int i = lane; i < KW * (ROW / 16); i += 32) {
                const int c = c0 + i / (ROW / 16), key = c < s_end ? c : c + skip;
                if (key < ctx + 1 - p.window && key >= p.sinks) clear(i);
            }
            __syncwarp();
            ptx::fence_proxy_async_smem();
        }
        if (c0 + KW > c_to) {
            // behind the last key: whatever the page or the ring held there, times a weight of zero, must be zero
            for (int i = (c_to - c0) * (ROW / 16) + lane; i < KW * (ROW / 16); i += 32) clear(i);
            __syncwarp();
            ptx::fence_proxy_async_smem();                        // before the copy that refills the stage
        }
        // s[g][r][2 u + i]: key 16 g + 8 u + key_n, row 8 r + 2 t4 + i
        float s[NG][NR][4];
#pragma unroll
        for (int i = 0; i < NG * NR * 4; ++i) s[i / (NR * 4)][i / 4 % NR][i % 4] = 0.f;
#pragma unroll
        for (int c = 0; c < ROW / 64; ++c) {
            uint32_t kw[NG][2][4];
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(k_s + kv_at<ROW>(16 * g + 8 * u + key_n, t4 + 4 * c));
                    kw[g][u][0] = x.x; kw[g][u][1] = x.y; kw[g][u][2] = x.z; kw[g][u][3] = x.w;
                }
#pragma unroll
            for (int e = 0; e < (PLAIN ? 2 : 4); ++e) {
                constexpr int STEPS = PLAIN ? 2 : 4;              // of a chunk
                uint32_t a[NG][4];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    if constexpr (PLAIN) {
                        a[g][0] = kw[g][0][2 * e]; a[g][2] = kw[g][0][2 * e + 1];
                        a[g][1] = kw[g][1][2 * e]; a[g][3] = kw[g][1][2 * e + 1];
                    } else {
                        kv_halves<FMT>(kw[g][0][e], a[g][0], a[g][2]);
                        kv_halves<FMT>(kw[g][1][e], a[g][1], a[g][3]);
                    }
                }
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    uint2 q;
                    if constexpr (Cfg::Q_IN_REGS) q = qr[STEPS * c + e][r];
                    else q = q_s[((4 * c + e) * NR + r) * 32 + lane];
#pragma unroll
                    for (int g = 0; g < NG; ++g) kv_mma(s[g][r], a[g], q.x, q.y);
                    if constexpr (F32) {
                        const uint2 q2 = q_s[Q_LO + ((4 * c + e) * NR + r) * 32 + lane];
#pragma unroll
                        for (int g = 0; g < NG; ++g) kv_mma(s[g][r], a[g], q2.x, q2.y);
                    }
                }
            }
        }
        // scores in units of log2, masks
        const bool need_mask = key1 >= ctx || (key0 < all_see && key1 >= p.sinks);
        float mx[NR][2];
#pragma unroll
        for (int r = 0; r < NR; ++r) mx[r][0] = mx[r][1] = -FLT_MAX;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float f = F32 ? 1.f : p.scale_log2;
                if constexpr (!PLAIN) f *= ksc[16 * g + 8 * u + key_n];
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int i = 0; i < 2; ++i) s[g][r][2 * u + i] *= F32 ? f * rowf[F32 ? r : 0][i] : f;
                if (need_mask) {
                    const int c = c0 + 16 * g + 8 * u + key_n, key = c < s_end ? c : c + skip;
#pragma unroll
                    for (int r = 0; r < NR; ++r)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int row = 8 * r + 2 * t4 + i;
                            bool sees;
                            if constexpr (PLAIN) sees = c < c_to && key < lows[row] + p.window && (key >= lows[row] || key < p.sinks);
                            else sees = key < ctx ? (key >= lows[row] || key < p.sinks) : (c < c_to && (words[row] >> (key - ctx) & 1));
                            if (!sees) s[g][r][2 * u + i] = -INFINITY;
                        }
                }
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int i = 0; i < 2; ++i) mx[r][i] = fmaxf(mx[r][i], s[g][r][2 * u + i]);
            }
        // the largest scale of the step's values; one that is not finite counts for the rows that see it only
        uint32_t top = 0;
        if constexpr (!PLAIN) {
            float my_vs = lane < KW && c0 + lane < c_to ? vsc[lane] : 0.f;
            if (!(my_vs < INFINITY)) my_vs = 0.f;
            top = __reduce_max_sync(0xffffffffu, __float_as_uint(my_vs));
        }
        float alpha[NR][2];
        bool rescale = false;
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) mx[r][i] = fmaxf(mx[r][i], __shfl_xor_sync(0xffffffffu, mx[r][i], w));
                const float next = mx[r][i] > m[r][i] + kKvLazy ? mx[r][i] : m[r][i];
                alpha[r][i] = ptx::ex2_approx(m[r][i] - next);
                rescale |= next != m[r][i];
                m[r][i] = next;
                l[r][i] *= alpha[r][i];
            }
        if (!PLAIN && top > ref) {
            const uint32_t next = min((top + 0x7fffffu) & 0x7f800000u, 253u << 23);
            const float f = __uint_as_float(ref) * __uint_as_float((254u << 23) - next);      // powers of two
            ref = next;
            inv_ref = __uint_as_float((254u << 23) - next);
#pragma unroll
            for (int r = 0; r < NR; ++r) { alpha[r][0] *= f; alpha[r][1] *= f; }
            rescale = true;
        }
        if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
            for (int d = 0; d < OT; ++d)
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[d][r][e] *= alpha[r][e & 1];
        }
        // weights, as operands of the second product
        uint32_t pa[NG][NR][2], pl[P2 ? NG : 1][NR][2];
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float f = PLAIN ? 1.f : vsc[16 * g + 8 * u + key_n] * inv_ref;
#pragma unroll
                for (int r = 0; r < NR; ++r) {
                    float x[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float w = ptx::ex2_approx(s[g][r][2 * u + i] - m[r][i] + kKvShift);
                        l[r][i] += w;
                        x[i] = w * f;
                        if (need_mask && s[g][r][2 * u + i] == -INFINITY) x[i] = 0.f;         // 0 times a scale that is not finite
                    }
                    const uint32_t hi = ptx::pack_half2(x[0], x[1]);
                    pa[g][r][u] = kv_transpose(hi);
                    if constexpr (P2) {
                        const float2 back = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                        pl[g][r][u] = kv_transpose(ptx::pack_half2(x[0] - back.x, x[1] - back.y));
                    }
                }
            }
        // O^T += V^T P^T: the two tiles of a word's four columns at a time
#pragma unroll
        for (int c = 0; c < (ROW + 127) / 128; ++c) {
            constexpr int WORDS = ROW == 64 ? 2 : 4;
            uint32_t v[NG][4][WORDS];
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int row = g * 16 + key_t[x & 1] + (x >> 1) * 8;
                    if constexpr (ROW == 64) {
                        const uint2 u = *reinterpret_cast<const uint2 *>(v_s + kv_at<ROW>(row, n >> 1) + (n & 1) * 8);
                        v[g][x][0] = u.x; v[g][x][1] = u.y;
                    } else {
                        const uint4 u = *reinterpret_cast<const uint4 *>(v_s + kv_at<ROW>(row, n + 8 * c));
                        v[g][x][0] = u.x; v[g][x][1] = u.y; v[g][x][2] = u.z; v[g][x][3] = u.w;
                    }
                }
#pragma unroll
            for (int w = 0; w < WORDS; ++w) {
                float part[F32 ? 2 : 1][NR][4];
                if constexpr (F32)
#pragma unroll
                    for (int e = 0; e < 2 * NR * 4; ++e) part[e / (NR * 4)][e / 4 % NR][e % 4] = 0.f;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    constexpr int TILES = PLAIN ? 1 : 2;          // of a word's columns
                    uint32_t a[2][4];
                    if constexpr (PLAIN) {
                        a[0][0] = __byte_perm(v[g][0][w], v[g][1][w], 0x5410); a[0][1] = __byte_perm(v[g][0][w], v[g][1][w], 0x7632);
                        a[0][2] = __byte_perm(v[g][2][w], v[g][3][w], 0x5410); a[0][3] = __byte_perm(v[g][2][w], v[g][3][w], 0x7632);
                    } else {
                        uint32_t a0[4], a1[4];                    // bytes 0 .. 3 of keys 2 t4, 2 t4 + 1 and of keys 8 further
                        kv_pairs<FMT>(v[g][0][w], v[g][1][w], a0);
                        kv_pairs<FMT>(v[g][2][w], v[g][3][w], a1);
#pragma unroll
                        for (int e = 0; e < 2; ++e) { a[e][0] = a0[2 * e]; a[e][1] = a0[2 * e + 1]; a[e][2] = a1[2 * e]; a[e][3] = a1[2 * e + 1]; }
                    }
#pragma unroll
                    for (int e = 0; e < TILES; ++e)
#pragma unroll
                        for (int r = 0; r < NR; ++r) {
                            float *acc = F32 ? part[F32 ? e : 0][r] : o[(c * 4 + w) * TILES + e][r];
                            kv_mma(acc, a[e], pa[g][r][0], pa[g][r][1]);
                            if constexpr (P2) kv_mma(acc, a[e], pl[g][r][0], pl[g][r][1]);
                        }
                }
                if constexpr (F32)
#pragma unroll
                    for (int e = 0; e < 2 * NR * 4; ++e) o[c * 8 + w * 2 + e / (NR * 4)][e / 4 % NR][e % 4] += part[e / (NR * 4)][e / 4 % NR][e % 4];
            }
        }
    };
    for (int j = 0; j < n_steps && ok; ++j) {
        if (j + NS - 1 < n_steps) request(j + NS - 1);            // over step j - 1: the warp has met since
        kv_copy_commit();
        kv_copy_wait<NS - 1>();                                   // this lane's scales of step j
        ok = ptx::mbar_wait(full + 8 * (j % NS), (uint32_t)(j / NS) & 1u, abort_flag);
        if (!ok) break;
        __syncwarp();                                             // the other lanes' scales
        step(j);
        __syncwarp();
    }
    if (run && !ok) { *abort_flag = 1; ptx::report(p.status, KV_ERR_ROWS); }

    // ------------------------------------------------------------ partial results
    // o[8 c + i][r][2 u + k]: element 128 c + 16 n + 2 i + u (at D = 64: 8 n + 2 i + u) of row 8 r + 2 t4 + k; plain keys:
    // o[4 c + i], element 64 c + 8 n + 2 i + u
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) l[r][i] += __shfl_xor_sync(0xffffffffu, l[r][i], w);
    kv_copy_wait<0>();
    __syncthreads();                                              // the rings are drained
    {
        constexpr int RUN = D == 64 || PLAIN ? 8 : 16, SPAN = D < 8 * RUN ? D : 8 * RUN;
        const float unit = __uint_as_float(ref);
        float *mine = part + warp * MR * D;
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int row = 8 * r + 2 * t4 + k;
                if (n == 0) ml[warp * MR + row] = make_float2(m[r][k], l[r][k]);
#pragma unroll
                for (int c = 0; c < D / SPAN; ++c)
#pragma unroll
                    for (int x = 0; x < RUN / 2; x += 2) {
                        const int i = RUN / 2 * c + x;
                        *reinterpret_cast<float4 *>(mine + row * D + SPAN * c + RUN * n + 2 * x) =
                            make_float4(o[i][r][k] * unit, o[i][r][2 + k] * unit, o[i + 1][r][k] * unit, o[i + 1][r][2 + k] * unit);
                    }
            }
    }
    __syncthreads();
    // Warps of the CTA: number `i` of MR x D / 4 float4s over them, into the first one's place
    constexpr int QUADS = D / 4;
    const int asked = PLAIN ? p.tokens : kv_nodes_asked(p, b);
    auto write = [&](int r, int quad, float4 v, float sum) {
        const int row = row0 + r, node = row % p.tokens;
        if (row >= rows || node >= asked) return;
        const float f = *bad || *abort_flag || node >= nodes ? __int_as_float(0x7fc00000) : 1.f / sum;               // no visible key: 0 * inf = NaN
        v.x *= f; v.y *= f; v.z *= f; v.w *= f;
        const int64_t to = ((int64_t)kvh * rows + row) * D + quad * 4;
        if (p.out_f16)
            *reinterpret_cast<uint2 *>(static_cast<__half *>(p.out) + to) = make_uint2(ptx::pack_half2(v.x, v.y), ptx::pack_half2(v.z, v.w));
        else
            *reinterpret_cast<float4 *>(static_cast<float *>(p.out) + to) = v;
    };
    auto add = [](float4 &a, const float4 &x, float f) { a.x += x.x * f; a.y += x.y * f; a.z += x.z * f; a.w += x.w * f; };
    for (int i = tid; i < MR * QUADS; i += Cfg::THREADS) {
        const int r = i / QUADS, quad = i % QUADS;
        float mn = -FLT_MAX, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < Cfg::WARPS; ++w) mn = fmaxf(mn, ml[w * MR + r].x);
#pragma unroll
        for (int w = 0; w < Cfg::WARPS; ++w) {
            const float2 s = ml[w * MR + r];
            const float f = ptx::ex2_approx(s.x - mn);
            add(acc, *reinterpret_cast<const float4 *>(part + (w * MR + r) * D + quad * 4), f);
            sum += s.y * f;
        }
        if (splits == 1) write(r, quad, acc, sum);
        else {
            *reinterpret_cast<float4 *>(part + r * D + quad * 4) = acc;
            if (quad == 0) cta_ml[r] = make_float2(mn, *bad || *abort_flag ? __int_as_float(0x7fc00000) : sum);
        }
    }
    if (*abort_flag)
        for (int i = 0; i < 64; ++i) __nanosleep(2000);           // let copies in flight land
    if (splits == 1) return;
    cluster.sync();
    for (int i = split * Cfg::THREADS + tid; i < MR * QUADS; i += splits * Cfg::THREADS) {
        const int r = i / QUADS, quad = i % QUADS;
        const float *at_part = part + r * D + quad * 4;
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
