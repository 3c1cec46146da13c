// Gradients of the sinks' keys and values (window.cuh): the few keys that every later row sees.
//
// With s_ij = q_i . k_j / sqrt(D), P = 2^(s log2e - lse_i), dS = P o (dO V^T - delta_i) / sqrt(D), summed over all rows i that
// see key j:      dV_j = sum_i P_ij dO_i        dK_j = sum_i dS_ij Q_i
// A key tile of the dK/dV kernel has 64 or 128 keys, so that tile's work over all rows is nearly all spent on keys that the
// rows do not see: 51 us alone (B4 H16 S2048 d128, window 512, four sinks), 24 us here, where a tile is sixteen keys.
//
// Bound: Q and dO are read once (L2, as the dQ and dK/dV kernels have just read them).  A warp takes sixteen rows at a time
// through a ring of its own and keeps its sums of both gradients in registers (mma m16n8k16, fp32 sums):
//     S^T = K Q^T, dP^T = V dO^T    keys are the products' rows, so that the results are, converted to fp16, the left operands of
//     dV += P^T dO, dK += dS^T Q    whose right operands are the same rows, transposed as they are read from shared memory.
// P and dS are rounded to fp16 as in the dK/dV kernel.  Warps, then the CTAs of a cluster, are added in a fixed order: the same
// bits on every run.  The launch stands between those of the dQ and the dK/dV kernel, starts under the first and lets the second
// start beside it: neither reads what it writes, and the dK/dV kernel leaves the sinks' rows out.
#pragma once
#include <cooperative_groups.h>

#include "ptx.cuh"
#include "sdpa_bwd.cuh"

namespace txb {

struct SinkGradParams {
    const __half *q, *k, *v, *dout;    // [B,Hq,Sq,D], [B,Hkv,Sk,D] x 2, [B,Hq,Sq,D]
    const float *lse, *delta;          // [B,Hq,Sq]
    KvLens kv_lens;
    int *prepared;
    void *dk, *dv;                     // [B,Hkv,Sk,D], fp32 or fp16 (grads_f16); rows below `sinks` are written
    WindowRule win;
    int Hkv, group, Sq, Sk;            // group = Hq / Hkv
    int grads_f16;
    float scale, scale_log2;
};

template <int D_>
struct SinkGradCfg {
    static constexpr int D = D_, WARPS = 8, THREADS = 32 * WARPS, NS = 3;
    static constexpr uint32_t TILE = 16 * D * 2;                         // sixteen rows
    static constexpr uint32_t STAGE = 2 * TILE + 128;                    // Q, dO, lse, delta
    static constexpr uint32_t OFF_K = WARPS * NS * STAGE, OFF_V = OFF_K + TILE;
    static constexpr uint32_t SMEM = OFF_V + TILE;
    static constexpr int CTAS_PER_SM = 2 * (SMEM + 1024) <= 233472 ? 2 : 1;
    static constexpr uint32_t PART = 2 * 16 * D * 4;                     // partial dK, dV of a warp, over the drained rings
    static_assert(D == 64 || D == 128, "both gradients of sixteen keys are registers of one warp");
    static_assert(SMEM <= 232448 && WARPS * PART <= OFF_K, "shared memory");
};

__device__ __forceinline__ void sink_mma(float *c, const uint32_t *a, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void sink_load4(uint32_t *r, uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void sink_load4_trans(uint32_t *r, uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, Cfg::CTAS_PER_SM)
sdpa_bwd_sinks_kernel(const __grid_constant__ SinkGradParams p)
{
    constexpr int D = Cfg::D, NS = Cfg::NS, CHUNKS = D / 8;
    namespace cg = cooperative_groups;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sbase = ptx::smem_u32(smem);
    cg::cluster_group cluster = cg::this_cluster();
    const int split = (int)cluster.block_rank(), splits = (int)cluster.num_blocks();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = lane >> 2, t4 = lane & 3;

    const int kvh = (int)blockIdx.x / splits, last = min(p.win.sinks, p.Sk);           // batch element and K/V head
    const int limit = p.kv_lens.limit(kvh / p.Hkv, p.Sk), off = p.win.offset(limit, p.Sq), front = p.win.front(off);
    const int64_t rows = (int64_t)p.group * p.Sq, first_row = (int64_t)kvh * rows;    // a head's rows follow the one before's
    const int steps = limit > 0 ? (int)((rows + 15) / 16) : 0;

    ptx::grid_trigger();
    // What the preprocess wrote is there once the dQ kernel says so (sdpa_bwd.cuh)
    if (tid == 0 && ptx::load_acquire(p.prepared) != 1) ptx::grid_wait();
    __syncthreads();

    // rows of D halves in 16-byte chunks, chunk c of row r at c ^ (r % 8): reads of eight rows touch every bank once
    auto at = [](int r, int c) { return (uint32_t)(r * CHUNKS + (c ^ (r & 7))) * 16u; };
    for (int i = tid; i < 2 * 16 * CHUNKS; i += Cfg::THREADS) {
        const int r = i / CHUNKS % 16, c = i % CHUNKS;
        const __half *src = i < 16 * CHUNKS ? p.k : p.v;
        const uint32_t dst = (i < 16 * CHUNKS ? Cfg::OFF_K : Cfg::OFF_V) + at(r, c);
        // keys behind the last may hold anything: zero
        *reinterpret_cast<uint4 *>(smem + dst) =
            r < limit ? __ldg(reinterpret_cast<const uint4 *>(src + ((int64_t)kvh * p.Sk + r) * D) + c) : make_uint4(0u, 0u, 0u, 0u);
    }

    // the warp's steps: number rank, rank + every, ... of all
    const int every = splits * Cfg::WARPS, rank = split * Cfg::WARPS + warp;
    const uint32_t ring = warp * NS * Cfg::STAGE;
    auto request = [&](int j) {
        const uint32_t stage = ring + j % NS * Cfg::STAGE;
        const int64_t row0 = ((int64_t)rank + (int64_t)j * every) * 16;
        auto copy = [&](auto there) {
#pragma unroll 4
            for (int i = lane; i < 2 * 16 * CHUNKS; i += 32) {
                const int r = i / CHUNKS % 16, c = i % CHUNKS;
                const __half *src = i < 16 * CHUNKS ? p.q : p.dout;
                const uint32_t dst = stage + (i < 16 * CHUNKS ? 0 : Cfg::TILE) + at(r, c);
                if (there(r)) ptx::cp_async16(sbase + dst, src + (first_row + row0 + r) * D + c * 8);
                else *reinterpret_cast<uint4 *>(smem + dst) = make_uint4(0u, 0u, 0u, 0u);
            }
        };
        // queries in front of the first key see none and may hold anything: zero
        if (front > 0) copy([&](int r) { return row0 + r < rows && (int)((row0 + r) % p.Sq) >= front; });
        else copy([&](int r) { return row0 + r < rows; });
        if (row0 + (lane & 15) < rows)
            ptx::cp_async4(sbase + stage + 2 * Cfg::TILE + lane * 4, (lane < 16 ? p.lse : p.delta) + first_row + row0 + (lane & 15));
    };
    const int mine = steps > rank ? (steps - rank + every - 1) / every : 0;
#pragma unroll
    for (int j = 0; j < NS - 1; ++j) {
        if (j < mine) request(j);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    __syncthreads();                                              // K and V

    float dk[D / 8][4], dv[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8 * 4; ++i) dk[i / 4][i % 4] = dv[i / 4][i % 4] = 0.f;
    for (int j = 0; j < mine; ++j) {
        if (j + NS - 1 < mine) request(j + NS - 1);               // over step j - 1: the warp has met since
        asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group %0;" ::"n"(NS - 1) : "memory");
        __syncwarp();
        const uint32_t stage = ring + j % NS * Cfg::STAGE, q_s = sbase + stage, do_s = q_s + Cfg::TILE;
        // element [x][2 u + i]: key n + 8 u, row 8 x + 2 t4 + i
        float s[2][4] = {}, dp[2][4] = {};
#pragma unroll
        for (int c = 0; c < CHUNKS; c += 2) {
            uint32_t ka[4], va[4], qb[4], ob[4];
            const uint32_t left = at(lane & 15, c + (lane >> 4)), right = at((lane & 7) + (lane >> 4) * 8, c + (lane >> 3 & 1));
            sink_load4(ka, sbase + Cfg::OFF_K + left);
            sink_load4(qb, q_s + right);
            sink_mma(s[0], ka, qb[0], qb[1]);
            sink_mma(s[1], ka, qb[2], qb[3]);
            sink_load4(va, sbase + Cfg::OFF_V + left);
            sink_load4(ob, do_s + right);
            sink_mma(dp[0], va, ob[0], ob[1]);
            sink_mma(dp[1], va, ob[2], ob[3]);
        }
        const float *stat = reinterpret_cast<const float *>(smem + stage + 2 * Cfg::TILE);
        const int64_t row0 = ((int64_t)rank + (int64_t)j * every) * 16;
        const int at0 = (int)(row0 % p.Sq);
        uint32_t pa[4], da[4];                                    // as left operands: rows are keys, columns the sixteen rows
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            float w[4], ds[4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 8 * x + 2 * t4 + i;
                int at_r = at0 + r;
                if (at_r >= p.Sq) at_r %= p.Sq;
                const int pos = row0 + r < rows ? off + at_r : -1;
                const float lse = stat[r], delta = stat[16 + r];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int key = n + 8 * u;
                    const bool sees = key <= pos && key < limit;  // a row that sees nothing has no statistics
                    const float e = ptx::ex2_approx(s[x][2 * u + i] * p.scale_log2 - lse);
                    w[2 * u + i] = sees ? e : 0.f;
                    ds[2 * u + i] = sees ? e * ((dp[x][2 * u + i] - delta) * p.scale) : 0.f;
                }
            }
            pa[2 * x] = ptx::pack_half2(w[0], w[1]); pa[2 * x + 1] = ptx::pack_half2(w[2], w[3]);
            da[2 * x] = ptx::pack_half2(ds[0], ds[1]); da[2 * x + 1] = ptx::pack_half2(ds[2], ds[3]);
        }
#pragma unroll
        for (int c = 0; c < D / 8; c += 2) {
            uint32_t qb[4], ob[4];
            const uint32_t right = at(lane & 15, c + (lane >> 4));
            sink_load4_trans(ob, do_s + right);
            sink_mma(dv[c], pa, ob[0], ob[1]);
            sink_mma(dv[c + 1], pa, ob[2], ob[3]);
            sink_load4_trans(qb, q_s + right);
            sink_mma(dk[c], da, qb[0], qb[1]);
            sink_mma(dk[c + 1], da, qb[2], qb[3]);
        }
        __syncwarp();
    }

    // partial gradients [dK, dV][16][D] of the warps, of the CTA in the first one's place, of the cluster
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();
    float *part = reinterpret_cast<float *>(smem), *my_part = part + warp * (Cfg::PART / 4);
#pragma unroll
    for (int c = 0; c < D / 8; ++c)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int to = (n + 8 * u) * D + 8 * c + 2 * t4;
            *reinterpret_cast<float2 *>(my_part + to) = make_float2(dk[c][2 * u], dk[c][2 * u + 1]);
            *reinterpret_cast<float2 *>(my_part + 16 * D + to) = make_float2(dv[c][2 * u], dv[c][2 * u + 1]);
        }
    __syncthreads();
    constexpr int QUADS = Cfg::PART / 16;
    auto add = [](float4 &a, const float4 &x) { a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w; };
    for (int i = tid; i < QUADS; i += Cfg::THREADS) {
        float4 a = reinterpret_cast<const float4 *>(part)[i];
#pragma unroll
        for (int w = 1; w < Cfg::WARPS; ++w) add(a, reinterpret_cast<const float4 *>(part + w * (Cfg::PART / 4))[i]);
        reinterpret_cast<float4 *>(part)[i] = a;
    }
    cluster.sync();
    for (int i = split * Cfg::THREADS + tid; i < QUADS; i += splits * Cfg::THREADS) {
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < splits; ++c) add(a, *reinterpret_cast<const float4 *>(cluster.map_shared_rank(part + i * 4, c)));
        const int row = i / (D / 4) % 16, col = i % (D / 4) * 4;
        if (row >= last) continue;
        void *to = i < QUADS / 2 ? p.dk : p.dv;
        const int64_t e = ((int64_t)kvh * p.Sk + row) * D + col;
        if (p.grads_f16) *reinterpret_cast<uint2 *>(static_cast<__half *>(to) + e) = make_uint2(ptx::pack_half2(a.x, a.y), ptx::pack_half2(a.z, a.w));
        else *reinterpret_cast<float4 *>(static_cast<float *>(to) + e) = a;
    }
    if (tid == 0) ptx::grid_wait();                               // what follows in the stream takes the dQ kernel for done
    cluster.sync();                                               // nobody leaves while its shared memory is read
}

}  // namespace txb
