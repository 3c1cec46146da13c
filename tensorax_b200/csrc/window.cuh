// Sliding window with sinks: row i of batch element b stands at position p = i, or at len_b - Sq + i where the rows are the
// last ones of their sequence (align_end), and sees key j iff j < len_b, j <= p and (j > p - window or j < sinks).
//
// The kernels that take it walk lists of key tiles instead of all of them: first the tiles of the sinks, then those from
// the window of the tile's first row on.  What that leaves out is never loaded; the tiles at the list's edges are masked
// element by element.  Every instantiation without a window is the code it was before (if constexpr on Cfg::WINDOW).
#pragma once
#include <cstdint>

namespace txb {

struct WindowRule {
    int window = 0, sinks = 0, align_end = 0;
    // Position of row 0 of a batch element with `limit` keys
    __device__ __forceinline__ int offset(int limit, int Sq) const { return align_end ? limit - Sq : 0; }
    // Of a batch element with keys, the rows that see none: those in front of row `front`, and without sinks those from row
    // `behind` on
    __device__ __forceinline__ int front(int off) const { return max(0, -off); }
    __device__ __forceinline__ int behind(int limit, int off) const { return (int)min((int64_t)0x7fffffff, (int64_t)limit + window - 1 - off); }
};

// The key tiles of BN keys that rows at positions [pos0, pos0 + rows) walk: list entry j is tile j for j < n_sink, else
// tile j - n_sink + w_tile; tiles at `end` and beyond are not walked.
template <int BN>
struct WindowWalk {
    int n_sink, w_tile, end;
    __device__ __forceinline__ WindowWalk(const WindowRule &w, int limit, int pos0, int rows)
    {
        const int kv_end = max(0, min(limit, pos0 + rows));
        end = (kv_end + BN - 1) / BN;
        w_tile = min(max(0, pos0 - w.window + 1) / BN, end);
        n_sink = min((min(w.sinks, kv_end) + BN - 1) / BN, w_tile);
    }
    __device__ __forceinline__ int tile(int j) const { return j < n_sink ? j : j - n_sink + w_tile; }
    __device__ __forceinline__ int count() const { return n_sink + end - w_tile; }
    // entries that hold a key below kv_end
    __device__ __forceinline__ int count_below(int kv_end) const
    {
        const int e = (max(kv_end, 0) + BN - 1) / BN;
        return min(n_sink, e) + max(0, min(end, e) - w_tile);
    }
};

// Whether some row at [pos0, pos0 + rows) sees some key of [kv0, kv0 + BN) and another does not see another
__device__ __forceinline__ bool window_edge(const WindowRule &w, int limit, int pos0, int rows, int kv0, int BN)
{
    return kv0 + BN > limit || kv0 + BN - 1 > pos0 || (kv0 <= pos0 + rows - 1 - w.window && kv0 + BN > w.sinks);
}

// The columns of a tile that a row sees: [lo, hi) and, below hi, [0, s)
struct WindowColumns {
    int lo, hi, s;
    __device__ __forceinline__ WindowColumns(const WindowRule &w, int limit, int pos, int kv0)
        : lo(pos - w.window + 1 - kv0), hi(min(limit, pos + 1) - kv0), s(w.sinks - kv0) {}
};

// v where column i is seen, else -inf (else 0): compares and a select, no branch
__device__ __forceinline__ uint32_t keep_if_seen(uint32_t v, int i, const WindowColumns &c)
{
    uint32_t r;
    asm("{\n\t.reg .pred p;\n\tsetp.ge.s32 p, %2, %3;\n\tsetp.lt.or.s32 p, %2, %5, p;\n\tsetp.lt.and.s32 p, %2, %4, p;\n\t"
        "selp.b32 %0, %1, 0xff800000, p;\n\t}"
        : "=r"(r) : "r"(v), "r"(i), "r"(c.lo), "r"(c.hi), "r"(c.s));
    return r;
}
__device__ __forceinline__ float zero_unless_seen(float v, int i, const WindowColumns &c)
{
    float r;
    asm("{\n\t.reg .pred p;\n\tsetp.ge.s32 p, %2, %3;\n\tsetp.lt.or.s32 p, %2, %5, p;\n\tsetp.lt.and.s32 p, %2, %4, p;\n\t"
        "selp.f32 %0, %1, 0f00000000, p;\n\t}"
        : "=f"(r) : "f"(v), "r"(i), "r"(c.lo), "r"(c.hi), "r"(c.s));
    return r;
}
// v where lo <= i < hi, else 0
__device__ __forceinline__ float zero_unless_within(float v, int i, int lo, int hi)
{
    float r;
    asm("{\n\t.reg .pred p;\n\tsetp.ge.s32 p, %2, %3;\n\tsetp.lt.and.s32 p, %2, %4, p;\n\tselp.f32 %0, %1, 0f00000000, p;\n\t}"
        : "=f"(r) : "f"(v), "r"(i), "r"(lo), "r"(hi));
    return r;
}

// Rows [from, to) of a stage of `panels` panels [BN][128 bytes] become zero: keys behind a sequence's last, queries that see no
// key, whatever they hold (a zero weight times a NaN would be one).  THREADS threads share them; the caller orders the writes
// before the MMA that reads the stage.
template <int BN, int THREADS>
__device__ __forceinline__ void zero_stage_rows(uint8_t *stage, int panels, int from, int thread, int to = BN)
{
    const int chunks = (to - from) * 8;
    for (int pn = 0; pn < panels; ++pn)
        for (int i = thread; i < chunks; i += THREADS)
            *reinterpret_cast<uint4 *>(stage + pn * (BN * 128) + from * 128 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
}

}  // namespace txb
