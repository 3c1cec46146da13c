// C ABI of the quantised K/V cache: validation, kernel selection, launch.  Declarations: include/tensorax_b200.h.
#include "../../include/tensorax_b200.h"

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "api_internal.h"
#include "kv_attention.cuh"
#include "kv_attention_tc.cuh"
#include "kv_cache.cuh"

namespace {

using txb::api::fail;

#define TX_CUDA(call)                                                                     \
    do {                                                                                  \
        cudaError_t e_ = (call);                                                          \
        if (e_ != cudaSuccess)                                                            \
            return fail(TX_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(e_));     \
    } while (0)

bool aligned(const void *p, uintptr_t by) { return (reinterpret_cast<uintptr_t>(p) & (by - 1)) == 0; }

// What every call says: the cache, the page table, the batch
int pages_of(const char *who, const tx_kv_cache &c, const int32_t *table, int64_t batch, int64_t table_len, int32_t dtype,
             txb::KvPages *out)
{
    if (!c.k || !c.v || !c.k_scale || !c.v_scale || !table) return fail(TX_ERR_INVALID, "%s: null pointer", who);
    if (!aligned(c.k, 16) || !aligned(c.v, 16) || !aligned(c.k_scale, 16) || !aligned(c.v_scale, 16) || !aligned(table, 4))
        return fail(TX_ERR_INVALID, "%s: the cache's codes and scales must be 16-byte aligned, the page table 4-byte", who);
    if (c.pages <= 0 || c.kv_heads <= 0 || batch <= 0 || table_len <= 0) return fail(TX_ERR_INVALID, "%s: every dimension must be positive", who);
    if (c.d != 64 && c.d != 128 && c.d != 256) return fail(TX_ERR_UNSUPPORTED, "%s: head dim must be 64, 128 or 256", who);
    if (c.page_size < 16 || c.page_size > 65536 || (c.page_size & (c.page_size - 1)))
        return fail(TX_ERR_INVALID, "%s: page_size must be a power of two from 16 to 65536", who);
    if (c.format != TX_KV_E4M3 && c.format != TX_KV_INT8) return fail(TX_ERR_INVALID, "%s: format must be TX_KV_E4M3 or TX_KV_INT8", who);
    if (dtype != TX_DTYPE_F32 && dtype != TX_DTYPE_F16) return fail(TX_ERR_INVALID, "%s: dtype must be float32 or float16", who);
    // positions, rows of the cache and its 128-byte lines are 32-bit numbers, byte offsets 64-bit
    if (c.pages > 0x7fffffffLL || c.kv_heads > 65535 || batch > 0xffffffLL || batch * c.kv_heads > 0x3fffffffLL || table_len > 0x7fffffffLL ||
        table_len * c.page_size > 0x7fffffffLL || c.pages * c.kv_heads > 0x7fffffffLL / (c.page_size * (c.d / 64)))
        return fail(TX_ERR_UNSUPPORTED, "%s: dimension too large", who);
    out->k = static_cast<uint8_t *>(c.k); out->v = static_cast<uint8_t *>(c.v);
    out->ks = c.k_scale; out->vs = c.v_scale;
    out->table = table; out->table_len = table_len;
    out->pages = (int)c.pages; out->Hkv = (int)c.kv_heads;
    out->page_shift = 0;
    while ((int64_t{1} << out->page_shift) < c.page_size) out->page_shift++;
    return TX_OK;
}

// f(T(), integral format, integral head dim) for the call's types
template <class F>
int for_types(int32_t dtype, int32_t format, int64_t d, F f)
{
    auto with_d = [&](auto t, auto fmt) -> int {
        if (d == 64) return f(t, fmt, std::integral_constant<int, 64>());
        if (d == 128) return f(t, fmt, std::integral_constant<int, 128>());
        return f(t, fmt, std::integral_constant<int, 256>());
    };
    auto with_fmt = [&](auto t) -> int {
        if (format == TX_KV_E4M3) return with_d(t, std::integral_constant<int, txb::KV_E4M3>());
        return with_d(t, std::integral_constant<int, txb::KV_INT8>());
    };
    return dtype == TX_DTYPE_F16 ? with_fmt(__half()) : with_fmt(float());
}

// Write and read: one launch over batch * kv_heads * tokens rows
template <bool WRITE>
int move_rows(const char *who, const tx_kv_cache &c, const void *k, const void *v, const int32_t *table, const int32_t *start,
              const int32_t *counts, const int32_t *pick, int64_t batch, int64_t tokens, int64_t src_tokens, int64_t table_len,
              int32_t dtype, int32_t flags, void *stream)
{
    txb::KvMoveParams p;
    if (!k || !v) return fail(TX_ERR_INVALID, "%s: null pointer", who);
    if (int rc = pages_of(who, c, table, batch, table_len, dtype, &p.pages)) return rc;
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(TX_ERR_INVALID, "%s: k and v must be 16-byte aligned", who);
    if (flags != 0) return fail(TX_ERR_INVALID, "%s: unknown flags", who);
    if (tokens <= 0 || src_tokens < 0) return fail(TX_ERR_INVALID, "%s: every dimension must be positive", who);
    if (src_tokens == 0) src_tokens = tokens;
    if (!pick && src_tokens < tokens) return fail(TX_ERR_INVALID, "%s: k and v hold fewer rows than tokens", who);
    if (tokens > 0x3fffffffLL || src_tokens > 0x3fffffffLL) return fail(TX_ERR_UNSUPPORTED, "%s: dimension too large", who);
    if (int rc = txb::api::ensure_device()) return rc;
    if (int rc = txb::api::page_word(&p.page_status)) return rc;
    p.k = const_cast<void *>(k); p.v = const_cast<void *>(v);
    p.start = start; p.counts = counts; p.pick = pick;
    p.tokens = (int)tokens; p.src_tokens = (int)src_tokens;
    return for_types(dtype, c.format, c.d, [&](auto t, auto fmt, auto d) -> int {
        using T = decltype(t);
        constexpr int per_cta = txb::KvMoveItem<d()>::PER_CTA;
        p.ctas = (int)((tokens + per_cta - 1) / per_cta);
        const int64_t ctas = batch * c.kv_heads * p.ctas;
        if (ctas > 0x7fffffffLL) return fail(TX_ERR_UNSUPPORTED, "%s: dimension too large", who);
        const cudaStream_t st = static_cast<cudaStream_t>(stream);
        if constexpr (WRITE) txb::kv_write_kernel<T, fmt(), d()><<<(unsigned)ctas, txb::KV_MOVE_THREADS, 0, st>>>(p);
        else txb::kv_read_kernel<T, fmt(), d()><<<(unsigned)ctas, txb::KV_MOVE_THREADS, 0, st>>>(p);
        txb::api::launched();
        TX_CUDA(cudaGetLastError());
        return TX_OK;
    });
}

// cudaFuncSetAttribute once per kernel and device
template <auto Kernel>
int allow_launch(int smem)
{
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    if (int rc = txb::api::current_device(&dev)) return rc;
    if (done.load(std::memory_order_acquire) >> dev & 1u) return TX_OK;
    TX_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    TX_CUDA(cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    done.fetch_or(uint64_t{1} << dev, std::memory_order_release);
    return TX_OK;
}

// CTAs of a cluster that share the keys of an item: as many as one wave holds -- up to eight, or sixteen -- as long as each has
// a tile of KT of the most keys that the call can see.  B16 Hkv8, 4096 to 8192 keys, d128, a row a head: in two 50.2 us, in three
// 45.5 (all places of one wave), in four 57.0, in six 49.7.
int splits_of(int64_t keys, int64_t items, int64_t places, int most, int kt)
{
    const int64_t splits = std::max<int64_t>(1, std::min({(int64_t)most, places / items, (keys + kt - 1) / kt}));
    return splits >= 16 ? 16 : (int)std::min<int64_t>(splits, 8);
}

int64_t keys_seen(const tx_kv_attention_desc *d)
{
    const int64_t keys = d->table_len * d->cache.page_size;
    return d->window > 0 ? std::min(keys, std::min<int64_t>(d->window, 0x7fffffff) + std::min<int64_t>(d->sinks, 0x7fffffff) + d->tokens) : keys;
}

template <class... Params, class... Args>
int launch_cluster(void (*kernel)(Params...), int64_t ctas, int cluster, int threads, size_t smem, void *stream, const Args &...args)
{
    if (ctas > 0x7fffffffLL) return fail(TX_ERR_UNSUPPORTED, "K/V cache attention: more than 2^31 work items");
    // (the kernels wait for what is in front of them in the stream before they read anything)
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cluster; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cfg.attrs = at;
    cfg.numAttrs = 2;
    TX_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    txb::api::launched();
    return TX_OK;
}

template <class Cfg>
int launch_attention_t(txb::KvAttnParams p, const tx_kv_attention_desc *d)
{
    const int64_t rows = (int64_t)p.group * p.tokens;
    p.row_parts = (int)((rows + Cfg::MR - 1) / Cfg::MR);
    const int64_t items = d->batch * d->cache.kv_heads * p.row_parts;
    int sms = 0;
    if (int rc = txb::api::sm_count(&sms)) return rc;
    const int splits = splits_of(keys_seen(d), items, (int64_t)Cfg::CTAS_PER_SM * sms, Cfg::MAX_SPLITS, Cfg::KT);
    if (int rc = allow_launch<txb::kv_attention_kernel<Cfg>>((int)Cfg::SMEM)) return rc;
    CUtensorMap tk, tv;
    const int64_t cache_rows = d->cache.pages * d->cache.kv_heads * d->cache.page_size;
    if (int rc = txb::api::map_of_codes(&tk, d->cache.k, cache_rows, d->cache.d)) return rc;
    if (int rc = txb::api::map_of_codes(&tv, d->cache.v, cache_rows, d->cache.d)) return rc;
    return launch_cluster(txb::kv_attention_kernel<Cfg>, items * splits, splits, Cfg::THREADS, Cfg::SMEM, d->stream, tk, tv, p);
}

template <class Cfg>
int launch_attention_tc(txb::KvAttnParams p, const tx_kv_attention_desc *d)
{
    const int64_t rows = (int64_t)p.group * p.tokens;
    p.row_parts = (int)((rows + Cfg::MR - 1) / Cfg::MR);
    const int64_t items = d->batch * d->cache.kv_heads * p.row_parts;
    int sms = 0;
    if (int rc = txb::api::sm_count(&sms)) return rc;
    const int splits = splits_of(keys_seen(d), items, sms, Cfg::MAX_SPLITS, Cfg::BN);
    if (int rc = allow_launch<txb::kv_attention_tc_kernel<Cfg>>((int)Cfg::SMEM)) return rc;
    return launch_cluster(txb::kv_attention_tc_kernel<Cfg>, items * splits, splits, Cfg::THREADS, Cfg::SMEM, d->stream, p);
}

// More query rows per K/V head than this: the tcgen05 kernel, whose CTA takes 256 at once.  Hkv8, us there and here, e4m3:
// B8, 8192 keys, d128: 32 rows 81 and 50, 64 rows 82 and 86; d64: 65 and 35, 65 and 63; B1, 2000 keys, d128: 18 and 16, 19 and 26;
// B16, 1000 keys: 28 and 24, 29 and 31.  int8, whose codes take longer to turn into fp16: 64 rows 105 and 94, 73 and 65, 20 and 26,
// 35 and 33.  128 rows, e4m3, B8: 83 and 162.  d256 and fp32 queries have the other kernel only, whose parts of up to 16 or 32
// rows read and convert the keys each for itself.
template <int FMT>
constexpr int kTcRows = FMT == txb::KV_E4M3 ? 32 : 64;

template <typename T, int FMT, int D>
int launch_attention(const txb::KvAttnParams &p, const tx_kv_attention_desc *d)
{
    const int64_t rows = (int64_t)p.group * p.tokens;
    if constexpr (sizeof(T) == 2 && D <= 128)
        if (rows > kTcRows<FMT>) return launch_attention_tc<txb::KvTcCfg<FMT, D, D == 64 ? 0x0303 : 0x0003>>(p, d);
    // Rows of a part: eight at a time up to 32 (16 at d = 256), as registers hold them.  Steps of 32 keys where registers allow
    // (B16 Hkv8, 8192 keys, d128: four rows 67.6 us with 32 keys a step and three CTAs an SM, 69.7 with 16 and four; sixteen
    // rows 71.7 and 101; 32 rows a head at 256 in all 352 and 463).
    constexpr bool F32 = sizeof(T) == 4;
    if constexpr (D == 256) {
        if (rows <= 8) return launch_attention_t<txb::KvAttnCfg<T, FMT, D, 1, 4, 16, 3, F32 ? 1 : 2>>(p, d);
        return launch_attention_t<txb::KvAttnCfg<T, FMT, D, 2, 4, 16, 3, F32 ? 1 : 2>>(p, d);
    } else {
        constexpr int NS1 = D == 64 ? 4 : F32 ? 3 : 2, NS = D == 64 ? 4 : 3;
        if (rows <= 8) return launch_attention_t<txb::KvAttnCfg<T, FMT, D, 1, 4, 32, NS1, F32 ? 2 : 3>>(p, d);
        if (rows <= 16) return launch_attention_t<txb::KvAttnCfg<T, FMT, D, 2, 4, F32 ? 16 : 32, F32 ? 4 : NS, 2>>(p, d);
        return launch_attention_t<txb::KvAttnCfg<T, FMT, D, 4, 4, F32 ? 16 : 32, F32 ? 4 : NS, 2>>(p, d);
    }
}

}  // namespace

namespace txb {
namespace api {

bool window_step_fits(const tx_sdpa_desc *d)
{
    if (d->dtype != TX_DTYPE_F16 || d->lse || (d->d_k != 64 && d->d_k != 128) || !aligned(d->out, 16)) return false;
    return d->q_heads / d->kv_heads * d->seq_q <= 16 && d->batch * d->kv_heads * d->seq_k * d->d_k / 64 <= 0x7fffffffLL;
}

int window_step(const tx_sdpa_desc *d, const KvLens &lens, int window, int sinks, int align_end, int *status)
{
    KvPlainParams p = {};
    p.lens = lens;
    p.Sk = (int)d->seq_k; p.align_end = align_end;
    p.pages.Hkv = (int)d->kv_heads;
    p.q = d->q; p.out = d->out; p.status = status;
    p.tokens = (int)d->seq_q; p.group = (int)(d->q_heads / d->kv_heads);
    p.window = window; p.sinks = sinks;
    p.out_f16 = (d->flags & TX_SDPA_OUT_F16) ? 1 : 0;
    p.scale_log2 = (1.0f / std::sqrt((float)d->d_k)) * 1.4426950408889634f;
    auto launch = [&](auto cfg) -> int {
        using Cfg = decltype(cfg);
        p.row_parts = (p.group * p.tokens + Cfg::MR - 1) / Cfg::MR;
        const int64_t heads = d->batch * d->kv_heads, items = heads * p.row_parts;
        int sms = 0;
        if (int rc = sm_count(&sms)) return rc;
        const int splits = splits_of(std::min<int64_t>(d->seq_k, (int64_t)window + sinks + d->seq_q), items, (int64_t)Cfg::CTAS_PER_SM * sms,
                                     Cfg::MAX_SPLITS, Cfg::KT);
        if (int rc = allow_launch<kv_attention_kernel<Cfg>>((int)Cfg::SMEM)) return rc;
        CUtensorMap tk, tv;
        if (int rc = map_of_codes(&tk, d->k, heads * d->seq_k, 2 * d->d_k)) return rc;
        if (int rc = map_of_codes(&tv, d->v, heads * d->seq_k, 2 * d->d_k)) return rc;
        return launch_cluster(kv_attention_kernel<Cfg>, items * splits, splits, Cfg::THREADS, Cfg::SMEM, d->stream, tk, tv, p);
    };
    if (d->d_k == 64) return launch(KvAttnCfg<__half, KV_PLAIN, 64, 1, 4, 32, 2, 3>());
    return launch(KvAttnCfg<__half, KV_PLAIN, 128, 1, 4, 16, 2, 3>());
}

}  // namespace api
}  // namespace txb

extern "C" {

int tx_kv_cache_write(const tx_kv_write_desc *d)
{
    if (!d) return fail(TX_ERR_INVALID, "K/V cache write: null descriptor");
    return move_rows<true>("K/V cache write", d->cache, d->k, d->v, d->page_table, d->start, d->counts, d->rows, d->batch, d->tokens,
                           d->src_tokens, d->table_len, d->dtype, d->flags, d->stream);
}

int tx_kv_cache_read(const tx_kv_read_desc *d)
{
    if (!d) return fail(TX_ERR_INVALID, "K/V cache read: null descriptor");
    return move_rows<false>("K/V cache read", d->cache, d->k, d->v, d->page_table, d->start, d->counts, nullptr, d->batch, d->tokens, 0,
                            d->table_len, d->dtype, d->flags, d->stream);
}

int tx_kv_cache_attention(const tx_kv_attention_desc *d)
{
    const char *who = "K/V cache attention";
    if (!d) return fail(TX_ERR_INVALID, "%s: null descriptor", who);
    if (!d->q || !d->out || !d->kv_lens) return fail(TX_ERR_INVALID, "%s: null pointer", who);
    txb::KvAttnParams p;
    if (int rc = pages_of(who, d->cache, d->page_table, d->batch, d->table_len, d->dtype, &p.pages)) return rc;
    if (!aligned(d->q, 16) || !aligned(d->out, 16) || !aligned(d->tree, 8)) return fail(TX_ERR_INVALID, "%s: q and out must be 16-byte aligned, tree 8-byte", who);
    if (d->tokens < 1 || d->tokens > 64) return fail(TX_ERR_UNSUPPORTED, "%s: 1 to 64 tokens a call", who);
    if (d->q_heads <= 0 || d->q_heads % d->cache.kv_heads) return fail(TX_ERR_INVALID, "%s: q_heads must be a multiple of kv_heads", who);
    if (d->q_heads > 0xffffffLL) return fail(TX_ERR_UNSUPPORTED, "%s: dimension too large", who);
    if (d->window < 0 || d->sinks < 0) return fail(TX_ERR_INVALID, "%s: window and sinks must not be negative", who);
    if (d->window > 0 && d->window < d->tokens) return fail(TX_ERR_INVALID, "%s: a window must hold the call's tokens", who);
    if (d->flags & ~TX_SDPA_OUT_F16) return fail(TX_ERR_INVALID, "%s: unknown flags", who);
    if (int rc = txb::api::ensure_device()) return rc;
    if (int rc = txb::api::status_word(&p.status)) return rc;
    if (int rc = txb::api::page_word(&p.page_status)) return rc;
    p.q = d->q; p.out = d->out;
    p.kv_lens = d->kv_lens; p.q_lens = d->q_lens; p.tree = d->tree;
    p.tokens = (int)d->tokens; p.group = (int)(d->q_heads / d->cache.kv_heads);
    p.row_parts = 0;
    p.most_keys = (int)(d->table_len * d->cache.page_size);
    // a window longer than any sequence is none
    p.window = (int)std::min<int64_t>(d->window, 0x7fffffffLL); p.sinks = (int)std::min<int64_t>(d->sinks, 0x7fffffffLL);
    p.out_f16 = (d->flags & TX_SDPA_OUT_F16) ? 1 : 0;
    p.scale_log2 = (1.0f / std::sqrt((float)d->cache.d)) * 1.4426950408889634f;
    return for_types(d->dtype, d->cache.format, d->cache.d, [&](auto t, auto fmt, auto dim) -> int {
        return launch_attention<decltype(t), fmt(), dim()>(p, d);
    });
}

}  // extern "C"
