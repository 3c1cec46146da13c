// What the entry points of every translation unit of the library share; defined in sdpa_api.cu.
#pragma once
#include <cuda.h>

#include <cstdint>

#include "../../include/tensorax_b200.h"
#include "kv_lens.cuh"

namespace txb {

enum : int { KV_ERR_PAGE = 51 };      // the only code of api::page_word

namespace api {

int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));   // sets tx_last_error(), returns code
int ensure_device();
int status_word(int **out);          // the current device's failure word: while it is set, kernels that look at it stop
int page_word(int **out);            // ... and the word for pages and rows that do not exist, which stops nothing
int sm_count(int *n);
int current_device(int *dev);
// `rows` rows of d one-byte codes as 128-byte lines, copied sixteen rows at a time with a 128-byte swizzle
int map_of_codes(CUtensorMap *m, const void *base, int64_t rows, int64_t d);
void launched();                     // counts one kernel launch
// kv_cache_api.cu: a decoding step of fp16 rows with a window over plain K and V, by the kernel of the cache's attention
bool window_step_fits(const tx_sdpa_desc *d);
int window_step(const tx_sdpa_desc *d, const KvLens &lens, int window, int sinks, int align_end, int *status);

}  // namespace api
}  // namespace txb
