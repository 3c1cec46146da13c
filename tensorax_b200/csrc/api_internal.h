// What the entry points of every translation unit of the library share; defined in sdpa_api.cu.
#pragma once
#include <cuda.h>

#include <cstdint>

namespace txb {

enum : int { KV_ERR_PAGE = 51 };      // failure word: see kv_cache.cuh

namespace api {

int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));   // sets tx_last_error(), returns code
int ensure_device();
int status_word(int **out);          // the current device's failure word
int sm_count(int *n);
int current_device(int *dev);
// `rows` rows of d one-byte codes as 128-byte lines, copied sixteen rows at a time with a 128-byte swizzle
int map_of_codes(CUtensorMap *m, const void *base, int64_t rows, int64_t d);
void launched();                     // counts one kernel launch

}  // namespace api
}  // namespace txb
