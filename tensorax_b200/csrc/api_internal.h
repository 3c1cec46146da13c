// What the entry points of every translation unit of the library share; defined in sdpa_api.cu.
#pragma once

namespace txb {

enum : int { KV_ERR_PAGE = 51 };      // failure word: see kv_cache.cuh

namespace api {

int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));   // sets tx_last_error(), returns code
int ensure_device();
int status_word(int **out);          // the current device's failure word
int sm_count(int *n);
int current_device(int *dev);
void launched();                     // counts one kernel launch

}  // namespace api
}  // namespace txb
