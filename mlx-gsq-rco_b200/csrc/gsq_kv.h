// The quantised key/value cache, as the kernels that write and read it share it.
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace gsq {

enum KvFormat : int { KV_INT8 = 0, KV_FP8 = 1 };  // gsq_kv_format

// Host-side checks every entry point with a cache makes; GSQ_OK or the recorded error.
int kv_check(const char* who, int fmt, const void* kc, const void* vc, const void* ks, const void* vs, int64_t batch,
             int64_t heads, int64_t dim, int64_t cap);

}  // namespace gsq
