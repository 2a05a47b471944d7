// kv_cache.h — what a KV cache handle holds (see kv_slab.cu for the layout).
#pragma once

#include <cstddef>
#include <cstdint>

#include <cuda_runtime.h>

#include "../../include/b200_fattn.h"

struct b200_kv_cache {
    b200_kv_config cfg;
    uint8_t* arena;   // cudaMalloc'ed
    uint8_t* base;    // arena rounded up to 1024
    size_t slab_bytes;
    size_t row_bytes;
    int64_t ctx_rows;
    int device;
};

namespace b200 {
// Whether the cache lives on the current device: a kernel of another one must not be given its rows.
inline bool on_current_device(const b200_kv_cache* kv) {
    int device = -1;
    return cudaGetDevice(&device) == cudaSuccess && device == kv->device;
}
}  // namespace b200
