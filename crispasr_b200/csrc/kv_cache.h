// kv_cache.h — what a KV cache handle holds (see kv_slab.cu for the layout).
#pragma once

#include <cstddef>
#include <cstdint>

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
