// Launch parameters of the row kernels of a 4-bit K/V cache (kv4_cache.hip):
// rows quantised into their page slots, read back, or copied slot to slot.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stdint.h>

#include "fast_div.h"

namespace xhip {

enum Kv4RowOp : int { KV4_WRITE = 0, KV4_READ = 1, KV4_COPY = 2 };

struct Kv4RowParams {
    char *key_cache;           // 4-bit pages (kv4_layout.h)
    char *value_cache;
    void *key;                 // [num_tokens][num_kv_heads][head_size], element type
    void *value;               // (KV4_WRITE reads them, KV4_READ writes them)
    const int *slots;          // [num_tokens] flat slots, or null: use block_tables + positions
    const int *src_slots;      // [num_tokens] KV4_COPY: the slots the rows come from
    const int *block_tables;   // [num_tokens][max_blocks]
    const int *positions;      // [num_tokens]
    long long kv_block_stride; // bytes
    long long kv_head_stride;  // bytes
    int num_tokens;
    int num_kv_heads;
    int head_size;
    int block_size;            // power of two, >= 16
    int bs_shift;
    int max_blocks;
    int max_ctx;               // max_blocks * block_size
    // set by launch_kv4_rows for each of its launches:
    int tok0;                  // first token of the launch
    uint32_t items;            // 8-channel pieces of K (and of V) rows of 4 tokens each
    DivMagic row_div;          // division by the pieces of a row
    DivMagic head_div;         // division by num_kv_heads
};

// dtype: KV_F16 / KV_BF16 / KV_F32, the rows' element type (KV4_COPY: unused).
hipError_t launch_kv4_rows(const Kv4RowParams &p, int op, int dtype, hipStream_t stream);

}  // namespace xhip
