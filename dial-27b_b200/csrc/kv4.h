// Host interface of the 4-bit KV cache operators (kv4_cache.cu, kv4_attn.cu,
// kv4_evict.cu): argument blocks shared by their kernels.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "../../include/dial_b200.h"

namespace dialb200 {

// A slab: one 16-token page of one kv head.
constexpr int kKv4Slab = DIAL_B200_KV4_SLAB_BYTES;
constexpr int kKv4VCodes = 1024;   // byte offsets inside a slab; k codes at 0
constexpr int kKv4KScales = 2048;
constexpr int kKv4VScales = 2176;

// The cache of a call: pool, tables and the sessions the rows name.
struct Kv4Cache {
  uint8_t* pages;              // [num_blocks][kv_heads][kKv4Slab]
  float* weights;              // [num_blocks][kv_heads][16] or null
  int32_t* positions;          // [num_blocks][kv_heads][16] or null
  const int32_t* block_table;  // [sessions][max_blocks]
  int sessions, max_blocks, num_blocks;
  int q_heads, kv_heads;
  float k_scale, v_scale;
  int* status;
};

// Looks up the operators' device status word on the current device for `c`
// (no allocation), once a call's arguments are found good.
int kv4_ready(Kv4Cache* c, char* err, size_t n);
// Its value on device `dev` (0 where no operator ran), cleared if asked.
cudaError_t kv4_status(int dev, bool clear, int* out);

// Writes a message and returns `code`.
int kv4_fail(char* err, size_t n, int code, const char* f, ...);
// Checks a shape and the pool arguments, and fills `c` but for the status
// word; DIAL_OK or an error.
int kv4_cache_of(const dial_b200_kv4_shape* sh, const void* pages, float* weights,
                 int32_t* positions, const int32_t* block_table, int64_t sessions, Kv4Cache* c,
                 char* err, size_t n);

}  // namespace dialb200
