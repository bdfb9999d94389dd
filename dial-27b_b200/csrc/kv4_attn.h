// Argument block of the attention kernels over the 4-bit KV cache.
#pragma once

#include "kv4.h"

namespace dialb200 {

struct Kv4AttnArgs {
  Kv4Cache c;
  const void* q;
  const int32_t* sids;
  const int32_t* lens;
  const int32_t* q_starts;
  void* out;
  void* scratch;
  long long q_ld, out_ld;
  int seqs, rows, max_q, max_len;
  float scale;
};

// Few queries a sequence: mma.sync, the cache streamed once for up to 16
// (query, head) columns (kv4_decode.cu).
constexpr int kKv4DecodeCols = 512;  // (query, head) columns of a kv head at most
size_t kv4_decode_scratch(int q_heads, int kv_heads, long long seqs, long long max_q,
                          long long max_len, bool weights);
cudaError_t kv4_decode_launch(const Kv4AttnArgs& a, int act, cudaStream_t s);

// Many queries a sequence: tcgen05, 256 (query, head) rows over each key block
// (kv4_prefill.cu).  With weights it leaves each row's log-sum-exp, base 2, in
// scratch at kv4_prefill_lse.
size_t kv4_prefill_scratch(int q_heads, long long rows, bool weights);
float* kv4_prefill_lse(const Kv4AttnArgs& a);
cudaError_t kv4_prefill_launch(const Kv4AttnArgs& a, int act, cudaStream_t s);

}  // namespace dialb200
