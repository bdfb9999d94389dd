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
  // unit 2^unit_exp = softmax_scale k_scale log2(e), unit in [1/2, 1]: from q . k of the
  // codes and e4m3 scales to base-2 scores
  float unit;
  int unit_exp;
  uint64_t zeros;  // two f32 zeros, not known when the kernels are compiled (score2)
};

// Few queries a sequence: mma.sync, the cache streamed once for up to 16
// (query, head) columns (kv4_decode.cu).
//
// (query, head of the group) columns of a sequence up to which it takes a call: its
// MMAs are 8 columns wide and a page costs it about the same instructions for each 16,
// while the tcgen05 kernels have 128 rows a tile whatever a sequence brings.
// Measured, decode / tcgen05, 32 heads of 8, 8 sessions of 4096 slots: 32 columns 38 / 52
// us, 64 61 / 53, 96 85 / 54; one of 65536: 61 / 84, 100 / 85, 144 / 86; with weights, 8
// of 4096: 61 / 99, 113 / 101, 193 / 102.
constexpr int kKv4FewCols = 48;
size_t kv4_decode_scratch(int q_heads, int kv_heads, long long seqs, long long max_q,
                          long long max_len, bool weights);
cudaError_t kv4_decode_launch(const Kv4AttnArgs& a, int act, cudaStream_t s);

// Many queries a sequence: tcgen05, 256 (query, head) rows over each key block
// (kv4_prefill.cu).  With weights it leaves in scratch, for every row and head,
// the f16 queries, their scale to base-2 scores and minus the log-sum-exp.
struct Kv4Rows {
  uint16_t* q16;  // [kv_heads][rows][heads of a group][128]
  float* fac;     // [kv_heads][rows][heads of a group]
  float* off;     // the same, minus the log-sum-exp, base 2
};
constexpr int kKv4RowBytes = 128 * 2 + 4 + 4;
size_t kv4_prefill_scratch(int q_heads, long long rows, bool weights);
Kv4Rows kv4_prefill_rows(const Kv4AttnArgs& a);
cudaError_t kv4_prefill_launch(const Kv4AttnArgs& a, int act, cudaStream_t s);

// The running weights of those queries (kv4_colsum.cu); `scratch` of its own.
size_t kv4_colsum_scratch(int q_heads, int kv_heads, long long seqs, long long max_q,
                          long long max_len);
cudaError_t kv4_colsum_launch(const Kv4AttnArgs& a, const Kv4Rows& rows, void* scratch,
                              cudaStream_t s);

}  // namespace dialb200
