// Attention over the 4-bit KV cache: argument checks and the choice of kernel.
//
//   o = sum_j p_j v_j,  p_j = exp(s_j - m) / l,  s_j = scale * q . k_j
//
// over the slots j a query sees.
#include <cmath>

#include "kv4_dev.cuh"

namespace dialb200 {
namespace {

// Scratch of the attention of many queries; that of their weights follows.
size_t rows_part(int q_heads, long long rows) {
  return (kv4_prefill_scratch(q_heads, rows, true) + 127) & ~static_cast<size_t>(127);
}

// The caller's scratch starts on a 16-byte boundary, what is laid out in it on this
// one: the tensor-core kernel stores its parts 32 bytes at a time.
constexpr size_t kScratchAlign = 128;

cudaError_t launch(const Kv4AttnArgs& a, int act, cudaStream_t s) {
  if (a.max_q * (a.c.q_heads / a.c.kv_heads) <= kKv4FewCols) return kv4_decode_launch(a, act, s);
  const cudaError_t e = kv4_prefill_launch(a, act, s);
  if (e != cudaSuccess || !a.c.weights) return e;
  return kv4_colsum_launch(a, kv4_prefill_rows(a),
                           static_cast<uint8_t*>(a.scratch) + rows_part(a.c.q_heads, a.rows), s);
}

}  // namespace
}  // namespace dialb200

using namespace dialb200;

extern "C" int64_t dial_b200_kv4_attention_scratch_bytes(const dial_b200_kv4_shape* sh,
                                                         int64_t seqs, int64_t rows, int64_t max_q,
                                                         int64_t max_len, int32_t with_weights) {
  if (!sh || sh->q_heads < 1 || sh->kv_heads < 1 || sh->kv_heads > 1024 || sh->q_heads % sh->kv_heads != 0 ||
      sh->q_heads / sh->kv_heads > 16 || seqs < 0 || seqs > 65535 || rows < 0 || rows > (1 << 26) || max_q < 0 ||
      max_q > (1 << 24) || max_len < 0 || max_len > 16LL << 26 || rows * sh->q_heads > INT32_MAX)
    return -1;
  if (seqs == 0 || rows == 0 || max_q == 0) return 0;  // the call does nothing
  // enough for every call within the sizes, whichever kernels it takes
  const int rep = sh->q_heads / sh->kv_heads;
  const int64_t few = max_q < kKv4FewCols / rep ? max_q : kKv4FewCols / rep;
  size_t bytes = kv4_decode_scratch(sh->q_heads, sh->kv_heads, seqs, few, max_len, with_weights != 0);
  if (max_q * rep > kKv4FewCols) {
    const size_t many = with_weights ? rows_part(sh->q_heads, rows) +
                                           kv4_colsum_scratch(sh->q_heads, sh->kv_heads, seqs, max_q, max_len)
                                     : kv4_prefill_scratch(sh->q_heads, rows, false);
    bytes = bytes > many ? bytes : many;
  }
  return static_cast<int64_t>(bytes > 0 ? bytes + kScratchAlign - 16 : 0);
}

extern "C" int dial_b200_kv4_attention(const dial_b200_kv4_shape* sh, const void* q, int64_t q_ld,
                                       const void* pages, float* weights,
                                       const int32_t* block_table, int64_t sessions,
                                       const int32_t* sids, const int32_t* lens,
                                       const int32_t* q_starts, int64_t seqs, int64_t rows,
                                       int64_t max_q, int64_t max_len, void* out, int64_t out_ld,
                                       void* scratch, void* stream, char* err, size_t n) {
  Kv4AttnArgs a{};
  int rc = kv4_cache_of(sh, pages, weights, nullptr, block_table, sessions, &a.c, err, n);
  if (rc != DIAL_OK) return rc;
  if (seqs != 0 && rows != 0 && (!q || !sids || !lens || !out))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "null pointer argument");
  if (seqs < 0 || seqs > 65535)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "seqs %lld outside [0, 65535]", (long long)seqs);
  if (rows < 0 || rows > (1 << 26) || max_q < 0 || max_q > (1 << 24))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "rows %lld / max_q %lld out of range",
                    (long long)rows, (long long)max_q);
  if (rows * sh->q_heads > INT32_MAX)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "rows %lld times q_heads out of range", (long long)rows);
  if (!q_starts && rows != seqs)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "without q_starts rows %lld must equal seqs %lld",
                    (long long)rows, (long long)seqs);
  if (max_len < 0 || max_len > 16LL * sh->max_blocks)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "max_len %lld exceeds the block table's %lld slots",
                    (long long)max_len, 16LL * sh->max_blocks);
  if (!(sh->softmax_scale >= 0.f && sh->softmax_scale < 1e30f))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "softmax_scale %g out of range", sh->softmax_scale);
  const int64_t width = 1LL * sh->q_heads * kHeadDim;
  if (q_ld < width || out_ld < width || q_ld % 8 != 0 || out_ld % 8 != 0 ||
      (reinterpret_cast<uintptr_t>(q) & 15) != 0 || (reinterpret_cast<uintptr_t>(out) & 15) != 0)
    return kv4_fail(err, n, DIAL_ERR_INVALID,
                    "q and out rows must hold q_heads heads and start on 16-byte boundaries");
  if (!q_starts) max_q = 1;  // row i is sequence i's
  if (seqs == 0 || rows == 0 || max_q == 0) return DIAL_OK;
  if (dial_b200_kv4_attention_scratch_bytes(sh, seqs, rows, max_q, max_len, weights != nullptr) > 0 &&
      (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 15) != 0))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "scratch must be given, 16-byte aligned");
  a.q = q;
  a.sids = sids;
  a.lens = lens;
  a.q_starts = q_starts;
  a.out = out;
  a.scratch = reinterpret_cast<void*>((reinterpret_cast<uintptr_t>(scratch) + kScratchAlign - 1) &
                                      ~static_cast<uintptr_t>(kScratchAlign - 1));
  a.q_ld = q_ld;
  a.out_ld = out_ld;
  a.seqs = static_cast<int>(seqs);
  a.rows = static_cast<int>(rows);
  a.max_q = static_cast<int>(max_q);
  a.max_len = static_cast<int>(max_len);
  const float scale = sh->softmax_scale > 0.f ? sh->softmax_scale : 1.f / sqrtf(static_cast<float>(kHeadDim));
  a.zeros = 0;
  a.unit = static_cast<float>(frexp(1.4426950408889634 * scale * sh->k_scale, &a.unit_exp));
  if ((rc = kv4_ready(&a.c, err, n)) != DIAL_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = launch(a, sh->act, s);
  if (e != cudaSuccess)
    return kv4_fail(err, n, DIAL_ERR_CUDA, "kv4 attention launch failed: %s", cudaGetErrorString(e));
  return DIAL_OK;
}
