// Attention over the 4-bit KV cache: argument checks, the choice of kernel, and
// the running weights of many queries.
//
//   o = sum_j p_j v_j,  p_j = exp(s_j - m) / l,  s_j = scale * q . k_j
//
// over the slots j a query sees.
#include <cmath>

#include "kv4_dev.cuh"

namespace dialb200 {
namespace {

constexpr int kFewCols = 64;

template <typename Act>
__global__ void __launch_bounds__(256) kv4_weights_kernel(const Kv4AttnArgs a, const float* lse) {
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int kvh = blockIdx.y, rep = a.c.q_heads / a.c.kv_heads;
  Kv4Seq s;
  if (!kv4_seq(a, blockIdx.z, s) || t >= s.len) return;
  const int block = kv4_block(a.c, a.c.block_table, s.sid, t / kPageTokens);
  const size_t si = kv4_slab_index(a.c, max(block, 0), kvh);
  float k[4], sum = 0.f;
  kv4_decode(a.c.pages + si * kKv4Slab, 0, kKv4KScales, t % kPageTokens, lane, a.c.k_scale, k);
  for (int j = max(0, t - (s.len - s.n)); j < s.n; ++j)
    for (int r = 0; r < rep; ++r) {
      const int h = kvh * rep + r;
      const size_t row = s.row0 + j;
      float q[4];
      load4(static_cast<const Act*>(a.q) + row * a.q_ld + h * kHeadDim + lane * 4, q);
      const float sc =
          warp_sum(fmaf(q[0], k[0], q[1] * k[1]) + fmaf(q[2], k[2], q[3] * k[3])) * a.scale;
      sum += exp2f(sc * 1.4426950408889634f - lse[row * a.c.q_heads + h]);
    }
  if (lane == 0 && block >= 0) a.c.weights[si * kPageTokens + t % kPageTokens] += sum;
}

cudaError_t launch(const Kv4AttnArgs& a, int act, cudaStream_t s) {
  if (a.max_q * (a.c.q_heads / a.c.kv_heads) <= kFewCols) return kv4_decode_launch(a, act, s);
  cudaError_t e = kv4_prefill_launch(a, act, s);
  if (e != cudaSuccess || !a.c.weights) return e;
  const dim3 grid((a.max_len + 7) / 8, a.c.kv_heads, a.seqs);
  if (act == DIAL_ACT_BF16) kv4_weights_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(a, kv4_prefill_lse(a));
  else kv4_weights_kernel<__half><<<grid, 256, 0, s>>>(a, kv4_prefill_lse(a));
  return cudaGetLastError();
}

}  // namespace
}  // namespace dialb200

using namespace dialb200;

extern "C" int64_t dial_b200_kv4_attention_scratch_bytes(const dial_b200_kv4_shape* sh,
                                                         int64_t seqs, int64_t rows, int64_t max_q,
                                                         int64_t max_len, int32_t with_weights) {
  if (!sh || sh->q_heads < 1 || sh->kv_heads < 1 || sh->q_heads % sh->kv_heads != 0 || seqs < 0 || rows < 0 || max_q < 0 ||
      max_len < 0)
    return -1;
  if (max_q * (sh->q_heads / sh->kv_heads) <= kFewCols)
    return static_cast<int64_t>(kv4_decode_scratch(sh->q_heads, sh->kv_heads, seqs, max_q, max_len,
                                                   with_weights != 0));
  return static_cast<int64_t>(kv4_prefill_scratch(sh->q_heads, rows, with_weights != 0));
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
  if (!q || !sids || !lens || !out)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "null pointer argument");
  if (seqs < 0 || seqs > 65535)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "seqs %lld outside [0, 65535]", (long long)seqs);
  if (rows < 0 || rows > (1 << 26) || max_q < 0 || max_q > (1 << 24))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "rows %lld / max_q %lld out of range",
                    (long long)rows, (long long)max_q);
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
  if (seqs == 0 || rows == 0 || max_q == 0) return DIAL_OK;
  if (dial_b200_kv4_attention_scratch_bytes(sh, seqs, rows, max_q, max_len, weights != nullptr) > 0 &&
      (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 15) != 0))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "scratch must be given, 16-byte aligned");
  a.q = q;
  a.sids = sids;
  a.lens = lens;
  a.q_starts = q_starts;
  a.out = out;
  a.scratch = scratch;
  a.q_ld = q_ld;
  a.out_ld = out_ld;
  a.seqs = static_cast<int>(seqs);
  a.rows = static_cast<int>(rows);
  a.max_q = static_cast<int>(q_starts ? max_q : 1);
  a.max_len = static_cast<int>(max_len);
  a.scale = sh->softmax_scale > 0.f ? sh->softmax_scale : 1.f / sqrtf(static_cast<float>(kHeadDim));
  if ((rc = kv4_ready(&a.c, err, n)) != DIAL_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = launch(a, sh->act, s);
  if (e != cudaSuccess)
    return kv4_fail(err, n, DIAL_ERR_CUDA, "kv4 attention launch failed: %s", cudaGetErrorString(e));
  return DIAL_OK;
}
