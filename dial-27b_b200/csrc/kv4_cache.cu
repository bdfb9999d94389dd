// 4-bit KV cache: append (q/k RMSNorm, RoPE, quantisation into the slots) and
// read back (slots as the values they stand for), with the argument checks and
// the status word that the cache's operators share.
#include <atomic>
#include <cstdarg>
#include <cstdio>

#include "kv4_dev.cuh"

namespace dialb200 {
namespace {

constexpr int kMaxDevices = 64;
__device__ int g_kv4_status;
std::atomic<int*> g_kv4_status_addr[kMaxDevices];

struct AppendArgs {
  Kv4Cache c;
  const void* qkv;
  const void* q_norm_w;
  const void* k_norm_w;
  const void* cos;
  const void* sin;
  const int32_t* sids;
  const int32_t* slots;
  const int32_t* pos;
  void* q_out;
  long long qkv_ld, q_out_ld;
  int rows, units, max_pos;
  float eps;
};

// RMSNorm and RoPE of the head held four dims a lane, each step rounded to the
// activation dtype (the decode op's steps).  The sum of squares is exact in 64
// bits, so that a value next to a code's border falls on one side of it
// whatever the order of the sum.
template <typename Act>
__device__ __forceinline__ void norm_rope64(float (&x)[4], const Act* w, float eps, const Act* cos,
                                            const Act* sin, int lane) {
  using AT = ActTraits<Act>;
  if (w) {
    double ss = 0.;
#pragma unroll
    for (int e = 0; e < 4; ++e) ss = fma(static_cast<double>(x[e]), static_cast<double>(x[e]), ss);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float m = AT::round(static_cast<float>(sqrt(ss / kHeadDim + static_cast<double>(eps))));
    float wv[4];
    load4(w + lane * 4, wv);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = AT::round(AT::round(__fdiv_rn(x[e], m)) * wv[e]);
  }
  if (cos) {
    float c[4], s[4];
    load4(cos + (lane & 15) * 4, c);
    load4(sin + (lane & 15) * 4, s);
    const bool first = lane < 16;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float other = __shfl_xor_sync(0xffffffffu, x[e], 16);
      const float x1 = first ? x[e] : other, x2 = first ? other : x[e];
      x[e] = first ? AT::round(AT::round(x1 * c[e]) - AT::round(x2 * s[e]))
                   : AT::round(AT::round(x1 * s[e]) + AT::round(x2 * c[e]));
    }
  }
}

// One warp per (row, head unit): unit u < kv_heads is a kv head (k and v),
// the others query heads.
template <typename Act>
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendArgs a) {
  const int lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (item >= static_cast<long long>(a.rows) * a.units) return;
  const int m = static_cast<int>(item / a.units), u = static_cast<int>(item % a.units);
  const int slot = a.slots[m];
  if (slot < 0) return;
  const int sid = a.sids[m], pos = a.pos ? a.pos[m] : 0;
  const int page = slot / kPageTokens, t = slot % kPageTokens;
  if (static_cast<unsigned>(sid) >= static_cast<unsigned>(a.c.sessions) ||
      page >= a.c.max_blocks ||
      (a.cos && static_cast<unsigned>(pos) >= static_cast<unsigned>(a.max_pos))) {
    if (lane == 0) set_status(a.c.status, kStatusBadArgs);
    return;
  }
  const Act* row = static_cast<const Act*>(a.qkv) + m * a.qkv_ld;
  const size_t rope = static_cast<size_t>(pos) * (kHeadDim / 2);
  const Act* cos = a.cos ? static_cast<const Act*>(a.cos) + rope : nullptr;
  const Act* sin = a.cos ? static_cast<const Act*>(a.sin) + rope : nullptr;
  float x[4];
  if (u >= a.c.kv_heads) {
    const int h = u - a.c.kv_heads;
    load4(row + h * kHeadDim + lane * 4, x);
    norm_rope64(x, static_cast<const Act*>(a.q_norm_w), a.eps, cos, sin, lane);
    store4(static_cast<Act*>(a.q_out) + m * a.q_out_ld + h * kHeadDim + lane * 4, x);
    return;
  }
  const int block = kv4_block(a.c, a.c.block_table, sid, page);
  if (block < 0) return;
  const size_t si = kv4_slab_index(a.c, block, u);
  uint8_t* slab = a.c.pages + si * kKv4Slab;
  uint32_t codes, scale;
  load4(row + (a.c.q_heads + u) * kHeadDim + lane * 4, x);
  norm_rope64(x, static_cast<const Act*>(a.k_norm_w), a.eps, cos, sin, lane);
  kv4_encode(x, a.c.k_scale, codes, scale);
  *reinterpret_cast<uint16_t*>(slab + t * 64 + lane * 2) = static_cast<uint16_t>(codes);
  if ((lane & 3) == 0) slab[kKv4KScales + t * 8 + (lane >> 2)] = static_cast<uint8_t>(scale);
  load4(row + (a.c.q_heads + a.c.kv_heads + u) * kHeadDim + lane * 4, x);
  kv4_encode(x, a.c.v_scale, codes, scale);
  *reinterpret_cast<uint16_t*>(slab + kKv4VCodes + t * 64 + lane * 2) =
      static_cast<uint16_t>(codes);
  if ((lane & 3) == 0) slab[kKv4VScales + t * 8 + (lane >> 2)] = static_cast<uint8_t>(scale);
  if (lane == 0 && a.c.weights) a.c.weights[si * kPageTokens + t] = 0.f;
  if (lane == 1 && a.c.positions) a.c.positions[si * kPageTokens + t] = pos;
}

struct ReadArgs {
  Kv4Cache c;
  const int32_t* sids;
  const int32_t* first;
  const int32_t* lens;
  void* k_out;
  void* v_out;
  int seqs, count;
};

// One warp per (sequence, slot, kv head).
template <typename Act>
__global__ void __launch_bounds__(256) kv4_read_kernel(const ReadArgs a) {
  const int lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int H = a.c.kv_heads;
  if (item >= static_cast<long long>(a.seqs) * a.count * H) return;
  const int h = static_cast<int>(item % H);
  const long long r = item / H;
  const int i = static_cast<int>(r / a.count);
  const long long slot = (a.first ? a.first[i] : 0) + r % a.count;
  const int sid = a.sids[i];
  float k[4] = {0.f, 0.f, 0.f, 0.f}, v[4] = {0.f, 0.f, 0.f, 0.f};
  if (slot >= 0 && slot < a.lens[i]) {
    if (static_cast<unsigned>(sid) >= static_cast<unsigned>(a.c.sessions) ||
        slot >= static_cast<long long>(a.c.max_blocks) * kPageTokens) {
      if (lane == 0) set_status(a.c.status, kStatusBadArgs);
      return;
    }
    const int t = static_cast<int>(slot % kPageTokens);
    const int block = max(0, kv4_block(a.c, a.c.block_table, sid, static_cast<int>(slot / kPageTokens)));
    const uint8_t* slab = a.c.pages + kv4_slab_index(a.c, block, h) * kKv4Slab;
    kv4_decode(slab, 0, kKv4KScales, t, lane, a.c.k_scale, k);
    kv4_decode(slab, kKv4VCodes, kKv4VScales, t, lane, a.c.v_scale, v);
  }
  store4(static_cast<Act*>(a.k_out) + item * kHeadDim + lane * 4, k);
  store4(static_cast<Act*>(a.v_out) + item * kHeadDim + lane * 4, v);
}

cudaError_t kv4_status_word(int** word) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  int* p = g_kv4_status_addr[dev].load(std::memory_order_acquire);
  if (!p) {
    e = cudaGetSymbolAddress(reinterpret_cast<void**>(&p), g_kv4_status);
    if (e != cudaSuccess) return e;
    g_kv4_status_addr[dev].store(p, std::memory_order_release);
  }
  *word = p;
  return cudaSuccess;
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace

cudaError_t kv4_status(int dev, bool clear, int* out) {
  *out = 0;
  if (dev < 0 || dev >= kMaxDevices) return cudaErrorInvalidDevice;
  int* p = g_kv4_status_addr[dev].load(std::memory_order_acquire);
  if (!p) return cudaSuccess;
  cudaError_t e = cudaMemcpy(out, p, sizeof(int), cudaMemcpyDeviceToHost);
  if (e == cudaSuccess && clear && *out != 0) e = cudaMemset(p, 0, sizeof(int));
  return e;
}

int kv4_fail(char* err, size_t n, int code, const char* f, ...) {
  if (err && n) {
    va_list ap;
    va_start(ap, f);
    std::vsnprintf(err, n, f, ap);
    va_end(ap);
  }
  return code;
}

int kv4_ready(Kv4Cache* c, char* err, size_t n) {
  const cudaError_t e = kv4_status_word(&c->status);
  if (e != cudaSuccess)
    return kv4_fail(err, n, DIAL_ERR_CUDA, "kv4 status word: %s", cudaGetErrorString(e));
  return DIAL_OK;
}

int kv4_cache_of(const dial_b200_kv4_shape* sh, const void* pages, float* weights,
                 int32_t* positions, const int32_t* block_table, int64_t sessions, Kv4Cache* c,
                 char* err, size_t n) {
  if (!sh || !pages || !block_table)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "null pointer argument");
  if (sh->head_dim != kHeadDim)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "head_dim must be 128 (got %d)", sh->head_dim);
  if (sh->q_heads < 1 || sh->kv_heads < 1 || sh->q_heads % sh->kv_heads != 0 ||
      sh->q_heads / sh->kv_heads > 16 || sh->kv_heads > 1024)
    return kv4_fail(err, n, DIAL_ERR_INVALID,
                    "q_heads %d must be 1 to 16 times kv_heads %d (at most 1024)", sh->q_heads,
                    sh->kv_heads);
  // slabs and pages of a sequence are counted in 32 bits
  if (sh->max_blocks < 1 || sh->num_blocks < 1 || sh->max_blocks > (1 << 26) ||
      1LL * sh->max_blocks * sh->kv_heads > INT32_MAX ||
      1LL * sh->num_blocks * sh->kv_heads > INT32_MAX)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "max_blocks %d / num_blocks %d out of range",
                    sh->max_blocks, sh->num_blocks);
  if (!(sh->k_scale > 0.f && sh->k_scale < 1e30f && sh->v_scale > 0.f && sh->v_scale < 1e30f))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "k_scale %g / v_scale %g must be positive",
                    sh->k_scale, sh->v_scale);
  if (sh->act != DIAL_ACT_BF16 && sh->act != DIAL_ACT_F16)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "act must be BF16 or F16");
  if (sessions < 1 || sessions > INT32_MAX)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "sessions %lld out of range", (long long)sessions);
  if (!aligned(pages, 16))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "pages must be 16-byte aligned");
  *c = Kv4Cache{};
  c->pages = static_cast<uint8_t*>(const_cast<void*>(pages));
  c->weights = weights;
  c->positions = positions;
  c->block_table = block_table;
  c->sessions = static_cast<int>(sessions);
  c->max_blocks = sh->max_blocks;
  c->num_blocks = sh->num_blocks;
  c->q_heads = sh->q_heads;
  c->kv_heads = sh->kv_heads;
  c->k_scale = sh->k_scale;
  c->v_scale = sh->v_scale;
  return DIAL_OK;
}

}  // namespace dialb200

using namespace dialb200;

extern "C" int dial_b200_kv4_append(const dial_b200_kv4_shape* sh, const void* qkv, int64_t qkv_ld,
                                    const void* q_norm_w, const void* k_norm_w, const void* cos,
                                    const void* sin, void* pages, float* weights,
                                    int32_t* positions_pool, const int32_t* block_table,
                                    int64_t sessions, const int32_t* sids, const int32_t* slots,
                                    const int32_t* positions, void* q_out, int64_t q_out_ld,
                                    int64_t rows, void* stream, char* err, size_t n) {
  AppendArgs a{};
  int rc = kv4_cache_of(sh, pages, weights, positions_pool, block_table, sessions, &a.c, err, n);
  if (rc != DIAL_OK) return rc;
  if (!qkv || !sids || !slots)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "null pointer argument");
  if (!q_norm_w != !k_norm_w || !cos != !sin)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "q_norm_w and k_norm_w, cos and sin go in pairs");
  if ((cos || positions_pool) && !positions)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "RoPE and a positions pool need positions");
  if (cos && sh->max_pos < 1)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "max_pos %d must be positive with RoPE", sh->max_pos);
  if (q_norm_w && !(sh->eps >= 0.f && sh->eps < 1e30f))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "eps %g out of range", sh->eps);
  if (rows < 0 || rows > (1 << 26))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "rows %lld outside [0, 2^26]", (long long)rows);
  const int64_t width = (sh->q_heads + 2LL * sh->kv_heads) * kHeadDim;
  if (qkv_ld < width || qkv_ld % 4 != 0 || !aligned(qkv, 8) || (q_out && !aligned(q_out, 8)) ||
      (q_out && (q_out_ld < 1LL * sh->q_heads * kHeadDim || q_out_ld % 4 != 0)))
    return kv4_fail(err, n, DIAL_ERR_INVALID,
                    "qkv and q_out rows must hold their heads and start on 8-byte boundaries");
  if (!aligned(q_norm_w, 8) || !aligned(k_norm_w, 8) || !aligned(cos, 8) || !aligned(sin, 8))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "norm weights and RoPE tables must be 8-byte aligned");
  if (rows == 0) return DIAL_OK;
  a.qkv = qkv;
  a.q_norm_w = q_norm_w;
  a.k_norm_w = k_norm_w;
  a.cos = cos;
  a.sin = sin;
  a.sids = sids;
  a.slots = slots;
  a.pos = positions;
  a.q_out = q_out;
  a.qkv_ld = qkv_ld;
  a.q_out_ld = q_out_ld;
  a.rows = static_cast<int>(rows);
  a.units = sh->kv_heads + (q_out ? sh->q_heads : 0);
  a.max_pos = sh->max_pos;
  a.eps = sh->eps;
  const long long grid = (rows * a.units + 7) / 8;
  if (grid > INT32_MAX)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "rows %lld times heads out of range", (long long)rows);
  if ((rc = kv4_ready(&a.c, err, n)) != DIAL_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (sh->act == DIAL_ACT_BF16)
    kv4_append_kernel<__nv_bfloat16><<<static_cast<unsigned>(grid), 256, 0, s>>>(a);
  else
    kv4_append_kernel<__half><<<static_cast<unsigned>(grid), 256, 0, s>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return kv4_fail(err, n, DIAL_ERR_CUDA, "kv4 append launch failed: %s", cudaGetErrorString(e));
  return DIAL_OK;
}

extern "C" int dial_b200_kv4_read(const dial_b200_kv4_shape* sh, const void* pages,
                                  const int32_t* block_table, int64_t sessions,
                                  const int32_t* sids, const int32_t* first, const int32_t* lens,
                                  int64_t seqs, int64_t count, void* k_out, void* v_out,
                                  void* stream, char* err, size_t n) {
  ReadArgs a{};
  int rc = kv4_cache_of(sh, pages, nullptr, nullptr, block_table, sessions, &a.c, err, n);
  if (rc != DIAL_OK) return rc;
  if (!sids || !lens || !k_out || !v_out)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "null pointer argument");
  if (!aligned(k_out, 8) || !aligned(v_out, 8))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "k_out and v_out must be 8-byte aligned");
  if (seqs < 0 || seqs > (1 << 20) || count < 0 || count > INT32_MAX / 2)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "seqs %lld / count %lld out of range",
                    (long long)seqs, (long long)count);
  if (seqs == 0 || count == 0) return DIAL_OK;
  a.sids = sids;
  a.first = first;
  a.lens = lens;
  a.k_out = k_out;
  a.v_out = v_out;
  a.seqs = static_cast<int>(seqs);
  a.count = static_cast<int>(count);
  if (seqs * count > (1LL << 31) * 8 / sh->kv_heads - 8)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "seqs %lld times count %lld out of range",
                    (long long)seqs, (long long)count);
  const long long grid = (seqs * count * sh->kv_heads + 7) / 8;
  if ((rc = kv4_ready(&a.c, err, n)) != DIAL_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (sh->act == DIAL_ACT_BF16)
    kv4_read_kernel<__nv_bfloat16><<<static_cast<unsigned>(grid), 256, 0, s>>>(a);
  else
    kv4_read_kernel<__half><<<static_cast<unsigned>(grid), 256, 0, s>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    return kv4_fail(err, n, DIAL_ERR_CUDA, "kv4 read launch failed: %s", cudaGetErrorString(e));
  return DIAL_OK;
}
