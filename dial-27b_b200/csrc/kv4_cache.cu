// 4-bit KV cache: append (q/k RMSNorm, RoPE, quantisation into the slots) and
// read back (slots as the values they stand for), with the argument checks and
// the status word that the cache's operators share.
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <type_traits>

#include "kv4_dev.cuh"
#include "kv4_launch.h"

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

// Packed pairs of the activation dtype, each operation rounded once (never
// contracted).
template <typename Act>
struct Pair;
template <>
struct Pair<__nv_bfloat16> {
  using T = __nv_bfloat162;
  static __device__ __forceinline__ T of(float lo, float hi) { return __floats2bfloat162_rn(lo, hi); }
  static __device__ __forceinline__ T mul(T a, T b) { return __hmul2_rn(a, b); }
  static __device__ __forceinline__ T add(T a, T b) { return __hadd2_rn(a, b); }
};
template <>
struct Pair<__half> {
  using T = __half2;
  static __device__ __forceinline__ T of(float lo, float hi) { return __floats2half2_rn(lo, hi); }
  static __device__ __forceinline__ T mul(T a, T b) { return __hmul2_rn(a, b); }
  static __device__ __forceinline__ T add(T a, T b) { return __hadd2_rn(a, b); }
};

// A head held by 16 lanes, eight dims each (dims 8 * l ..), as four pairs.
template <typename Act>
struct Head {
  typename Pair<Act>::T v[4];
  __device__ __forceinline__ void load(const Act* p, int l) {
    *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(p + l * 8);
  }
  __device__ __forceinline__ void store(Act* p, int l) const {
    *reinterpret_cast<uint4*>(p + l * 8) = *reinterpret_cast<const uint4*>(v);
  }
  __device__ __forceinline__ void floats(float (&x)[8]) const {
    const Act* h = reinterpret_cast<const Act*>(v);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = ActTraits<Act>::to_f(h[e]);
  }
};

// act(sqrt(sum x^2 / 128 + eps)) of each half warp's head, as from an exact sum: the f32
// form (off by less than 2^-20: 9 roundings of the sum, halved by the root, and 3
// more) unless a border of the dtype lies within 2^-19 of it, else 64 bits.
template <typename Act>
__device__ __forceinline__ float rms_of(const float (&x)[8], float eps) {
  using AT = ActTraits<Act>;
  float ss = fmaf(x[0], x[0], x[1] * x[1]) + fmaf(x[2], x[2], x[3] * x[3]);
  ss += fmaf(x[4], x[4], x[5] * x[5]) + fmaf(x[6], x[6], x[7] * x[7]);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float m = __fsqrt_rn(ss * (1.f / kHeadDim) + eps);
  const float lo = AT::round(m * (1.f - 0x1p-19f)), hi = AT::round(m * (1.f + 0x1p-19f));
  // sums near the ends of f32's range lose more than that
  const bool near = !(lo == hi && ss > 1e-30f && ss < 1e37f);
  if (!__any_sync(0xffffffffu, near)) return lo;
  double sum = 0.;
#pragma unroll
  for (int e = 0; e < 8; ++e) sum = fma(static_cast<double>(x[e]), static_cast<double>(x[e]), sum);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return AT::round(static_cast<float>(sqrt(sum / kHeadDim + static_cast<double>(eps))));
}

// act(x / m).  A quotient of two bf16 values is never within 2^-17 of the middle of
// two bf16 values, so a product with 1 / m rounds as the quotient does; f16's
// quotients come as near as 2^-23 and are divided.
template <typename Act>
__device__ __forceinline__ void divide(const float (&x)[8], float m, typename Pair<Act>::T (&v)[4]) {
  float q[8];
  if (std::is_same<Act, __nv_bfloat16>::value && m > 1e-37f && m < 1e37f) {
    const float inv = __frcp_rn(m);
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = x[e] * inv;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] = __fdiv_rn(x[e], m);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = Pair<Act>::of(q[2 * e], q[2 * e + 1]);
}

// RMSNorm and RoPE, each step rounded to the activation dtype (the decode op's
// steps); sin has the sign of the lane's half of the dims.
template <typename Act>
__device__ __forceinline__ void norm_rope(Head<Act>& x, const Head<Act>& w, const Head<Act>& c, const Head<Act>& s,
                                          float eps, bool norm, bool rope) {
  using P = Pair<Act>;
  if (norm) {
    float f[8];
    x.floats(f);
    divide<Act>(f, rms_of<Act>(f, eps), x.v);
#pragma unroll
    for (int e = 0; e < 4; ++e) x.v[e] = P::mul(x.v[e], w.v[e]);
  }
  if (rope) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t own = *reinterpret_cast<const uint32_t*>(&x.v[e]);
      const uint32_t far = __shfl_xor_sync(0xffffffffu, own, 8);
      x.v[e] = P::add(P::mul(x.v[e], c.v[e]), P::mul(*reinterpret_cast<const typename P::T*>(&far), s.v[e]));
    }
  }
}

// The lane's eight values quantised: four code bytes, and the scale code of its
// 16-dim group (two lanes).
__device__ __forceinline__ void encode8(const float (&x)[8], float mult, uint32_t& codes, uint32_t& scale) {
  float v[8], amax = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = isnan(x[e]) ? 0.f : x[e];
    amax = fmaxf(amax, fabsf(v[e]));
  }
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  scale = e4m3_of(__fdiv_rn(quotient(amax, 6.f, 1.f / 6.f), mult));
  const float s = e4m3_value(scale) * mult;
  codes = 0;
  if (s > 0.f) {
    const float y = __frcp_rn(s);
#pragma unroll
    for (int e = 0; e < 8; e += 2)
      codes |= e2m1x2_of(quotient(v[e], s, y), quotient(v[e + 1], s, y)) << (4 * e);
  }
}

// A CTA for a row and a share (blockIdx.y) of its head units, a half warp a unit: unit
// u < kv_heads is a kv head (k and v), the others query heads.  A warp's norm weights,
// cos and sin serve all its units, U of which are loaded at once.
// 2048 rows: 14.6 M instructions, about half of them the quantisation, at 2.45 of 4 a
// clock: a row's loads are waited for (DRAM 12 %, ALU 42 %).  A token: latency (7 us cold).
template <typename Act, int U>
__global__ void __launch_bounds__(256) kv4_append_kernel(const AppendArgs a) {
  const int lane = threadIdx.x & 31, l = lane & 15, m = blockIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  const Act* row = static_cast<const Act*>(a.qkv) + m * a.qkv_ld;
  const int step = gridDim.y * 16, H = a.c.kv_heads, Q = a.c.q_heads;
  const int u0 = (blockIdx.y * 8 + (threadIdx.x >> 5)) * 2 + (lane >> 4);
  const bool norm = a.q_norm_w != nullptr, rope = a.cos != nullptr;
  // the first units' loads beside the look-ups
  Head<Act> x[U], y{};
  auto fetch = [&](int base) {
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int u = base + e * step;
      x[e] = Head<Act>{};
      if (u < a.units) x[e].load(row + (u < H ? Q + u : u - H) * kHeadDim, l);
    }
    if (base < H && base < a.units) y.load(row + (Q + H + base) * kHeadDim, l);
  };
  fetch(u0);
  const int slot = a.slots[m], sid = a.sids[m], pos = a.pos ? a.pos[m] : 0;
  if (slot < 0) return;
  const int page = slot / kPageTokens, t = slot % kPageTokens;
  if (static_cast<unsigned>(sid) >= static_cast<unsigned>(a.c.sessions) || page >= a.c.max_blocks ||
      (rope && static_cast<unsigned>(pos) >= static_cast<unsigned>(a.max_pos))) {
    if (threadIdx.x == 0) set_status(a.c.status, kStatusBadArgs);
    return;
  }
  const int block = kv4_block(a.c, a.c.block_table, sid, page);
  Head<Act> qw{}, kw{}, c{}, s{};
  if (norm) {
    qw.load(static_cast<const Act*>(a.q_norm_w), l);
    kw.load(static_cast<const Act*>(a.k_norm_w), l);
  }
  if (rope) {
    const size_t at = static_cast<size_t>(pos) * (kHeadDim / 2);
    c.load(static_cast<const Act*>(a.cos) + at, l & 7);
    s.load(static_cast<const Act*>(a.sin) + at, l & 7);
    if (l < 8) {  // dims below 64: x c - far s; above: x c + far s
#pragma unroll
      for (int e = 0; e < 4; ++e) s.v[e] = __hneg2(s.v[e]);
    }
  }
  for (int base = u0; base - (lane >> 4) < a.units; base += U * step) {  // warp-uniform
    if (base != u0) fetch(base);
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int u = base + e * step;
      const bool kv = u < H && u < a.units;
      const bool some_kv = __any_sync(0xffffffffu, kv);
      if (e > 0 && kv) y.load(row + (Q + H + u) * kHeadDim, l);
      norm_rope(x[e], u < H ? kw : qw, c, s, a.eps, norm, rope);
      if (!kv && u < a.units) x[e].store(static_cast<Act*>(a.q_out) + m * a.q_out_ld + (u - H) * kHeadDim, l);
      if (!some_kv) continue;
      uint32_t kc, ks, vc, vs;
      float f[8];
      x[e].floats(f);
      encode8(f, a.c.k_scale, kc, ks);
      y.floats(f);
      encode8(f, a.c.v_scale, vc, vs);
      if (!kv || block < 0) continue;
      const size_t si = kv4_slab_index(a.c, block, u);
      uint8_t* slab = a.c.pages + si * kKv4Slab;
      *reinterpret_cast<uint32_t*>(slab + t * 64 + l * 4) = kc;
      *reinterpret_cast<uint32_t*>(slab + kKv4VCodes + t * 64 + l * 4) = vc;
      if ((l & 1) == 0) {
        slab[kKv4KScales + t * 8 + (l >> 1)] = static_cast<uint8_t>(ks);
        slab[kKv4VScales + t * 8 + (l >> 1)] = static_cast<uint8_t>(vs);
      }
      if (l == 1 && a.c.weights) a.c.weights[si * kPageTokens + t] = 0.f;
      if (l == 3 && a.c.positions) a.c.positions[si * kPageTokens + t] = pos;
    }
  }
}

struct ReadArgs {
  Kv4Cache c;
  const int32_t* sids;
  const int32_t* first;
  const int32_t* lens;
  void* k_out;
  void* v_out;
  unsigned rows;  // seqs * count
  int count;
};

// Lanes 0-15 of a warp take k and 16-31 v, 8 dims each: 4 bytes of codes in, 16 bytes
// out, so that its stores are whole lines.  HEADS: a warp takes rows (slots) and goes
// over their kv heads, which shares a row's table look-ups; else one (slot, kv head).
template <typename Act, bool HEADS>
__global__ void __launch_bounds__(256) kv4_read_kernel(const ReadArgs a) {
  const int lane = threadIdx.x & 31, part = lane >> 4, l = lane & 15;
  const unsigned H = a.c.kv_heads;
  pdl_wait();
  pdl_launch_dependents();
  const float mult = part ? a.c.v_scale : a.c.k_scale;
  const int codes_at = (part ? kKv4VCodes : 0) + l * 4;
  const int scales_at = (part ? kKv4VScales : kKv4KScales) + (l >> 1);
  const unsigned unit = blockIdx.x * 8 + (threadIdx.x >> 5);
  constexpr unsigned R = HEADS ? 2 : 1, B = HEADS ? 4 : 1;  // rows, and heads at once
  const unsigned h0 = HEADS ? 0 : unit % H, h1 = HEADS ? H : h0 + 1;
  // the rows' look-ups beside each other, then the loads of B heads of them
  bool write[R], there[R];
  const uint8_t* slab[R];
  int t[R];
#pragma unroll
  for (unsigned e = 0; e < R; ++e) {
    const unsigned row = HEADS ? unit * R + e : unit / H;
    write[e] = row < a.rows;
    const unsigned i = write[e] ? row / static_cast<unsigned>(a.count) : 0;
    const int sid = a.sids[i];
    const long long slot = (a.first ? a.first[i] : 0) + static_cast<long long>(row - i * a.count);
    there[e] = write[e] && slot >= 0 && slot < a.lens[i];
    if (write[e] && (static_cast<unsigned>(sid) >= static_cast<unsigned>(a.c.sessions) ||
                     (there[e] && slot >= static_cast<long long>(a.c.max_blocks) * kPageTokens))) {
      if (lane == 0) set_status(a.c.status, kStatusBadArgs);
      write[e] = there[e] = false;
    }
    t[e] = there[e] ? static_cast<int>(slot % kPageTokens) : 0;
    const int block = there[e] ? max(0, kv4_block(a.c, a.c.block_table, sid, static_cast<int>(slot / kPageTokens))) : 0;
    slab[e] = a.c.pages + kv4_slab_index(a.c, block, 0) * kKv4Slab;
  }
  for (unsigned h = h0; h < h1; h += B) {
    uint32_t w[R][B], sc[R][B];
#pragma unroll
    for (unsigned e = 0; e < R; ++e)
#pragma unroll
      for (unsigned u = 0; u < B; ++u) {
        w[e][u] = sc[e][u] = 0;
        if (there[e] && h + u < h1) {
          const uint8_t* from = slab[e] + (h + u) * kKv4Slab;
          w[e][u] = *reinterpret_cast<const uint32_t*>(from + codes_at + t[e] * 64);
          sc[e][u] = from[scales_at + t[e] * 8];
        }
      }
#pragma unroll
    for (unsigned e = 0; e < R; ++e)
#pragma unroll
      for (unsigned u = 0; u < B; ++u) {
        if (!write[e] || h + u >= h1) continue;
        const float f = e4m3_value(sc[e][u]) * mult;
        uint32_t o[4];
        e2m1x8_to_f16x2x4(w[e][u], o);
        uint4 r;
        typename Pair<Act>::T* p = reinterpret_cast<typename Pair<Act>::T*>(&r);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&o[q]));
          p[q] = Pair<Act>::of(v.x * f, v.y * f);
        }
        const size_t row = HEADS ? unit * R + e : unit / H;
        *reinterpret_cast<uint4*>(static_cast<Act*>(part ? a.v_out : a.k_out) + (row * H + h + u) * kHeadDim + l * 8) = r;
      }
  }
}

template <typename Act>
cudaError_t launch_read(const ReadArgs& a, cudaStream_t s) {
  const long long units = static_cast<long long>(a.rows) * a.c.kv_heads;
  // Few: every (slot, kv head) a warp of its own, for latency; many: a warp two rows.
  // 8 kv heads, own / shared: 256 rows 2.5 / 4.1 us, 2048 5.3 / 4.3, 4096 9.1 / 5.6, 65536
  // 115 / 59 (302 MB: 5.1 TB/s).  Four heads of two rows are loaded before the first is
  // stored (stores hold back the loads behind them): 59 against 67; eight 60.
  if (a.rows <= 148 * 8)
    return kv4_start(kv4_read_kernel<Act, false>, dim3(static_cast<unsigned>((units + 7) / 8)), 256, 0, s, a);
  return kv4_start(kv4_read_kernel<Act, true>, dim3((a.rows + 15) / 16), 256, 0, s, a);
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
      (1LL * sh->max_blocks + 64) * sh->kv_heads > INT32_MAX ||
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
  if (rows != 0 && (!qkv || !sids || !slots))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "null pointer argument");
  if (!q_norm_w != !k_norm_w || !cos != !sin)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "q_norm_w and k_norm_w, cos and sin go in pairs");
  if ((cos || positions_pool) && !positions && rows != 0)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "RoPE and a positions pool need positions");
  if (cos && sh->max_pos < 1)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "max_pos %d must be positive with RoPE", sh->max_pos);
  if (q_norm_w && !(sh->eps >= 0.f && sh->eps < 1e30f))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "eps %g out of range", sh->eps);
  if (rows < 0 || rows > (1 << 26))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "rows %lld outside [0, 2^26]", (long long)rows);
  const int64_t width = (sh->q_heads + 2LL * sh->kv_heads) * kHeadDim;
  if (qkv_ld < width || qkv_ld % 8 != 0 || !aligned(qkv, 16) || (q_out && !aligned(q_out, 16)) ||
      (q_out && (q_out_ld < 1LL * sh->q_heads * kHeadDim || q_out_ld % 8 != 0)))
    return kv4_fail(err, n, DIAL_ERR_INVALID,
                    "qkv and q_out rows must hold their heads and start on 16-byte boundaries");
  if (!aligned(q_norm_w, 16) || !aligned(k_norm_w, 16) || !aligned(cos, 16) || !aligned(sin, 16))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "norm weights and RoPE tables must be 16-byte aligned");
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
  if ((rc = kv4_ready(&a.c, err, n)) != DIAL_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  const int most = (a.units + 15) / 16;
  // A unit a half warp up to twice the 592 CTAs that are resident (four an SM, at 64
  // registers a thread); from there on a row a CTA, three of a half warp's units in
  // flight.  32 heads of 8 (3 CTAs a row), unit / row: 16 rows 3.0 / 4.0 us, 256 4.9 / 4.8,
  // 394 (1182 CTAs) 6.0 / 6.4, 1024 13.3 / 10.3, 2048 24.7 / 18.5.
  if (rows * most <= 2 * 592) {
    const dim3 grid(static_cast<unsigned>(rows), most);
    e = sh->act == DIAL_ACT_BF16 ? kv4_start(kv4_append_kernel<__nv_bfloat16, 1>, grid, 256, 0, s, a)
                                 : kv4_start(kv4_append_kernel<__half, 1>, grid, 256, 0, s, a);
  } else {
    const dim3 grid(static_cast<unsigned>(rows), 1);
    e = sh->act == DIAL_ACT_BF16 ? kv4_start(kv4_append_kernel<__nv_bfloat16, 3>, grid, 256, 0, s, a)
                                 : kv4_start(kv4_append_kernel<__half, 3>, grid, 256, 0, s, a);
  }
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
  if (seqs != 0 && count != 0 && (!sids || !lens || !k_out || !v_out))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "null pointer argument");
  if (!aligned(k_out, 16) || !aligned(v_out, 16))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "k_out and v_out must be 16-byte aligned");
  if (seqs < 0 || seqs > (1 << 20) || count < 0 || count > INT32_MAX / 2)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "seqs %lld / count %lld out of range",
                    (long long)seqs, (long long)count);
  if (seqs == 0 || count == 0) return DIAL_OK;
  a.sids = sids;
  a.first = first;
  a.lens = lens;
  a.k_out = k_out;
  a.v_out = v_out;
  if (seqs * count > INT32_MAX / sh->kv_heads)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "seqs %lld times count %lld out of range",
                    (long long)seqs, (long long)count);
  a.rows = static_cast<unsigned>(seqs * count);
  a.count = static_cast<int>(count);
  if ((rc = kv4_ready(&a.c, err, n)) != DIAL_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = sh->act == DIAL_ACT_BF16 ? launch_read<__nv_bfloat16>(a, s) : launch_read<__half>(a, s);
  if (e != cudaSuccess)
    return kv4_fail(err, n, DIAL_ERR_CUDA, "kv4 read launch failed: %s", cudaGetErrorString(e));
  return DIAL_OK;
}
