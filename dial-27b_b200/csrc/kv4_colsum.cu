// Running weights of many queries over the 4-bit KV cache: for every slot, the sum
// of its probabilities over the queries that see it and the heads of its group.
//
//   weights[t] += sum_r 2^(fac_r q_r . k_t - lse_r)
//
// with the f16 queries, scales and log-sum-exps that the attention before it left
// (kv4_prefill.cu).  Half that attention's MMAs and all of its exponentials; bound
// by the exponentials (16 a clock and SM).  S^T = K Q^T has a key in every TMEM
// lane, so a thread adds up its own key's row and nothing is exchanged.
// Measured: 512 tokens each on 9500 and 16897 slots, 40 heads of 8, 258 us cold,
// the exponentials' unit 69 % busy, tensor pipe 34 %.  With one warp a key and
// tile (8, not 16) 325; with scores in runs of 32, not 16, 280.
//
// Items: two 128-key blocks of a (sequence, kv head), so that a query tile fetched
// from L2 serves 256 keys, and up to kChunk tiles of 128 rows that see them, dealt
// to the CTAs in turn.  Warps 0-15 add up: warp w the keys of block (w / 4) % 2 over
// half w / 8 of a tile's rows; kv4_colsum_add_kernel adds the sums to the weights in a
// fixed order.  Warps 16-19: K codes -> f16 once an item, loaded during the item
// before; warp 20: query tiles by TMA into four buffers, and their constants; warp
// 21: tcgen05.mma into four TMEM buffers.
#include <cuda.h>

#include "kv4_attn.h"
#include "kv4_launch.h"
#include "kv4_tc.cuh"

namespace dialb200 {
namespace {

constexpr int kThreads = 22 * 32;
constexpr int kSeqChunk = 512;  // sequences a launch
constexpr int kKeys = 256;      // of an item
constexpr int kChunk = 32;      // query tiles of an item at most
constexpr int kQBufs = 4, kSBufs = 4, kCBufs = 8;  // query tiles, scores, constants
constexpr int kOffK = 0;                     // [2], the item's two key blocks
constexpr int kOffQ = 2 * kTile;             // [kQBufs]
constexpr int kOffMisc = (2 + kQBufs) * kTile;
constexpr int kStatusKv4Colsum = 0x602;
constexpr float kLarge = 4096.f;

struct Misc {
  uint64_t kfull, kfree, qfull[kQBufs], qfree[kQBufs], sfull[kSBufs], sfree[kSBufs], cfull[kCBufs], cfree[kCBufs], fin;
  uint32_t tmem;
  int failed;
  alignas(16) float fac[kCBufs][128];
  alignas(16) float off[kCBufs][128];
  alignas(16) int seen[kCBufs][128];    // slots the row sees
  // slots that all of a tile's 128 rows see; 0 for fewer rows, and for a log-sum-exp above
  // kLarge, of whose rounding an fma would keep too much in the exponent (2^-13 at kLarge;
  // rounding every score first, in the path of whole tiles too, takes 290 us)
  int all_see[kCBufs];
  long long cum[kSeqChunk + 1];         // items of one kv head of the sequences before
};
constexpr int kSmemBytes = kOffMisc + sizeof(Misc) + 1024;

struct ColsumArgs {
  Kv4AttnArgs a;
  Kv4Rows r;
  float* part;  // [seqs][kv_heads][kb_max][chunks][2][256]
  int kb_max, chunks;
};

__device__ __forceinline__ void tma2d(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}

struct Item {
  Kv4Seq s;
  int i, h, kb, t0, t1;  // tiles t0 .. t1 - 1
  size_t part;
};

__device__ __forceinline__ int tiles_of(const Kv4Seq& s, int rep) { return (s.n * rep + 127) / 128; }
__device__ __forceinline__ int blocks_of(const Kv4Seq& s) { return s.n > 0 ? (s.len + kKeys - 1) / kKeys : 0; }
__device__ __forceinline__ int chunks_of(const Kv4Seq& s, int rep) { return (tiles_of(s, rep) + kChunk - 1) / kChunk; }

// Tiles of chunk c that see the keys from kb * kKeys on: t1 <= t0 for none.
__device__ __forceinline__ void tiles_seeing(const Kv4Seq& s, int rep, int kb, int c, int& t0, int& t1) {
  const int first = max(0, kb * kKeys - (s.len - s.n));  // the first query that does
  t0 = static_cast<int>(static_cast<unsigned>(first * rep) / 128u) + c * kChunk;
  t1 = min(t0 + kChunk, tiles_of(s, rep));
}

__device__ __forceinline__ size_t part_at(const ColsumArgs& d, int i, int h, int kb, int c) {
  return (((static_cast<size_t>(i) * d.a.c.kv_heads + h) * d.kb_max + kb) * d.chunks + c) * 2 * kKeys;
}

// Item f of all (cum: items of a kv head of the sequences before).
__device__ __forceinline__ Item item_at(const ColsumArgs& d, const long long* cum, long long f) {
  const Kv4AttnArgs& a = d.a;
  const int H = a.c.kv_heads, rep = a.c.q_heads / H;
  int lo = 0, hi = a.seqs;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cum[mid] * H <= f) lo = mid;
    else hi = mid;
  }
  Item w;
  w.i = lo;
  kv4_seq(a, lo, w.s);
  const long long per = cum[lo + 1] - cum[lo], r = f - cum[lo] * H;
  w.h = static_cast<int>(r / per);
  const int q = static_cast<int>(r - w.h * per), nc = chunks_of(w.s, rep);
  // later blocks are seen by fewer tiles: the long ones first
  w.kb = q / nc;
  const int c = q - w.kb * nc;
  tiles_seeing(w.s, rep, w.kb, c, w.t0, w.t1);
  w.part = part_at(d, w.i, w.h, w.kb, c);
  return w;
}

// The first item from f on (in steps of the grid) that has tiles.
__device__ __forceinline__ long long next_with_tiles(const ColsumArgs& d, const long long* cum, long long f,
                                                     long long total) {
  for (; f < total; f += gridDim.x) {
    const Item w = item_at(d, cum, f);
    if (w.t1 > w.t0) break;
  }
  return f;
}

__global__ void __launch_bounds__(kThreads, 1) kv4_colsum_kernel(const __grid_constant__ CUtensorMap q_map, const ColsumArgs d) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  Misc& sm = *reinterpret_cast<Misc*>(smem + kOffMisc);
  const Kv4AttnArgs& a = d.a;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int H = a.c.kv_heads, rep = a.c.q_heads / H;
  if (tid == 0) {
    mbar_init(&sm.kfull, 4);
    mbar_init(&sm.kfree, 1);
    for (int i = 0; i < kQBufs; ++i) {
      mbar_init(&sm.qfull[i], 1);
      mbar_init(&sm.qfree[i], 1);
    }
    for (int i = 0; i < kSBufs; ++i) {
      mbar_init(&sm.sfull[i], 1);
      mbar_init(&sm.sfree[i], 8);
    }
    for (int i = 0; i < kCBufs; ++i) {
      mbar_init(&sm.cfull[i], 1);
      mbar_init(&sm.cfree[i], 16);
    }
    mbar_init(&sm.fin, 1);
    sm.failed = 0;
    fence_mbar_init();
  }
  if (warp == 21) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sm.tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  pdl_wait();
  pdl_launch_dependents();
  for (int i = tid; i < a.seqs; i += kThreads) {
    Kv4Seq s;
    sm.cum[i + 1] = kv4_seq(a, i, s) ? static_cast<long long>(blocks_of(s)) * chunks_of(s, rep) : 0;
  }
  if (tid == 0) sm.cum[0] = 0;
  __syncthreads();
  if (warp == 0) {
    long long carry = 0;
    for (int i0 = 1; i0 <= a.seqs; i0 += 32) {
      long long v = i0 + lane <= a.seqs ? sm.cum[i0 + lane] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (i0 + lane <= a.seqs) sm.cum[i0 + lane] = v + carry;
      carry += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  const long long total = sm.cum[a.seqs] * H;
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    bool ok = mbar_try_wait(bar, parity);
    if (!ok && !*reinterpret_cast<volatile int*>(&sm.failed)) {
      ok = mbar_wait_sleep(bar, parity, a.c.status, kStatusKv4Colsum);
      if (!ok) *reinterpret_cast<volatile int*>(&sm.failed) = 1;
    }
    return __all_sync(0xffffffffu, ok) != 0;
  };

  if (warp < 16) {
    // --------------------------- sums, one key and half of a tile's rows a thread
    const int half = warp >> 3, grp = warp >> 2 & 1, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(32 * quarter) << 16;
    uint32_t n = 0;  // tiles so far
    for (long long f = blockIdx.x; f < total; f += gridDim.x) {
      const Item w = item_at(d, sm.cum, f);
      const int key0 = w.kb * kKeys + grp * 128, key = key0 + r;
      uint64_t s0 = 0, s1 = 0;
      bool ok = true;
      for (int T = w.t0; T < w.t1; ++T, ++n) {
        const uint32_t sb = n % 2 * 2 + grp, cb = n % kCBufs;
        ok = ok && wait(&sm.cfull[cb], n / kCBufs & 1u) && wait(&sm.sfull[sb], n / 2 & 1u);
        if (!ok) continue;
        fence_after();
        const uint32_t tS = sm.tmem + sb * 128 + half * 64 + lane_off;
        const float *fc = sm.fac[cb] + half * 64, *of = sm.off[cb] + half * 64;
        const int* seen = sm.seen[cb] + half * 64;
        auto free_scores = [&]() {
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.sfree[sb]);
        };
        if (sm.all_see[cb] >= key0 + 128) {
          uint32_t x[16], y[16];
          auto add = [&](const uint32_t* v, int c0) {
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              const ulonglong2 f2 = *reinterpret_cast<const ulonglong2*>(fc + c0 + e);
              const ulonglong2 o2 = *reinterpret_cast<const ulonglong2*>(of + c0 + e);
              const uint64_t z0 = fma2(pair(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), f2.x, o2.x);
              const uint64_t z1 = fma2(pair(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])), f2.y, o2.y);
              s0 = add2(s0, pair(ex2(lo_of(z0)), ex2(hi_of(z0))));
              s1 = add2(s1, pair(ex2(lo_of(z1)), ex2(hi_of(z1))));
            }
          };
          ld16(tS, x);
          ld_wait16(x);
          ld16(tS + 16, y);
          add(x, 0);
          ld_wait16(y);
          ld16(tS + 32, x);
          add(y, 16);
          ld_wait16(x);
          ld16(tS + 48, y);
          add(x, 32);
          ld_wait16(y);
          free_scores();
          add(y, 48);
        } else {
#pragma unroll 1
          for (int c = 0; c < 64; c += 16) {
            uint32_t x[16];
            ld16(tS + c, x);
            ld_wait16(x);
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              // scores rounded as the log-sum-exps have them
              const float z0 = __fmul_rn(__uint_as_float(x[e]), fc[c + e]) + of[c + e];
              const float z1 = __fmul_rn(__uint_as_float(x[e + 1]), fc[c + e + 1]) + of[c + e + 1];
              s0 = add2(s0, pair(key < seen[c + e] ? ex2(z0) : 0.f, key < seen[c + e + 1] ? ex2(z1) : 0.f));
            }
            __syncwarp();
          }
          free_scores();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.cfree[cb]);
      }
      const uint64_t s = add2(s0, s1);
      if (w.t1 > w.t0) d.part[w.part + half * kKeys + grp * 128 + r] = lo_of(s) + hi_of(s);
    }
  } else if (warp < 20) {
    // ------------------------------------------------------- K codes, once an item
    const int dw = warp - 16, q = lane & 3, tok = lane >> 2;
    uint4 kc[2][4];
    uint32_t ks[2][4], items = 0;
    auto fetch = [&](const Item& w) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int g = i >> 2, e = i & 3, key = w.kb * kKeys + g * 128 + dw * 32 + e * 8 + tok, tt = key % kPageTokens;
        const bool there = key < w.s.len;
        const int block = there ? max(0, kv4_block(a.c, a.c.block_table, w.s.sid, key / kPageTokens)) : 0;
        const uint8_t* slab = a.c.pages + kv4_slab_index(a.c, block, w.h) * kKv4Slab;
        kc[g][e] = *reinterpret_cast<const uint4*>(slab + tt * 64 + q * 16);
        // slots past the end may hold anything: scale 0
        ks[g][e] = there ? *reinterpret_cast<const uint16_t*>(slab + kKv4KScales + tt * 8 + q * 2) : 0u;
      }
    };
    long long f = next_with_tiles(d, sm.cum, blockIdx.x, total);
    if (f < total) fetch(item_at(d, sm.cum, f));
    for (; f < total; ++items) {
      if (!wait(&sm.kfree, (items & 1u) ^ 1u)) break;
      codes_to_tile(smem + kOffK, dw, kc[0], ks[0]);
      codes_to_tile(smem + kOffK + kTile, dw, kc[1], ks[1]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.kfull);
      f = next_with_tiles(d, sm.cum, f + gridDim.x, total);
      if (f < total) fetch(item_at(d, sm.cum, f));
    }
  } else if (warp == 20) {
    // ------------------------------------- query tiles (TMA) and their constants
    uint32_t n = 0, issued = 0;
    bool ok = true;
    for (long long f = blockIdx.x; f < total && ok; f += gridDim.x) {
      const Item w = item_at(d, sm.cum, f);
      const int y0 = (w.h * a.rows + w.s.row0) * rep;  // the sequence's first row of the kv head
      for (int T = w.t0; T < w.t1; ++T, ++n) {
        const uint32_t qb = n % kQBufs, cb = n % kCBufs;
        float fv[4], ov[4];
        int sv[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int R = T * 128 + e * 32 + lane;
          const bool live = R < w.s.n * rep;
          fv[e] = live ? d.r.fac[y0 + R] : 0.f;
          ov[e] = live ? d.r.off[y0 + R] : -INFINITY;
          sv[e] = live ? w.s.len - w.s.n + 1 + R / rep : 0;
        }
        ok = wait(&sm.qfree[qb], (n / kQBufs & 1u) ^ 1u);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&sm.qfull[qb], kTile);
          tma2d(smem + kOffQ + qb * kTile, &q_map, 0, y0 + T * 128, &sm.qfull[qb]);
          tma2d(smem + kOffQ + qb * kTile + kHalf, &q_map, 64, y0 + T * 128, &sm.qfull[qb]);
        }
        ++issued;
        ok = wait(&sm.cfree[cb], (n / kCBufs & 1u) ^ 1u);
        if (!ok) break;
        bool large = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          large |= fabsf(ov[e]) > kLarge && ov[e] != -INFINITY;
          sm.fac[cb][e * 32 + lane] = fv[e];
          sm.off[cb][e * 32 + lane] = ov[e];
          sm.seen[cb][e * 32 + lane] = sv[e];
        }
        large = __any_sync(0xffffffffu, large);
        if (lane == 0)
          sm.all_see[cb] = large || (T + 1) * 128 > w.s.n * rep ? 0 : w.s.len - w.s.n + 1 + T * 128 / rep;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.cfull[cb]);
      }
    }
    // every copy has landed before the block ends
    for (uint32_t i = issued > kQBufs ? issued - kQBufs : 0; i < issued; ++i)
      mbar_wait(&sm.qfull[i % kQBufs], i / kQBufs & 1u, a.c.status, kStatusKv4Colsum);
  } else {
    // ------------------------------------------------------------------ MMA
    const uint32_t tm = __shfl_sync(0xffffffffu, sm.tmem, 0);
    const uint64_t dk = kmajor_desc(smem_u32(smem + kOffK)), dq = kmajor_desc(smem_u32(smem + kOffQ));
    const bool leader = elect_one();
    uint32_t n = 0, items = 0;
    bool ok = true;
    for (long long f = blockIdx.x; f < total && ok; f += gridDim.x) {
      const Item w = item_at(d, sm.cum, f);
      const int t0 = __shfl_sync(0xffffffffu, w.t0, 0), t1 = __shfl_sync(0xffffffffu, w.t1, 0);
      if (t1 <= t0) continue;
      ok = wait(&sm.kfull, items & 1u);
      for (int T = t0; T < t1 && ok; ++T, ++n) {
        const uint32_t qb = n % kQBufs;
        ok = wait(&sm.qfull[qb], n / kQBufs & 1u);
        const uint64_t q0 = dq + qb * (kTile >> 4);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const uint32_t sb = n % 2 * 2 + g;
          ok = ok && wait(&sm.sfree[sb], (n / 2 & 1u) ^ 1u);
          if (!ok) break;
          fence_after();
          if (leader) {
#pragma unroll
            for (int i = 0; i < kHeadDim / 16; ++i) {
              const uint64_t off = ((i >> 2) * kHalf + (i & 3) * 32) >> 4;
              mma_ss(tm + sb * 128, dk + g * (kTile >> 4) + off, q0 + off, idesc(false), i > 0 ? 1u : 0u);
            }
            commit(&sm.sfull[sb]);
          }
          __syncwarp();
        }
        if (ok && leader) {
          commit(&sm.qfree[qb]);
          if (T + 1 == t1) commit(&sm.kfree);
        }
        __syncwarp();
      }
      ++items;
    }
    if (leader) {
      commit(&sm.fin);  // nothing may still write TMEM when it is freed
      mbar_wait(&sm.fin, 0, a.c.status, kStatusKv4Colsum);
    }
    __syncwarp();
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 21)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(sm.tmem));
}

// weights of 256 keys: their items' sums in order, one thread a slot.
__global__ void __launch_bounds__(kKeys) kv4_colsum_add_kernel(const ColsumArgs d) {
  const Kv4AttnArgs& a = d.a;
  const int kb = blockIdx.x, h = blockIdx.y, i = blockIdx.z, rep = a.c.q_heads / a.c.kv_heads;
  const int key = kb * kKeys + threadIdx.x;
  pdl_wait();
  Kv4Seq s;
  if (!kv4_seq(a, i, s) || s.n == 0 || key >= s.len) return;
  float sum = 0.f;
  for (int c = 0; c < chunks_of(s, rep); ++c) {
    int t0, t1;
    tiles_seeing(s, rep, kb, c, t0, t1);
    if (t1 <= t0) break;
    const float* part = d.part + part_at(d, i, h, kb, c) + threadIdx.x;
    sum += part[0] + part[kKeys];
  }
  const int block = kv4_block(a.c, a.c.block_table, s.sid, key / kPageTokens);
  if (block >= 0) a.c.weights[kv4_slab_index(a.c, block, h) * kPageTokens + key % kPageTokens] += sum;
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return static_cast<EncodeTiledFn>(nullptr);
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

// The f16 queries as rows of 128, boxes of 128 rows by 64 dims; rows past the end
// read as zeros.
bool q_map_of(const Kv4Rows& r, uint64_t rows, CUtensorMap* m) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  const cuuint64_t dims[2] = {kHeadDim, rows}, strides[1] = {kHeadDim * 2};
  const cuuint32_t box[2] = {64, 128}, one[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, r.q16, dims, strides, box, one,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

long long chunks_max(int rep, long long max_q) {
  const long long tiles = (max_q * rep + 127) / 128;
  return (tiles + kChunk - 1) / kChunk;
}

}  // namespace

size_t kv4_colsum_scratch(int q_heads, int kv_heads, long long seqs, long long max_q,
                          long long max_len) {
  const long long n = seqs < kSeqChunk ? seqs : kSeqChunk;
  return static_cast<size_t>(n) * kv_heads * ((max_len + kKeys - 1) / kKeys) * chunks_max(q_heads / kv_heads, max_q) *
         2 * kKeys * sizeof(float);
}

cudaError_t kv4_colsum_launch(const Kv4AttnArgs& a, const Kv4Rows& rows, void* scratch,
                              cudaStream_t s) {
  if (a.max_len == 0) return cudaSuccess;
  CUtensorMap map;
  if (!q_map_of(rows, static_cast<uint64_t>(a.rows) * a.c.q_heads, &map)) return cudaErrorNotSupported;
  cudaError_t e = kv4_allow_smem<kv4_colsum_kernel>(kSmemBytes);
  for (int at = 0; at < a.seqs && e == cudaSuccess; at += kSeqChunk) {
    ColsumArgs d{};
    d.a = a;
    d.a.seqs = a.seqs - at < kSeqChunk ? a.seqs - at : kSeqChunk;
    d.a.sids = a.sids + at;
    d.a.lens = a.lens + at;
    if (a.q_starts) d.a.q_starts = a.q_starts + at;
    d.r = rows;
    d.part = static_cast<float*>(scratch);
    d.kb_max = (a.max_len + kKeys - 1) / kKeys;
    d.chunks = static_cast<int>(chunks_max(a.c.q_heads / a.c.kv_heads, a.max_q));
    e = kv4_start(kv4_colsum_kernel, dim3(148), kThreads, kSmemBytes, s, map, d);
    if (e == cudaSuccess)
      e = kv4_start(kv4_colsum_add_kernel, dim3(d.kb_max, a.c.kv_heads, d.a.seqs), kKeys, 0, s, d);
  }
  return e;
}

}  // namespace dialb200
