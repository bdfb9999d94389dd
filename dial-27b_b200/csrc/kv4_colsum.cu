// Running weights of many queries over the 4-bit KV cache: for every slot, the sum
// of its probabilities over the queries that see it and the heads of its group.
//
//   weights[t] += sum_r 2^(fac_r q_r . k_t - lse_r)
//
// with the f16 queries, scales and log-sum-exps that the attention before it left
// (kv4_prefill.cu).  Half that attention's MMAs and all of its exponentials; bound
// by the exponentials (16 a clock and SM).  S^T = K Q^T has a key in every TMEM
// lane, so a thread adds up its own key's row and nothing is exchanged.
//
// Items: a 128-key block of a (sequence, kv head) and up to kChunk tiles of 128 rows
// that see it, dealt to the CTAs in turn.  Warps 0-3 and 4-7 take tiles in turn
// and leave a sum for each key; kv4_colsum_add_kernel adds an item's sums to the
// weights in a fixed order.  Warps 8-11: K codes -> f16 once an item (loaded during
// the item before), query tiles and their constants by cp.async into four buffers;
// warp 12: tcgen05.mma into four TMEM buffers.
#include "kv4_attn.h"
#include "kv4_tc.cuh"

namespace dialb200 {
namespace {

constexpr int kThreads = 13 * 32;
constexpr int kSeqChunk = 512;  // sequences a launch
constexpr int kChunk = 32;      // query tiles of an item at most
constexpr int kQBufs = 4, kSBufs = 4, kCBufs = 8;  // query tiles, scores, constants
constexpr int kOffK = 0;                     // [2]
constexpr int kOffQ = 2 * kTile;             // [kQBufs]
constexpr int kOffMisc = (2 + kQBufs) * kTile;
constexpr int kStatusKv4Colsum = 0x602;

struct Misc {
  uint64_t kfull[2], kfree[2], qfull[kQBufs], qfree[kQBufs], sfull[kSBufs], sfree[kSBufs], cfull[kCBufs], cfree[kCBufs], fin;
  uint32_t tmem;
  int failed;
  alignas(16) float fac[kCBufs][128];
  alignas(16) float off[kCBufs][128];
  alignas(16) int seen[kCBufs][128];    // slots the row sees
  long long cum[kSeqChunk + 1];         // items of one kv head of the sequences before
};
constexpr int kSmemBytes = kOffMisc + sizeof(Misc) + 1024;

struct ColsumArgs {
  Kv4AttnArgs a;
  Kv4Rows r;
  float* part;  // [seqs][kv_heads][kb_max][chunks][2][128]
  int kb_max, chunks;
};

__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}

struct Item {
  Kv4Seq s;
  int i, h, kb, t0, t1;  // tiles t0 .. t1 - 1
  size_t part;
};

__device__ __forceinline__ int tiles_of(const Kv4Seq& s, int rep) { return (s.n * rep + 127) / 128; }
__device__ __forceinline__ int blocks_of(const Kv4Seq& s) { return s.n > 0 ? (s.len + 127) / 128 : 0; }
__device__ __forceinline__ int chunks_of(const Kv4Seq& s, int rep) { return (tiles_of(s, rep) + kChunk - 1) / kChunk; }

// Tiles of chunk c that see key block kb: t1 <= t0 for none.
__device__ __forceinline__ void tiles_seeing(const Kv4Seq& s, int rep, int kb, int c, int& t0, int& t1) {
  const int first = max(0, kb * 128 - (s.len - s.n));  // the first query that sees the block
  t0 = static_cast<int>(static_cast<unsigned>(first * rep) / 128u) + c * kChunk;
  t1 = min(t0 + kChunk, tiles_of(s, rep));
}

__device__ __forceinline__ size_t part_at(const ColsumArgs& d, int i, int h, int kb, int c) {
  return ((((static_cast<size_t>(i) * d.a.c.kv_heads + h) * d.kb_max + kb) * d.chunks + c) * 2) * 128;
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

__global__ void __launch_bounds__(kThreads, 1) kv4_colsum_kernel(const ColsumArgs d) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  Misc& sm = *reinterpret_cast<Misc*>(smem + kOffMisc);
  const Kv4AttnArgs& a = d.a;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int H = a.c.kv_heads, rep = a.c.q_heads / H;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.kfull[i], 4);
      mbar_init(&sm.kfree[i], 1);
    }
    for (int i = 0; i < kQBufs; ++i) {
      mbar_init(&sm.qfull[i], 4);
      mbar_init(&sm.qfree[i], 1);
    }
    for (int i = 0; i < kSBufs; ++i) {
      mbar_init(&sm.sfull[i], 1);
      mbar_init(&sm.sfree[i], 4);
    }
    for (int i = 0; i < kCBufs; ++i) {
      mbar_init(&sm.cfull[i], 4);
      mbar_init(&sm.cfree[i], 4);
    }
    mbar_init(&sm.fin, 1);
    sm.failed = 0;
    fence_mbar_init();
  }
  if (warp == 12) {
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

  if (warp < 8) {
    // ------------------------------------------------ sums, one key a thread
    const int grp = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(32 * quarter) << 16;
    uint32_t n = 0;  // tiles so far
    for (long long f = blockIdx.x; f < total; f += gridDim.x) {
      const Item w = item_at(d, sm.cum, f);
      const int key = w.kb * 128 + r;
      uint64_t s0 = 0, s1 = 0;
      bool ok = true;
      for (int T = w.t0; T < w.t1; ++T, ++n) {
        if ((n & 1u) != static_cast<uint32_t>(grp)) continue;
        const uint32_t sb = n % kSBufs, cb = n % kCBufs;
        ok = ok && wait(&sm.cfull[cb], n / kCBufs & 1u) && wait(&sm.sfull[sb], n / kSBufs & 1u);
        if (!ok) continue;
        fence_after();
        const uint32_t tS = sm.tmem + sb * 128 + lane_off;
        const float *fc = sm.fac[cb], *of = sm.off[cb];
        // every row of the tile sees the whole block
        if (w.s.len - w.s.n + 1 + T * 128 / rep >= (w.kb + 1) * 128) {
          uint32_t x[32], y[32];
          auto add = [&](const uint32_t* v, int c0) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const ulonglong2 f2 = *reinterpret_cast<const ulonglong2*>(fc + c0 + e);
              const ulonglong2 o2 = *reinterpret_cast<const ulonglong2*>(of + c0 + e);
              const uint64_t z0 = fma2(pair(__uint_as_float(v[e]), __uint_as_float(v[e + 1])), f2.x, o2.x);
              const uint64_t z1 = fma2(pair(__uint_as_float(v[e + 2]), __uint_as_float(v[e + 3])), f2.y, o2.y);
              s0 = add2(s0, pair(ex2(lo_of(z0)), ex2(hi_of(z0))));
              s1 = add2(s1, pair(ex2(lo_of(z1)), ex2(hi_of(z1))));
            }
          };
          ld32(tS, x);
          ld_wait(x);
          ld32(tS + 32, y);
          add(x, 0);
          ld_wait(y);
          ld32(tS + 64, x);
          add(y, 32);
          ld_wait(x);
          ld32(tS + 96, y);
          add(x, 64);
          ld_wait(y);
          add(y, 96);
        } else {
#pragma unroll 1
          for (int c = 0; c < 128; c += 16) {
            uint32_t x[16];
            ld16(tS + c, x);
            ld_wait16(x);
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const float z0 = fmaf(__uint_as_float(x[e]), fc[c + e], of[c + e]);
              const float z1 = fmaf(__uint_as_float(x[e + 1]), fc[c + e + 1], of[c + e + 1]);
              s0 = add2(s0, pair(key < sm.seen[cb][c + e] ? ex2(z0) : 0.f, key < sm.seen[cb][c + e + 1] ? ex2(z1) : 0.f));
            }
            __syncwarp();
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sm.sfree[sb]);
          mbar_arrive(&sm.cfree[cb]);
        }
      }
      const uint64_t s = add2(s0, s1);
      d.part[w.part + grp * 128 + r] = w.t1 > w.t0 ? lo_of(s) + hi_of(s) : 0.f;
    }
  } else if (warp < 12) {
    // --------------------------------------------- K codes and query tiles
    const int dw = warp - 8, q = lane & 3, tok = lane >> 2, row = dw * 32 + lane;
    constexpr uint32_t kAhead = 2;         // tiles in flight behind the one being issued
    uint32_t n = 0, landed = 0, items = 0;  // tiles issued and handed on
    bool ok = true;
    auto hand_on = [&]() {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sm.qfull[landed % kQBufs]);
        mbar_arrive(&sm.cfull[landed % kCBufs]);
      }
      ++landed;
    };
    uint4 kc[4];
    uint32_t ks[4];
    auto next_item = [&](long long& f, Item& w) {  // the next with tiles, and its codes
      for (; f < total; f += gridDim.x) {
        w = item_at(d, sm.cum, f);
        if (w.t1 > w.t0) break;
      }
      if (f >= total) return;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = w.kb * 128 + dw * 32 + e * 8 + tok, tt = key % kPageTokens;
        const bool there = key < w.s.len;
        const int block = there ? max(0, kv4_block(a.c, a.c.block_table, w.s.sid, key / kPageTokens)) : 0;
        const uint8_t* slab = a.c.pages + kv4_slab_index(a.c, block, w.h) * kKv4Slab;
        kc[e] = *reinterpret_cast<const uint4*>(slab + tt * 64 + q * 16);
        // slots past the end may hold anything: scale 0
        ks[e] = there ? *reinterpret_cast<const uint16_t*>(slab + kKv4KScales + tt * 8 + q * 2) : 0u;
      }
    };
    long long f = blockIdx.x;
    Item w;
    next_item(f, w);
    while (f < total) {
      const int kbuf = items & 1;
      const uint32_t turn = (items >> 1 & 1u) ^ 1u;
      if (!__all_sync(0xffffffffu, mbar_try_wait(&sm.kfree[kbuf], turn))) {
        // the buffer's MMAs may need tiles that are still held back here
        cp_async_wait();
        while (landed < n) hand_on();
      }
      ok = wait(&sm.kfree[kbuf], turn);
      if (!ok) break;
      codes_to_tile(smem + kOffK + kbuf * kTile, dw, kc, ks);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.kfull[kbuf]);
      ++items;
      const Item cur = w;
      f += gridDim.x;
      next_item(f, w);
      for (int T = cur.t0; T < cur.t1; ++T, ++n) {
        const uint32_t qb = n % kQBufs, cb = n % kCBufs;
        ok = wait(&sm.qfree[qb], (n / kQBufs & 1u) ^ 1u) && wait(&sm.cfree[cb], (n / kCBufs & 1u) ^ 1u);
        if (!ok) break;
        const int R = T * 128 + row;
        const bool live = R < cur.s.n * rep;
        const int j = live ? R / rep : 0;
        const long long at = live ? static_cast<long long>(cur.s.row0 + j) * a.c.q_heads + cur.h * rep + (R - j * rep) : -1;
        uint8_t* tile = smem + kOffQ + qb * kTile;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int rr = 2 * e + (lane >> 4), c = lane & 15;
          const long long from = __shfl_sync(0xffffffffu, at, rr);
          cp_async16(tile + (c >> 3) * kHalf + (dw * 32 + rr) * 128 + (((c & 7) ^ (rr & 7)) << 4),
                     d.r.q16 + (from < 0 ? 0 : from) * kHeadDim + c * 8, from >= 0);
        }
        if (live) {
          cp_async4(&sm.fac[cb][row], d.r.fac + at);
          cp_async4(&sm.off[cb][row], d.r.off + at);
        } else {
          sm.fac[cb][row] = 0.f;
          sm.off[cb][row] = -INFINITY;
        }
        sm.seen[cb][row] = live ? cur.s.len - cur.s.n + 1 + j : 0;
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (n - landed >= kAhead) {
          asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
          hand_on();
        }
      }
      if (!ok) break;
    }
    cp_async_wait();
    while (landed < n) hand_on();
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
      const uint32_t kbuf = items & 1;
      ok = wait(&sm.kfull[kbuf], items >> 1 & 1u);
      const uint64_t k0 = dk + kbuf * (kTile >> 4);
      for (int T = t0; T < t1 && ok; ++T, ++n) {
        const uint32_t qb = n % kQBufs, sb = n % kSBufs;
        ok = wait(&sm.qfull[qb], n / kQBufs & 1u) && wait(&sm.sfree[sb], (n / kSBufs & 1u) ^ 1u);
        if (!ok) break;
        fence_after();
        const uint64_t q0 = dq + qb * (kTile >> 4);
        if (leader) {
#pragma unroll
          for (int i = 0; i < kHeadDim / 16; ++i) {
            const uint64_t off = ((i >> 2) * kHalf + (i & 3) * 32) >> 4;
            mma_ss(tm + sb * 128, k0 + off, q0 + off, idesc(false), i > 0 ? 1u : 0u);
          }
          commit(&sm.sfull[sb]);
          commit(&sm.qfree[qb]);
          if (T + 1 == t1) commit(&sm.kfree[kbuf]);
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
  if (warp == 12)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(sm.tmem));
}

// weights of a key block: its items' sums in order, one thread a slot.
__global__ void __launch_bounds__(128) kv4_colsum_add_kernel(const ColsumArgs d) {
  const Kv4AttnArgs& a = d.a;
  const int kb = blockIdx.x, h = blockIdx.y, i = blockIdx.z, rep = a.c.q_heads / a.c.kv_heads;
  const int key = kb * 128 + threadIdx.x;
  pdl_wait();
  Kv4Seq s;
  if (!kv4_seq(a, i, s) || s.n == 0 || key >= s.len) return;
  float sum = 0.f;
  for (int c = 0; c < chunks_of(s, rep); ++c) {
    int t0, t1;
    tiles_seeing(s, rep, kb, c, t0, t1);
    if (t1 <= t0) break;
    const float* p = d.part + part_at(d, i, h, kb, c) + threadIdx.x;
    sum += p[0] + p[128];
  }
  const int block = kv4_block(a.c, a.c.block_table, s.sid, key / kPageTokens);
  if (block >= 0) a.c.weights[kv4_slab_index(a.c, block, h) * kPageTokens + key % kPageTokens] += sum;
}

template <typename K>
cudaError_t start(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t s, const ColsumArgs& d) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, d);
}

long long chunks_max(int rep, long long max_q) {
  const long long tiles = (max_q * rep + 127) / 128;
  return (tiles + kChunk - 1) / kChunk;
}

}  // namespace

size_t kv4_colsum_scratch(int q_heads, int kv_heads, long long seqs, long long max_q,
                          long long max_len) {
  const long long n = seqs < kSeqChunk ? seqs : kSeqChunk;
  return static_cast<size_t>(n) * kv_heads * ((max_len + 127) / 128) * chunks_max(q_heads / kv_heads, max_q) * 2 *
         128 * sizeof(float);
}

cudaError_t kv4_colsum_launch(const Kv4AttnArgs& a, const Kv4Rows& rows, void* scratch,
                              cudaStream_t s) {
  if (a.max_len == 0) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kv4_colsum_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
  for (int at = 0; at < a.seqs && e == cudaSuccess; at += kSeqChunk) {
    ColsumArgs d{};
    d.a = a;
    d.a.seqs = a.seqs - at < kSeqChunk ? a.seqs - at : kSeqChunk;
    d.a.sids = a.sids + at;
    d.a.lens = a.lens + at;
    if (a.q_starts) d.a.q_starts = a.q_starts + at;
    d.r = rows;
    d.part = static_cast<float*>(scratch);
    d.kb_max = (a.max_len + 127) / 128;
    d.chunks = static_cast<int>(chunks_max(a.c.q_heads / a.c.kv_heads, a.max_q));
    e = start(kv4_colsum_kernel, dim3(148), kThreads, kSmemBytes, s, d);
    if (e == cudaSuccess)
      e = start(kv4_colsum_add_kernel, dim3(d.kb_max, a.c.kv_heads, d.a.seqs), 128, 0, s, d);
  }
  return e;
}

}  // namespace dialb200
