// Attention of many queries over the 4-bit KV cache on the 5th-generation
// tensor cores (prompts, chunks of prompts).
//
// Tensor-bound: 4 * 128 FLOP a (query, head, slot) against 144 bytes a slot and
// kv head, which 256 rows share.  A row is a (query, head of the group) pair, so
// that a tile of 128 rows uses one kv head whatever the group's size, and a CTA
// takes two tiles over the same keys.  Its 13 warps:
//   0-3, 4-7  one row of tile 0 / 1 a thread: the row's queries into shared
//             memory (f16 after an exact power-of-two scale), softmax, output
//   8-11      codes -> f16 operands: registers one block ahead, e2m1 * e4m3
//             (exact in f16), 128-byte swizzled tiles, K and V double-buffered
//   12        tcgen05.mma: S_t = Q_t K^T into TMEM, O_t += P_t V with P from TMEM
// P (f16) takes the first 64 of its own S's 128 columns, 32 for each half of the
// keys, once the scores there are read.  S_t of block j + 1 is issued right after P V
// of block j, so one tile's softmax runs beside the other's MMAs.
// The exponent's reference moves only when a score exceeds the one it was set by by more
// than 8 (base 2): a block is taken in one pass, without its maximum first, and O in
// TMEM is rarely rescaled.  P is f16 (2^-11 relative), which its MMA's rate asks for; scores,
// sums and O are f32.
// A block goes in halves of 64 keys, so that the first half's P is stored beside the
// second's work (332 us against 363 for the 512-token chunk); code that runs once
// an item is kept in rolled loops, since its instructions are fetched anew each time
// (290 against 332).
//
// Measured: a 2048-token prompt, 32 heads of 8 (34 GFLOP) 73 us with the join of 14; 512
// tokens each on 9500 and 16897 slots, 40 heads of 8 (271 GFLOP) 290-317 by the
// clock.  Two tiles' 128-key block takes 2.4 us against 1.1 for its MMAs and 1.1 for
// its exponentials: bound by the chain S, softmax, P V of each tile, of which two
// are all that TMEM's 512 columns hold.  Sixteen softmax warps, two a row, took 420
// (80 registers a thread); scores in runs of 32 380 (spills).
//
// Work split: the 128-key blocks of all items (sequence, kv head, pair of tiles)
// laid end to end, one range a CTA, an item counted as kPad blocks more for its
// start and output; the parts of items that cross ranges are added by
// kv4_prefill_join_kernel.
#include <cmath>

#include "kv4_attn.h"
#include "kv4_launch.h"
#include "kv4_tc.cuh"

namespace dialb200 {
namespace {

constexpr int kRows = 128;                  // rows of a tile
constexpr int kKeys = 128;                  // keys of a block
constexpr int kThreads = 13 * 32;
// An item's own cost (its start and output), in blocks.  At 2 / 4 / 6: a prompt of 1024
// tokens 41.1 / 39.3 / 36.5 us, of 2048 81.1 / 72.9 / 75.8, of 4096 195 / 181 / 186; 300
// queries each of 4 sessions of 2000 to 6000 slots 137 / 140 / 142; 512 each on 9500
// and 16897 the same within 0.4 %.
constexpr int kPad = 4;
constexpr int kSeqChunk = 512;              // sequences a launch
constexpr int kOffQ = 0;                    // [2]
constexpr int kOffK = 2 * kTile;            // [2]
constexpr int kOffV = 4 * kTile;            // [2]
constexpr int kOffMisc = 6 * kTile;
// Probabilities are taken against a reference kLift below a row's largest score, base 2:
// f16 keeps them to 2^-32 of the largest, and the f32 sums lose more over as many slots.
// The reference moves when one would exceed 2^kTop.
constexpr float kLift = 7.f, kTop = 15.f;
constexpr int kStatusKv4Prefill = 0x601;

struct Misc {
  uint64_t kfull[2], kfree[2], vfull[2], vfree[2];  // by buffer
  uint64_t qfull[2], sfull[2], pready[2], odone[2], fin;  // by tile
  uint32_t tmem;
  int failed;
  long long cum[kSeqChunk + 1];  // cost of one kv head of the sequences before
  long long cut[2];
  alignas(16) unsigned char share[8][2][96];  // of the softmax warps: this item and the next
};
constexpr int kSmemBytes = kOffMisc + sizeof(Misc) + 1024;

struct PrefillArgs {
  Kv4AttnArgs a;
  int ctas;
  // [ctas]: (sequence, kv head, pair) of the item that starts in a range and
  // goes on, or -1; and whether the item the range begins inside ends in it
  int4* desc;
  float* part_o;    // [2 * ctas][256][128]
  float2* part_ml;  // [2 * ctas][256]
  // with weights (else null), for every row and head: the queries as f16, their
  // scale to base-2 scores, and minus the log-sum-exp, base 2
  uint16_t* q16;
  float* fac;
  float* off;
};

// Place of (row, query head) in the arrays that the weights' kernel reads.
__device__ __forceinline__ size_t row_at(const Kv4AttnArgs& a, int row, int head) {
  const int rep = a.c.q_heads / a.c.kv_heads, h = head / rep;
  return (static_cast<size_t>(h) * a.rows + row) * rep + (head - h * rep);
}

// --------------------------------------------------------------- work items
// Key blocks that tile T (128 rows) of the sequence sees.  n * rep < 2^29.
__device__ __forceinline__ int tile_blocks(const Kv4Seq& s, unsigned rep, int T) {
  const int all = s.n * static_cast<int>(rep), r0 = T * kRows;
  if (r0 >= all) return 0;
  const int last = static_cast<int>(static_cast<unsigned>(min(r0 + kRows, all) - 1) / rep);
  const int seen = s.len - s.n + 1 + last;
  return seen > 0 ? (seen + kKeys - 1) / kKeys : 0;
}
// Blocks of the pair of tiles tp: its last row sees the most.
__device__ __forceinline__ int pair_blocks(const Kv4Seq& s, unsigned rep, int tp) {
  const int t1 = 2 * tp + 1;
  return tile_blocks(s, rep, t1 * kRows < s.n * static_cast<int>(rep) ? t1 : t1 - 1);
}
__device__ __forceinline__ int pairs_of(const Kv4Seq& s, int rep) {
  return (s.n * rep + 2 * kRows - 1) / (2 * kRows);
}
// An item's length in the order of work.
__device__ __forceinline__ int item_cost(int blocks) { return blocks > 0 ? blocks + kPad : 0; }

// One item's share of a range: blocks j0 .. j1 - 1 of the item's nb.
struct Share {
  Kv4Seq s;
  int i, h, tp, nb, j0, j1;
  int blocks[2];     // of the two tiles
  long long start;   // the item's first block among all
};

// The item that holds place f of the order of work (f < total); warp-collective.
__device__ Share item_at(const Kv4AttnArgs& a, const long long* cum, long long f) {
  const int lane = threadIdx.x & 31, H = a.c.kv_heads, rep = a.c.q_heads / H;
  int lo = 0, hi = a.seqs;  // cum[lo] * H <= f < cum[hi] * H
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cum[mid] * H <= f) lo = mid;
    else hi = mid;
  }
  Share w;
  w.i = lo;
  kv4_seq(a, lo, w.s);
  const long long per = cum[lo + 1] - cum[lo];
  long long r = f - cum[lo] * H;
  w.h = static_cast<int>(r / per);
  r -= w.h * per;
  w.start = f - r;
  w.tp = 0;
  w.nb = 1;
  for (int tp = 0; tp < pairs_of(w.s, rep); tp += 32) {  // the pair whose blocks hold r
    const int own = pair_blocks(w.s, rep, tp + lane);
    int v = item_cost(own);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    const unsigned past = __ballot_sync(0xffffffffu, v > r);
    if (past) {
      const int at = __ffs(past) - 1;
      w.tp = tp + at;
      w.nb = __shfl_sync(0xffffffffu, own, at);
      w.start += __shfl_sync(0xffffffffu, v, at) - item_cost(w.nb);
      break;
    }
    const int all = __shfl_sync(0xffffffffu, v, 31);
    r -= all;
    w.start += all;
  }
  return w;
}

// The share of [f, end) that begins at f in item w.
__device__ __forceinline__ void set_share(const Kv4AttnArgs& a, Share& w, long long f, long long end) {
  const int rep = a.c.q_heads / a.c.kv_heads;
  w.j0 = max(0, static_cast<int>(f - w.start) - kPad);
  w.j1 = static_cast<int>(min(static_cast<long long>(w.nb), end - w.start - kPad));
  w.blocks[0] = tile_blocks(w.s, rep, 2 * w.tp);
  w.blocks[1] = tile_blocks(w.s, rep, 2 * w.tp + 1);
}

// The item after w, which is not the last.
__device__ __forceinline__ void next_item(const Kv4AttnArgs& a, const long long* cum, Share& w) {
  const int rep = a.c.q_heads / a.c.kv_heads;
  w.start += item_cost(w.nb);
  do {
    if (++w.tp >= pairs_of(w.s, rep)) {
      w.tp = 0;
      if (++w.h >= a.c.kv_heads) {
        w.h = 0;
        do ++w.i;
        while (cum[w.i + 1] == cum[w.i]);
        kv4_seq(a, w.i, w.s);
      }
    }
    w.nb = pair_blocks(w.s, rep, w.tp);
  } while (w.nb == 0);
}

__device__ void work_prefix(const Kv4AttnArgs& a, long long* cum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int rep = a.c.q_heads / a.c.kv_heads;
  for (int i = warp; i < a.seqs; i += warps) {
    Kv4Seq s;
    long long sum = 0;
    if (kv4_seq(a, i, s))
      for (int tp = lane; tp < pairs_of(s, rep); tp += 32) sum += item_cost(pair_blocks(s, rep, tp));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) cum[i + 1] = sum;
  }
  if (threadIdx.x == 0) cum[0] = 0;
  __syncthreads();
  if (warp == 0) {
    long long carry = 0;
    for (int i0 = 1; i0 <= a.seqs; i0 += 32) {
      long long v = i0 + lane <= a.seqs ? cum[i0 + lane] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (i0 + lane <= a.seqs) cum[i0 + lane] = v + carry;
      carry += __shfl_sync(0xffffffffu, v, 31);
    }
  }
  __syncthreads();
}

// 32 bytes, on a 32-byte boundary: a row's stores are whole sectors.
__device__ __forceinline__ void st_global8(void* to, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]),
               "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

template <typename Act>
__global__ void __launch_bounds__(kThreads, 1) kv4_prefill_kernel(const PrefillArgs d) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  Misc& sm = *reinterpret_cast<Misc*>(smem + kOffMisc);
  const Kv4AttnArgs& a = d.a;
  const int tid = threadIdx.x, lane = tid & 31, b = blockIdx.x;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // known to be one value a warp
  const int H = a.c.kv_heads, rep = a.c.q_heads / H;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.kfull[i], 4);
      mbar_init(&sm.vfull[i], 4);
      mbar_init(&sm.kfree[i], 1);
      mbar_init(&sm.vfree[i], 1);
      mbar_init(&sm.qfull[i], 4);
      mbar_init(&sm.pready[i], 4);
      mbar_init(&sm.sfull[i], 1);
      mbar_init(&sm.odone[i], 1);
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
  work_prefix(a, sm.cum);
  const long long total = sm.cum[a.seqs] * H;
  // queries that see no slot: zeros
  for (int i = b; i < a.seqs; i += d.ctas) {
    Kv4Seq s;
    if (!kv4_seq(a, i, s)) continue;
    for (int r = 0; r < min(s.n, s.n - s.len); ++r) {
      for (int e = tid * 8; e < a.c.q_heads * kHeadDim; e += kThreads * 8)
        *reinterpret_cast<uint4*>(static_cast<Act*>(a.out) + (s.row0 + r) * a.out_ld + e) =
            make_uint4(0, 0, 0, 0);
      if (d.off)
        for (int e = tid; e < a.c.q_heads; e += kThreads)
          d.off[row_at(a, s.row0 + r, e)] = -INFINITY;
    }
  }
  const int ctas = static_cast<int>(min(static_cast<long long>(d.ctas), total));
  if (warp < 2 && b < ctas) {
    // this CTA's two cuts, none before an item's first block
    long long f = total * (b + warp) / ctas;
    if (f < total) {
      const Share w = item_at(a, sm.cum, f);
      if (f - w.start <= kPad) f = w.start;
    }
    if (lane == 0) sm.cut[warp] = f;
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sm.tmem;
  const long long f0 = b < ctas ? sm.cut[0] : 0, f1 = b < ctas ? sm.cut[1] : 0;
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (mbar_try_wait(bar, parity)) return true;
    if (*reinterpret_cast<volatile int*>(&sm.failed)) return false;
    if (mbar_wait_sleep(bar, parity, a.c.status, kStatusKv4Prefill)) return true;
    *reinterpret_cast<volatile int*>(&sm.failed) = 1;
    return false;
  };

  if (f0 >= f1) {
    if (tid == 0) d.desc[b] = make_int4(-1, 0, 0, -1);
  } else if (warp < 8) {
    // ------------------------------------------- queries, softmax and output
    const int t = warp >> 2, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(32 * quarter) << 16;
    const uint32_t tS = tmem + t * 128 + lane_off, tO = tmem + 256 + t * 128 + lane_off;
    uint8_t* q_tile = smem + kOffQ + t * kTile;
    uint8_t* q_row = q_tile + r * 128;
    uint32_t sphase = 0, ophase = 0;
    // kept in shared memory: registers are for the scores
    static_assert(sizeof(Share) <= sizeof(sm.share[0][0]), "a share's place");
    Share* cur = reinterpret_cast<Share*>(sm.share[warp][0]);
    Share* next = reinterpret_cast<Share*>(sm.share[warp][1]);
    {
      Share w = item_at(a, sm.cum, f0);
      set_share(a, w, f0, f1);
      if (lane == 0) *cur = w;
      __syncwarp();
    }
    auto find_next = [&](long long f) {
      Share w = *cur;
      next_item(a, sm.cum, w);
      set_share(a, w, f, f1);
      if (lane == 0) *next = w;
      __syncwarp();
    };
    bool ok = true, fetched = false;
    const bool wide = (reinterpret_cast<uintptr_t>(a.out) & 31) == 0 && a.out_ld % 16 == 0;
    // whether the item the range begins inside ends in it (1) or not (0)
    const int first = cur->j0 == 0 ? -1 : cur->j1 == cur->nb;
    // the warp's 32 rows of the tile's queries, raw, where their f16 form will be
    auto fetch_q = [&](const Share& x) {
      const int R = (2 * x.tp + t) * kRows + r;
      const bool mine = R < x.s.n * rep;
      const int j = mine ? R / rep : 0;
      long long at = (x.s.row0 + j) * a.q_ld + (x.h * rep + (mine ? R - j * rep : 0)) * kHeadDim;
      if (!mine) at = -1;
#pragma unroll 4
      for (int e = 0; e < 16; ++e) {
        const int row = 2 * e + (lane >> 4), c = lane & 15;
        const long long from = __shfl_sync(0xffffffffu, at, row);
        cp_async16(q_tile + (c >> 3) * kHalf + (quarter * 32 + row) * 128 + (((c & 7) ^ (row & 7)) << 4),
                   static_cast<const Act*>(a.q) + (from < 0 ? 0 : from) + c * 8, from >= 0);
      }
    };
    for (;;) {
      const Share& w = *cur;
      const int R = (2 * w.tp + t) * kRows + r;
      const bool live = R < w.s.n * rep;
      const int j = live ? R / rep : 0, head = w.h * rep + (live ? R - j * rep : 0);
      const int seen = live ? max(0, w.s.len - w.s.n + 1 + j) : 0;
      const int begin = w.j0, last = min(w.j1, w.blocks[t]);
      const long long f = w.start + kPad + w.j1;
      float m = -INFINITY, ref = 0.f, fac = 0.f;
      uint64_t l2 = 0;
      if (begin < last) {
        if (!fetched) fetch_q(w);
        cp_async_wait();
        __syncwarp();
        // to f16 (query_exp)
        float top = 0.f;
#pragma unroll 2
        for (int e = 0; e < 16; ++e) {
          const uint4 raw = *reinterpret_cast<const uint4*>(q_row + (e >> 3) * kHalf + (((e & 7) ^ (r & 7)) << 4));
          const Act* v = reinterpret_cast<const Act*>(&raw);
#pragma unroll
          for (int u = 0; u < 8; ++u) top = fmaxf(top, fabsf(ActTraits<Act>::to_f(v[u])));
        }
        const int ex = query_exp(top);
        const float down = exp2i(-ex);
        fac = score_scale(a, ex);
        const bool keep_q = d.off && live && begin == 0;
#pragma unroll 2
        for (int e = 0; e < 16; ++e) {
          uint4* at = reinterpret_cast<uint4*>(q_row + (e >> 3) * kHalf + (((e & 7) ^ (r & 7)) << 4));
          const uint4 raw = *at;
          const Act* v = reinterpret_cast<const Act*>(&raw);
          uint32_t o[4];
#pragma unroll
          for (int u = 0; u < 4; ++u)
            o[u] = pack_f16(ActTraits<Act>::to_f(v[2 * u]) * down, ActTraits<Act>::to_f(v[2 * u + 1]) * down);
          *at = make_uint4(o[0], o[1], o[2], o[3]);
          if (keep_q)
            reinterpret_cast<uint4*>(d.q16 + row_at(a, w.s.row0 + j, head) * kHeadDim)[e] = *at;
        }
        if (keep_q) d.fac[row_at(a, w.s.row0 + j, head)] = fac;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.qfull[t]);
      }
      fetched = false;
      if (f < f1) find_next(f);  // beside the first S
      const uint64_t fac2 = pair(fac, fac);
      for (int kb = begin; kb < last; ++kb) {
        ok = __all_sync(0xffffffffu, ok && wait(&sm.sfull[t], sphase & 1u));
        if (!ok) break;
        ++sphase;
        fence_after();
        const int open = seen - kb * kKeys;  // slots of the block that the row sees
        if (__any_sync(0xffffffffu, open < kKeys)) {  // few blocks are not whole: masked in place
#pragma unroll 1
          for (int c = 0; c < 8; ++c) {
            uint32_t x[16];
            ld16(tS + 16 * c, x);
            ld_wait16(x);
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (e + 16 * c >= open) x[e] = 0xFF800000u;  // -inf
            __syncwarp();  // tcgen05.ld and .st are warp-collective
            st16(tS + 16 * c, x);
          }
          st_wait();
        }
        // a half of the block after the other: the probabilities under the reference
        // so far, 16 scores at a time, the load of one chunk beside the work on the
        // other; where one would exceed 2^kTop the reference moves to kLift below the
        // row's maximum and the half is done again.  References are whole numbers, so that
        // sums and O are rescaled exactly, and the P of the half before to f16's smallest step.
#pragma unroll 1
        for (int hf = 0; hf < 2; ++hf) {
          uint32_t p[32];
          uint64_t sum0, sum1;
          float top;
          const uint32_t tH = tS + 64 * hf;
          auto probs = [&]() {
            const uint64_t off2 = pair(-ref, -ref);
            uint32_t x[16], y[16];
            float t0 = -INFINITY, t1 = -INFINITY;
            sum0 = sum1 = 0;
            auto chunk = [&](const uint32_t* v, uint32_t* to) {
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const uint64_t s = score2(a, pair(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), fac2);
                if (e & 1) t1 = max3(t1, lo_of(s), hi_of(s));
                else t0 = max3(t0, lo_of(s), hi_of(s));
                const uint64_t z = add2(s, off2);
                const float p0 = ex2(lo_of(z)), p1 = ex2(hi_of(z));
                if (e & 1) sum1 = add2(sum1, pair(p0, p1));
                else sum0 = add2(sum0, pair(p0, p1));
                to[e] = pack_f16(p0, p1);
              }
            };
            ld16(tH, x);
            ld_wait16(x);
            ld16(tH + 16, y);
            chunk(x, p);
            ld_wait16(y);
            ld16(tH + 32, x);
            chunk(y, p + 8);
            ld_wait16(x);
            ld16(tH + 48, y);
            chunk(x, p + 16);
            ld_wait16(y);
            chunk(y, p + 24);
            top = fmaxf(t0, t1);
          };
          probs();
          if (__any_sync(0xffffffffu, top > __fadd_rd(m, kTop))) {
            const float mn = fmaxf(m, ceilf(top) - kLift);
            const float al = m == -INFINITY ? 0.f : ex2(m - mn);
            m = mn;
            ref = mn == -INFINITY ? 0.f : mn;
            l2 = pair(lo_of(l2) * al, hi_of(l2) * al);
            if (kb > begin) {  // S of this block was issued after P V of the one before
#pragma unroll 1
              for (int cb = 0; cb < 8; ++cb) {
                uint32_t o[16];
                ld16(tO + cb * 16, o);
                ld_wait16(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * al);
                __syncwarp();
                st16(tO + cb * 16, o);
              }
            }
            if (hf == 1) {
              st_wait();
#pragma unroll 1
              for (int cb = 0; cb < 2; ++cb) {
                uint32_t o[16];
                ld16(tS + cb * 16, o);
                ld_wait16(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&o[e]));
                  o[e] = pack_f16(x.x * al, x.y * al);
                }
                __syncwarp();
                st16(tS + cb * 16, o);
              }
            }
            probs();
          }
          l2 = add2(l2, add2(sum0, sum1));
          __syncwarp();
          st16(tS + 32 * hf, p);
          st16(tS + 32 * hf + 16, p + 16);
        }
        st_wait();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.pready[t]);
        if (kb + 1 == last && f < f1) {
          // the tile's queries are read: the next item's may take their place
          fetched = next->j0 < min(next->j1, next->blocks[t]);
          if (fetched) fetch_q(*next);
        }
      }
      // ------------------------------------------------------------ output
      const bool whole = w.j0 == 0 && w.j1 == w.nb;
      const int slot = 2 * b + (w.j0 == 0 ? 1 : 0);
      const float l = lo_of(l2) + hi_of(l2);
      if (ok && w.j0 < last) {
        ok = __all_sync(0xffffffffu, wait(&sm.odone[t], ophase & 1u));
        ++ophase;
        if (ok) {
          fence_after();
          const float inv = l != 0.f ? a.c.v_scale / l : 0.f;
          Act* dst = static_cast<Act*>(a.out) + (w.s.row0 + j) * a.out_ld + head * kHeadDim;
          float* part = d.part_o + (static_cast<size_t>(slot) * 2 * kRows + t * kRows + r) * kHeadDim;
#pragma unroll 1
          for (int cb = 0; cb < 4; ++cb) {
            uint32_t o[32];
            ld32(tO + cb * 32, o);
            ld_wait(o);
            if (live && whole) {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                uint32_t v[8];
                Act* h = reinterpret_cast<Act*>(v);
#pragma unroll
                for (int u = 0; u < 16; ++u)
                  h[u] = ActTraits<Act>::from_f(l != 0.f ? __uint_as_float(o[16 * e + u]) * inv : 0.f);
                Act* to = dst + cb * 32 + e * 16;
                if (wide) {
                  st_global8(to, v);
                } else {
                  reinterpret_cast<uint4*>(to)[0] = make_uint4(v[0], v[1], v[2], v[3]);
                  reinterpret_cast<uint4*>(to)[1] = make_uint4(v[4], v[5], v[6], v[7]);
                }
              }
            } else if (live) {
#pragma unroll
              for (int e = 0; e < 4; ++e) st_global8(part + cb * 32 + e * 8, o + 8 * e);
            }
            __syncwarp();
          }
          __syncwarp();
          fence_before();
        }
      }
      if (live) {
        if (!whole)
          d.part_ml[static_cast<size_t>(slot) * 2 * kRows + t * kRows + r] = make_float2(l > 0.f || l != l ? m : -INFINITY, l);
        else if (d.off)
          d.off[row_at(a, w.s.row0 + j, head)] = l > 0.f ? -(m + log2f(l)) : -INFINITY;
      }
      if (f >= f1 || !ok) {
        // the only item of the range that can start in it and go on
        if (tid == 0)
          d.desc[b] = w.j0 == 0 && w.j1 < w.nb ? make_int4(w.i, w.h, w.tp, first) : make_int4(-1, 0, 0, first);
        break;
      }
      __syncwarp();  // every lane has read *cur, which takes the item after the next one
      Share* was = cur;
      cur = next;
      next = was;
    }
    cp_async_wait();
  } else if (warp < 12) {
    // ------------------------------------------------- codes to f16 operands
    // 4 lanes a token: lane q of a token holds dims 32q .. 32q + 31 (two scale
    // groups); a warp's load covers 8 tokens, 4 loads a warp and block
    const int dw = warp - 8, q = lane & 3, tok = lane >> 2;
    uint4 kc[4], vc[4];
    uint32_t ks[4], vs[4];
    // the block whose page numbers are being fetched: its item, slots, slabs
    Share w = item_at(a, sm.cum, f0);
    set_share(a, w, f0, f1);
    int kb = w.j0, slab[4], left = 0;
    bool more = true;
    auto fetch_pages = [&]() {  // of block kb, then on to the next block
      if (!more) return;
      left = w.s.len - kb * kKeys;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = dw * 32 + e * 8 + tok;
        const int block =
            at < left ? max(0, kv4_block(a.c, a.c.block_table, w.s.sid, (kb * kKeys + at) / kPageTokens)) : 0;
        slab[e] = block * H + w.h;
      }
      if (++kb >= w.j1) {
        const long long f = w.start + kPad + w.j1;
        more = f < f1;
        if (more) {
          next_item(a, sm.cum, w);
          set_share(a, w, f, f1);
          kb = w.j0;
        }
      }
    };
    auto load = [&]() {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = dw * 32 + e * 8 + tok, tt = at % kPageTokens;
        const uint8_t* src = a.c.pages + static_cast<size_t>(static_cast<unsigned>(slab[e])) * kKv4Slab;
        kc[e] = *reinterpret_cast<const uint4*>(src + tt * 64 + q * 16);
        vc[e] = *reinterpret_cast<const uint4*>(src + kKv4VCodes + tt * 64 + q * 16);
        // slots past the end may hold anything: scale 0
        ks[e] = at < left ? *reinterpret_cast<const uint16_t*>(src + kKv4KScales + tt * 8 + q * 2) : 0u;
        vs[e] = at < left ? *reinterpret_cast<const uint16_t*>(src + kKv4VScales + tt * 8 + q * 2) : 0u;
      }
    };
    fetch_pages();
    load();
    for (uint32_t n = 0;; ++n) {
      const bool again = more;
      fetch_pages();  // of the block after this one
      const int buf = n & 1;
      const uint32_t turn = (n >> 1) & 1u;
      if (!__all_sync(0xffffffffu, wait(&sm.kfree[buf], turn ^ 1u))) break;
      codes_to_tile(smem + kOffK + buf * kTile, dw, kc, ks);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.kfull[buf]);
      if (!__all_sync(0xffffffffu, wait(&sm.vfree[buf], turn ^ 1u))) break;
      codes_to_tile(smem + kOffV + buf * kTile, dw, vc, vs);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.vfull[buf]);
      if (!again) break;
      load();
    }
  } else {
    // ------------------------------------------------------------------ MMA
    // the whole warp runs this, on values that are the same in all its lanes, and
    // one lane issues: operands stay in uniform registers
    Share w = item_at(a, sm.cum, f0);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t dq = kmajor_desc(smem_u32(smem + kOffQ)), dk = kmajor_desc(smem_u32(smem + kOffK)),
                   dv = mnmajor_desc(smem_u32(smem + kOffV));
    const bool leader = elect_one();
    uint32_t n = 0, qphase[2] = {0, 0}, pphase[2] = {0, 0};
    auto all_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
    auto issue_s = [&](int t, uint32_t kn) {
      const uint64_t k0 = dk + (kn & 1) * (kTile >> 4), q0 = dq + t * (kTile >> 4);
      if (leader) {
#pragma unroll
        for (int i = 0; i < kHeadDim / 16; ++i) {
          const uint64_t off = ((i >> 2) * kHalf + (i & 3) * 32) >> 4;
          mma_ss(tm + t * 128, q0 + off, k0 + off, idesc(false), i > 0 ? 1u : 0u);
        }
        commit(&sm.sfull[t]);
      }
      __syncwarp();
    };
    bool ok = true;
    for (long long f = f0; ok;) {
      set_share(a, w, f, f1);
      const int j0 = __shfl_sync(0xffffffffu, w.j0, 0), j1 = __shfl_sync(0xffffffffu, w.j1, 0);
      const int last0 = min(j1, __shfl_sync(0xffffffffu, w.blocks[0], 0));
      const int last1 = min(j1, __shfl_sync(0xffffffffu, w.blocks[1], 0));
      if (j0 < last0) ok = ok && all_wait(&sm.qfull[0], qphase[0]++ & 1u);
      if (j0 < last1) ok = ok && all_wait(&sm.qfull[1], qphase[1]++ & 1u);
      ok = ok && all_wait(&sm.kfull[n & 1], (n >> 1) & 1u);
      if (!ok) break;
      fence_after();
      if (j0 < last0) issue_s(0, n);
      if (j0 < last1) issue_s(1, n);
      if (leader) commit(&sm.kfree[n & 1]);
      for (int kb = j0; kb < j1; ++kb, ++n) {
        ok = all_wait(&sm.vfull[n & 1], (n >> 1) & 1u);
        const uint64_t v0 = dv + (n & 1) * (kTile >> 4);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int last = t == 0 ? last0 : last1;
          if (kb < last && ok) {
            ok = all_wait(&sm.pready[t], pphase[t]++ & 1u);
            if (!ok) break;
            fence_after();
            if (leader) {
#pragma unroll
              for (int i = 0; i < kKeys / 16; ++i)
                mma_ts(tm + 256 + t * 128, tm + t * 128 + i * 8, v0 + (i * 2048 >> 4), idesc(true),
                       (kb > j0 || i > 0) ? 1u : 0u);
              if (kb + 1 == last) commit(&sm.odone[t]);
            }
            __syncwarp();
          }
          if (kb + 1 < last && ok) {
            ok = all_wait(&sm.kfull[(n + 1) & 1], ((n + 1) >> 1) & 1u);
            if (!ok) break;
            fence_after();
            issue_s(t, n + 1);
          }
        }
        if (!ok) break;
        if (leader) {
          commit(&sm.vfree[n & 1]);
          if (kb + 1 < j1) commit(&sm.kfree[(n + 1) & 1]);
        }
        __syncwarp();
      }
      f = w.start + kPad + j1;
      if (f >= f1) break;
      next_item(a, sm.cum, w);
    }
    if (leader) {
      commit(&sm.fin);  // nothing may still write TMEM when it is freed
      mbar_wait(&sm.fin, 0, a.c.status, kStatusKv4Prefill);
    }
    __syncwarp();
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 12)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// Adds the parts of the item that starts in range blockIdx.x and goes on in
// others: one warp a row, parts in order.
template <typename Act>
__global__ void __launch_bounds__(256) kv4_prefill_join_kernel(const PrefillArgs d) {
  const Kv4AttnArgs& a = d.a;
  const int b = blockIdx.x, lane = threadIdx.x & 31, row = blockIdx.y * 8 + (threadIdx.x >> 5);
  const int rep = a.c.q_heads / a.c.kv_heads;
  pdl_wait();
  const int4 it = d.desc[b];
  if (it.x < 0) return;
  Kv4Seq s;
  kv4_seq(a, it.x, s);
  const long long R = static_cast<long long>(it.z) * 2 * kRows + row;
  if (R >= static_cast<long long>(s.n) * rep) return;
  // the ranges after this one that go on with the item, up to the one it ends in
  int parts = 1;
  for (;; parts += 32) {
    const bool end = b + parts + lane >= d.ctas || d.desc[b + parts + lane].w != 0;
    const unsigned ends = __ballot_sync(0xffffffffu, end);
    if (ends) {
      parts += __ffs(ends);
      break;
    }
  }
  float M = -INFINITY, L = 0.f;
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  auto slot = [&](int p) { return static_cast<size_t>(p == 0 ? 2 * b + 1 : 2 * (b + p)) * 2 * kRows + row; };
  for (int p = 0; p < parts; ++p) M = fmaxf(M, d.part_ml[slot(p)].x);
  for (int p = 0; p < parts; ++p) {
    const float2 ml = d.part_ml[slot(p)];
    if (ml.x == -INFINITY && ml.y == 0.f) continue;  // the row sees nothing there
    // scores that are all NaN leave no maximum, but a sum
    const float f = ml.x == -INFINITY ? 1.f : ex2(ml.x - M);
    const float4 v = reinterpret_cast<const float4*>(d.part_o)[slot(p) * (kHeadDim / 4) + lane];
    L = fmaf(f, ml.y, L);
    O.x = fmaf(f, v.x, O.x);
    O.y = fmaf(f, v.y, O.y);
    O.z = fmaf(f, v.z, O.z);
    O.w = fmaf(f, v.w, O.w);
  }
  const int j = static_cast<int>(R / rep), head = it.y * rep + static_cast<int>(R % rep);
  const float inv = L != 0.f ? a.c.v_scale / L : 0.f;
  const float o[4] = {O.x * inv, O.y * inv, O.z * inv, O.w * inv};
  store4(static_cast<Act*>(a.out) + (s.row0 + j) * a.out_ld + head * kHeadDim + lane * 4, o);
  if (d.off && lane == 0)
    d.off[row_at(a, s.row0 + j, head)] = L > 0.f ? -(M + log2f(L)) : -INFINITY;
}

int range_count() {
  static int n = [] {
    int v = 0, dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v < 1 || v > 148)
      v = 148;
    return v;
  }();
  return n;
}

constexpr size_t kDescBytes = 148 * 16 + 128 - (148 * 16) % 128;
constexpr size_t kPartBytes = 2ull * 148 * 2 * kRows * kHeadDim * 4;
constexpr size_t kMlBytes = 2ull * 148 * 2 * kRows * 8;

template <typename Act>
cudaError_t launch(const PrefillArgs& d, cudaStream_t s) {
  cudaError_t e = kv4_allow_smem<kv4_prefill_kernel<Act>>(kSmemBytes);
  if (e != cudaSuccess) return e;
  e = kv4_start(kv4_prefill_kernel<Act>, dim3(d.ctas), kThreads, kSmemBytes, s, d);
  if (e != cudaSuccess) return e;
  return kv4_start(kv4_prefill_join_kernel<Act>, dim3(d.ctas, 2 * kRows / 8), 256, 0, s, d);
}

}  // namespace

size_t kv4_prefill_scratch(int q_heads, long long rows, bool weights) {
  return kDescBytes + kPartBytes + kMlBytes + (weights ? static_cast<size_t>(rows) * q_heads * kKv4RowBytes : 0);
}

Kv4Rows kv4_prefill_rows(const Kv4AttnArgs& a) {
  Kv4Rows r;
  uint8_t* w = static_cast<uint8_t*>(a.scratch) + kDescBytes + kPartBytes + kMlBytes;
  const size_t n = static_cast<size_t>(a.rows) * a.c.q_heads;
  r.q16 = reinterpret_cast<uint16_t*>(w);
  r.fac = reinterpret_cast<float*>(w + n * kHeadDim * 2);
  r.off = r.fac + n;
  return r;
}

cudaError_t kv4_prefill_launch(const Kv4AttnArgs& a, int act, cudaStream_t s) {
  for (int at = 0; at < a.seqs; at += kSeqChunk) {
    PrefillArgs d{};
    d.a = a;
    d.a.seqs = a.seqs - at < kSeqChunk ? a.seqs - at : kSeqChunk;
    d.a.sids = a.sids + at;
    d.a.lens = a.lens + at;
    if (a.q_starts) d.a.q_starts = a.q_starts + at;
    d.ctas = range_count();
    uint8_t* w = static_cast<uint8_t*>(a.scratch);
    d.desc = reinterpret_cast<int4*>(w);
    d.part_o = reinterpret_cast<float*>(w + kDescBytes);
    d.part_ml = reinterpret_cast<float2*>(w + kDescBytes + kPartBytes);
    if (a.c.weights) {
      const Kv4Rows r = kv4_prefill_rows(a);
      d.q16 = r.q16;
      d.fac = r.fac;
      d.off = r.off;
    }
    const cudaError_t e = act == DIAL_ACT_BF16 ? launch<__nv_bfloat16>(d, s) : launch<__half>(d, s);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace dialb200
