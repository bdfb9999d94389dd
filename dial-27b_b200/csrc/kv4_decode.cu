// Attention of few queries over the 4-bit KV cache (single tokens, drafts).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(x_j - m),  x_j = log2(e) scale q.k_j
//
// HBM-bound: 144 bytes a slot and kv head against 512 FLOP a column.  What
// decides is the instructions a page takes, so its codes go from shared memory
// straight into MMA operand registers, in the order the page has them:
//   S^T = K Q^T  m16n8k16, A = 16 tokens x 16 dims.  Lane (g, c) holds row g's
//                dims 32c .. 32c + 31 (16 bytes); MMA step t takes 4 of them, and
//                the query operand is loaded in the same order of dims.
//   O^T = V^T P^T  A = 16 dims x 16 tokens.  Lane (g, c) holds scale group g of 4
//                tokens; nibbles of two tokens are interleaved before the
//                conversion, which then gives the operand's token pairs.
// e2m1 times e4m3 is exact in f16 (6 significant bits, 2^-10 .. 2688), so K and V
// enter the MMA as the values the cache stands for; queries enter as f16 after
// an exact power-of-two scale, P as f16 (2^-11 relative, for the rate of its MMA, and
// lifted by 2^7 so that a long tail of small ones counts), and scores, sums and
// accumulators are f32.  Columns are (query, head of the group) pairs, so the
// 8 columns of an MMA cost the same for 1 and for 8.
// The softmax reference m moves only when a score exceeds the one it was set by by more
// than 8 (base 2), found by one vote a page instead of a shuffle tree.
//
// Work split: the pages of all (sequence, kv head) segments laid end to end and
// cut into ranges of equal cost, one a CTA, so ragged lengths balance; the pages of a
// range go round its warps, each with its own ring of bulk copies that runs on
// across segment borders.  A segment inside one range is finished there; the
// others leave (m, l, O) parts that kv4_join_kernel adds in order.  With running
// weights the scores are kept in scratch (16 bytes a slot at 4 heads a group, a ninth
// of the page's) and the join turns them into probabilities once m and l are known, a
// slot a thread, no atomics.
//
// Measured, kernel and join by themselves with cold caches: 32 sessions of 128 to 8192
// slots (180 MB) 48 + 4 us, one of 131071 (151 MB) 38 + 6, 9 of 900 to 30001 with weights
// 46 + 16, five queries of 8 sessions of 700 to 4099 with weights 34 + 14, 201 slots 7.
// No unit is full: a page and column tile takes 320 instructions (16 MMAs, 64
// conversions and 64 packed products of the codes with what arranges them, the softmax
// of 128 scores), each waiting for one before it, and the 16 warps an SM that registers
// leave issue 2.45 of 4 a clock (ALU 52 %, DRAM 46 %, tensor pipe 21 %).
#include <cmath>
#include <type_traits>

#include "kv4_attn.h"
#include "kv4_dev.cuh"
#include "kv4_launch.h"

namespace dialb200 {
namespace {

// Warps a CTA: 16 warps an SM fit at up to 128 registers (one column tile) as two
// CTAs of 8, 12 at 164 (two tiles) as three of 4.
template <int NT>
constexpr int kWarpsOf = NT == 1 ? 8 : 4;
template <int NT>
constexpr int kPages = NT == 1 ? 2 : 1;  // pages of a ring slot, taken at once
template <int NT>
constexpr int kCtasPerSm = NT == 1 ? 2 : 3;
constexpr int kRing = 4;           // pages in flight a warp
constexpr int kSeqChunk = 256;     // sequences a launch
// A segment's own cost (its start, and the merge of its parts), in pages.  At 10 / 20 / 30
// / 45: 32 sessions of 128 to 8192 slots 50.1 / 48.1 / 47.9 / 49.3 us; 100 of 1200 to 2500
// 63.1 / 61.7 / 61.4 / 61.4, with weights 90.3 / 87.7 / 86.9 / 87.0; five queries of 8
// sessions with weights 44.8 / 42.7 / 43.0 / 45.1; four of 20 sessions of 1000 to 9000
// slots 56.0 / 54.7 / 55.3 / 56.5.
constexpr int kSegPad = 20;
constexpr int kInfo = 6;           // sequences of a range kept in shared memory
constexpr int kOneLen = 1024;      // slots up to which a CTA takes a whole segment
// Probabilities are taken against a reference kLift below the largest score, base 2:
// f16 keeps them to 2^-32 of the largest, and the f32 sums lose more over as many slots.
// The reference moves when one would exceed 2^kTop.
constexpr float kLift = 7.f, kTop = 15.f;
constexpr int kColStride = kHeadDim + 8;

// A range's share of a segment, for its weights.
struct Rec {
  int seg, seg0, page0, page1;  // segment, its first page, the share's pages in it
  int sid, h, len, cols;
};

struct DecodeArgs {
  Kv4AttnArgs a;
  int groups;       // column groups of NT * 8
  int ctas;         // ranges
  int one;          // every CTA takes one whole segment: ctas = segments, no join
  int pages_max;    // of a sequence
  int score_ld;     // floats a slot in `scores`
  int join_y;       // CTAs of the join that a segment's columns are dealt to
  // [ctas]: the segment that starts in a range and goes on (or -1), its first row
  // and columns; and of the segment that the range begins inside (if it does)
  // whether it ends there: 1 yes, 0 no, -1 the range begins with a segment
  int4* desc;
  int rec_ld;       // records a range can have
  int* rec_n;       // [ctas], with weights
  Rec* rec;         // [ctas][rec_ld]
  float* part_o;    // [ctas + segments][groups][NT * 8][128]
  float* part_ml;   // [ctas + segments][groups][NT * 8][2]
  float* scores;    // [pages of all segments][16][score_ld] or null
};

// cum[i]: pages of the sequences before i; the block's threads share the scan, and
// each keeps its sequences in `s`.
template <int THREADS>
__device__ __forceinline__ void page_prefix(const Kv4AttnArgs& a, int* cum, int* sums,
                                            Kv4Seq (&s)[kSeqChunk / THREADS]) {
  constexpr int PER = kSeqChunk / THREADS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, seqs = a.seqs;
  int v[PER], total = 0;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int i = tid * PER + e;
    v[e] = 0;
    if (i < seqs && kv4_seq(a, i, s[e]) && s[e].n > 0) v[e] = (s[e].len + kPageTokens - 1) / kPageTokens;
    total += v[e];
  }
  int run = total;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += u;
  }
  if (lane == 31) sums[warp] = run;
  __syncthreads();
  int before = run - total;
  for (int w = 0; w < warp; ++w) before += sums[w];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int i = tid * PER + e;
    if (i <= seqs) cum[i] = before;
    before += v[e];
  }
  if (tid == THREADS - 1 && seqs == kSeqChunk) cum[kSeqChunk] = before;
  __syncthreads();
}

// The sequence whose pages hold page `fp` of the prefix.
__device__ __forceinline__ int seq_at(const int* cum, int seqs, int fp) {
  int lo = 0, hi = seqs;  // cum[lo] <= fp < cum[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cum[mid] <= fp) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Ranges that `total` pages are cut into: no range is empty, and each warp of
// a CTA has a page where the pages do not go round all CTAs.
__device__ __forceinline__ int ranges_of(int total, int ctas, int warps) {
  return min(ctas, (total + warps - 1) / warps);
}
// First page (over all segments) of range b of `ctas`.  Ranges are equal in cost, a
// segment's own counted before its first page; a cut inside that falls on the page.
// Costs are below 2^31 (chunk_of).
__device__ __forceinline__ int range_start(const int* cum, int seqs, int H, int b, int ctas) {
  if (b >= ctas) return cum[seqs] * H;
  const unsigned all = H * (cum[seqs] + kSegPad * seqs);
  const int x = static_cast<int>(static_cast<double>(static_cast<unsigned long long>(all) * b) / ctas);
  int lo = 0, hi = seqs;  // cost before sequence lo <= x < cost before sequence hi
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (H * (cum[mid] + kSegPad * mid) <= x) lo = mid;
    else hi = mid;
  }
  const int np = cum[lo + 1] - cum[lo], r = x - H * (cum[lo] + kSegPad * lo), h = r / (np + kSegPad);
  return cum[lo] * H + h * np + max(0, r - h * (np + kSegPad) - kSegPad);
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Token of the page in row r of the K operand (and of the probabilities): the
// row order in which a lane's 4 V tokens lie in both halves of a bank line.
__device__ __forceinline__ int row_token(int r) { return r ^ ((r >> 1) & 1); }

// Dim at place p of a part's row: the order in which the accumulators' lanes
// reach shared memory without bank conflicts, kept up to the output.
__device__ __forceinline__ int place_dim(int p) { return (p >> 1 & 7) * 16 + (p >> 4) * 2 + (p & 1); }

// D = A B + C with the accumulator's first use: C zero.
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                             uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src),
               "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

template <int NT>
struct DecodeSmem {
  static constexpr int kWarps = kWarpsOf<NT>, kSlots = kRing / kPages<NT>;
  uint8_t ring[kWarps][kRing][kKv4Slab];
  float o[kWarps][8][kColStride];
  uint8_t q[2][NT * 8][kHeadDim * 2];  // this segment's queries and the next one's
  float ml[kWarps][8][2];
  float2 fin[NT * 8];  // (m, 1 / l) of the only segment
  uint64_t full[kWarps][kSlots];
  uint64_t merged;  // every warp has read the parts in o and ml
  Kv4Seq info[kInfo];  // the range's first sequences
  int cum[kSeqChunk + 1];
  int sums[kWarps];
};

// The probabilities of slots t, t + step .. below `upto` of segment (sid, h) into
// their running weights: scores x [slot][score_ld], the columns' (m, 1 / l) in ml.
// B slots at once, whose loads all precede the stores.
template <int B>
__device__ __forceinline__ void add_weights(const DecodeArgs& d, int sid, int h, int t, int step, int upto,
                                            const float* x, const float2* ml, int cols) {
  const Kv4AttnArgs& a = d.a;
  for (; t < upto; t += B * step) {
    int block[B];
    float* to[B];
    float old[B], sum[B];
#pragma unroll
    for (int e = 0; e < B; ++e) {
      const int at = t + e * step;
      block[e] = at < upto ? kv4_block(a.c, a.c.block_table, sid, at / kPageTokens) : -1;
    }
#pragma unroll
    for (int e = 0; e < B; ++e) {
      const int at = t + e * step;
      to[e] = a.c.weights + kv4_slab_index(a.c, max(block[e], 0), h) * kPageTokens + at % kPageTokens;
      old[e] = block[e] >= 0 ? *to[e] : 0.f;
      sum[e] = 0.f;
    }
    int col = 0;
    if ((d.score_ld & 3) == 0)
      for (; col + 4 <= cols; col += 4) {
        float4 v[B];
#pragma unroll
        for (int e = 0; e < B; ++e)
          v[e] = *reinterpret_cast<const float4*>(x + static_cast<size_t>(min(t + e * step, upto - 1)) * d.score_ld + col);
#pragma unroll
        for (int e = 0; e < B; ++e) {
          sum[e] = fmaf(ex2(v[e].x - ml[col].x), ml[col].y, sum[e]);
          sum[e] = fmaf(ex2(v[e].y - ml[col + 1].x), ml[col + 1].y, sum[e]);
          sum[e] = fmaf(ex2(v[e].z - ml[col + 2].x), ml[col + 2].y, sum[e]);
          sum[e] = fmaf(ex2(v[e].w - ml[col + 3].x), ml[col + 3].y, sum[e]);
        }
      }
    for (; col < cols; ++col)
#pragma unroll
      for (int e = 0; e < B; ++e)
        sum[e] = fmaf(ex2(x[static_cast<size_t>(min(t + e * step, upto - 1)) * d.score_ld + col] - ml[col].x),
                      ml[col].y, sum[e]);
#pragma unroll
    for (int e = 0; e < B; ++e)
      if (block[e] >= 0) *to[e] = old[e] + sum[e];
  }
}

// One segment's share of a range.
struct Share {
  Kv4Seq s;
  int h, seg, seg0, seg1, end;  // kv head, number, first and last page, end of the share
};

template <typename Act>
__device__ __forceinline__ void zero_rows(const Kv4AttnArgs& a, const Kv4Seq& s, int tid, int threads) {
  for (int r = 0; r < s.n; ++r)
    for (int e = tid * 8; e < a.c.q_heads * kHeadDim; e += threads * 8)
      *reinterpret_cast<uint4*>(static_cast<Act*>(a.out) + (s.row0 + r) * a.out_ld + e) = make_uint4(0, 0, 0, 0);
}

template <typename Act, int NT, bool SCORES>
__global__ void __launch_bounds__(kWarpsOf<NT> * 32, kCtasPerSm<NT>)
    kv4_decode_kernel(const DecodeArgs d) {
  constexpr int kWarps = kWarpsOf<NT>, U = kPages<NT>, kSlots = kRing / U;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  DecodeSmem<NT>& sm = *reinterpret_cast<DecodeSmem<NT>*>(smem_raw);
  const Kv4AttnArgs& a = d.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  const int H = a.c.kv_heads, rep = a.c.q_heads / H;
  const int b = blockIdx.x, col0 = blockIdx.y * NT * 8;
  pdl_wait();
  pdl_launch_dependents();
  if (lane == 0) {
    for (int i = 0; i < kSlots; ++i) mbar_init(&sm.full[warp][i], 1);
    if (warp == 0) mbar_init(&sm.merged, kWarps);
    fence_mbar_init();
  }
  // sequences of this CTA's work: all of the call, or one
  const int si0 = d.one ? b / H : 0, seqs = d.one ? 1 : a.seqs, b_of = d.one ? b - si0 * H : b;
  Kv4Seq own[kSeqChunk / (kWarps * 32)];
  int f0, f1, first_seq = 0;
  if (d.one) {
    const bool good = kv4_seq(a, si0, own[0]);
    const int np = good && own[0].n > 0 ? (own[0].len + kPageTokens - 1) / kPageTokens : 0;
    if (tid == 0) {
      sm.cum[0] = 0;
      sm.cum[1] = np;
      sm.info[0] = own[0];
    }
    f0 = b_of * np;
    f1 = f0 + np;
    if (good && np == 0 && b_of == 0 && blockIdx.y == 0) zero_rows<Act>(a, own[0], tid, kWarps * 32);
  } else {
    page_prefix<kWarps * 32>(a, sm.cum, sm.sums, own);
    const int ctas = ranges_of(sm.cum[seqs] * H, d.ctas, kWarps);
    f0 = range_start(sm.cum, seqs, H, min(b, ctas), ctas);
    f1 = range_start(sm.cum, seqs, H, min(b + 1, ctas), ctas);
    first_seq = f0 < f1 ? seq_at(sm.cum, seqs, f0 / H) : 0;
#pragma unroll
    for (int e = 0; e < kSeqChunk / (kWarps * 32); ++e) {
      const int i = tid * (kSeqChunk / (kWarps * 32)) + e;
      if (i >= first_seq && i < min(seqs, first_seq + kInfo)) sm.info[i - first_seq] = own[e];
    }
    // sequences without a slot: zeros
    for (int i = b; i < seqs; i += d.ctas) {
      Kv4Seq s;
      if (sm.cum[i + 1] == sm.cum[i] && blockIdx.y == 0 && kv4_seq(a, i, s)) zero_rows<Act>(a, s, tid, kWarps * 32);
    }
    if (f0 == f1 && tid == 0 && blockIdx.y == 0) {
      d.desc[b] = make_int4(-1, 0, 0, -1);
      if (SCORES) d.rec_n[b] = 0;
    }
  }
  if (f0 == f1) return;
  __syncthreads();
  auto seq_info = [&](int i, Kv4Seq& s) {
    if (i - first_seq < kInfo) s = sm.info[i - first_seq];
    else kv4_seq(a, i, s);
  };

  // this warp's pages: f0 + warp + kWarps * i, i < mine; each lane holds the slab
  // number of one page of a window of 32 and copies that page itself; the next
  // window's table loads go out a window ahead
  const int mine = f1 - f0 > warp ? (f1 - f0 - warp + kWarps - 1) / kWarps : 0;
  // table entry of the warp's page i (past its last: of a page of the range), and its kv head
  auto entry_of = [&](int i, int& h) -> const int32_t* {
    const int f = min(f0 + warp + kWarps * min(i, max(mine - 1, 0)), f1 - 1);
    const int s = seq_at(sm.cum, seqs, f / H);
    const int np = sm.cum[s + 1] - sm.cum[s], r = f - sm.cum[s] * H;
    Kv4Seq q;
    seq_info(s, q);
    h = r / np;
    return a.c.block_table + static_cast<size_t>(q.sid) * a.c.max_blocks + (r - h * np);
  };
  auto slab_of = [&](int block, int h) -> int {
    if (static_cast<unsigned>(block) >= static_cast<unsigned>(a.c.num_blocks)) {
      set_status(a.c.status, kStatusBadArgs);
      block = 0;
    }
    return block * H + h;
  };
  int win = 0, block_next = 0, head_next = 0, issued = 0;
  auto issue = [&]() {  // the next U pages into their slot; warp-uniform
    if (issued > 0 && (issued & 31) == 0) {
      win = slab_of(block_next, head_next);
      block_next = *entry_of(issued + 32 + lane, head_next);
    }
    const int n = min(U, mine - issued), at = lane - (issued & 31);
    uint64_t* bar = &sm.full[warp][issued / U % kSlots];
    if (at == 0) mbar_arrive_expect_tx(bar, n * kKv4Slab);
    if (at >= 0 && at < n)
      bulk_g2s(sm.ring[warp][(issued + at) % kRing],
               a.c.pages + static_cast<size_t>(static_cast<unsigned>(win)) * kKv4Slab, kKv4Slab, bar);
    issued += n;
  };
  auto share_at = [&](int f) {
    Share w;
    const int si = seq_at(sm.cum, seqs, f / H);
    const int np = sm.cum[si + 1] - sm.cum[si], base = sm.cum[si] * H;
    w.h = (f - base) / np;
    w.seg = si * H + w.h;
    w.seg0 = base + w.h * np;
    w.seg1 = w.seg0 + np;
    w.end = min(f1, w.seg1);
    seq_info(si, w.s);
    return w;
  };
  auto load_q = [&](const Share& w, int buf) {
    for (int e = tid; e < NT * 8 * 16; e += kWarps * 32) {
      const int cl = e >> 4, col = col0 + cl, there = col < w.s.n * rep;
      const int cc = there ? col : 0;
      cp_async16(sm.q[buf][cl] + (e & 15) * 16,
                 static_cast<const Act*>(a.q) + (w.s.row0 + cc / rep) * a.q_ld +
                     (w.h * rep + cc % rep) * kHeadDim + (e & 15) * 8,
                 there);
    }
  };

  // scores of the sequences before this CTA's (one segment a CTA)
  const size_t score0 = static_cast<size_t>(si0) * H * d.pages_max * kPageTokens;
  int done = 0, buf = 0;
  uint32_t shares = 0;
  bool ok = true;
  Share w = share_at(f0);
  load_q(w, 0);
  {
    int h;
    const int32_t *e0 = entry_of(lane, h), *e1 = entry_of(32 + lane, head_next);
    const int block = *e0;
    block_next = *e1;
    win = slab_of(block, h);
  }
  while (issued < kRing && issued < mine) issue();
  cp_async_wait();
  __syncthreads();
  // the segment that the range begins inside: ends in it (1) or not (0)
  const int first_ends = f0 == w.seg0 ? -1 : w.seg1 <= f1;
  int recs = 0;
  for (int fc = f0;; buf ^= 1, ++shares) {
    // ------------------------------------------------ one segment's share
    const int fe = w.end, cols = w.s.n * rep;
    Share next = w;
    if (fe < f1) {
      next = share_at(fe);
      load_q(next, buf ^ 1);
    }
    uint32_t qf[NT][16];
    float fac[NT][2], m[NT][2], ref[NT][2], high[NT][2], l[NT][2], o[NT][8][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint4* src = reinterpret_cast<const uint4*>(sm.q[buf][nt * 8 + g] + 64 * c);
      float qv[32], top = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint4 raw = src[e];
        const Act* v = reinterpret_cast<const Act*>(&raw);
#pragma unroll
        for (int u = 0; u < 8; ++u) qv[8 * e + u] = ActTraits<Act>::to_f(v[u]);
      }
#pragma unroll
      for (int e = 0; e < 32; ++e) top = fmaxf(top, fabsf(qv[e]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int ex = query_exp(top);
      const float down = exp2i(-ex);
#pragma unroll
      for (int e = 0; e < 16; ++e) qf[nt][e] = pack_f16(qv[2 * e] * down, qv[2 * e + 1] * down);
      const float mine_f = score_scale(a, ex);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        fac[nt][e] = __shfl_sync(0xffffffffu, mine_f, (2 * c + e) * 4);
        m[nt][e] = high[nt][e] = -INFINITY;
        ref[nt][e] = l[nt][e] = 0.f;
      }
#pragma unroll
      for (int mt = 0; mt < 8; ++mt)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][mt][e] = 0.f;
    }
    // ------------------------------------------------------------- pages
    const int t0 = row_token(g), ta = row_token(2 * c), tb = row_token(2 * c + 1);
    const int open_end = w.s.len - w.s.n + 1;  // slots every query sees
    // N pages from `done` on, all of one slot: their score chains and
    // exponentials overlap, and one vote does for all
    auto step = [&](auto count) {
      constexpr int N = decltype(count)::value;
      const int page0 = f0 + warp + kWarps * done - w.seg0;
      const uint8_t* pg0 = sm.ring[warp][done % kRing];
      // after a wait that ran out (status recorded) the rest is computed on
      // whatever the slots hold, without more waiting
      if (ok)
        ok = mbar_wait(&sm.full[warp][done / U % kSlots], static_cast<uint32_t>(done / kRing) & 1u,
                       a.c.status, kStatusAttnRing);
      __syncwarp();
      float x[N][NT][4];
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const uint8_t* pg = pg0 + u * kKv4Slab;
        const uint4 k0 = *reinterpret_cast<const uint4*>(pg + t0 * 64 + c * 16);
        const uint4 k1 = *reinterpret_cast<const uint4*>(pg + t0 * 64 + 512 + c * 16);
        const uint32_t s0 = e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t*>(pg + kKv4KScales + t0 * 8 + c * 2));
        const uint32_t s1 = e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t*>(pg + kKv4KScales + t0 * 8 + 64 + c * 2));
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t sc0 = __byte_perm(s0, 0, i < 2 ? 0x1010 : 0x3232);
          const uint32_t sc1 = __byte_perm(s1, 0, i < 2 ? 0x1010 : 0x3232);
          uint32_t r0[4], r1[4];
          e2m1x8_to_f16x2x4(w0[i], r0);
          e2m1x8_to_f16x2x4(w1[i], r1);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const uint32_t af[4] = {hmul2(r0[2 * hf], sc0), hmul2(r1[2 * hf], sc1),
                                    hmul2(r0[2 * hf + 1], sc0), hmul2(r1[2 * hf + 1], sc1)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (i == 0 && hf == 0) mma_f16_zero(x[u][nt], af, qf[nt][0], qf[nt][1]);
              else mma_f16(x[u][nt], af, qf[nt][4 * i + 2 * hf], qf[nt][4 * i + 2 * hf + 1]);
            }
          }
        }
      }
      // scores, rounded: the same in the reference and here, so that the largest one's
      // difference is right however large they are (an fma would keep the rounding of the
      // reference, 2^-24 of it, in the exponent)
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[u][nt][e] = __fmul_rn(x[u][nt][e], fac[nt][e & 1]);
      uint32_t there[N][2];  // V scales to keep: slots past the end may hold anything
#pragma unroll
      for (int u = 0; u < N; ++u) there[u][0] = there[u][1] = 0xFFFFFFFFu;
      if ((page0 + kWarps * (N - 1) + 1) * kPageTokens > open_end) {  // causal border or the end
#pragma unroll
        for (int u = 0; u < N; ++u) {
          const int left = w.s.len - (page0 + kWarps * u) * kPageTokens;
          there[u][0] = (ta < left ? 0xFFFFu : 0u) | (tb < left ? 0xFFFF0000u : 0u);
          there[u][1] = (ta + 8 < left ? 0xFFFFu : 0u) | (tb + 8 < left ? 0xFFFF0000u : 0u);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int cc = col0 + nt * 8 + 2 * c + e;
            const int seen = cc < cols ? open_end + cc / rep : 0;
#pragma unroll
            for (int u = 0; u < N; ++u) {
              const int t = (page0 + kWarps * u) * kPageTokens + t0;
              if (t >= seen) x[u][nt][e] = -INFINITY;
              if (t + 8 >= seen) x[u][nt][e + 2] = -INFINITY;
            }
          }
      }
      if constexpr (SCORES) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int cc = col0 + nt * 8 + 2 * c;
          if (cc < cols)
#pragma unroll
            for (int u = 0; u < N; ++u) {
              float* to = d.scores + (score0 + static_cast<size_t>(w.seg0 + page0 + kWarps * u) * kPageTokens + t0) * d.score_ld + cc;
              *reinterpret_cast<float2*>(to) = make_float2(x[u][nt][0], x[u][nt][1]);
              *reinterpret_cast<float2*>(to + 8 * d.score_ld) = make_float2(x[u][nt][2], x[u][nt][3]);
            }
        }
      }
      // m is the reference, `high` m + kTop
      float top[NT][2];
      bool raise = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          top[nt][e] = fmaxf(x[0][nt][e], x[0][nt][e + 2]);
#pragma unroll
          for (int u = 1; u < N; ++u) top[nt][e] = fmaxf(top[nt][e], fmaxf(x[u][nt][e], x[u][nt][e + 2]));
          raise |= top[nt][e] > high[nt][e];
        }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float t = top[nt][e];
#pragma unroll
            for (int i = 4; i < 32; i <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, i));
            const float mn = fmaxf(m[nt][e], t - kLift);
            const float al = m[nt][e] == -INFINITY ? 0.f : ex2(m[nt][e] - mn);
            m[nt][e] = mn;
            ref[nt][e] = mn == -INFINITY ? 0.f : mn;
            high[nt][e] = __fadd_rd(mn, kTop);
            l[nt][e] *= al;
#pragma unroll
            for (int mt = 0; mt < 8; ++mt) {
              o[nt][mt][e] *= al;
              o[nt][mt][e + 2] *= al;
            }
          }
      }
      uint32_t pf[N][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int u = 0; u < N; ++u) {
          const float p0 = ex2(x[u][nt][0] - ref[nt][0]);
          const float p1 = ex2(x[u][nt][1] - ref[nt][1]);
          const float p2 = ex2(x[u][nt][2] - ref[nt][0]);
          const float p3 = ex2(x[u][nt][3] - ref[nt][1]);
          l[nt][0] += p0 + p2;
          l[nt][1] += p1 + p3;
          pf[u][nt][0] = transpose8(pack_f16(p0, p1));
          pf[u][nt][1] = transpose8(pack_f16(p2, p3));
        }
      // V: rows 2c, 2c + 1 and 2c + 8, 2c + 9 of the page, scale group g
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const uint8_t* vp = pg0 + u * kKv4Slab + kKv4VCodes + g * 8;
        const uint2 va = *reinterpret_cast<const uint2*>(vp + ta * 64);
        const uint2 vb = *reinterpret_cast<const uint2*>(vp + tb * 64);
        const uint2 vc = *reinterpret_cast<const uint2*>(vp + ta * 64 + 512);
        const uint2 vd = *reinterpret_cast<const uint2*>(vp + tb * 64 + 512);
        const uint8_t* sp = pg0 + u * kKv4Slab + kKv4VScales + g;
        const uint32_t sab = e4m3x2_to_f16x2(static_cast<uint16_t>(sp[ta * 8] | sp[tb * 8] << 8)) & there[u][0];
        const uint32_t scd = e4m3x2_to_f16x2(static_cast<uint16_t>(sp[ta * 8 + 64] | sp[tb * 8 + 64] << 8)) & there[u][1];
        constexpr uint32_t kLow = 0x0F0F0F0Fu;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t A = i ? va.y : va.x, B = i ? vb.y : vb.x, C = i ? vc.y : vc.x, D = i ? vd.y : vd.x;
          uint32_t lo0[4], hi0[4], lo1[4], hi1[4];
          e2m1x8_to_f16x2x4((A & kLow) | ((B << 4) & ~kLow), lo0);
          e2m1x8_to_f16x2x4(((A >> 4) & kLow) | (B & ~kLow), hi0);
          e2m1x8_to_f16x2x4((C & kLow) | ((D << 4) & ~kLow), lo1);
          e2m1x8_to_f16x2x4(((C >> 4) & kLow) | (D & ~kLow), hi1);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t af[4] = {hmul2(lo0[e], sab), hmul2(hi0[e], sab), hmul2(lo1[e], scd),
                                    hmul2(hi1[e], scd)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][4 * i + e], af, pf[u][nt][0], pf[u][nt][1]);
          }
        }
      }
      done += N;
      if (done % U == 0 && issued < mine) {
        // the slot's reads before the copies that refill it
        fence_proxy_async_smem();
        __syncwarp();
        issue();
      }
    };
    const int upto = fe - f0 > warp ? (fe - f0 - warp + kWarps - 1) / kWarps : 0;  // of `mine`
    while (done < upto) {
      if (U == 2 && done % 2 == 0 && done + 1 < upto) step(std::integral_constant<int, U>{});
      else step(std::integral_constant<int, 1>{});
    }
    // ------------------------------------- the warps' parts of the segment
    const bool whole = fc == w.seg0 && fe == w.seg1;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // the parts before these have been read (the first wait passes at once)
      const uint32_t turn = shares * NT + nt;
      mbar_wait(&sm.merged, (turn & 1u) ^ 1u, a.c.status, kStatusAttnRing);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[nt][e];
#pragma unroll
        for (int i = 4; i < 32; i <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
        if (g == 0) {
          sm.ml[warp][2 * c + e][0] = m[nt][e];
          sm.ml[warp][2 * c + e][1] = sum;
        }
#pragma unroll
        for (int mt = 0; mt < 8; ++mt)
          *reinterpret_cast<float2*>(&sm.o[warp][2 * c + e][16 * mt + 2 * g]) =
              make_float2(o[nt][mt][e], o[nt][mt][e + 2]);
      }
      cp_async_wait();  // the next segment's queries, for the barrier to publish
      __syncthreads();
      const size_t part = (static_cast<size_t>(b + w.seg) * d.groups + blockIdx.y) * NT * 8 + nt * 8;
      const int at = tid % kHeadDim, dim = place_dim(at);
      for (int cl = tid / kHeadDim; cl < 8; cl += kWarps * 32 / kHeadDim) {
        const int col = col0 + nt * 8 + cl;
        if (col >= cols) break;
        float M = -INFINITY, L = 0.f, O = 0.f;
#pragma unroll
        for (int i = 0; i < kWarps; ++i) M = fmaxf(M, sm.ml[i][cl][0]);
#pragma unroll
        for (int i = 0; i < kWarps; ++i) {
          const float mw = sm.ml[i][cl][0];
          const float f = mw == -INFINITY ? 0.f : ex2(mw - M);
          L = fmaf(f, sm.ml[i][cl][1], L);
          O = fmaf(f, sm.o[i][cl][at], O);
        }
        if (whole)
          static_cast<Act*>(a.out)[(w.s.row0 + col / rep) * a.out_ld + (w.h * rep + col % rep) * kHeadDim + dim] =
              ActTraits<Act>::from_f(L != 0.f ? O / L * a.c.v_scale : 0.f);
        else
          d.part_o[(part + cl) * kHeadDim + at] = O;
        if (SCORES && at == 0 && d.one)
          sm.fin[nt * 8 + cl] = make_float2(M == -INFINITY ? 0.f : M, L > 0.f ? 1.f / L : 0.f);
        else if ((!whole || SCORES) && at == 0)
          *reinterpret_cast<float2*>(d.part_ml + (part + cl) * 2) = make_float2(M, L);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.merged);
    }
    if (SCORES && d.one) {  // this CTA's scores, all of the segment's columns
      __syncthreads();
      add_weights<2>(d, w.s.sid, w.h, tid, kWarps * 32, w.s.len,
                     d.scores + (score0 + static_cast<size_t>(w.seg0) * kPageTokens) * d.score_ld, sm.fin, cols);
      break;
    }
    if (d.one) break;
    if (tid == 0 && blockIdx.y == 0) {
      if (SCORES && recs < d.rec_ld)
        d.rec[static_cast<size_t>(b) * d.rec_ld + recs] =
            Rec{w.seg, w.seg0, fc - w.seg0, fe - w.seg0, w.s.sid, w.h, w.s.len, cols};
      if (SCORES && recs >= d.rec_ld) set_status(a.c.status, kStatusBadArgs);
      if (fe == f1) {
        // the only segment of the range that can start in it and go on
        d.desc[b] = make_int4(fc == w.seg0 && fe < w.seg1 ? w.seg : -1, w.s.row0, cols, first_ends);
        if (SCORES) d.rec_n[b] = min(recs + 1, d.rec_ld);
      }
    }
    ++recs;
    if (fe == f1) break;
    fc = fe;
    w = next;
  }
  if (!ok)  // a copy did not land in time: wait (bounded) for each slot's last one
    for (int i = 0, n = (mine + U - 1) / U; i < kSlots && i < n; ++i)
      mbar_wait(&sm.full[warp][i], static_cast<uint32_t>((n - 1 - i) / kSlots) & 1u, a.c.status,
                kStatusAttnRing);
}

constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32;
constexpr int kWeightCtas = 4;  // of a range, scheduled first: 17 us against 20 when last
// Parts of a segment up to which a warp joins a column by itself (more: a CTA).  Five
// queries of 8 sessions, 4 parts a segment: the join takes 14 us against 21.
constexpr int kFewParts = 16;

// max over a segment's parts of a column, and the sum l under it; G lanes share them.
template <int G>
__device__ __forceinline__ float2 join_ml(const float2* ml, size_t stride, int parts) {
  const int lane = threadIdx.x % G;
  float2 own = lane < parts ? ml[lane * stride] : make_float2(-INFINITY, 0.f);
  float M = own.x;
  for (int p = lane + G; p < parts; p += G) M = fmaxf(M, ml[p * stride].x);
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  float L = own.x == -INFINITY ? 0.f : ex2(own.x - M) * own.y;
  for (int p = lane + G; p < parts; p += G) {
    const float2 v = ml[p * stride];
    if (v.x != -INFINITY) L = fmaf(ex2(v.x - M), v.y, L);
  }
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  return make_float2(M, L);
}

// (m, 1 / l) of a segment's columns, G lanes a column.
template <int G>
__device__ __forceinline__ void column_ml(const float2* first, size_t stride, int parts, int cols, float2* ml) {
  for (int c0 = threadIdx.x / 32 * (32 / G); c0 < cols; c0 += kJoinThreads / G) {  // warp-uniform
    const int col = c0 + threadIdx.x % 32 / G;
    const float2 v = join_ml<G>(first + min(col, cols - 1), stride, parts);
    if (threadIdx.x % G == 0 && col < cols)
      ml[col] = make_float2(v.x == -INFINITY ? 0.f : v.x, v.y > 0.f ? 1.f / v.y : 0.f);
  }
}

// Ranges after b that go on with the segment that b begins or continues and does not
// end; `ends`: whether it ends in range b + 1 + lane.
__device__ __forceinline__ int parts_after(const DecodeArgs& d, int b, bool ends) {
  const int lane = threadIdx.x & 31;
  for (int n = 0;; n += 32) {
    if (n > 0) ends = b + 1 + n + lane >= d.ctas || d.desc[b + 1 + n + lane].w != 0;
    const unsigned any = __ballot_sync(0xffffffffu, ends);
    if (any) return n + __ffs(any);
  }
}
// The range before b in which segment `seg` starts; `starts`: the segment that starts
// in range b - 1 - lane and goes on.
__device__ __forceinline__ int owner_before(const DecodeArgs& d, int b, int seg, int starts) {
  const int lane = threadIdx.x & 31;
  for (int n = b - 1;; n -= 32) {
    const int at = n - lane;
    if (n < b - 1) starts = at < 0 ? seg : d.desc[at].x;
    const unsigned hit = __ballot_sync(0xffffffffu, starts == seg || at < 0);
    if (hit) return max(n - (__ffs(hit) - 1), 0);
  }
}

// With weights, blockIdx.y < kWeightCtas: adds the probabilities of the slots of
// range blockIdx.x to the running weights.  The other blockIdx.y: joins the parts
// of the segment that starts in the range and goes on in others, a column a CTA,
// parts over the warps.
template <typename Act, int NT>
__global__ void __launch_bounds__(kJoinThreads, 4) kv4_join_kernel(const DecodeArgs d) {
  const Kv4AttnArgs& a = d.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.x;
  const int H = a.c.kv_heads, rep = a.c.q_heads / H;
  const size_t stride = static_cast<size_t>(d.groups) * NT * 8;  // columns of a part
  pdl_wait();
  // what range b and its neighbours hold, loaded at once
  const int4 ds = d.desc[b];
  const bool ends = b + 1 + lane >= d.ctas || d.desc[b + 1 + lane].w != 0;
  const int ys = d.scores ? kWeightCtas : 0;
  if (blockIdx.y >= ys) {
    __shared__ float4 red[kJoinWarps][kHeadDim / 4];
    if (ds.x < 0) return;
    const int parts = 1 + parts_after(d, b, ends);
    // few parts: a column a warp; else a column a CTA, its parts over the warps
    const bool few = parts <= kFewParts;
    const int y = blockIdx.y - ys, gy = gridDim.y - ys, W = few ? 1 : kJoinWarps, part0 = few ? 0 : warp;
    for (int col = few ? y * kJoinWarps + warp : y; col < ds.z; col += few ? gy * kJoinWarps : gy) {
      const size_t first = static_cast<size_t>(b + ds.x) * stride + col;
      const float4* po = reinterpret_cast<const float4*>(d.part_o) + first * (kHeadDim / 4) + lane;
      const float2* ml = reinterpret_cast<const float2*>(d.part_ml) + first;
      constexpr int PRE = 4;  // parts a warp loads before the maximum is known
      float4 pre[PRE];
      float pm[PRE];
#pragma unroll
      for (int e = 0; e < PRE; ++e) {
        const int p = part0 + W * e;
        pre[e] = p < parts ? po[p * stride * (kHeadDim / 4)] : make_float4(0.f, 0.f, 0.f, 0.f);
        pm[e] = p < parts ? ml[p * stride].x : -INFINITY;
      }
      const float2 all = join_ml<32>(ml, stride, parts);
      float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
      auto add = [&](const float4& v, float mp) {
        const float f = mp == -INFINITY ? 0.f : ex2(mp - all.x);
        O.x = fmaf(f, v.x, O.x);
        O.y = fmaf(f, v.y, O.y);
        O.z = fmaf(f, v.z, O.z);
        O.w = fmaf(f, v.w, O.w);
      };
#pragma unroll
      for (int e = 0; e < PRE; ++e) add(pre[e], pm[e]);
#pragma unroll 4
      for (int p = part0 + W * PRE; p < parts; p += W)
        add(po[p * stride * (kHeadDim / 4)], ml[p * stride].x);
      Act* out = static_cast<Act*>(a.out) + (ds.y + col / rep) * a.out_ld + ((ds.x % H) * rep + col % rep) * kHeadDim;
      const float scale = all.y != 0.f ? a.c.v_scale / all.y : 0.f;
      if (few) {
        const float v[4] = {O.x, O.y, O.z, O.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) out[place_dim(lane * 4 + e)] = ActTraits<Act>::from_f(v[e] * scale);
        continue;
      }
      red[warp][lane] = O;
      __syncthreads();
      if (tid < kHeadDim) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) v += reinterpret_cast<const float*>(red[w])[tid];
        out[place_dim(tid)] = ActTraits<Act>::from_f(v * scale);
      }
      __syncthreads();
    }
    return;
  }
  __shared__ float2 ml[kKv4FewCols];  // (m, 1 / l) of the segment's columns
  const Rec* recs = d.rec + static_cast<size_t>(b) * d.rec_ld;
  const int n = d.rec_n[b];
  const int starts = b - 1 - lane >= 0 ? d.desc[b - 1 - lane].x : -1;
  Rec r = recs[0];
  for (int k = 0; k < n; ++k) {
    // ranges that hold parts of the segment: from the one it starts in, b0, on
    const int b0 = r.page0 == 0 ? b : owner_before(d, b, r.seg, starts);
    const bool here = k + 1 < n || (r.page0 == 0 ? ds.x != r.seg : ds.w != 0);  // it ends in this range
    const int parts = b - b0 + 1 + (here ? 0 : parts_after(d, b, ends));
    const float2* first = reinterpret_cast<const float2*>(d.part_ml) + static_cast<size_t>(b0 + r.seg) * stride;
    if (parts <= kFewParts) column_ml<8>(first, stride, parts, r.cols, ml);
    else column_ml<32>(first, stride, parts, r.cols, ml);
    __syncthreads();
    add_weights<4>(d, r.sid, r.h, r.page0 * kPageTokens + blockIdx.y * kJoinThreads + tid, kWeightCtas * kJoinThreads,
                   min(r.page1 * kPageTokens, r.len),
                   d.scores + static_cast<size_t>(r.seg0) * kPageTokens * d.score_ld, ml, r.cols);
    if (k + 1 < n) r = recs[k + 1];
    __syncthreads();
  }
}

int sm_count() {
  static int n = [] {
    int v = 0, dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v < 1)
      v = 148;
    return v;
  }();
  return n;
}

// Sizes of one launch over `seqs` sequences.
struct Plan {
  int nt, groups, ctas, cols, score_ld, pages_max;
  bool one;
  long long pages;  // pages of all segments at most
  int rec_ld;
  size_t desc, rec, part_o, part_ml, scores;
};

Plan plan_of(int q_heads, int kv_heads, long long seqs, long long max_q, long long max_len,
             bool weights, int sms) {
  Plan p{};
  const int rep = q_heads / kv_heads;
  p.cols = static_cast<int>(max_q * rep);
  p.nt = p.cols <= 8 ? 1 : 2;
  p.groups = (p.cols + p.nt * 8 - 1) / (p.nt * 8);
  const long long per = (max_len + kPageTokens - 1) / kPageTokens;
  p.pages = seqs * per * kv_heads;
  // a page a warp at least, as many CTAs as are resident at once at most
  p.pages_max = static_cast<int>(per);
  // Short sequences: a CTA for each segment, which nothing has to join; without the
  // second launch, the prefix and the parts.  A CTA a segment / ranges, 32 heads of 8:
  // one session of 256 slots 5.4 / 7.5 us, of 1024 9.1 / 9.3; 32 sessions of 256 7.7 /
  // 15.1, of 1024 13.6 / 20.7; 128 of 1024 44.7 / 52.3.  The weights of several column
  // groups need the join.
  p.one = max_len <= kOneLen && !(weights && p.groups > 1);
  const int warps = p.nt == 1 ? kWarpsOf<1> : kWarpsOf<2>;
  const long long want = (p.pages + warps - 1) / warps;
  const long long most = static_cast<long long>(sms) * (p.nt == 1 ? kCtasPerSm<1> : kCtasPerSm<2>) / p.groups;
  p.ctas = static_cast<int>(want < 1 ? 1 : want < most ? want : most);
  if (p.one) p.ctas = static_cast<int>(seqs * kv_heads);
  p.score_ld = (p.cols + 1) & ~1;
  auto up = [](size_t v) { return (v + 127) & ~static_cast<size_t>(127); };
  const size_t rows = p.one ? 0 : static_cast<size_t>(p.ctas + seqs * kv_heads) * p.groups * p.nt * 8;
  p.desc = p.one ? 0 : up(static_cast<size_t>(p.ctas) * sizeof(int4));
  p.part_o = up(rows * kHeadDim * 4);
  p.part_ml = up(rows * 8);
  // a share costs kSegPad pages at least, and a segment has one in a range; with
  // k < ctas ranges (few pages: 8 k at most) a range has 8 k shares at most
  const long long segs = seqs * kv_heads;
  long long shares = (p.pages + kSegPad * segs) / (static_cast<long long>(p.ctas) * kSegPad) + 8;
  shares += static_cast<long long>(sqrt(8. * static_cast<double>(segs))) + 1;
  p.rec_ld = static_cast<int>(shares < segs ? shares : segs);
  p.rec = weights && !p.one ? up(static_cast<size_t>(p.ctas) * (4 + static_cast<size_t>(p.rec_ld) * sizeof(Rec)) + 128) : 0;
  p.scores = weights ? up(static_cast<size_t>(p.pages) * kPageTokens * p.score_ld * 4) : 0;
  return p;
}

// Sequences a launch takes: the prefix in shared memory holds kSeqChunk, and
// page numbers are 32-bit.
long long chunk_of(int kv_heads, long long seqs, long long max_len) {
  const long long per = ((max_len + kPageTokens - 1) / kPageTokens + kSegPad) * kv_heads;
  long long n = INT32_MAX / per;
  n = n < kSeqChunk ? n : kSeqChunk;
  return n < seqs ? n : seqs;
}

template <typename Act, int NT>
cudaError_t launch_nt(const DecodeArgs& d, cudaStream_t s) {
  const size_t smem = sizeof(DecodeSmem<NT>);
  cudaError_t e;
  if (d.scores) {
    e = kv4_allow_smem<kv4_decode_kernel<Act, NT, true>>(smem);
    if (e == cudaSuccess)
      e = kv4_start(kv4_decode_kernel<Act, NT, true>, dim3(d.ctas, d.groups), kWarpsOf<NT> * 32, smem, s, d);
  } else {
    e = kv4_allow_smem<kv4_decode_kernel<Act, NT, false>>(smem);
    if (e == cudaSuccess)
      e = kv4_start(kv4_decode_kernel<Act, NT, false>, dim3(d.ctas, d.groups), kWarpsOf<NT> * 32, smem, s, d);
  }
  if (e != cudaSuccess || d.one) return e;
  return kv4_start(kv4_join_kernel<Act, NT>, dim3(d.ctas, d.join_y + (d.scores ? kWeightCtas : 0)), kJoinThreads, 0, s, d);
}

}  // namespace

size_t kv4_decode_scratch(int q_heads, int kv_heads, long long seqs, long long max_q,
                          long long max_len, bool weights) {
  // no fewer sequences than a launch with a shorter max_len takes
  const long long n = seqs < kSeqChunk ? seqs : kSeqChunk;
  if (n < 1) return 0;
  const Plan p = plan_of(q_heads, kv_heads, n, max_q, max_len, weights, 148);
  return p.desc + p.rec + p.part_o + p.part_ml + p.scores;
}

cudaError_t kv4_decode_launch(const Kv4AttnArgs& a, int act, cudaStream_t s) {
  const long long n = chunk_of(a.c.kv_heads, a.seqs, a.max_len);
  if (n < 1) return cudaErrorInvalidValue;
  const int sms = sm_count() < 148 ? sm_count() : 148;  // as the scratch was sized
  for (long long at = 0; at < a.seqs; at += n) {
    DecodeArgs d{};
    d.a = a;
    d.a.seqs = static_cast<int>(a.seqs - at < n ? a.seqs - at : n);
    d.a.sids = a.sids + at;
    d.a.lens = a.lens + at;
    if (a.q_starts) {
      d.a.q_starts = a.q_starts + at;
    } else {
      d.a.q = static_cast<const uint8_t*>(a.q) + at * a.q_ld * 2;
      d.a.out = static_cast<uint8_t*>(a.out) + at * a.out_ld * 2;
    }
    const Plan p = plan_of(a.c.q_heads, a.c.kv_heads, d.a.seqs, a.max_q, a.max_len,
                           a.c.weights != nullptr, sms);
    d.groups = p.groups;
    d.ctas = p.ctas;
    d.one = p.one;
    d.pages_max = p.pages_max;
    d.score_ld = p.score_ld;
    uint8_t* w = static_cast<uint8_t*>(a.scratch);
    d.desc = reinterpret_cast<int4*>(w);
    w += p.desc;
    d.rec_ld = p.rec_ld;
    d.rec = reinterpret_cast<Rec*>(w);
    d.rec_n = reinterpret_cast<int*>(w + static_cast<size_t>(p.ctas) * p.rec_ld * sizeof(Rec));
    w += p.rec;
    d.part_o = reinterpret_cast<float*>(w);
    d.part_ml = reinterpret_cast<float*>(w + p.part_o);
    d.scores = a.c.weights ? reinterpret_cast<float*>(w + p.part_o + p.part_ml) : nullptr;
    d.join_y = p.cols < 8 ? p.cols : 8;
    const bool bf = act == DIAL_ACT_BF16;
    const cudaError_t e = p.nt == 1 ? (bf ? launch_nt<__nv_bfloat16, 1>(d, s) : launch_nt<__half, 1>(d, s))
                                    : (bf ? launch_nt<__nv_bfloat16, 2>(d, s) : launch_nt<__half, 2>(d, s));
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace dialb200
