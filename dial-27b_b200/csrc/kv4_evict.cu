// Eviction from the 4-bit KV cache by accumulated attention weight.
//
// Per (sequence, kv head) the entries are ranked by (protected, weight, lowest
// slot) and the first `keep` stay.  Only the set matters to attention, so the
// kept entries below slot `keep` do not move and those beyond it fill the
// holes: in place the copies are at most the evicted entries, and no copy's
// source (at or past `keep`) is another's destination (below it).
//
//  1. kv4_select_kernel, one CTA per (sequence, kv head): keys (the weights as
//     integers of the same order) in shared memory where they fit, the key of
//     rank `keep` by four passes of 8-bit digits over a shared histogram, then
//     the slots in order, a run of 32 a warp and step, holes and movers counted by
//     ballots.
//  2. kv4_move_kernel: eight lanes an entry, four entries a warp and step.
//
// Measured: 16 sessions of 3500 to 8192 slots, 8 kv heads, halved: select 30 us (128 CTAs,
// one wave: the passes take about 330 instructions for 32 slots, 1.96 of 4 a clock), move
// 37 (waits for its loads of 64-byte pieces; DRAM at 48 %).  Keys in shared memory / read anew each pass, both kernels:
// one session of 4096 19 / 27 us, 16 of 8192 40 / 57, 4 of 24576 63 / 127.
#include "kv4_dev.cuh"
#include "kv4_launch.h"

namespace dialb200 {
namespace {

constexpr int kSelectThreads = 1024, kSelectWarps = kSelectThreads / 32;
constexpr int kStaged = 24 * 1024;  // slots whose keys and positions fit shared memory

struct EvictArgs {
  Kv4Cache c;
  const int32_t* dst_table;
  const int32_t* sids;
  const int32_t* lens;
  int32_t* lens_out;
  int seqs, max_len, keep, recent;
  int32_t* count;   // [seqs][kv_heads]: entries kept, -1 for a bad sequence
  int32_t* whole;   // [seqs][kv_heads]: 1 where no entry is dropped
  int32_t* source;  // [seqs][kv_heads][keep]: source slot, or -1 - (rank of the hole)
  int32_t* mover;   // [seqs][kv_heads][keep]: source slot of the hole of that rank
};

// Rising with the weight; NaN below every number, -0 equal to 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (isnan(w)) return 0u;
  const uint32_t b = __float_as_uint(w + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Sum of `v` over the threads of the block before this one, and over all.
__device__ __forceinline__ int block_before(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int run = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += u;
  }
  if (lane == 31) warp_sums[warp] = run;
  __syncthreads();
  int w = warp_sums[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += u;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const int before = warp > 0 ? __shfl_sync(0xffffffffu, w, max(warp - 1, 0)) : 0;
  __syncthreads();
  return before + run - v;
}

// STAGED: at most kStaged slots, whose keys are kept in shared memory.  Otherwise
// every pass reads the weights again.
template <bool STAGED>
__global__ void __launch_bounds__(kSelectThreads) kv4_select_kernel(const EvictArgs a) {
  extern __shared__ uint32_t keys[];  // STAGED: [max_len], and the positions after it
  __shared__ uint32_t safe_bits[STAGED ? kStaged / 32 : 1];
  __shared__ int hist[256];
  __shared__ int sums[32];
  __shared__ int newest, found_digit, found_above;
  const int h = blockIdx.x, i = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int item = i * a.c.kv_heads + h;
  pdl_wait();
  pdl_launch_dependents();
  const int sid = a.sids[i], n = a.lens[i];
  if (static_cast<unsigned>(sid) >= static_cast<unsigned>(a.c.sessions) || n < 0 || n > a.max_len) {
    if (tid == 0) {
      set_status(a.c.status, kStatusBadArgs);
      a.count[item] = -1;
    }
    return;
  }
  if (tid == 0) {
    a.count[item] = min(n, a.keep);
    a.whole[item] = n <= a.keep;
  }
  if (n <= a.keep || a.keep == 0) return;  // the move takes every entry, or none
  int32_t* source = a.source + static_cast<size_t>(item) * a.keep;
  int32_t* mover = a.mover + static_cast<size_t>(item) * a.keep;
  auto index = [&](int s) {
    return kv4_slab_index(a.c, max(0, kv4_block(a.c, a.c.block_table, sid, s / kPageTokens)), h) *
               kPageTokens + s % kPageTokens;
  };
  if (tid == 0) newest = INT32_MIN;
  __syncthreads();
  // keys, and the newest position
  int32_t* staged_pos = reinterpret_cast<int32_t*>(keys) + a.max_len;
  int top = INT32_MIN;
#pragma unroll 8
  for (int s = tid; s < n; s += kSelectThreads) {
    const size_t at = index(s);
    const int p = a.recent > 0 ? a.c.positions[at] : 0;
    if (STAGED) {
      keys[s] = weight_key(a.c.weights[at]);
      staged_pos[s] = p;
    }
    top = max(top, p);
  }
  if (a.recent > 0) {
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) atomicMax(&newest, top);
    __syncthreads();
    top = newest;
  }
  const long long bar = a.recent > 0 ? static_cast<long long>(top) - a.recent : INT64_MAX;
  auto is_new = [&](int s) {
    return a.recent > 0 && static_cast<long long>(STAGED ? staged_pos[s] : a.c.positions[index(s)]) > bar;
  };
  __syncthreads();
  // runs of 32 slots, in order over the warps: warp w takes runs w * per ..
  const int runs = (n + 31) / 32, per = (runs + kSelectWarps - 1) / kSelectWarps;
  const int run0 = min(warp * per, runs), run1 = min(run0 + per, runs);
  int protects = 0;
  for (int r = run0; r < run1; ++r) {
    const int s = r * 32 + lane;
    const uint32_t bits = __ballot_sync(0xffffffffu, s < n && is_new(min(s, n - 1)));
    if (STAGED && lane == 0) safe_bits[r] = bits;
    if (lane == 0) protects += __popc(bits);
  }
  int all;
  block_before(protects, sums, all);  // also: every key and bit is written
  protects = all;
  auto key_of = [&](int s) { return STAGED ? keys[s] : weight_key(a.c.weights[index(s)]); };
  auto safe = [&](int s) {
    return STAGED ? (safe_bits[s >> 5] >> (s & 31) & 1u) != 0 : is_new(s);
  };
  // the class whose entries compete for `want` places
  const bool cls = protects >= a.keep;
  int want = cls ? a.keep : a.keep - protects;
  uint32_t prefix = 0;  // digits of the key of rank `want` found so far
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int r = warp; r < runs; r += kSelectWarps) {
      const int s = r * 32 + lane;
      uint32_t digit = 256;  // none
      if (s < n) {
        const uint32_t key = key_of(s);
        if ((shift == 24 || key >> (shift + 8) == prefix >> (shift + 8)) && safe(s) == cls)
          digit = key >> shift & 255u;
      }
      if (shift == 24) {  // weights share their sign and exponent: one addition for the lanes that do
        const uint32_t same = __match_any_sync(0xffffffffu, digit);
        if (digit < 256 && lane == __ffs(same) - 1) atomicAdd(&hist[digit], __popc(same));
      } else if (digit < 256) {
        atomicAdd(&hist[digit], 1);
      }
    }
    __syncthreads();
    // entries with a higher digit, from the top down: warp 0, eight digits a lane
    if (warp == 0) {
      int c[8], sum = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += c[e] = hist[255 - lane * 8 - e];
      int above = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, above, o);
        if (lane >= o) above += u;
      }
      above -= sum;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (above < want && above + c[e] >= want) {
          found_digit = 255 - lane * 8 - e;
          found_above = above;
        }
        above += c[e];
      }
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(found_digit) << shift;
    want -= found_above;
    __syncthreads();
  }
  // `want` entries equal to the key of that rank stay, the first ones
  int ties = 0;
  for (int r = run0; r < run1; ++r) {
    const int s = r * 32 + lane;
    const bool tie = s < n && key_of(s) == prefix && safe(s) == cls;
    ties += __popc(__ballot_sync(0xffffffffu, tie));
  }
  int tie0 = block_before(lane == 0 ? ties : 0, sums, all);
  tie0 = __shfl_sync(0xffffffffu, tie0, 0);
  // holes below `keep` and movers from it on, counted, then placed
  int holes = 0, movers = 0, hole0 = 0, mover0 = 0;
  const uint32_t below = (1u << lane) - 1u;
  for (int pass = 0; pass < 2; ++pass) {
    int tie_at = tie0;
    for (int r = run0; r < run1; ++r) {
      const int s = r * 32 + lane;
      bool tie = false, stay = false;
      if (s < n) {
        const uint32_t key = key_of(s);
        const bool in = safe(s) == cls;
        tie = in && key == prefix;
        stay = in ? key > prefix : !cls;
      }
      const uint32_t tied = __ballot_sync(0xffffffffu, tie);
      if (tie) stay = tie_at + __popc(tied & below) < want;
      tie_at += __popc(tied);
      const bool low = s < a.keep;
      const uint32_t hole = __ballot_sync(0xffffffffu, s < n && low && !stay);
      const uint32_t move = __ballot_sync(0xffffffffu, s < n && !low && stay);
      if (pass == 0) {
        holes += __popc(hole);
        movers += __popc(move);
      } else {
        if (s < n && low) source[s] = stay ? s : -1 - (hole0 + __popc(hole & below));
        if (s < n && !low && stay) mover[mover0 + __popc(move & below)] = s;
        hole0 += __popc(hole);
        mover0 += __popc(move);
      }
    }
    if (pass == 0) {
      hole0 = __shfl_sync(0xffffffffu, block_before(lane == 0 ? holes : 0, sums, all), 0);
      mover0 = __shfl_sync(0xffffffffu, block_before(lane == 0 ? movers : 0, sums, all), 0);
    }
  }
}

constexpr int kMoveEntries = 64;  // of a CTA of 4 warps: 16 a warp, four at a time

__global__ void __launch_bounds__(128) kv4_move_kernel(const EvictArgs a) {
  const int h = blockIdx.y, i = blockIdx.z, lane = threadIdx.x & 31, l = lane & 7;
  const int item = i * a.c.kv_heads + h;
  pdl_wait();
  pdl_launch_dependents();
  const int kept = a.count[item];
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0 && kept >= 0) a.lens_out[i] = kept;
  const int d0 = blockIdx.x * kMoveEntries + (threadIdx.x >> 5) * 16;
  if (d0 >= kept) return;
  const int sid = a.sids[i];
  // lanes 0-15: the warp's entries, source and destination slab and token
  size_t fi = 0, ti = 0;
  int st = 0, dt = 0;
  bool moves = false;
  if (lane < 16 && d0 + lane < kept) {
    const int d = d0 + lane;
    int s = a.whole[item] ? d : a.source[static_cast<size_t>(item) * a.keep + d];
    if (s < 0) s = a.mover[static_cast<size_t>(item) * a.keep - s - 1];
    const int from = max(0, kv4_block(a.c, a.c.block_table, sid, s / kPageTokens));
    const int to = kv4_block(a.c, a.dst_table, sid, d / kPageTokens);
    moves = to >= 0 && !(to == from && s == d);
    st = s % kPageTokens;
    dt = d % kPageTokens;
    fi = kv4_slab_index(a.c, from, h);
    ti = kv4_slab_index(a.c, max(to, 0), h);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int src = e * 4 + (lane >> 3);
    const size_t f = __shfl_sync(0xffffffffu, fi, src), t = __shfl_sync(0xffffffffu, ti, src);
    const int ft = __shfl_sync(0xffffffffu, st, src), tt = __shfl_sync(0xffffffffu, dt, src);
    if (!__shfl_sync(0xffffffffu, moves, src)) continue;
    const uint8_t* from = a.c.pages + f * kKv4Slab;
    uint8_t* to = a.c.pages + t * kKv4Slab;
    const uint2 k = *reinterpret_cast<const uint2*>(from + ft * 64 + l * 8);
    const uint2 v = *reinterpret_cast<const uint2*>(from + kKv4VCodes + ft * 64 + l * 8);
    // lanes 0 and 1 the scales, 2 and 3 weight and position
    uint2 x = make_uint2(0, 0);
    if (l < 2) x = *reinterpret_cast<const uint2*>(from + (l == 0 ? kKv4KScales : kKv4VScales) + ft * 8);
    else if (l == 2) x.x = __float_as_uint(a.c.weights[f * kPageTokens + ft]);
    else if (l == 3 && a.c.positions) x.x = a.c.positions[f * kPageTokens + ft];
    *reinterpret_cast<uint2*>(to + tt * 64 + l * 8) = k;
    *reinterpret_cast<uint2*>(to + kKv4VCodes + tt * 64 + l * 8) = v;
    if (l < 2) *reinterpret_cast<uint2*>(to + (l == 0 ? kKv4KScales : kKv4VScales) + tt * 8) = x;
    else if (l == 2) a.c.weights[t * kPageTokens + tt] = __uint_as_float(x.x);
    else if (l == 3 && a.c.positions) a.c.positions[t * kPageTokens + tt] = static_cast<int>(x.x);
  }
}

}  // namespace
}  // namespace dialb200

using namespace dialb200;

extern "C" int64_t dial_b200_kv4_evict_scratch_bytes(const dial_b200_kv4_shape* sh, int64_t seqs,
                                                     int64_t max_len, int64_t keep) {
  if (!sh || sh->kv_heads < 1 || sh->kv_heads > 1024 || seqs < 0 || seqs > 65535 || max_len < 0 ||
      max_len > 16LL << 26 || keep < 0 || keep > INT32_MAX)
    return -1;
  const int64_t most = keep < max_len ? keep : max_len;
  return seqs * sh->kv_heads * (2 + 2 * most) * 4 + 16;
}

extern "C" int dial_b200_kv4_evict(const dial_b200_kv4_shape* sh, void* pages, float* weights,
                                   int32_t* positions, const int32_t* block_table,
                                   const int32_t* dst_table, int64_t sessions, const int32_t* sids,
                                   const int32_t* lens, int32_t* lens_out, int64_t seqs,
                                   int64_t max_len, int64_t keep, int64_t recent, void* scratch,
                                   void* stream, char* err, size_t n) {
  EvictArgs a{};
  int rc = kv4_cache_of(sh, pages, weights, positions, block_table, sessions, &a.c, err, n);
  if (rc != DIAL_OK) return rc;
  if (!weights || (seqs != 0 && (!sids || !lens || !lens_out)))
    return kv4_fail(err, n, DIAL_ERR_INVALID, "null pointer argument");
  if (seqs < 0 || seqs > 65535)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "seqs %lld outside [0, 65535]", (long long)seqs);
  if (max_len < 0 || max_len > 16LL * sh->max_blocks)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "max_len %lld exceeds the block table's %lld slots",
                    (long long)max_len, 16LL * sh->max_blocks);
  if (keep < 0 || keep > INT32_MAX || recent < 0 || recent > keep)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "keep %lld / recent %lld: 0 <= recent <= keep",
                    (long long)keep, (long long)recent);
  if (recent > 0 && !positions)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "recent > 0 needs positions");
  if (seqs == 0) return DIAL_OK;
  if (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 15) != 0)
    return kv4_fail(err, n, DIAL_ERR_INVALID, "scratch must be given, 16-byte aligned");
  const int64_t most = keep < max_len ? keep : max_len;  // nothing is dropped above max_len
  a.dst_table = dst_table ? dst_table : block_table;
  a.sids = sids;
  a.lens = lens;
  a.lens_out = lens_out;
  a.seqs = static_cast<int>(seqs);
  a.max_len = static_cast<int>(max_len);
  a.keep = static_cast<int>(most);
  a.recent = static_cast<int>(recent < most ? recent : most);
  a.count = static_cast<int32_t*>(scratch);
  a.whole = a.count + seqs * sh->kv_heads;
  a.source = a.whole + seqs * sh->kv_heads;
  a.mover = a.source + seqs * sh->kv_heads * most;
  if ((rc = kv4_ready(&a.c, err, n)) != DIAL_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid(sh->kv_heads, a.seqs);
  cudaError_t e;
  if (max_len <= kStaged) {
    e = kv4_allow_smem<kv4_select_kernel<true>>(kStaged * 8);
    if (e == cudaSuccess)
      e = kv4_start(kv4_select_kernel<true>, grid, kSelectThreads, static_cast<size_t>(max_len) * 8, s, a);
  } else {
    e = kv4_start(kv4_select_kernel<false>, grid, kSelectThreads, 0, s, a);
  }
  if (e == cudaSuccess) {
    const unsigned groups = static_cast<unsigned>(most > 0 ? (most + kMoveEntries - 1) / kMoveEntries : 1);
    e = kv4_start(kv4_move_kernel, dim3(groups, sh->kv_heads, a.seqs), 128, 0, s, a);
  }
  if (e != cudaSuccess)
    return kv4_fail(err, n, DIAL_ERR_CUDA, "kv4 evict launch failed: %s", cudaGetErrorString(e));
  return DIAL_OK;
}
