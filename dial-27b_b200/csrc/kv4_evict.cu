// Eviction from the 4-bit KV cache by accumulated attention weight.
//
// Per (sequence, kv head) the entries are ranked by (protected, weight, lowest
// slot) and the first `keep` stay.  Only the set matters to attention, so the
// kept entries below slot `keep` do not move and those beyond it fill the
// holes: in place the copies are at most the evicted entries, and no copy's
// source (at or past `keep`) is another's destination (below it).
//
//  1. kv4_select_kernel, one CTA per (sequence, kv head): the key of rank
//     `keep` by four passes of 8-bit digits over a shared histogram, then the
//     slots in order with a running count of holes and of movers.
//  2. kv4_move_kernel: one warp per destination slot and kv head.
#include "kv4_dev.cuh"

namespace dialb200 {
namespace {

constexpr int kSelectThreads = 1024;

struct EvictArgs {
  Kv4Cache c;
  const int32_t* dst_table;
  const int32_t* sids;
  const int32_t* lens;
  int32_t* lens_out;
  int seqs, max_len, keep, recent;
  int32_t* count;   // [seqs][kv_heads]: entries kept, -1 for a bad sequence
  int32_t* source;  // [seqs][kv_heads][keep]: source slot, or -1 - (rank of the hole)
  int32_t* mover;   // [seqs][kv_heads][keep]: source slot of the hole of that rank
};

// Rising with the weight; NaN below every number, -0 equal to 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (isnan(w)) return 0u;
  const uint32_t b = __float_as_uint(w + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// Inclusive sum of `v` over the block's threads; `total` is the whole sum.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) warp_sums[warp] = v;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  total = warp_sums[31];
  const int before = warp > 0 ? warp_sums[warp - 1] : 0;
  __syncthreads();
  return v + before;
}

__global__ void __launch_bounds__(kSelectThreads) kv4_select_kernel(const EvictArgs a) {
  __shared__ int hist[256];
  __shared__ int sums[32];
  __shared__ int newest, found_digit, found_above;
  const int h = blockIdx.x, i = blockIdx.y, tid = threadIdx.x;
  const int item = i * a.c.kv_heads + h;
  const int sid = a.sids[i], n = a.lens[i];
  if (static_cast<unsigned>(sid) >= static_cast<unsigned>(a.c.sessions) || n < 0 || n > a.max_len) {
    if (tid == 0) {
      set_status(a.c.status, kStatusBadArgs);
      a.count[item] = -1;
    }
    return;
  }
  const int kept = min(n, a.keep);
  int32_t* source = a.source + static_cast<size_t>(item) * a.keep;
  int32_t* mover = a.mover + static_cast<size_t>(item) * a.keep;
  if (tid == 0) a.count[item] = kept;
  if (n <= a.keep) {
    for (int s = tid; s < n; s += kSelectThreads) source[s] = s;
    return;
  }
  if (a.keep == 0) return;
  auto index = [&](int s) {
    return kv4_slab_index(a.c, max(0, kv4_block(a.c, a.c.block_table, sid, s / kPageTokens)), h) *
               kPageTokens + s % kPageTokens;
  };
  // the newest position, then how many entries it protects
  int top = INT32_MIN;
  if (a.recent > 0) {
    if (tid == 0) newest = INT32_MIN;
    __syncthreads();
    for (int s = tid; s < n; s += kSelectThreads) top = max(top, a.c.positions[index(s)]);
    atomicMax(&newest, top);
    __syncthreads();
    top = newest;
  }
  auto safe = [&](size_t at) {
    return a.recent > 0 &&
           static_cast<long long>(a.c.positions[at]) > static_cast<long long>(top) - a.recent;
  };
  int mine = 0, protects = 0;
  for (int s = tid; s < n; s += kSelectThreads) mine += safe(index(s));
  block_scan(mine, sums, protects);
  // the class whose entries compete for `want` places
  const bool cls = protects >= a.keep;
  int want = cls ? a.keep : a.keep - protects;
  uint32_t prefix = 0;  // digits of the key of rank `want` found so far
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int b = tid; b < 256; b += kSelectThreads) hist[b] = 0;
    __syncthreads();
    for (int s = tid; s < n; s += kSelectThreads) {
      const size_t at = index(s);
      const uint32_t key = weight_key(a.c.weights[at]);
      if (safe(at) == cls && (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8)))
        atomicAdd(&hist[key >> shift & 255u], 1);
    }
    __syncthreads();
    // entries with a higher digit, from the top down
    const int d = 255 - tid;
    int all;
    const int upto = block_scan(tid < 256 ? hist[d] : 0, sums, all);
    if (tid < 256 && upto >= want && upto - hist[d] < want) {
      found_digit = d;
      found_above = upto - hist[d];
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(found_digit) << shift;
    want -= found_above;
    __syncthreads();
  }
  // slots in order: `want` entries equal to the key of that rank stay, the first ones
  int ties = 0, holes = 0, movers = 0;
  for (int base = 0; base < n; base += kSelectThreads) {
    const int s = base + tid;
    bool tie = false, stay = false;
    if (s < n) {
      const size_t at = index(s);
      const uint32_t key = weight_key(a.c.weights[at]);
      if (safe(at) == cls) {
        tie = key == prefix;
        stay = key > prefix;
      } else {
        stay = !cls;
      }
    }
    int total;
    const int rank = ties + block_scan(tie, sums, total);
    ties += total;
    if (tie) stay = rank <= want;
    const bool low = s < a.keep;
    const int hole = holes + block_scan(s < n && low && !stay, sums, total);
    holes += total;
    const int move = movers + block_scan(s < n && !low && stay, sums, total);
    movers += total;
    if (s < n && low) source[s] = stay ? s : -hole;
    if (s < n && !low && stay) mover[move - 1] = s;
  }
}

__global__ void __launch_bounds__(256) kv4_move_kernel(const EvictArgs a) {
  const int d = blockIdx.x * 8 + (threadIdx.x >> 5), h = blockIdx.y, i = blockIdx.z;
  const int lane = threadIdx.x & 31, item = i * a.c.kv_heads + h;
  const int kept = a.count[item];
  if (d == 0 && h == 0 && lane == 0 && kept >= 0) a.lens_out[i] = kept;
  if (d >= kept) return;
  int s = a.source[static_cast<size_t>(item) * a.keep + d];
  if (s < 0) s = a.mover[static_cast<size_t>(item) * a.keep - s - 1];
  const int sid = a.sids[i];
  const int from = max(0, kv4_block(a.c, a.c.block_table, sid, s / kPageTokens));
  const int to = kv4_block(a.c, a.dst_table, sid, d / kPageTokens);
  if (to < 0 || (to == from && s == d)) return;
  const int st = s % kPageTokens, dt = d % kPageTokens;
  const size_t fi = kv4_slab_index(a.c, from, h), ti = kv4_slab_index(a.c, to, h);
  const uint8_t* src = a.c.pages + fi * kKv4Slab;
  uint8_t* dst = a.c.pages + ti * kKv4Slab;
  if (lane < 16) {  // k codes (lanes 0-7) and v codes, 8 bytes a lane
    const int part = (lane >> 3) * kKv4VCodes + (lane & 7) * 8;
    *reinterpret_cast<uint2*>(dst + part + dt * 64) =
        *reinterpret_cast<const uint2*>(src + part + st * 64);
  } else if (lane < 18) {
    const int part = lane == 16 ? kKv4KScales : kKv4VScales;
    *reinterpret_cast<uint2*>(dst + part + dt * 8) =
        *reinterpret_cast<const uint2*>(src + part + st * 8);
  } else if (lane == 18) {
    a.c.weights[ti * kPageTokens + dt] = a.c.weights[fi * kPageTokens + st];
  } else if (lane == 19 && a.c.positions) {
    a.c.positions[ti * kPageTokens + dt] = a.c.positions[fi * kPageTokens + st];
  }
}

}  // namespace
}  // namespace dialb200

using namespace dialb200;

extern "C" int64_t dial_b200_kv4_evict_scratch_bytes(const dial_b200_kv4_shape* sh, int64_t seqs,
                                                     int64_t max_len, int64_t keep) {
  if (!sh || sh->kv_heads < 1 || seqs < 0 || max_len < 0 || keep < 0) return -1;
  const int64_t most = keep < max_len ? keep : max_len;
  return seqs * sh->kv_heads * (1 + 2 * most) * 4 + 16;
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
  if (!weights || !sids || !lens || !lens_out)
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
  a.source = a.count + seqs * sh->kv_heads;
  a.mover = a.source + seqs * sh->kv_heads * most;
  if ((rc = kv4_ready(&a.c, err, n)) != DIAL_OK) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  kv4_select_kernel<<<dim3(sh->kv_heads, a.seqs), kSelectThreads, 0, s>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) {
    const unsigned groups = static_cast<unsigned>(most > 0 ? (most + 7) / 8 : 1);
    kv4_move_kernel<<<dim3(groups, sh->kv_heads, a.seqs), 256, 0, s>>>(a);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess)
    return kv4_fail(err, n, DIAL_ERR_CUDA, "kv4 evict launch failed: %s", cudaGetErrorString(e));
  return DIAL_OK;
}
