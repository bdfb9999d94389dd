// Device helpers of the 4-bit KV cache operators: the e2m1 / e4m3 codec and
// the checked way from a session's slot to its slab.
#pragma once

#include "attn_dev.cuh"
#include "common.cuh"
#include "kv4_attn.h"

namespace dialb200 {

// Page of slot `slot`, or -1 (with the status recorded) for a block id outside
// the pool.  sid and slot / 16 are within the table.
__device__ __forceinline__ int kv4_block(const Kv4Cache& c, const int32_t* table, int sid,
                                         int page) {
  const int b = table[static_cast<size_t>(sid) * c.max_blocks + page];
  if (static_cast<unsigned>(b) >= static_cast<unsigned>(c.num_blocks)) {
    set_status(c.status, kStatusBadArgs);
    return -1;
  }
  return b;
}

__device__ __forceinline__ size_t kv4_slab_index(const Kv4Cache& c, int block, int head) {
  return static_cast<size_t>(block) * c.kv_heads + head;
}

// e4m3 code nearest to a non-negative v, saturating at 448.
__device__ __forceinline__ uint32_t e4m3_of(float v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.f), "f"(v));
  return r & 0xFFu;
}

__device__ __forceinline__ float e4m3_value(uint32_t code) {
  const uint32_t h = e4m3x2_to_f16x2(static_cast<uint16_t>(code));
  return __low2float(*reinterpret_cast<const __half2*>(&h));
}

// Two e2m1 codes, lo in the low nibble, nearest even, saturating at 6.
__device__ __forceinline__ uint32_t e2m1x2_of(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 b;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %1, %2;\n\t"
      "cvt.u32.u8 %0, b;\n\t}"
      : "=r"(r)
      : "f"(hi), "f"(lo));
  return r;
}

// x / s correctly rounded, with y = 1 / s correctly rounded: the remainder of x y
// is exact, and its product with y corrects the last place (Markstein).  Quotients
// that overflow are divided.
__device__ __forceinline__ float quotient(float x, float s, float y) {
  const float q = x * y;
  return fabsf(q) < 1e30f ? fmaf(fmaf(-q, s, x), y, q) : __fdiv_rn(x, s);
}

// Queries enter the MMAs as f16 after 2^-e, e the exponent of the row's largest value
// `top` (within f32's normal powers): exact for values down to 2^-14 of it, and off by
// at most 2^-25 of it below.
__device__ __forceinline__ int query_exp(float top) {
  return min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -126), 126);
}
// What such a row's sums are multiplied by to become base-2 scores.  Kept within f32's
// normal numbers, so that a masked score, -inf, stays -inf under any scale.
__device__ __forceinline__ float score_scale(const Kv4AttnArgs& a, int e) {
  return a.unit * exp2i(min(max(e + a.unit_exp, -125), 127));
}

// A sequence of an attention call: its session, slots, first row and rows.
struct Kv4Seq {
  int sid, len, row0, n;
};

// The sequence's rows and slots; false (with the status recorded) for one
// whose session, rows or length are out of range.
__device__ __forceinline__ bool kv4_seq(const Kv4AttnArgs& a, int i,
                                        Kv4Seq& s) {
  s.sid = a.sids[i];
  s.len = a.lens[i];
  s.row0 = a.q_starts ? a.q_starts[i] : i;
  const int end = a.q_starts ? a.q_starts[i + 1] : i + 1;
  if (static_cast<unsigned>(s.sid) >= static_cast<unsigned>(a.c.sessions) || s.len < 0 ||
      s.len > a.max_len || s.row0 < 0 || end < s.row0 || end > a.rows || end - s.row0 > a.max_q) {
    set_status(a.c.status, kStatusBadArgs);
    return false;
  }
  s.n = end - s.row0;
  return true;
}

}  // namespace dialb200
