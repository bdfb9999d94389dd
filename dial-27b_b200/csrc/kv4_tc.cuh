// Shared by the tensor-core kernels over the 4-bit KV cache: tcgen05 wrappers,
// pair arithmetic, and the way from codes to a swizzled f16 operand tile.
#pragma once

#include "kv4_dev.cuh"

namespace dialb200 {
namespace {

constexpr int kTile = 128 * 128 * 2;  // f16 tile: two 64-column halves of 128-byte rows
constexpr int kHalf = kTile / 2;

// ------------------------------------------------------------ tcgen05 forms
constexpr uint32_t idesc(bool b_mn_major) {  // f16 x f16 -> f32, M = N = 128
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
}
// K-major operand: 128-byte rows, 128-byte swizzle, 8-row groups 1 KB apart.
__device__ __forceinline__ uint64_t kmajor_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (1ull << 16) | (64ull << 32) |
         (1ull << 46) | (2ull << 61);
}
// MN-major operand (keys x dims, dims contiguous): 64-dim halves kHalf apart.
__device__ __forceinline__ uint64_t mnmajor_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(kHalf >> 4) << 16) |
         (64ull << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(da), "l"(db), "r"(id), "r"(acc));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t ta, uint64_t db, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(ta), "l"(db), "r"(id), "r"(acc));
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_u32(bar))
               : "memory");
}
// One lane of the warp, the same on every call.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// The wait for the tcgen05.ld before it; naming the registers keeps their uses
// behind it.
#define KV4_RW32(v)                                                                              \
  "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), \
      "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]),   \
      "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]),  \
      "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]),  \
      "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
__device__ __forceinline__ void ld_wait(uint32_t* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : KV4_RW32(v)::"memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src),
               "r"(there ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define KV4_R32(v)                                                                              \
  "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), \
      "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]),  \
      "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), \
      "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), \
      "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
// 32 columns of the thread's TMEM lane, without the wait.
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];"
      : KV4_R32(v)
      : "r"(taddr));
}
__device__ __forceinline__ void ld16(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}
__device__ __forceinline__ void ld_wait16(uint32_t* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]),
                 "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]),
                 "+r"(v[13]), "+r"(v[14]), "+r"(v[15])::"memory");
}
__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, "
      "%12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]));
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// (x0, x1) * f + c, and a + b, on pairs.
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  return static_cast<uint64_t>(__float_as_uint(lo)) | static_cast<uint64_t>(__float_as_uint(hi)) << 32;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// x f, rounded, two at a time: scores as their references and log-sum-exps have them,
// so that what is subtracted from the largest one leaves the right exponent however
// large they are (an fma would keep a reference's rounding, 2^-24 of it, in the
// exponent).  Written with a zero that the compiler does not know: a product and the
// sum after it are made into one fma, in this form too.
__device__ __forceinline__ uint64_t score2(const Kv4AttnArgs& a, uint64_t x, uint64_t f) {
  return fma2(x, f, a.zeros);
}
__device__ __forceinline__ float lo_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float hi_of(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }

// 32 tokens of a 128-token block (warp dw of four, token 32 dw + 8 e + lane / 4,
// dims 32 q .. 32 q + 31 with q = lane % 4) as rows of a 128-byte-swizzled tile.
__device__ __forceinline__ void codes_to_tile(uint8_t* tile, int dw, const uint4 (&c)[4],
                                              const uint32_t (&s)[4]) {
  const int lane = threadIdx.x & 31, q = lane & 3, tok = lane >> 2;
  const bool swap = (q & 2) != 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int row = dw * 32 + e * 8 + tok;
    const uint32_t sc = e4m3x2_to_f16x2(static_cast<uint16_t>(s[e]));
    const uint32_t first = __byte_perm(sc, 0, swap ? 0x3232 : 0x1010);
    const uint32_t second = __byte_perm(sc, 0, swap ? 0x1010 : 0x3232);
    uint8_t* to = tile + (q >> 1) * kHalf + row * 128;
    // lanes of the upper half take their words two on: no two lanes of a
    // quarter warp meet in a bank
    const uint32_t words[4] = {swap ? c[e].z : c[e].x, swap ? c[e].w : c[e].y,
                               swap ? c[e].x : c[e].z, swap ? c[e].y : c[e].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t o[4];
      e2m1x8_to_f16x2x4(words[i], o);
      const uint32_t sx = i < 2 ? first : second;
      const int chunk = (q & 1) * 4 + (swap ? i ^ 2 : i);
      *reinterpret_cast<uint4*>(to + ((chunk ^ (row & 7)) << 4)) =
          make_uint4(hmul2(o[0], sx), hmul2(o[1], sx), hmul2(o[2], sx), hmul2(o[3], sx));
    }
  }
}

}  // namespace
}  // namespace dialb200
