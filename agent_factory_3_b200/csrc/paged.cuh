// Device view of one layer's KV pages, shared by the kernels that read or write them.
//
// A pool is a tensor [pages, page_size, Hkv, D] of bf16 or of e4m3 codes whose rows of D
// elements are contiguous; the other strides are free (e4m3 pools usually keep a KV head's rows
// of a page together).  e4m3 pools come with one e8m0 byte b per row, [pages, Hkv, page_size]
// with free strides: the row's values are code * 2^(b - 127), exact in bf16.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

namespace af3 {
namespace paged {

struct Pool {
  uint8_t* k;
  uint8_t* v;
  uint8_t* ks;  // scale bytes, null for bf16 pages
  uint8_t* vs;
  // strides in bytes, the same for K and V
  int64_t page, token, head;
  int64_t s_page, s_head, s_token;
  int num_pages, page_size, page_shift;  // page_shift: log2(page_size), -1 if not a power of two
};

__device__ __forceinline__ void split_slot(const Pool& p, uint32_t slot, uint32_t& page,
                                           uint32_t& off) {
  if (p.page_shift >= 0) {
    page = slot >> p.page_shift;
    off = slot & (uint32_t)(p.page_size - 1);
  } else {
    page = slot / (uint32_t)p.page_size;
    off = slot - page * (uint32_t)p.page_size;
  }
}

__device__ __forceinline__ float ex2a(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^e for integer e in [-127, 127]; 2^-127 is a denormal.
__device__ __forceinline__ float pow2i(int e) {
  return e > -127 ? __uint_as_float((uint32_t)(e + 127) << 23) : __uint_as_float(0x00400000u);
}

// Two e4m3 codes (low byte first) -> f16 pair, exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t c) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
  return r;
}

// Four e4m3 codes -> f16 pairs of the low two and of the high two.
__device__ __forceinline__ void e4m3x4_to_f16x2(uint32_t c, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}"
      : "=r"(lo), "=r"(hi)
      : "r"(c));
}

__device__ __forceinline__ float2 f16x2_to_float2(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// Asynchronous copies of 16 bytes into shared memory, and its 16-byte loads.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;  // 0: the 16 bytes are filled with zeros and src is not read
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a));
  return r;
}

// A byte, 0 where not on, in one predicated load: no branch for the result to be waited for in.
__device__ __forceinline__ uint32_t load_byte(const uint8_t* p, bool on) {
  uint32_t r;
  asm volatile("{\n.reg .pred q;\nsetp.ne.b32 q, %2, 0;\nmov.b32 %0, 0;\n@q ld.global.nc.u8 %0, [%1];\n}"
               : "=r"(r)
               : "l"(p), "r"((int)on));
  return r;
}

}  // namespace paged
}  // namespace af3
