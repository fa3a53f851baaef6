// Writing keys and values into e4m3 cache pages and reading them back.
//
// Per row of D elements (one token, one KV head), over its finite entries: a = max |x|, e = the
// smallest integer in [-127, 120] with a <= 448 * 2^e, code = e4m3(x * 2^-e) rounded to nearest
// even, scale byte = e + 127 (e8m0).  A power of two as scale costs no relative precision, since
// e4m3 is a floating type itself, and leaves nothing to round on the way back: code * 2^e is a
// bf16 number.  At e = 120 codes end at 240, because 256 * 2^120 is past the largest bf16.  Entries
// that are not finite become the NaN code, so that a broken token stays visible.
//
// Both kernels are bound by memory (and by the launch for a decode step's few rows): one pass, one warp
// a token, 16-byte accesses on the bf16 side, 8-byte ones on the e4m3 side, D / 8 lanes a row, every
// load of a token before its first store.  Measured with 8 KV heads of 64 and slots in random order:
// store of 16384 tokens 16.4 us (3.1 TB/s), where each row's 64 codes and its scale byte are writes of
// their own; gather of 131072 rows 89 us (4.5 TB/s).
#include "common.h"
#include "host_utils.h"
#include "paged.cuh"
#include "paged_host.h"

namespace af3 {
namespace paged {

constexpr int kCacheThreads = 128;

struct RowArgs {
  __nv_bfloat16* qkv;
  int64_t ld;
  int k_off, v_off;
  const int* slots;
  int n, hkv, lanes_log2;  // lanes per row: D / 8
  uint32_t n_slots;
};

// The smallest e in [-127, 120] with a <= 448 * 2^e, of a = 1.m * 2^E >= 0 given by its fp32 bits:
// 448 * 2^e = 1.75 * 2^(e + 8).
__device__ __forceinline__ int exponent_of(uint32_t bits) {
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return min(max(e, -127), 120);
}

// One warp per row of qkv; its lanes walk the row's Hkv * D / 8 pieces of K and of V, 32 at a time.
// The loads of both go out before anything waits, for the slot too.
__global__ void __launch_bounds__(kCacheThreads) kv_store_fp8_kernel(const RowArgs a, const Pool p) {
  const int row = (int)blockIdx.x * (kCacheThreads / 32) + (int)(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= a.n) return;
  const uint32_t slot = (uint32_t)a.slots[row];
  const __nv_bfloat16* src = a.qkv + (int64_t)row * a.ld;
  const uint4* from[2] = {reinterpret_cast<const uint4*>(src + a.k_off), reinterpret_cast<const uint4*>(src + a.v_off)};
  const int pieces = a.hkv << a.lanes_log2, per_row = 1 << a.lanes_log2;
  for (int base = 0; base < pieces; base += 64) {
    uint4 w[4];  // K, V of piece base + lane, then of base + 32 + lane
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = base + 32 * (u >> 1) + lane;
      w[u] = i < pieces ? __ldcs(from[u & 1] + i) : make_uint4(0u, 0u, 0u, 0u);
    }
    if (slot >= a.n_slots) return;  // negative or past the pool
    uint32_t page, off;
    split_slot(p, slot, page, off);
    const int64_t at = (int64_t)page * p.page + (int64_t)off * p.token;
    const int64_t sat = (int64_t)page * p.s_page + (int64_t)off * p.s_token;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = base + 32 * (u >> 1) + lane;
      const bool on = i < pieces;  // a row's lanes are all on or all off: per_row divides 32
      const uint32_t h[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
      // largest magnitude as bf16 bits: integers order like the values
      const uint32_t m2 = __vmaxu2(__vmaxu2(h[0] & 0x7fff7fffu, h[1] & 0x7fff7fffu),
                                   __vmaxu2(h[2] & 0x7fff7fffu, h[3] & 0x7fff7fffu));
      uint32_t m = max(m2 & 0xffffu, m2 >> 16);
      for (int o = per_row >> 1; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      float x[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = __uint_as_float(h[j] << 16);
        x[2 * j + 1] = __uint_as_float(h[j] & 0xffff0000u);
      }
      int e = exponent_of(m << 16);
      // Rows with entries that are not finite, and the largest exponent, go the long way (all rows
      // going it: 18.1 us for 16384 tokens, bound by its instructions).
      if (__any_sync(0xffffffffu, m >= 0x7f80u || e == 120)) {
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float f = fabsf(x[j]);
          if (f < INFINITY) amax = fmaxf(amax, f);  // false for NaN
        }
        for (int o = per_row >> 1; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        e = exponent_of(__float_as_uint(amax));
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
        const float lim = e == 120 ? 240.f : 448.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool fin = fabsf(x[j]) < INFINITY;
          x[j] = fin ? fminf(fmaxf(x[j] * inv, -lim), lim) : __uint_as_float(0x7fc00000u);
        }
      } else {
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);  // |x| * inv <= 448
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] *= inv;
      }
      uint32_t out[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint16_t lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x[4 * j + 1]), "f"(x[4 * j]));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x[4 * j + 3]), "f"(x[4 * j + 2]));
        out[j] = (uint32_t)lo | ((uint32_t)hi << 16);
      }
      if (on) {
        const int head = i >> a.lanes_log2, piece = i & (per_row - 1);
        *reinterpret_cast<uint2*>(((u & 1) ? p.v : p.k) + at + head * p.head + piece * 8) = make_uint2(out[0], out[1]);
        if (piece == 0) ((u & 1) ? p.vs : p.ks)[sat + head * p.s_head] = (uint8_t)(e + 127);
      }
    }
  }
}

// One warp per row of qkv, 64 pieces of K and of V at a time, every load before the first store.
__global__ void __launch_bounds__(kCacheThreads) kv_gather_fp8_kernel(const RowArgs a, const Pool p) {
  const int row = (int)blockIdx.x * (kCacheThreads / 32) + (int)(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= a.n) return;
  const uint32_t slot = (uint32_t)a.slots[row];
  if (slot >= a.n_slots) return;
  uint32_t page, off;
  split_slot(p, slot, page, off);
  __nv_bfloat16* dst = a.qkv + (int64_t)row * a.ld;
  uint4* to[2] = {reinterpret_cast<uint4*>(dst + a.k_off), reinterpret_cast<uint4*>(dst + a.v_off)};
  const int64_t at = (int64_t)page * p.page + (int64_t)off * p.token;
  const int64_t sat = (int64_t)page * p.s_page + (int64_t)off * p.s_token;
  const int pieces = a.hkv << a.lanes_log2, per_row = 1 << a.lanes_log2;
  for (int base = 0; base < pieces; base += 64) {
    uint2 c[4];
    uint32_t byte[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = base + 32 * (u >> 1) + lane;
      const bool on = i < pieces;
      const int head = i >> a.lanes_log2, piece = i & (per_row - 1);
      c[u] = make_uint2(0u, 0u);
      if (on) c[u] = __ldg(reinterpret_cast<const uint2*>(((u & 1) ? p.v : p.k) + at + head * p.head + piece * 8));
      byte[u] = load_byte(((u & 1) ? p.vs : p.ks) + sat + head * p.s_head, on);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = base + 32 * (u >> 1) + lane;
      const float s = pow2i((int)byte[u] - 127);
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t word = j < 2 ? c[u].x : c[u].y;
        const float2 f = f16x2_to_float2(e4m3x2_to_f16x2((uint16_t)(word >> (16 * (j & 1)))));
        const __nv_bfloat162 r = __floats2bfloat162_rn(f.x * s, f.y * s);
        o[j] = *reinterpret_cast<const uint32_t*>(&r);
      }
      if (i < pieces) __stcs(to[u & 1] + i, make_uint4(o[0], o[1], o[2], o[3]));
    }
  }
}

static RowArgs row_args(const torch::Tensor& qkv, int64_t k_off, int64_t v_off,
                        const torch::Tensor& slots, const torch::Tensor& k_pages) {
  check_cuda_bf16(qkv, "qkv");
  const int64_t hkv = k_pages.size(2), d = k_pages.size(3);
  AF3_CHECK(qkv.dim() == 2 && qkv.stride(1) == 1, "qkv must be [n, width] with contiguous rows");
  AF3_CHECK(d >= 8 && d <= 256 && (d & (d - 1)) == 0, "head_dim must be a power of two from 8 to 256");
  AF3_CHECK(slots.is_cuda() && slots.scalar_type() == torch::kInt && slots.dim() == 1 && slots.is_contiguous(),
            "slots must be a contiguous int32 CUDA vector");
  AF3_CHECK(slots.get_device() == qkv.get_device() && k_pages.get_device() == qkv.get_device(),
            "qkv, slots and pages must be on one device");
  AF3_CHECK(slots.numel() <= qkv.size(0), "more slots than rows");
  AF3_CHECK(k_off >= 0 && v_off >= 0 && k_off + hkv * d <= qkv.size(1) && v_off + hkv * d <= qkv.size(1),
            "k_off / v_off past the row");
  AF3_CHECK(k_off % 8 == 0 && v_off % 8 == 0 && (qkv.stride(0) % 8 == 0 || qkv.size(0) <= 1) &&
                reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 == 0,
            "qkv rows and k_off / v_off must be 16-byte aligned");
  AF3_CHECK(slots.numel() < (int64_t(1) << 30), "too many rows");
  RowArgs a;
  a.qkv = reinterpret_cast<__nv_bfloat16*>(qkv.data_ptr());
  a.ld = qkv.stride(0);
  a.k_off = (int)k_off;
  a.v_off = (int)v_off;
  a.slots = slots.data_ptr<int>();
  a.n = (int)slots.numel();
  a.hkv = (int)hkv;
  a.lanes_log2 = 0;
  while ((8 << a.lanes_log2) < d) ++a.lanes_log2;
  a.n_slots = (uint32_t)std::min<int64_t>(k_pages.size(0) * k_pages.size(1), INT32_MAX);
  return a;
}

}  // namespace paged

void kv_store_fp8(torch::Tensor qkv, int64_t k_off, int64_t v_off, torch::Tensor slots,
                  torch::Tensor k_pages, torch::Tensor v_pages, c10::optional<torch::Tensor> k_scales,
                  c10::optional<torch::Tensor> v_scales) {
  using namespace paged;
  const Pool p = make_pool(k_pages, v_pages, k_scales, v_scales, 8);
  AF3_CHECK(p.ks != nullptr, "kv_store_fp8 needs float8_e4m3fn pages");
  const RowArgs a = row_args(qkv, k_off, v_off, slots, k_pages);
  if (a.n == 0) return;
  const c10::cuda::CUDAGuard guard(qkv.device());
  const unsigned blocks = (unsigned)(((int64_t)a.n * 32 + kCacheThreads - 1) / kCacheThreads);
  kv_store_fp8_kernel<<<blocks, kCacheThreads, 0, at::cuda::getCurrentCUDAStream()>>>(a, p);
  AF3_CUDA_CHECK(cudaGetLastError());
}

void kv_gather_fp8(torch::Tensor qkv, int64_t k_off, int64_t v_off, torch::Tensor slots,
                   torch::Tensor k_pages, torch::Tensor v_pages, c10::optional<torch::Tensor> k_scales,
                   c10::optional<torch::Tensor> v_scales) {
  using namespace paged;
  const Pool p = make_pool(k_pages, v_pages, k_scales, v_scales, 8);
  AF3_CHECK(p.ks != nullptr, "kv_gather_fp8 needs float8_e4m3fn pages");
  const RowArgs a = row_args(qkv, k_off, v_off, slots, k_pages);
  if (a.n == 0) return;
  const c10::cuda::CUDAGuard guard(qkv.device());
  const unsigned blocks = (unsigned)(((int64_t)a.n * 32 + kCacheThreads - 1) / kCacheThreads);
  kv_gather_fp8_kernel<<<blocks, kCacheThreads, 0, at::cuda::getCurrentCUDAStream()>>>(a, p);
  AF3_CUDA_CHECK(cudaGetLastError());
}

}  // namespace af3
