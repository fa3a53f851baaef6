// Attention of each sequence's new tokens over its cache pages: arguments, the visibility rule
// and the attention of one (row, head) by one warp, key by key.
//
// Sequence b has seq_lens[b] tokens, the last q_b = cu_q[b + 1] - cu_q[b] of which are queries.
// Query row t of b is at position p = seq_lens[b] - cu_q[b + 1] + t and sees the keys
//   max(0, p - window + 1) <= j <= p     (window 0: 0 <= j <= p)
// whose page exists, i.e. whose page-table entry is in [0, pages); entries past the table's
// width do not exist either.
//   o = sum_j e^{s_j} v_j / (sum_j e^{s_j} + e^{sink_h}),  s_j = scale * q . k_j
// A row that sees nothing gets 0.
#pragma once
#include "paged.cuh"

namespace af3 {
namespace paged {

constexpr int kD = 64;  // head dim
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const __nv_bfloat16* q;  // [T, >= Hq * 64]
  int64_t ld_q;
  __nv_bfloat16* out;
  int64_t ld_out;
  const int* table;  // [B, max_pages]
  int64_t ld_table;
  int max_pages;
  const int* lens;     // [B]
  const int* cu;       // [B + 1]
  const float* sinks;  // [Hq], null: no sink
  int B, T, hq, hkv, group, window;
  float scale_log2;  // softmax scale * log2(e)
  Pool p;
};

// One sequence's rows and lengths, read from device memory and clamped to the tensors.
struct Seq {
  int t0, t1;    // query rows
  int first;     // position of row t0 (may be negative: such rows see nothing)
  int key_end;   // keys [0, key_end) have a page-table entry
};

__device__ __forceinline__ Seq load_seq(const Args& a, int b) {
  Seq s;
  s.t0 = min(max(a.cu[b], 0), a.T);
  s.t1 = min(max(a.cu[b + 1], s.t0), a.T);
  const int len = min(max(a.lens[b], 0), 1 << 30);
  s.first = len - (s.t1 - s.t0);
  const int64_t cap = (int64_t)a.max_pages * a.p.page_size;
  s.key_end = (int)min((int64_t)len, cap);
  return s;
}

// Byte offset of key j's row of KV head g, and of its scale byte; false if its page does not
// exist.  j must be in [0, key_end).
__device__ __forceinline__ bool key_row(const Args& a, const int* table, int j, int g, int64_t& row,
                                        int64_t& scale) {
  uint32_t pi, off;
  split_slot(a.p, (uint32_t)j, pi, off);
  const uint32_t page = (uint32_t)table[pi];
  if (page >= (uint32_t)a.p.num_pages) return false;
  row = (int64_t)page * a.p.page + (int64_t)off * a.p.token + (int64_t)g * a.p.head;
  scale = (int64_t)page * a.p.s_page + (int64_t)off * a.p.s_token + (int64_t)g * a.p.s_head;
  return true;
}

// Attention of query row t (position pos, of the sequence with this page table) and head h by one
// warp: lane l scores key l of each 32, then owns dims 2l, 2l + 1 of the output.  Exact in what it
// touches: a key that is not visible is never read.  Reads keys [lo, hi) only, which the caller
// has cut to the visible ones.
template <bool FP8>
__device__ void warp_row(const Args& a, const int* table, int t, int h, int lo, int hi, float& o0,
                         float& o1) {
  const int lane = threadIdx.x & 31;
  const int g = h / a.group;
  const uint4* qrow = reinterpret_cast<const uint4*>(a.q + (int64_t)t * a.ld_q + (int64_t)h * kD);
  float m = -INFINITY, l = 0.f;
  o0 = o1 = 0.f;
  for (int base = lo; base < hi; base += 32) {
    const int j = base + lane;
    int64_t row = 0, sc = 0;
    const bool vis = j < hi && key_row(a, table, j, g, row, sc);
    float s = -INFINITY, vscale = 1.f;
    if (vis) {
      float dot = 0.f;
#pragma unroll 1
      for (int c = 0; c < kD / 8; ++c) {
        const uint4 qw = qrow[c];
        const __nv_bfloat162* q2 = reinterpret_cast<const __nv_bfloat162*>(&qw);
        if constexpr (FP8) {
          const uint2 kw = reinterpret_cast<const uint2*>(a.p.k + row)[c];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 qf = __bfloat1622float2(q2[e]);
            const uint32_t w = e < 2 ? kw.x : kw.y;
            const float2 kf = f16x2_to_float2(e4m3x2_to_f16x2((uint16_t)(w >> (16 * (e & 1)))));
            dot = fmaf(qf.x, kf.x, fmaf(qf.y, kf.y, dot));
          }
        } else {
          const uint4 kw = reinterpret_cast<const uint4*>(a.p.k + row)[c];
          const __nv_bfloat162* k2 = reinterpret_cast<const __nv_bfloat162*>(&kw);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 qf = __bfloat1622float2(q2[e]);
            const float2 kf = __bfloat1622float2(k2[e]);
            dot = fmaf(qf.x, kf.x, fmaf(qf.y, kf.y, dot));
          }
        }
      }
      if constexpr (FP8) {
        dot *= pow2i((int)a.p.ks[sc] - 127);
        vscale = pow2i((int)a.p.vs[sc] - 127);
      }
      s = dot * a.scale_log2;
    }
    float mx = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float mn = fmaxf(m, mx);
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float alpha = ex2a(m - mu);
    const float pr = vis ? ex2a(s - mu) : 0.f;
    l = l * alpha + pr;  // this lane's keys
    o0 *= alpha;
    o1 *= alpha;
    m = mn;
    const uint32_t there = __ballot_sync(0xffffffffu, vis);
    for (uint32_t left = there; left; left &= left - 1) {
      const int k = __ffs(left) - 1;
      const float pk = __shfl_sync(0xffffffffu, pr, k) * (FP8 ? __shfl_sync(0xffffffffu, vscale, k) : 1.f);
      const int64_t rk = __shfl_sync(0xffffffffu, row, k);
      float2 v;
      if constexpr (FP8) {
        v = f16x2_to_float2(e4m3x2_to_f16x2(reinterpret_cast<const uint16_t*>(a.p.v + rk)[lane]));
      } else {
        v = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(a.p.v + rk)[lane]);
      }
      o0 = fmaf(pk, v.x, o0);
      o1 = fmaf(pk, v.y, o1);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  const float sk = a.sinks != nullptr ? a.sinks[h] * kLog2e : -INFINITY;
  const float top = fmaxf(m, sk);
  if (top == -INFINITY && l == 0.f) {  // nothing visible (or only scores of -inf) and no sink
    o0 = o1 = 0.f;
    return;
  }
  const float f = ex2a(m - top);
  const float inv = f / (l * f + ex2a(sk - top));
  o0 *= inv;
  o1 *= inv;
}

}  // namespace paged
}  // namespace af3
