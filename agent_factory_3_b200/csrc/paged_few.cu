// Attention over cache pages for few query rows a KV head (decoding, short verify blocks).  It reads
// every visible key and value once for each tile of up to 16 rows: 4 KB (e4m3) or 8 KB (bf16) of pages
// against 400 to 500 instructions of a warp for 32 keys, so that memory and issue are both near.
//
// Work: one cluster of S CTAs per (sequence, KV head, tile); the CTAs take contiguous parts of the keys
// and join over distributed shared memory, so there is one launch, no workspace, and a fixed order
// of every sum.  In a CTA each warp runs on its own: every fourth or eighth block of 32 keys,
// copied by cp.async into the warp's ring, with its own running maximum, sum
// and output, merged at the end.
//
// The matrix instructions (m16n8k16) run with the keys as M and the query rows as N, so 8 rows
// waste nothing:
//   S^T = K Q^T      M = 16 keys,  N = 8 rows, K = 64 dims in 4 steps
//   O^T = V^T P^T    M = 16 dims (4 tiles), N = 8 rows, K = 16 keys
// Index permutations make each load of a thread (group g = lane / 4, t = lane % 4) contiguous: in S
// the thread feeds step s with dims 16t + 4s + {0,1} and 16t + 4s + {2,3} of key rows and query
// rows; in O row g of dim tile i is dim 8g + 2i and row g + 8 is dim 8g + 2i + 1.  P^T comes out of
// S^T's accumulator layout by movmatrix (an 8x8 transpose of 16-bit elements).
//
// e4m3 pages: codes are expanded to f16 (exact).  K's scale multiplies the score in fp32.  V's scale
// is folded into P: P' = p * 2^(e - E) with E the largest V exponent seen by this warp so far; O is
// rescaled when E grows.  The largest p is 2^15, so P' keeps f16's 11 bits down to 2^-29 of it (a key of
// less weight counts with fewer bits, below 2^-39 not at all); rows that met exponents more than
// kWideRange apart are taken key by key (the values of the largest may have next to no weight).  Codes
// as bf16 and P' as two bf16 numbers would hold any range, at 18 % more time of the long decode (259 us).
// The query rows are brought to f16 after a power-of-two scaling to [1, 2), undone in fp32.
// (An e4m3 code costs one conversion of half rate; integer conversions took three times as long.)
// bf16 pages: K, V, Q as they are; P as the sum of two bf16 numbers (16 bits), since one alone would
// cost as much precision as the rounding of the output.  The 8 more instructions of 32 keys hide
// behind the copies.
//
// Measured with 64 query heads on 8 KV heads, pages of 64: 128 sequences of 7k tokens on average, e4m3,
// 224 us (4.5 TB/s; at 64-key blocks the kernel issues 390 instructions for 32 keys, bound by latency
// and issue, 45 % of the slots); 2 sequences of 131072, bf16, 97 us (5.5 TB/s, on the 96 SMs that 16
// clusters of 6 take); 128 sequences with a window of 128, bf16, 18.4 us, three round trips to memory
// and the launch.
#include <cooperative_groups.h>

#include <type_traits>

#include "host_utils.h"
#include "paged_attention.h"

namespace cg = cooperative_groups;

namespace af3 {
namespace paged {

constexpr int kMaxSplits = 8;  // the largest portable cluster

// Two shapes of CTA.  Long: 8 warps with 3 blocks of 32 keys in flight each (bf16, tiles of 32 rows) or
// 4 warps with 2 blocks of 64 (e4m3: half the votes, reductions and branches a key).  Short (a part of
// at most 8 blocks: short contexts, sliding windows): 4 warps with 2 blocks of 32 each, small enough
// that four CTAs share an SM; bf16 gets there with one block a warp (128 sequences x 8 KV heads with a
// window of 128, L2 flushed: 24.6 us, against 27.5 us with two).
template <bool FP8, int NT, bool LONG>
struct FewCfg {
  static constexpr int kSub = LONG && FP8 && NT <= 2 ? 2 : 1;  // a block is kSub x 32 keys
  static constexpr int kKeys = 32 * kSub;
  static constexpr int kWarps = LONG && kSub == 1 ? 8 : 4;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kStages = LONG ? (kSub == 1 ? 3 : 2) : (NT == 1 && !FP8 ? 1 : 2);
  static constexpr int kRowBytes = FP8 ? 64 : 128;
  static constexpr int kSubBytes = 2 * 32 * kRowBytes;  // K then V of 32 keys
  static constexpr int kStageBytes = kSub * kSubBytes;
  static constexpr int kRingBytes = kStages * kStageBytes;
  static constexpr int kBlocksPerSm = LONG ? (kSub == 2 ? 3 : 1) : (NT == 1 ? 4 : NT == 2 ? 3 : 2);
  static constexpr float kTop = FP8 ? 15.f : 0.f;  // the largest p of a row is 2^kTop
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a));
  return r;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}
template <bool FP8>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  if constexpr (FP8) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}
template <bool FP8>
__device__ __forceinline__ uint32_t pack16x2(float lo, float hi) {
  uint32_t r;
  if constexpr (FP8)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Byte offset of 16-byte chunk c of key row r inside a block.  e4m3: two 64-byte rows share a
// 128-byte line, chunks xored by twice the line's low bits; bf16: chunks xored by the row's low
// bits.  Both leave the copies and both access patterns below free of bank conflicts.
template <bool FP8>
__device__ __forceinline__ uint32_t chunk_at(int r, int c) {
  if constexpr (FP8) {
    const int line = r >> 1;
    return (uint32_t)(line * 128 + ((((r & 1) * 4 + c) ^ ((line & 3) << 1)) << 4));
  } else {
    return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4));
  }
}

// Zeroes what is not finite in 16 bytes of V; true if there was something.
template <bool FP8>
__device__ __forceinline__ bool clear_nonfinite(uint32_t addr) {
  uint4 w = lds128(addr);
  uint32_t* x = reinterpret_cast<uint32_t*>(&w);
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t m = FP8 ? __vcmpeq4(x[i] & 0x7f7f7f7fu, 0x7f7f7f7fu) : __vcmpeq2(x[i] & 0x7f807f80u, 0x7f807f80u);
    bad |= m != 0;
    x[i] &= ~m;
  }
  if (bad)
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
  return bad;
}

// What is remembered of 32 keys on their way: the ones that exist, and lane l's scale bytes of key l.
// The bytes stay as loaded until the block is used; combining them at once would wait for them.
struct Keys {
  uint32_t there, k, v;
};

// Page of key base + lane (of key base where a block lies in one page), -1 when the key is out of
// range.  Loaded a block before it is needed.
template <bool ONE>
__device__ __forceinline__ int block_page(const Args& a, const int* table, int base, int lo, int hi) {
  const int j = ONE ? base : base + (int)(threadIdx.x & 31);
  if (!ONE && (j < lo || j >= hi)) return -1;
  return table[a.p.page_shift >= 0 ? j >> a.p.page_shift : j / a.p.page_size];
}

// Starts the copies of keys base .. base + 31.
// ONE: the block lies in one page (pages of a multiple of 32 keys), so that the rows' addresses
// differ by constants: a third of the instructions.  kb, vb: the pools at this lane's piece of row 0.
template <class C, bool FP8, bool ONE>
__device__ __forceinline__ Keys issue_block(const Args& a, const uint8_t* kb, const uint8_t* vb, const uint8_t* ksb,
                                                const uint8_t* vsb, int page, int g, int base, int lo, int hi, uint32_t dst) {
  const int lane = threadIdx.x & 31;
  constexpr int kChunks = C::kRowBytes / 16, kRowsPer = 32 / kChunks;
  const int c = lane % kChunks, r0 = lane / kChunks;
  bool there = (uint32_t)page < (uint32_t)a.p.num_pages;
  uint32_t pi, off;
  Keys info{0, 0, 0};
  if constexpr (ONE) {
    const bool inside = base >= lo && base + 32 <= hi;
    if (there) {
      split_slot(a.p, (uint32_t)base, pi, off);
      const int64_t start = (int64_t)page * a.p.page + (int64_t)off * a.p.token;
      const uint8_t *ks = kb + start, *vs = vb + start;
      const int64_t step = (int64_t)kRowsPer * a.p.token;
      if (inside) {
#pragma unroll
        for (int i = 0; i < 32 / kRowsPer; ++i) {
          const uint32_t d = dst + chunk_at<FP8>(i * kRowsPer + r0, c);
          cp_async16(d, ks);
          cp_async16(d + 32 * C::kRowBytes, vs);
          ks += step;
          vs += step;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 32 / kRowsPer; ++i) {
          const int key = base + i * kRowsPer + r0;
          const bool on = key >= lo && key < hi;
          const uint32_t d = dst + chunk_at<FP8>(i * kRowsPer + r0, c);
          cp_async16(d, ks, on);
          cp_async16(d + 32 * C::kRowBytes, vs, on);
          ks += step;
          vs += step;
        }
      }
      const bool mine = inside || (base + lane >= lo && base + lane < hi);
      info.there = __ballot_sync(0xffffffffu, mine);
      if constexpr (FP8) {
        const int64_t sc = (int64_t)page * a.p.s_page + (int64_t)off * a.p.s_token;
        info.k = load_byte(ksb + sc, mine);
        info.v = load_byte(vsb + sc, mine);
      }
      return info;
    }
#pragma unroll
    for (int i = 0; i < 32 / kRowsPer; ++i) {
      const uint32_t d = dst + chunk_at<FP8>(i * kRowsPer + r0, c);
      cp_async16(d, kb, false);
      cp_async16(d + 32 * C::kRowBytes, vb, false);
    }
    return info;
  } else {
    int64_t row = 0, sc = 0;
    if (there) {
      split_slot(a.p, (uint32_t)(base + lane), pi, off);
      row = (int64_t)page * a.p.page + (int64_t)off * a.p.token + (int64_t)g * a.p.head;
      sc = (int64_t)page * a.p.s_page + (int64_t)off * a.p.s_token + (int64_t)g * a.p.s_head;
    }
    if constexpr (FP8) {
      info.k = load_byte(a.p.ks + sc, there);
      info.v = load_byte(a.p.vs + sc, there);
    }
    // the rows' offsets travel by shuffle; a missing row has offset 0 and is filled with zeros
    const uint32_t mask = __ballot_sync(0xffffffffu, there);
    info.there = mask;
#pragma unroll
    for (int i = 0; i < 32 / kRowsPer; ++i) {
      const int r = i * kRowsPer + r0;
      const int64_t at = __shfl_sync(0xffffffffu, row, r) + c * 16;
      const bool on = (mask >> r) & 1u;
      const uint32_t d = dst + chunk_at<FP8>(r, c);
      cp_async16(d, a.p.k + at, on);
      cp_async16(d + 32 * C::kRowBytes, a.p.v + at, on);
    }
    return info;
  }
}

template <bool FP8, int NT, bool LONG, bool ONE>
__global__ void __launch_bounds__(FewCfg<FP8, NT, LONG>::kThreads, FewCfg<FP8, NT, LONG>::kBlocksPerSm)
    paged_few_kernel(const Args a, const int rows_per_tile, const int tiles, const int splits) {
  using C = FewCfg<FP8, NT, LONG>;
  constexpr int kWarps = C::kWarps, kStages = C::kStages;
  constexpr int R = NT * 8;  // query rows of a tile
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_m[kWarps][R], s_l[kWarps][R];
  __shared__ float c_m[R], c_l[R];
  __shared__ int s_wide[kWarps];
  float* c_o = reinterpret_cast<float*>(smem + kWarps * C::kRingBytes);  // [R][64], this CTA's part
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int grp = lane >> 2, tig = lane & 3;
  const int rank = splits > 1 ? (int)blockIdx.x : 0;
  const int g = blockIdx.y / tiles, b = blockIdx.z;
  const Seq sq = load_seq(a, b);
  const int tokens_per_tile = rows_per_tile / a.group;
  const int* table = a.table + (int64_t)b * a.ld_table;
  uint8_t* ring = smem + warp * C::kRingBytes;
  const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring);
  constexpr int kChunks = C::kRowBytes / 16;
  const int64_t piece = (int64_t)g * a.p.head + (lane / kChunks) * a.p.token + (lane % kChunks) * 16;
  const int64_t byte = (int64_t)g * a.p.s_head + lane * a.p.s_token;
  const uint8_t *kb0 = a.p.k + piece, *vb0 = a.p.v + piece, *ksb = a.p.ks + byte, *vsb = a.p.vs + byte;

  // (one round when the caller's longest q is right)
  for (int tok0 = sq.t0 + (int)(blockIdx.y % tiles) * tokens_per_tile; tok0 < sq.t1; tok0 += tiles * tokens_per_tile) {
    const int ntok = min(tokens_per_tile, sq.t1 - tok0);
    const int nrows = ntok * a.group;
    const bool several = ntok > 1;  // rows differ in what they see
    const int pos0 = sq.first + (tok0 - sq.t0);  // position of the tile's first token
    // keys that any row of the tile may see
    const int lo = a.window > 0 ? max(0, pos0 - a.window + 1) : 0;
    const int hi = min(pos0 + ntok, sq.key_end);
    const int blk0 = lo / C::kKeys, blk1 = max((hi + C::kKeys - 1) / C::kKeys, blk0);
    const int per = (blk1 - blk0 + splits - 1) / splits;
    const int my0 = min(blk0 + rank * per, blk1), my1 = min(my0 + per, blk1);

    // ---- the first copies, before anything waits for the query rows
    Keys info[kStages][C::kSub];
    const int first = my0 + warp;
    int ahead_page[C::kSub];  // pages of the next block to copy
    auto load_pages = [&](int blk) {
#pragma unroll
      for (int u = 0; u < C::kSub; ++u)
        if (C::kSub == 1 || (blk * C::kSub + u) * 32 < hi)
          ahead_page[u] = block_page<ONE>(a, table, (blk * C::kSub + u) * 32, lo, hi);
        else
          ahead_page[u] = -1;
    };
    auto copy_block = [&](int blk, Keys (&inf)[C::kSub], uint32_t dst) {
      int page[C::kSub];
#pragma unroll
      for (int u = 0; u < C::kSub; ++u) page[u] = ahead_page[u];
      if (blk + kWarps < my1) load_pages(blk + kWarps);
#pragma unroll
      for (int u = 0; u < C::kSub; ++u)
        inf[u] = issue_block<C, FP8, ONE>(a, kb0, vb0, ksb, vsb, page[u], g, (blk * C::kSub + u) * 32, lo, hi,
                                          dst + u * C::kSubBytes);
    };
    if (first < my1) load_pages(first);
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s) {
      if (first + s * kWarps < my1) copy_block(first + s * kWarps, info[s], ring_s + s * C::kStageBytes);
      cp_async_commit();
    }

    // ---- query rows: thread (grp, tig) holds dims [16 tig, 16 tig + 16) of rows nt * 8 + grp
    uint32_t qf[NT][8];
    float smul[NT][2];  // rows nt * 8 + 2 tig + {0, 1}: softmax scale * log2(e) * the row's scaling
    int rlo[NT][2], rhi[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + grp;
      uint4 w0 = make_uint4(0, 0, 0, 0), w1 = w0;
      if (r < nrows) {
        const uint4* src = reinterpret_cast<const uint4*>(
            a.q + (int64_t)(tok0 + r / a.group) * a.ld_q + (int64_t)(g * a.group + r % a.group) * kD + 16 * tig);
        w0 = src[0];
        w1 = src[1];
      }
      const uint32_t w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
      float back = 1.f;
      if constexpr (FP8) {
        uint32_t mx = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) mx = max(mx, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        int e = (int)(mx >> 7) - 127;  // largest magnitude in [2^e, 2^(e+1))
        if (e > 126 || e < -126) e = 0;  // zero, denormal, infinite or NaN rows: as they are
        const float f = pow2i(-e);
        back = pow2i(e);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float lo16 = __uint_as_float(w[i] << 16), hi16 = __uint_as_float(w[i] & 0xffff0000u);
          qf[nt][i] = pack16x2<true>(lo16 * f, hi16 * f);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) qf[nt][i] = w[i];
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        smul[nt][c] = a.scale_log2 * __shfl_sync(0xffffffffu, back, (2 * tig + c) * 4);
        const int rr = nt * 8 + 2 * tig + c;
        const int p = pos0 + (rr < nrows ? rr / a.group : 0);
        rhi[nt][c] = rr < nrows ? p : -1;
        rlo[nt][c] = a.window > 0 ? p - a.window + 1 : 0;
      }
    }
    // a block is full when every row sees all of it
    const int full_lo = a.window > 0 ? pos0 + ntok - a.window : 0, full_hi = min(pos0 + 1, sq.key_end);

    float m[NT][2], l[NT][2], o[NT][4][4];
    int vmax = 0, vmin = 255;  // V's scale bytes seen (blocks of this warp); vmin skips zero rows
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
    }

    for (int blk = first; blk < my1; blk += kStages * kWarps) {
#pragma unroll
      for (int s = 0; s < kStages; ++s) {
        const int cur = blk + s * kWarps;
        if (cur >= my1) break;
        {
          constexpr int ahead = kStages - 1;
          const int slot = (s + ahead) % kStages;
          const int nxt = cur + ahead * kWarps;
          __syncwarp();  // every lane has read the block that this slot held
          if (nxt < my1) copy_block(nxt, info[slot], ring_s + slot * C::kStageBytes);
          cp_async_commit();
        }
        cp_async_wait<kStages - 1>();
        __syncwarp();
        const uint32_t kv = ring_s + s * C::kStageBytes;
        const int base = cur * C::kKeys;

        uint32_t there[C::kSub], broken[C::kSub];  // a bit for each key
        bool full = base >= full_lo && base + C::kKeys <= full_hi;
#pragma unroll
        for (int u = 0; u < C::kSub; ++u) {
          there[u] = info[s][u].there;
          full &= there[u] == 0xffffffffu;
          broken[u] = 0;
        }
        // A value that is not finite would reach every row through 0 * inf.  Where rows differ in
        // what they see, such values are taken out of the block (which leaves the rows that do not
        // see them as they are), and the rows that see them are taken again at the end.
        if (several && !full) {
#pragma unroll
          for (int u = 0; u < C::kSub; ++u) {
            bool bad = false;
#pragma unroll 1
            for (int c = 0; c < C::kRowBytes / 16; ++c)
              bad |= clear_nonfinite<FP8>(kv + u * C::kSubBytes + 32 * C::kRowBytes + chunk_at<FP8>(lane, c));
            broken[u] = __ballot_sync(0xffffffffu, bad);
          }
          __syncwarp();
        }

        // ---- S^T, keys base + 16 mt + {grp, grp + 8}
        float sc[2 * C::kSub][NT][4];
#pragma unroll
        for (int mt = 0; mt < 2 * C::kSub; ++mt) {
          const uint32_t kb = kv + (mt >> 1) * C::kSubBytes;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) sc[mt][nt][0] = sc[mt][nt][1] = sc[mt][nt][2] = sc[mt][nt][3] = 0.f;
          const int r0 = (mt & 1) * 16 + grp, r1 = r0 + 8;
          if constexpr (FP8) {
            const uint4 x = lds128(kb + chunk_at<true>(r0, tig)), y = lds128(kb + chunk_at<true>(r1, tig));
            const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
              uint32_t a0, a1, a2, a3;
              e4m3x4_to_f16x2(xw[ks], a0, a2);
              e4m3x4_to_f16x2(yw[ks], a1, a3);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
                mma16816<true>(sc[mt][nt], a0, a1, a2, a3, qf[nt][2 * ks], qf[nt][2 * ks + 1]);
            }
          } else {
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              const uint4 x = lds128(kb + chunk_at<false>(r0, 2 * tig + hf));
              const uint4 y = lds128(kb + chunk_at<false>(r1, 2 * tig + hf));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816<false>(sc[mt][nt], x.x, y.x, x.y, y.y, qf[nt][4 * hf], qf[nt][4 * hf + 1]);
                mma16816<false>(sc[mt][nt], x.z, y.z, x.w, y.w, qf[nt][4 * hf + 2], qf[nt][4 * hf + 3]);
              }
            }
          }
        }
        // ---- scales of this thread's keys (computed by the key's lane), masks
        float kmul[4 * C::kSub], vmul[4 * C::kSub];
        bool grew = false;
        float shrink = 1.f;
        if constexpr (FP8) {
          int mine[C::kSub];
          int most = 0;
#pragma unroll
          for (int u = 0; u < C::kSub; ++u) {
            mine[u] = ((broken[u] >> lane) & 1u) ? 0 : (int)info[s][u].v;  // absent: 0
            vmin = min(vmin, mine[u] > 0 ? mine[u] : 255);
            most = max(most, mine[u]);
          }
          const int top = (int)__reduce_max_sync(0xffffffffu, (unsigned)most);
          grew = top > vmax;
          if (grew) {
            shrink = pow2i(max(vmax - top, -127));
            vmax = top;
          }
#pragma unroll
          for (int u = 0; u < C::kSub; ++u) {
            const float kf = __uint_as_float(max(info[s][u].k << 23, 0x400000u));  // (2^-127 is a denormal)
            const float vf = __uint_as_float((uint32_t)max(mine[u] - vmax + 127, 0) << 23);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              kmul[4 * u + k] = __shfl_sync(0xffffffffu, kf, grp + 8 * k);
              vmul[4 * u + k] = __shfl_sync(0xffffffffu, vf, grp + 8 * k);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 4 * C::kSub; ++k) {  // keys grp + 8 k: mt = k / 2, accumulator half k % 2
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) sc[k >> 1][nt][2 * (k & 1) + c] *= FP8 ? smul[nt][c] * kmul[k] : smul[nt][c];
          }
        }
        if (!full) {
#pragma unroll
          for (int k = 0; k < 4 * C::kSub; ++k) {
            const int bit = grp + 8 * (k & 3), key = base + grp + 8 * k;
            const bool on = (there[k >> 2] >> bit) & 1u, bad = (broken[k >> 2] >> bit) & 1u;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                if (!(on && key >= rlo[nt][c] && key <= rhi[nt][c]))
                  sc[k >> 1][nt][2 * (k & 1) + c] = -INFINITY;
                else if (bad)
                  l[nt][c] = __uint_as_float(0x7fc00000u);
              }
            }
          }
        }
        // ---- running reference
        bool need = false;
        float mx[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float x = fmaxf(sc[0][nt][c], sc[0][nt][2 + c]);
#pragma unroll
            for (int mt = 1; mt < 2 * C::kSub; ++mt) x = fmaxf(x, fmaxf(sc[mt][nt][c], sc[mt][nt][2 + c]));
            mx[nt][c] = x - C::kTop;
            need |= mx[nt][c] > m[nt][c];
          }
        }
        if (__any_sync(0xffffffffu, need)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float x = mx[nt][c];
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
              if (x > m[nt][c]) {
                const float f = ex2a(m[nt][c] - x);  // 0 from -inf
                m[nt][c] = x;
                l[nt][c] *= f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  o[nt][i][c] *= f;
                  o[nt][i][2 + c] *= f;
                }
              }
            }
          }
        }
        if (FP8 && grew) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
              for (int e = 0; e < 4; ++e) o[nt][i][e] *= shrink;
            }
        }
        // ---- P^T as B fragments
        uint32_t pb[2 * C::kSub][NT][2], pl[2 * C::kSub][NT][2];  // pl: what pb's bf16 leaves out
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float mu0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], mu1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
          for (int k = 0; k < 4 * C::kSub; ++k) {
            float p0 = ex2a(sc[k >> 1][nt][2 * (k & 1)] - mu0);
            float p1 = ex2a(sc[k >> 1][nt][2 * (k & 1) + 1] - mu1);
            l[nt][0] += p0;
            l[nt][1] += p1;
            if constexpr (FP8) {
              p0 *= vmul[k];
              p1 *= vmul[k];
            }
            const uint32_t w = pack16x2<FP8>(p0, p1);
            pb[k >> 1][nt][k & 1] = transpose8x8(w);
            if constexpr (!FP8)
              pl[k >> 1][nt][k & 1] = transpose8x8(
                  pack16x2<false>(p0 - __uint_as_float(w << 16), p1 - __uint_as_float(w & 0xffff0000u)));
          }
        }
        // ---- O^T += V^T P^T
#pragma unroll
        for (int mt = 0; mt < 2 * C::kSub; ++mt) {
          const uint32_t vb = kv + (mt >> 1) * C::kSubBytes + 32 * C::kRowBytes;
          const int r = (mt & 1) * 16 + 2 * tig;
          if constexpr (FP8) {
            // dims [8 grp, 8 grp + 8): half of chunk grp / 2
            const uint32_t in = (uint32_t)(grp & 1) * 8;
            const uint2 x = lds64(vb + chunk_at<true>(r, grp >> 1) + in);
            const uint2 y = lds64(vb + chunk_at<true>(r + 1, grp >> 1) + in);
            const uint2 z = lds64(vb + chunk_at<true>(r + 8, grp >> 1) + in);
            const uint2 u = lds64(vb + chunk_at<true>(r + 9, grp >> 1) + in);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              // bytes of dims 2i, 2i + 1 of two keys -> (key, key + 1) of dim 2i, then of dim 2i + 1
              const uint32_t sel = (i & 1) ? 0x7362u : 0x5140u;
              const uint32_t xy = __byte_perm(i < 2 ? x.x : x.y, i < 2 ? y.x : y.y, sel);
              const uint32_t zu = __byte_perm(i < 2 ? z.x : z.y, i < 2 ? u.x : u.y, sel);
              uint32_t a0, a1, a2, a3;
              e4m3x4_to_f16x2(xy, a0, a1);
              e4m3x4_to_f16x2(zu, a2, a3);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816<true>(o[nt][i], a0, a1, a2, a3, pb[mt][nt][0], pb[mt][nt][1]);
            }
          } else {
            const uint4 x = lds128(vb + chunk_at<false>(r, grp)), y = lds128(vb + chunk_at<false>(r + 1, grp));
            const uint4 z = lds128(vb + chunk_at<false>(r + 8, grp)), u = lds128(vb + chunk_at<false>(r + 9, grp));
            const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
            const uint32_t zw[4] = {z.x, z.y, z.z, z.w}, uw[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t a0 = __byte_perm(xw[i], yw[i], 0x5410), a1 = __byte_perm(xw[i], yw[i], 0x7632);
              const uint32_t a2 = __byte_perm(zw[i], uw[i], 0x5410), a3 = __byte_perm(zw[i], uw[i], 0x7632);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma16816<false>(o[nt][i], a0, a1, a2, a3, pb[mt][nt][0], pb[mt][nt][1]);
                mma16816<false>(o[nt][i], a0, a1, a2, a3, pl[mt][nt][0], pl[mt][nt][1]);
              }
            }
          }
        }
      }
    }
    cp_async_wait<0>();
    __syncwarp();

    // ---- this warp's part, normalised: (m, l, o / l)
    float* w_o = reinterpret_cast<float*>(ring);  // [R][64] over the warp's ring
    const float vscale = FP8 ? pow2i(vmax - 127) : 1.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float x = l[nt][c];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        const int r = nt * 8 + 2 * tig + c;
        const float inv = x == 0.f ? 0.f : 1.f / x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          *reinterpret_cast<float2*>(w_o + r * kD + 8 * grp + 2 * i) =
              make_float2(o[nt][i][c] * inv * vscale, o[nt][i][2 + c] * inv * vscale);
        }
        if (grp == 0) {
          s_m[warp][r] = m[nt][c];
          s_l[warp][r] = x;
        }
      }
    }
    if constexpr (FP8) {
      const int least = (int)__reduce_min_sync(0xffffffffu, (unsigned)vmin);
      if (lane == 0) s_wide[warp] = vmax - least > kWideRange;
    }
    __syncthreads();
    // ---- join the warps: one warp a row, lane l has dims 2l, 2l + 1
    bool wide = false;
    if constexpr (FP8) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) wide |= s_wide[w] != 0;
    }
    for (int r = warp; r < nrows; r += kWarps) {
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, s_m[w][r]);
      const float mu = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = s_l[w][r] * ex2a(s_m[w][r] - mu);
        const float2 v = reinterpret_cast<const float2*>(smem + w * C::kRingBytes)[r * (kD / 2) + lane];
        ll += f;
        x = fmaf(f, v.x, x);
        y = fmaf(f, v.y, y);
      }
      const float inv = ll == 0.f ? 0.f : 1.f / ll;
      reinterpret_cast<float2*>(c_o)[r * (kD / 2) + lane] = make_float2(x * inv, y * inv);
      if (lane == 0) {
        c_m[r] = mm;
        c_l[r] = wide ? __uint_as_float(0x7fc00000u) : ll;  // NaN: the row is taken key by key
      }
    }
    if (splits > 1) cg::this_cluster().sync(); else __syncthreads();
    // ---- join the CTAs; row r belongs to one warp of the cluster
    for (int r = rank * kWarps + warp; r < nrows; r += splits * kWarps) {
      const int h = g * a.group + r % a.group, t = tok0 + r / a.group;
      const float sk = a.sinks != nullptr ? a.sinks[h] * kLog2e : -INFINITY;
      float mc = -INFINITY, lc = 0.f;
      if (lane < splits) {
        mc = splits > 1 ? *cg::this_cluster().map_shared_rank(&c_m[r], lane) : c_m[r];
        lc = splits > 1 ? *cg::this_cluster().map_shared_rank(&c_l[r], lane) : c_l[r];
      }
      float top = fmaxf(mc, sk);
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float tu = top == -INFINITY ? 0.f : top;
      const float f = lc * ex2a(mc - tu);
      float den = f;
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) den += __shfl_xor_sync(0xffffffffu, den, x);
      den += ex2a(sk - tu);
      float x = 0.f, y = 0.f;
      const float2* mine = reinterpret_cast<const float2*>(c_o) + r * (kD / 2) + lane;
      float2 v[kMaxSplits];  // every CTA's part is asked for before the first is used
#pragma unroll
      for (int c = 0; c < kMaxSplits; ++c) {
        v[c] = make_float2(0.f, 0.f);
        if (c < splits) v[c] = splits > 1 ? *cg::this_cluster().map_shared_rank(mine, c) : *mine;
      }
#pragma unroll
      for (int c = 0; c < kMaxSplits; ++c) {
        const float fc = __shfl_sync(0xffffffffu, f, c);
        if (c < splits) {
          x = fmaf(fc, v[c].x, x);
          y = fmaf(fc, v[c].y, y);
        }
      }
      const float inv = den == 0.f ? 0.f : 1.f / den;
      x *= inv;
      y *= inv;
      // Rows that see a value that is not finite (an infinity comes out of the two halves of P as
      // NaN), and tiles of too wide a range: key by key.
      const bool bad = !(fabsf(x) < INFINITY && fabsf(y) < INFINITY);
      if (__any_sync(0xffffffffu, bad)) {
        const int p = pos0 + r / a.group;
        warp_row<FP8>(a, table, t, h, a.window > 0 ? max(0, p - a.window + 1) : 0, min(p + 1, sq.key_end), x, y);
      }
      reinterpret_cast<__nv_bfloat162*>(a.out + (int64_t)t * a.ld_out + (int64_t)h * kD)[lane] =
          __floats2bfloat162_rn(x, y);
    }
    // parts may be overwritten (next tile) or go away (exit) only when every CTA has read them
    if (splits > 1) cg::this_cluster().sync(); else __syncthreads();
  }
}

// How many clusters of `splits` CTAs the device holds at once.  Clusters lie within one GPC, so this
// is less than the number of CTAs that fit divided by the size (16 clusters of 6 fit, not of 7).
template <class K>
static int clusters_at_once(K kern, const cudaLaunchConfig_t& cfg) {
  int n = 0;
  AF3_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
  return std::max(n, 1);
}

template <bool FP8, int NT, bool LONG, bool ONE>
static void launch_few_nt(const Args& a, int rows_per_tile, int max_q, int64_t keys, cudaStream_t stream) {
  using C = FewCfg<FP8, NT, LONG>;
  constexpr int smem = C::kWarps * C::kRingBytes + NT * 8 * kD * 4;
  static_assert(NT * 8 * kD * 4 <= C::kRingBytes, "a warp's part has to fit its ring");
  auto kern = paged_few_kernel<FP8, NT, LONG, ONE>;
  static int at_once[64][kMaxSplits + 1] = {};
  int dev;
  AF3_CUDA_CHECK(cudaGetDevice(&dev));
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (at_once[dev][1] == 0) {
    AF3_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    for (int s = kMaxSplits; s >= 1; --s) {
      attr[0].val.clusterDim = {(unsigned)s, 1, 1};
      cfg.gridDim = dim3((unsigned)s, 1024, 1);
      at_once[dev][s] = clusters_at_once(kern, cfg);
    }
  }
  // The keys are split so that the number of rounds of clusters times the length of one is least:
  // a CTA takes as long as kFixed keys to begin and to end (5 us against some 150 keys a us), and
  // half a round is lost at the end when there are several.
  const int tokens = rows_per_tile / a.group, tiles = (max_q + tokens - 1) / tokens;
  const int64_t items = (int64_t)a.B * a.hkv * tiles;
  constexpr double kFixed = 768;
  int splits = 1;
  double best = 0;
  for (int s = 1; s <= kMaxSplits; ++s) {
    const double rounds = (double)items / at_once[dev][s];
    const double cost = (rounds <= 1 ? 1 : rounds + 0.5) * (kFixed + (double)keys / s);
    if (s == 1 || cost < best) {
      best = cost;
      splits = s;
    }
  }
  cfg.gridDim = dim3((unsigned)splits, (unsigned)(a.hkv * tiles), (unsigned)a.B);
  attr[0].val.clusterDim = {(unsigned)splits, 1, 1};
  cfg.numAttrs = splits > 1 ? 1 : 0;
  AF3_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, a, rows_per_tile, tiles, splits));
}

template <bool FP8, bool LONG, bool ONE>
static void launch_few_t(const Args& a, int max_q, int64_t keys, cudaStream_t stream) {
  // Up to 16 rows in one tile.  More rows take tiles of 16 that read the keys side by side, from L2
  // but for one of them: 64 sequences of 5 tokens (40 rows) on 4200 take 259 us so, 341 us in tiles of
  // 32, whose registers leave half the warps (e4m3; of 1 to 5 tokens on 210 to 4200, 115 and 133 us).  A group of more than 16 heads needs the larger tile.
  const int rows = a.group > 16 ? kFewRows : 16;
  const int want = std::max(std::min(max_q, rows / a.group), 1) * a.group;  // rows of a tile
  if (want <= 8)
    launch_few_nt<FP8, 1, LONG, ONE>(a, want, max_q, keys, stream);
  else if (want <= 16)
    launch_few_nt<FP8, 2, LONG, ONE>(a, want, max_q, keys, stream);
  else
    launch_few_nt<FP8, 4, LONG, ONE>(a, want, max_q, keys, stream);
}

void launch_few(const Args& a, int64_t max_q, int64_t max_len, cudaStream_t stream) {
  const int64_t keys = a.window > 0 ? std::min<int64_t>(max_len, a.window + max_q) : max_len;
  const int q = (int)std::min<int64_t>(max_q, kFewTotal);
  // 8 blocks of 32 keys for 4 warps; a part of more in the short shape only runs slower
  const bool is_long = keys > 256 && (keys > 8 * 256 || (int64_t)a.B * a.hkv * 8 > 3 * (int64_t)num_sms());
  const bool one = (a.p.page_size & 31) == 0;
  auto go = [&](auto fp8, auto lng, auto on) {
    launch_few_t<decltype(fp8)::value, decltype(lng)::value, decltype(on)::value>(a, q, keys, stream);
  };
  using T = std::true_type;
  using F = std::false_type;
  auto pick2 = [&](auto fp8, auto lng) { one ? go(fp8, lng, T{}) : go(fp8, lng, F{}); };
  auto pick = [&](auto fp8) { is_long ? pick2(fp8, T{}) : pick2(fp8, F{}); };
  a.p.ks != nullptr ? pick(T{}) : pick(F{});
}

}  // namespace paged
}  // namespace af3
