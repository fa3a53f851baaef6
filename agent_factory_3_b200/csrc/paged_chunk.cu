// Attention over cache pages for many query rows a KV head (prefill chunks, longer verify blocks),
// on the fifth-generation tensor cores.
//
// One CTA per (span of up to 2 x 128 query rows, KV head); a row is a (token, query head of the
// group) pair, floor(128 / group) tokens a tile, so the whole group shares every K/V block.  Few
// spans over a long context are split: the CTAs of a cluster take parts of the keys and join over
// distributed shared memory.
//   warps 0-2    loaders of 96-key blocks by cp.async, four ahead (any page size and stride), 32 keys each:
//                bf16 rows of K and V straight into 128B-swizzled tiles; e4m3 rows of V as raw pieces that
//                the thread which copied them expands into a bf16 tile, scale included (code * 2^e is a
//                bf16 number)
//   warps 4-11   softmax, one warpgroup per 128-row tile: thread t owns query row t
//   warp 12      tcgen05 issuer: S = Q K^T (M 128, N 96, K 64) of the next block is issued before
//                O += P V (M 128, N 64, K 96, P from TMEM) of this one
//   warps 13-15  e4m3: loaders of K, by the same instructions as V's
// One bf16 P would cost as much precision as the rounding of the output, and an f16 P (11 bits down to
// 2^-14, nothing below 2^-24) loses what a row gets from keys of little weight, which is all it has in a
// channel where the others' codes are 0; V scaled to f16 has the like trouble with its own range.  So K, V and
// Q are bf16 as they are, and P is two bf16 numbers, its first 8 bits and the next 8 (two products): nothing
// depends on the magnitudes met elsewhere.  The softmax reference is the running maximum itself, so that a
// row that one key dominates comes out as that key's value.
// P takes as many TMEM columns as S and lies over it; two S of 96 columns a tile let the next block's
// product start before this one's P is used (one S of 128: 2.04 ms where this takes 1.75).
// TMEM: S / P of tile A 0 and 96, of tile B 192 and 288, O 384 and 448.
//
// Measured with 64 query heads on 8 KV heads, 4096 rows over 12288 cached keys: bf16 pages 1.75 ms (550
// TFLOP/s), e4m3 1.92 ms, where the loaders' expansion takes issue slots from the softmax's dependent
// chains.  The exponentials alone take 0.86 ms (16 a cycle and SM).  e4m3 with f16 tiles and an f16 P took
// 1.60 ms, but 30 of 600 random batches of widely spread scores were off by up to all of a small element
// (of 32-bit torch's, 1).  Tried and slower for e4m3: one set of loaders for K and V (1.94 ms; a verify block
// of 9 rows 210 against 196 us), two with instructions of their own (2.15 ms); for both: four softmax
// streams of 64 keys, rolled loops in the issuer, spinning or sleeping waits.
//
// Rows that do not see a value must not meet it as 0 * inf: blocks that are not fully visible to
// the whole span have such values cleared by the loaders and their keys reported; rows that do see
// one are taken key by key at the end.
#include <cooperative_groups.h>

#include "common.h"
#include "host_utils.h"
#include "paged_attention.h"
#include "sm100.cuh"

namespace cg = cooperative_groups;

namespace af3 {
namespace paged {

constexpr int kChunkThreads = 512;
constexpr int kQTile = 128 * kD * 2;  // 16 KB: 128 rows of Q
constexpr uint32_t kColO = 384;
constexpr int kBK = 96;               // keys of a block
constexpr int kLoaders = kBK / 32;    // warps, 32 keys each
constexpr int kTile = kBK * kD * 2;   // 12 KB: a bf16 tile of K or V; e4m3: also a raw block

// Stages and where things lie in shared memory.
template <bool FP8>
struct Cfg {
  static constexpr int kST = FP8 ? 5 : 6;        // stages of K/V tiles
  static constexpr int kAhead = 4;               // blocks whose copies are in flight
  static constexpr int Q = 0;                    // 2 tiles
  static constexpr int K = Q + 2 * kQTile;       // kST tiles
  static constexpr int V = K + kST * kTile;      // kST tiles
  static constexpr int RAW = V + kST * kTile;    // e4m3: kAhead raw blocks, V's half and K's, own 16-byte pieces of each thread
  static constexpr int kBytes = RAW + (FP8 ? kAhead * kTile : 0);
  static_assert(256 * kD * 4 <= 2 * kST * kTile, "a CTA's parts lie over its K and V tiles");
};

// TMEM column of block c's S, and of the P over it, of tile x
__device__ __forceinline__ uint32_t col_s(int x, int c) { return x * 192 + (c & 1) * 96; }

struct StageInfo {
  uint32_t there[4];   // keys that exist and lie in the span's range, but for the broken ones
  uint32_t broken[4];  // those whose V is not finite (cleared), in blocks not seen by every row
};

constexpr int kMaxST = 6;
struct ChunkBars {
  uint64_t q_full, kv_full[kMaxST], kv_empty[kMaxST], s_full[2], p_full[2], o_ready[2];
  uint32_t tmem;
  int abort_flag;
  StageInfo info[kMaxST];
  float row_m[256], row_l[256];
};
static_assert(sizeof(ChunkBars) <= 4096, "");

// 16-byte chunk c of row r of a 128B-swizzled tile of 128-byte rows
__device__ __forceinline__ uint32_t sw128(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

__device__ __forceinline__ uint64_t pk2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void upk2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// bf16 pair of a scale byte's power of two, 2^(b - 127); 255: infinity
__device__ __forceinline__ uint32_t scale_bf16x2(uint32_t b) {
  const uint32_t h = b ? b << 7 : 0x40u;
  return h | (h << 16);
}

// The keys a tile's rows see, and its blocks within this CTA's part.
struct Tile {
  int tok0, ntok, pos0;
  int jlo, jhi;  // blocks, absolute; empty when jhi <= jlo
};

__device__ __forceinline__ Tile make_tile(const Args& a, const Seq& s, int tok0, int tokens, int kv_lo, int b0, int b1) {
  Tile t;
  t.tok0 = tok0;
  t.ntok = max(0, min(tokens, s.t1 - tok0));
  t.pos0 = s.first + (tok0 - s.t0);
  const int lo = a.window > 0 ? max(0, t.pos0 - a.window + 1) : 0;
  const int hi = min(t.pos0 + t.ntok, s.key_end);
  t.jlo = t.jhi = b0;
  if (t.ntok > 0 && hi > lo) {
    t.jlo = max(b0, (lo - kv_lo) / kBK);
    t.jhi = min(b1, (hi - 1 - kv_lo) / kBK + 1);
  }
  return t;
}

// The sequence of a span slot: the largest b with cu[b] / span + b <= slot (slots of b are at
// least as many as its spans, see launch_chunk).
__device__ __forceinline__ int seq_of_slot(const Args& a, int span, int slot) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = a.B;
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int i = lane * step;
    const bool le = i < n && min(max(a.cu[lo + i], 0), a.T) / span + (lo + i) <= slot;
    const int cnt = max(__popc(__ballot_sync(0xffffffffu, le)), 1);
    lo += (cnt - 1) * step;
    n = min(step, n - (cnt - 1) * step);
  }
  return lo;
}

// ------------------------------------------------------------------------------- issuer
struct Issue {
  int jlo, jhi, n_s, n_pv;
};

template <int X>
__device__ __forceinline__ bool issue_s(Issue& t, int j, int st, uint32_t tmem, uint32_t sq, uint32_t sk0, ChunkBars* b,
                                        int* err) {
  if (j < t.jlo || j >= t.jhi) return true;
  // the block before the last, whose P lies there, has to be done
  if (t.n_s > 1 && !mbar_wait(&b->o_ready[X], t.n_s & 1, err, &b->abort_flag)) return false;
  tc_fence_after();
  constexpr uint32_t idesc = make_idesc_bf16(128, kBK, false, false);
  const uint32_t q = sq + X * kQTile, k = sk0 + st * kTile, s = tmem + col_s(X, t.n_s);
#pragma unroll
  for (int kk = 0; kk < kD / 16; ++kk)
    umma_f16(s, make_smem_desc(q + kk * 32, 16, 1024, kLayoutSW128),
             make_smem_desc(k + kk * 32, 16, 1024, kLayoutSW128), idesc, kk > 0);
  umma_commit(&b->s_full[X]);
  ++t.n_s;
  return true;
}

template <int X>
__device__ __forceinline__ bool issue_pv(Issue& t, int j, int st, uint32_t tmem, uint32_t sv0, ChunkBars* b, int* err) {
  if (j < t.jlo || j >= t.jhi) return true;
  if (!mbar_wait(&b->p_full[X], t.n_pv & 1, err, &b->abort_flag)) return false;
  tc_fence_after();
  constexpr uint32_t idesc = make_idesc_bf16(128, kD, false, true);
  const uint32_t v = sv0 + st * kTile, p = tmem + col_s(X, t.n_pv);
  const uint32_t first = t.n_pv > 0 ? 1u : 0u;
#pragma unroll
  for (int term = 0; term < 2; ++term) {
#pragma unroll
    for (int kk = 0; kk < kBK / 16; ++kk)
      umma_f16_tmem_a(tmem + kColO + X * kD, p + term * (kBK / 2) + kk * 8,
                      make_smem_desc(v + kk * 2048, 8192, 1024, kLayoutSW128), idesc, term + kk > 0 ? 1u : first);
  }
  umma_commit(&b->o_ready[X]);
  ++t.n_pv;
  return true;
}

// ------------------------------------------------------------------------------- loaders
// A warp loads rows in groups of 32 keys; lane l looks up the group's key l.
struct Rows {
  uint32_t there;
  int64_t scale;  // offset of the lane's scale bytes
};

// Page of key j, -1 when it is out of range; loaded a block before it is needed.
__device__ __forceinline__ int page_of(const Args& a, const int* table, int j, int hi) {
  int page = -1;
  const int pi = a.p.page_shift >= 0 ? j >> a.p.page_shift : j / a.p.page_size;
  if (j < hi) page = table[pi];
  return page;
}

// Starts the copies of keys key0 .. key0 + 31.  e4m3: 16 codes a piece, piece i of lane l, of row
// 8 i + l / 4 of `pool`, goes to dst + i * kPitch.  bf16: 8 values a piece, of row 4 i + l / 8 of both
// pools, into rows r0 .. r0 + 31 of the swizzled tiles of K (dst) and V (as far behind).
constexpr int kPitch = kLoaders * 32 * 16;  // of a loader thread's own pieces
template <bool FP8>
__device__ __forceinline__ Rows load_rows(const Args& a, const uint8_t* pool, int page, int g, int key0, uint32_t dst, int r0) {
  const int lane = threadIdx.x & 31;
  const bool on = (uint32_t)page < (uint32_t)a.p.num_pages;
  int64_t row = 0, sc = 0;
  if (on) {
    uint32_t pi, off;
    split_slot(a.p, (uint32_t)(key0 + lane), pi, off);
    row = (int64_t)page * a.p.page + (int64_t)off * a.p.token + (int64_t)g * a.p.head;
    sc = (int64_t)page * a.p.s_page + (int64_t)off * a.p.s_token + (int64_t)g * a.p.s_head;
  }
  Rows h;
  h.there = __ballot_sync(0xffffffffu, on);
  h.scale = sc;
  constexpr int kPer = FP8 ? 4 : 8;  // pieces of a row
  const int c = lane % kPer;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int r = (32 / kPer) * i + lane / kPer;
    const int64_t off = __shfl_sync(0xffffffffu, row, r) + c * 16;
    const bool there = (h.there >> r) & 1u;
    if constexpr (FP8) {
      cp_async16(dst + i * kPitch, pool + off, there);
    } else {
      const uint32_t at = dst + sw128(r0 + r, c);
      cp_async16(at, a.p.k + off, there);
      cp_async16(at + (Cfg<false>::V - Cfg<false>::K), a.p.v + off, there);
    }
  }
  return h;
}

// Bits at 0, n, 2 n, ... of x: whether any of the n lanes from there on has its bit set.
__device__ __forceinline__ uint32_t any_of_groups(uint32_t x, int n) {
  for (int s = 1; s < n; s *= 2) x |= x >> s;
  return x & (n == 4 ? 0x11111111u : 0x01010101u);
}

__device__ __forceinline__ void st4(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t u) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(u));
}

// Zeroes what is not finite in rows r0 .. r0 + 31 of a bf16 tile of V, each lane in the pieces that
// it has copied; the keys (bits) that had something.
__device__ __forceinline__ uint32_t clear_tile_rows(uint32_t tile, int r0) {
  const int lane = threadIdx.x & 31;
  uint32_t broken = 0;
#pragma unroll 1
  for (int i = 0; i < 8; ++i) {
    const uint32_t at = tile + sw128(r0 + 4 * i + (lane >> 3), lane & 7);
    const uint4 w = lds128(at);
    uint32_t x[4] = {w.x, w.y, w.z, w.w}, bad = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t m = __vcmpeq2(x[e] & 0x7f807f80u, 0x7f807f80u);
      bad |= m;
      x[e] &= ~m;
    }
    if (bad) st4(at, x[0], x[1], x[2], x[3]);
    const uint32_t q = any_of_groups(__ballot_sync(0xffffffffu, bad != 0), 8);  // bit 8 r: key 4 i + r
#pragma unroll
    for (int r = 0; r < 4; ++r) broken |= ((q >> (8 * r)) & 1u) << (4 * i + r);
  }
  return broken;
}

// 16 e4m3 codes -> 16 bf16 scaled by mul (exact), into chunks 2c and 2c + 1 of row r.
__device__ __forceinline__ void expand16(uint32_t tile, int r, int c, const uint4& w, uint32_t mul) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t l, h;
    e4m3x4_to_f16x2(x[i], l, h);
    const float2 fl = f16x2_to_float2(l), fh = f16x2_to_float2(h);
    o[2 * i] = mul_bf16x2(pack_bf16x2(fl.x, fl.y), mul);
    o[2 * i + 1] = mul_bf16x2(pack_bf16x2(fh.x, fh.y), mul);
  }
  st4(tile + sw128(r, 2 * c), o[0], o[1], o[2], o[3]);
  st4(tile + sw128(r, 2 * c + 1), o[4], o[5], o[6], o[7]);
}

template <bool FP8>
__global__ void __launch_bounds__(kChunkThreads, 1) paged_chunk_kernel(const Args a, const int tokens, const int splits,
                                                                      int* err) {
  using C = Cfg<FP8>;
  constexpr int kST = C::kST, kAhead = C::kAhead;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ ChunkBars bars;
  ChunkBars* b = &bars;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = splits > 1 ? (int)(blockIdx.x % (unsigned)splits) : 0;
  const int slots = gridDim.x / splits;
  const int slot = slots - 1 - (int)(blockIdx.x / (unsigned)splits);  // the longest spans of a sequence first
  const int g = blockIdx.y;
  const int span = 2 * tokens;
  const int sb = seq_of_slot(a, span, slot);
  const Seq sq = load_seq(a, sb);
  const int idx = slot - (sq.t0 / span + sb);
  // (64-bit: a slot far past the sequence's rows must not wrap)
  const int64_t tok64 = (int64_t)sq.t0 + (int64_t)idx * span;
  if (idx < 0 || tok64 >= sq.t1) return;  // the whole cluster
  const int tok0 = (int)tok64;
  const int ntok = min(span, sq.t1 - tok0);
  const int pos0 = sq.first + (tok0 - sq.t0);
  const int lo = a.window > 0 ? max(0, pos0 - a.window + 1) : 0;
  const int hi = max(min(pos0 + ntok, sq.key_end), lo);
  const int nb = (hi - lo + kBK - 1) / kBK;
  const int per = (nb + splits - 1) / splits;
  const int b0 = min(rank * per, nb), b1 = min(b0 + per, nb);
  const int* table = a.table + (int64_t)sb * a.ld_table;
  const Tile tl[2] = {make_tile(a, sq, tok0, tokens, lo, b0, b1), make_tile(a, sq, tok0 + tokens, tokens, lo, b0, b1)};

  if (warp == 0 && lane == 0) {
    mbar_init(&b->q_full, 8);
    for (int s = 0; s < kST; ++s) {
      mbar_init(&b->kv_full[s], FP8 ? 2 * kLoaders : kLoaders);
      mbar_init(&b->kv_empty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&b->s_full[x], 1);
      mbar_init(&b->p_full[x], 4);
      mbar_init(&b->o_ready[x], 1);
    }
    b->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 13) {
    tmem_alloc(&b->tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = b->tmem;
  const uint32_t sbase = smem_u32(smem);

  // a block is seen in full by every row of the span when it lies in [full_lo, full_hi)
  const int full_lo = a.window > 0 ? pos0 + ntok - a.window : 0, full_hi = min(pos0 + 1, sq.key_end);

  auto issue = [&]() {
    if (b1 > b0 && elect_one_sync()) {
      const uint32_t sqa = sbase + C::Q, sk0 = sbase + C::K, sv0 = sbase + C::V;
      Issue ta{tl[0].jlo, tl[0].jhi, 0, 0}, tb{tl[1].jlo, tl[1].jhi, 0, 0};
      bool ok = mbar_wait(&b->q_full, 0, err, &b->abort_flag) && mbar_wait(&b->kv_full[0], 0, err, &b->abort_flag);
      ok = ok && issue_s<0>(ta, b0, 0, tmem, sqa, sk0, b, err) && issue_s<1>(tb, b0, 0, tmem, sqa, sk0, b, err);
      for (int j = b0; ok && j < b1; ++j) {
        const int n = j - b0, st = n % kST, sn = (n + 1) % kST;
        const bool next = j + 1 < b1;
        if (next) ok = mbar_wait(&b->kv_full[sn], ((n + 1) / kST) & 1, err, &b->abort_flag);
        if (ok && next) ok = issue_s<0>(ta, j + 1, sn, tmem, sqa, sk0, b, err);
        ok = ok && issue_pv<0>(ta, j, st, tmem, sv0, b, err);
        if (ok && next) ok = issue_s<1>(tb, j + 1, sn, tmem, sqa, sk0, b, err);
        ok = ok && issue_pv<1>(tb, j, st, tmem, sv0, b, err);
        umma_commit(&b->kv_empty[st]);
      }
    }
  };

  // registers (launch: 512 x 128): loaders and issuer 72, softmax 2 x 184
  if (!FP8 && warp < 4) {
    setmaxnreg_dec<72>();
    if (warp < kLoaders) {
      const int w = warp, key0 = lo + 32 * w;
      bool dead = false;
      uint32_t there[kAhead];
      int next_page = b0 < b1 ? page_of(a, table, key0 + lane + b0 * kBK, hi) : -1;
      auto load = [&](int j) -> uint32_t {
        const int page = next_page;
        if (j + 1 < b1) next_page = page_of(a, table, key0 + lane + (j + 1) * kBK, hi);
        return load_rows<false>(a, nullptr, page, g, key0 + j * kBK, sbase + C::K + ((j - b0) % kST) * kTile, 32 * w).there;
      };
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        there[i] = b0 + i < b1 ? load(b0 + i) : 0u;
        cp_async_commit();
      }
#pragma unroll 1
      for (int j = b0; j < b1; ++j) {
        const int n = j - b0, st = n % kST, m = n + kAhead, k0 = lo + j * kBK;
        cp_async_wait<kAhead - 1>();
        uint32_t broken = 0;  // keys of this warp
        if (k0 < full_lo || k0 + kBK > full_hi) broken = clear_tile_rows(sbase + C::V + st * kTile, 32 * w);
        if (lane == 0) {
          b->info[st].there[w] = there[0] & ~broken;
          b->info[st].broken[w] = broken;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b->kv_full[st]);
#pragma unroll
        for (int i = 0; i < kAhead - 1; ++i) there[i] = there[i + 1];
        there[kAhead - 1] = 0;
        if (j + kAhead < b1) {
          if (!dead && m >= kST && !mbar_wait(&b->kv_empty[m % kST], ((m / kST) & 1) ^ 1, err, &b->abort_flag)) dead = true;
          there[kAhead - 1] = load(j + kAhead);
        }
        cp_async_commit();
      }
    }
  } else if (FP8 && (warp < 4 || warp >= 12)) {
    setmaxnreg_dec<72>();
    if (warp < kLoaders || warp >= 13) {
      const bool is_v = warp < 4;
      const int w = is_v ? warp : warp - 13, key0 = lo + 32 * w;
      const uint8_t *pool = is_v ? a.p.v : a.p.k, *scales = is_v ? a.p.vs : a.p.ks;
      const uint32_t tile0 = sbase + (is_v ? C::V : C::K);
      bool dead = false;
      Rows ah[kAhead];
      // Scale bytes of the block to expand.  Those of the next block are asked for at the top of a round
      // and moved here at its end: a move right after the load would wait for it (1000 cycles a block).
      uint32_t byte = 0;
      auto fetch_scale = [&](const Rows& h) -> uint32_t {
        return load_byte(scales + h.scale, (h.there >> lane) & 1u);
      };
      int pages[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) pages[i] = b0 + i < b1 ? page_of(a, table, key0 + lane + (b0 + i) * kBK, hi) : -1;
      int next_page = b0 + kAhead < b1 ? page_of(a, table, key0 + lane + (b0 + kAhead) * kBK, hi) : -1;
      const uint32_t own0 = sbase + C::RAW + (is_v ? 0 : 4 * kPitch) + (32 * w + lane) * 16;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        ah[i] = Rows{0, 0};
        if (b0 + i < b1) ah[i] = load_rows<true>(a, pool, pages[i], g, key0 + (b0 + i) * kBK, own0 + i * kTile, 0);
        cp_async_commit();
      }
      byte = fetch_scale(ah[0]);
#pragma unroll 1
      for (int j = b0; j < b1; ++j) {
        const int n = j - b0, st = n % kST, k0 = lo + j * kBK;
        const uint32_t next_byte = fetch_scale(ah[1]);
        const uint32_t own = own0 + n % kAhead * kTile;
        cp_async_wait<kAhead - 1>();
        const bool partial = is_v && (k0 < full_lo || k0 + kBK > full_hi);
        uint32_t broken = 0;  // keys of this warp
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = lds128(own + i * kPitch);
        if (partial) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t* x = reinterpret_cast<uint32_t*>(&v[i]);
            bool bad = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t m = __vcmpeq4(x[e] & 0x7f7f7f7fu, 0x7f7f7f7fu);
              bad |= m != 0;
              x[e] &= ~m;
            }
            const uint32_t q = any_of_groups(__ballot_sync(0xffffffffu, bad), 4);  // bit 4 r: key 8 i + r
#pragma unroll
            for (int r = 0; r < 8; ++r) broken |= ((q >> (4 * r)) & 1u) << (8 * i + r);
          }
          broken |= __ballot_sync(0xffffffffu, byte == 255u);
        }
        if (!dead && n >= kST && !mbar_wait(&b->kv_empty[st], ((n / kST) & 1) ^ 1, err, &b->abort_flag)) dead = true;
        // ---- expand into the tiles
        // (each key's lane works out its factor, and all of them travel before the first store: left
        // to the loop below, the stores kept the rows one after the other)
        const uint32_t mine = (broken >> lane) & 1u ? 0u : scale_bf16x2(byte);
        uint32_t mul[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) mul[i] = __shfl_sync(0xffffffffu, mine, 8 * i + (lane >> 2));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          expand16(tile0 + st * kTile, 32 * w + 8 * i + (lane >> 2), lane & 3, v[i], mul[i]);
        if (is_v && lane == 0) {
          b->info[st].there[w] = ah[0].there & ~broken;
          b->info[st].broken[w] = broken;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b->kv_full[st]);
        // ---- refill
#pragma unroll
        for (int i = 0; i < kAhead - 1; ++i) ah[i] = ah[i + 1];
        ah[kAhead - 1] = Rows{0, 0};
        if (j + kAhead < b1) {
          const int page = next_page;
          if (j + kAhead + 1 < b1) next_page = page_of(a, table, key0 + lane + (j + kAhead + 1) * kBK, hi);
          ah[kAhead - 1] = load_rows<true>(a, pool, page, g, key0 + (j + kAhead) * kBK, own, 0);
        }
        cp_async_commit();
        byte = next_byte;
      }
    } else if (warp == 12) {
      issue();
    }
  } else if (warp >= 12) {
    setmaxnreg_dec<72>();
    if (warp == 12) issue();
  } else {
    setmaxnreg_inc<184>();
    const int x = (warp - 4) >> 2;
    const Tile t = x ? tl[1] : tl[0];
    const int row = (warp & 3) * 32 + lane;
    const int tr = row / a.group;
    const bool real = tr < t.ntok;
    const int tok = t.tok0 + tr, h = g * a.group + row % a.group;
    const int pos = t.pos0 + tr;
    // visible keys of this row, relative to lo
    const int see_lo = a.window > 0 ? max(pos - a.window + 1, 0) - lo : -lo;
    const int see_hi = real ? min(pos + 1, sq.key_end) - lo : -1;  // exclusive
    {  // this row of Q into its tile
      const uint4* src = reinterpret_cast<const uint4*>(a.q + (int64_t)tok * a.ld_q + (int64_t)h * kD);
      const uint32_t dst = sbase + C::Q + x * kQTile;
      uint4 w[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) w[c] = real ? src[c] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int c = 0; c < 8; ++c) st4(dst + sw128(row, c), w[c].x, w[c].y, w[c].z, w[c].w);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b->q_full);
    }
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_addr = tmem + lane_base + kColO + x * kD;
    // blocks [k0, k0 + 128) with every key visible to every row of the tile
    const int tile_lo = a.window > 0 ? max(t.pos0 + t.ntok - a.window, 0) - lo : -lo;
    const int tile_hi = min(t.pos0 + 1, sq.key_end) - lo;
    const float smul = fmaxf(a.scale_log2, 1.17549435e-38f);  // not 0: -inf * 0
    float m_ref = -INFINITY, l_run = 0.f;
    int c = 0;
    bool ok = true, broken_row = false;
    for (int j = t.jlo; j < t.jhi; ++j, ++c) {
      const int st = (j - b0) % kST;
      // (the block's tiles are complete when S is; the wait on them is for what info holds)
      if (!mbar_wait(&b->s_full[x], c & 1, err, &b->abort_flag) ||
          !mbar_wait(&b->kv_full[st], ((j - b0) / kST) & 1, err, &b->abort_flag)) { ok = false; break; }
      tc_fence_after();
      const StageInfo* info = &b->info[st];
      const uint32_t s_addr = tmem + lane_base + col_s(x, c);
      float sv[kBK];
      {
        uint32_t r[kBK / 32][32];
#pragma unroll
        for (int w = 0; w < kBK / 32; ++w) tmem_ld_32x32b_x32(s_addr + 32 * w, r[w]);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < kBK; ++e) sv[e] = __uint_as_float(r[e / 32][e % 32]);
      }
      const int k0 = j * kBK;  // relative to lo
      uint32_t all = info->there[0];
#pragma unroll
      for (int w = 1; w < kBK / 32; ++w) all &= info->there[w];
      // (a broken key is not in `there`: a tile may see all of a block that the span does not)
      const bool need_mask = k0 < tile_lo || k0 + kBK > tile_hi || all != 0xffffffffu;
      if (need_mask) {
        uint32_t hit = 0;
#pragma unroll
        for (int w = 0; w < kBK / 32; ++w) {
          // bits of keys k0 + 32 w + e in [see_lo, see_hi)
          const int f = min(max(see_lo - (k0 + 32 * w), 0), 32), e1 = min(max(see_hi - (k0 + 32 * w), 0), 32);
          uint32_t vis = info->there[w] | info->broken[w];
          vis &= f >= 32 ? 0u : 0xffffffffu << f;
          vis &= e1 >= 32 ? 0xffffffffu : (1u << e1) - 1u;
          hit |= vis & info->broken[w];
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (!((vis >> e) & 1u)) sv[32 * w + e] = -INFINITY;
        }
        broken_row |= hit != 0;
      }
      float mxp[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) mxp[u] = fmaxf(sv[u], sv[8 + u]);
#pragma unroll
      for (int cc = 16; cc < kBK; cc += 16) {
#pragma unroll
        for (int u = 0; u < 8; ++u) mxp[u] = fmax3(mxp[u], sv[cc + u], sv[cc + 8 + u]);
      }
      const float mraw = fmax3(fmax3(mxp[0], mxp[1], mxp[2]), fmax3(mxp[3], mxp[4], mxp[5]), fmaxf(mxp[6], mxp[7]));
      const float cand = mraw == -INFINITY ? -INFINITY : mraw * smul;
      float alpha = 1.f;
      bool resc = cand > m_ref;
      if (resc) {
        alpha = ex2a(m_ref - cand);
        m_ref = cand;
      }
      const float m_use = m_ref == -INFINITY ? 0.f : m_ref;
      const uint64_t negm2 = pk2(-m_use, -m_use), scale2 = pk2(smul, smul);
      uint32_t pk[kBK / 2], pl[kBK / 2];  // pk is cut off after 8 bits, pl is the rest
      uint64_t rs2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
      for (int c8 = 0; c8 < kBK / 8; ++c8) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          float x0, x1;
          upk2(fma2(pk2(sv[c8 * 8 + e], sv[c8 * 8 + e + 1]), scale2, negm2), x0, x1);
          x0 = ex2a(x0);
          x1 = ex2a(x1);
          rs2[e / 2] = add2(rs2[e / 2], pk2(x0, x1));
          const uint32_t u0 = __float_as_uint(x0), u1 = __float_as_uint(x1);
          pk[c8 * 4 + e / 2] = __byte_perm(u0, u1, 0x7632);
          upk2(fma2(pk2(__uint_as_float(u0 & 0xffff0000u), __uint_as_float(u1 & 0xffff0000u)), pk2(-1.f, -1.f), pk2(x0, x1)), x0, x1);
          pl[c8 * 4 + e / 2] = pack_bf16x2(x0, x1);
        }
      }
      float rs0, rs1;
      upk2(add2(add2(rs2[0], rs2[1]), add2(rs2[2], rs2[3])), rs0, rs1);
      l_run = l_run * alpha + (rs0 + rs1);
      if (c > 0) {
        if (!mbar_wait(&b->o_ready[x], (c - 1) & 1, err, &b->abort_flag)) { ok = false; break; }
        tc_fence_after();
        if (__any_sync(0xffffffffu, resc)) {
#pragma unroll
          for (int h32 = 0; h32 < kD / 32; ++h32) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(o_addr + h32 * 32, r);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
            tmem_st_32x32b_x32(o_addr + h32 * 32, r);
          }
        }
      }
      {
        uint32_t w0[32], w1[32], w2[32];  // 48 columns of pk, then 48 of pl
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          w0[e] = pk[e];
          w1[e] = e < 16 ? pk[32 + e] : pl[e - 16];
          w2[e] = pl[16 + e];
        }
        tmem_st_32x32b_x32(s_addr, w0);
        tmem_st_32x32b_x32(s_addr + 32, w1);
        tmem_st_32x32b_x32(s_addr + 64, w2);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&b->p_full[x]);
    }
    // ---- this CTA's part of the row: o / l in fp32
    uint32_t o0[32], o1[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) o0[e] = o1[e] = 0u;
    if (ok && c > 0 && mbar_wait(&b->o_ready[x], (c - 1) & 1, err, &b->abort_flag)) {
      tc_fence_after();
      tmem_ld_32x32b_x32(o_addr, o0);
      tmem_ld_32x32b_x32(o_addr + 32, o1);
      tmem_ld_wait();
    }
    tc_fence_before();
    named_barrier_sync(2, 256);  // every product of this CTA is done
    if (broken_row) l_run = __uint_as_float(0x7fc00000u);  // NaN: key by key below
    const float sk = a.sinks != nullptr ? a.sinks[h < a.hq ? h : 0] * kLog2e : -INFINITY;
    float inv, m_fin = m_ref;
    if (splits == 1) {
      m_fin = fmaxf(m_ref, sk);
      const float mu = m_fin == -INFINITY ? 0.f : m_fin;
      const float f = ex2a(m_ref - mu);
      const float den = l_run * f + ex2a(sk - mu);
      inv = den == 0.f ? 0.f : f / den;
    } else {
      inv = l_run == 0.f ? 0.f : 1.f / l_run;
    }
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      const float p0 = __uint_as_float(o0[e]) * inv, p1 = __uint_as_float(o1[e]) * inv;
      bad |= !(fabsf(p0) < INFINITY) || !(fabsf(p1) < INFINITY);
      o0[e] = __float_as_uint(p0);
      o1[e] = __float_as_uint(p1);
    }
    if (splits == 1) {
      if (real && !bad) {
        __nv_bfloat16* orow = a.out + (int64_t)tok * a.ld_out + (int64_t)h * kD;
#pragma unroll
        for (int c8 = 0; c8 < 8; ++c8) {
          const uint32_t* s = c8 < 4 ? o0 + c8 * 8 : o1 + (c8 - 4) * 8;
          uint4 w;
          w.x = pack_bf16x2(__uint_as_float(s[0]), __uint_as_float(s[1]));
          w.y = pack_bf16x2(__uint_as_float(s[2]), __uint_as_float(s[3]));
          w.z = pack_bf16x2(__uint_as_float(s[4]), __uint_as_float(s[5]));
          w.w = pack_bf16x2(__uint_as_float(s[6]), __uint_as_float(s[7]));
          *reinterpret_cast<uint4*>(orow + c8 * 8) = w;
        }
      }
    } else {
      // parts lie over the K/V tiles: [256 rows][64] fp32, 16-byte chunks swizzled by the row
      const int r = x * 128 + row;
      const uint32_t dst = sbase + C::K + r * 256;
#pragma unroll
      for (int c16 = 0; c16 < 16; ++c16) {
        const uint32_t* s = c16 < 8 ? o0 + c16 * 4 : o1 + (c16 - 8) * 4;
        st4(dst + ((c16 ^ (r & 15)) << 4), s[0], s[1], s[2], s[3]);
      }
      b->row_m[r] = m_ref;
      b->row_l[r] = bad ? __uint_as_float(0x7fc00000u) : l_run;
      bad = false;
      cg::this_cluster().sync();
      const float* part = reinterpret_cast<const float*>(smem + C::K);
      for (int rr = rank * 8 + (warp - 4); rr < 256; rr += splits * 8) {
        const Tile& tt = rr < 128 ? tl[0] : tl[1];
        const int rt = (rr & 127) / a.group;
        if (rt >= tt.ntok) continue;
        const int hh = g * a.group + (rr & 127) % a.group;
        const float sk2 = a.sinks != nullptr ? a.sinks[hh] * kLog2e : -INFINITY;
        float mc = -INFINITY, lc = 0.f;
        if (lane < splits) {
          mc = *cg::this_cluster().map_shared_rank(&b->row_m[rr], lane);
          lc = *cg::this_cluster().map_shared_rank(&b->row_l[rr], lane);
        }
        float mt = fmaxf(mc, sk2);
#pragma unroll
        for (int y = 16; y > 0; y >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, y));
        const float mu = mt == -INFINITY ? 0.f : mt;
        const float f = lc * ex2a(mc - mu);
        float den = f;
#pragma unroll
        for (int y = 16; y > 0; y >>= 1) den += __shfl_xor_sync(0xffffffffu, den, y);
        den += ex2a(sk2 - mu);
        float p0 = 0.f, p1 = 0.f;
        const float* src = part + rr * 64 + (((lane >> 1) ^ (rr & 15)) << 2) + (lane & 1) * 2;
        for (int q = 0; q < splits; ++q) {
          const float fq = __shfl_sync(0xffffffffu, f, q);
          const float2 v = *reinterpret_cast<const float2*>(cg::this_cluster().map_shared_rank(src, q));
          p0 = fmaf(fq, v.x, p0);
          p1 = fmaf(fq, v.y, p1);
        }
        const float iv = den == 0.f ? 0.f : 1.f / den;
        p0 *= iv;
        p1 *= iv;
        if (__any_sync(0xffffffffu, !(fabsf(p0) < INFINITY && fabsf(p1) < INFINITY))) {
          const int p = tt.pos0 + rt;
          warp_row<FP8>(a, table, tt.tok0 + rt, hh, a.window > 0 ? max(0, p - a.window + 1) : 0, min(p + 1, sq.key_end),
                        p0, p1);
        }
        reinterpret_cast<__nv_bfloat162*>(a.out + (int64_t)(tt.tok0 + rt) * a.ld_out + (int64_t)hh * kD)[lane] =
            __floats2bfloat162_rn(p0, p1);
      }
    }
    // rows to take key by key (splits == 1)
    for (uint32_t left = __ballot_sync(0xffffffffu, bad && real); left; left &= left - 1) {
      const int src = __ffs(left) - 1;
      const int bt = __shfl_sync(0xffffffffu, tok, src), bh = __shfl_sync(0xffffffffu, h, src);
      const int bp = __shfl_sync(0xffffffffu, pos, src);
      float p0, p1;
      warp_row<FP8>(a, table, bt, bh, a.window > 0 ? max(0, bp - a.window + 1) : 0, min(bp + 1, sq.key_end), p0, p1);
      reinterpret_cast<__nv_bfloat162*>(a.out + (int64_t)bt * a.ld_out + (int64_t)bh * kD)[lane] =
          __floats2bfloat162_rn(p0, p1);
    }
  }
  // the other warps of a cluster meet the softmax warps' first barrier here
  if (splits > 1) {
    __syncwarp();
    if (warp < 4 || warp >= 12) cg::this_cluster().sync();
    cg::this_cluster().sync();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 13) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <bool FP8>
static void launch_chunk_t(const Args& a, int tokens, int slots, int splits, cudaStream_t stream) {
  auto kern = paged_chunk_kernel<FP8>;
  constexpr int smem = Cfg<FP8>::kBytes + 1024;
  static bool ready[64] = {};
  int dev;
  AF3_CUDA_CHECK(cudaGetDevice(&dev));
  if (!ready[dev]) {
    AF3_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    ready[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(slots * splits), (unsigned)a.hkv);
  cfg.blockDim = dim3(kChunkThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)splits, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  AF3_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, a, tokens, splits, device_error_ptr()));
}

void launch_chunk(const Args& a, int64_t max_q, int64_t max_len, cudaStream_t stream) {
  const int tokens = 128 / a.group, span = 2 * tokens;
  // Sequence b has slots [cu[b] / span + b, cu[b + 1] / span + b + 1): at least ceil(q_b / span).
  const int slots = a.T / span + a.B;
  const int64_t keys = a.window > 0 ? std::min<int64_t>(max_len, a.window + std::min<int64_t>(max_q, span)) : max_len;
  const int64_t spans = std::max<int64_t>((a.T + span - 1) / span, 1) * a.hkv;
  int splits = 1;
  while (splits < 8 && spans * splits * 2 <= num_sms() && keys >= 2048 * splits) splits *= 2;
  if (a.p.ks != nullptr)
    launch_chunk_t<true>(a, tokens, slots, splits, stream);
  else
    launch_chunk_t<false>(a, tokens, slots, splits, stream);
}

}  // namespace paged
}  // namespace af3
