// Kernels of the attention over cache pages (see paged_attention.cuh for what they compute).
#pragma once
#include "paged_attention.cuh"

namespace af3 {
namespace paged {

constexpr int kFewRows = 32;  // query rows a KV head that launch_few takes in one tile

// Where the V (or K) scale bytes of keys that share a tile are further apart than this many
// powers of two, f16 no longer holds all of them well enough once a row does not see the largest;
// such a tile's rows are taken key by key.  Tokens of one sequence differ by far less.
constexpr int kWideRange = 14;
// bf16 V scaled to f16 keeps 2^-25 of 2^8; judged by 8 values at a time.
constexpr int kWideRangeBf16 = 18;

// At most kFewRows query rows a KV head and sequence: memory-bound, split over the keys.
void launch_few(const Args& a, int64_t max_q, int64_t max_len, cudaStream_t stream);

// Any number of rows, at most 128 query heads a KV head: tensor cores, split over the keys when
// there are few rows.
void launch_chunk(const Args& a, int64_t max_q, int64_t max_len, cudaStream_t stream);

}  // namespace paged
}  // namespace af3
