// Kernels of the attention over cache pages (see paged_attention.cuh for what they compute).
#pragma once
#include "paged_attention.cuh"

namespace af3 {
namespace paged {

constexpr int kFewRows = 32;  // query rows a KV head of launch_few's largest tile: its largest group

// Sequences of up to this many query rows a KV head go to launch_few.  Measured on 4200 tokens, 8
// heads a KV head, 64 sequences, launch_few against launch_chunk: 4 tokens (32 rows) 197 and 301 us in
// e4m3, 205 and 295 us in bf16; 5 (40 rows) 259 and 279 us, 301 and 260 us; ragged, 1 to 5 tokens on 210
// to 4200, 115 and 231 us, 125 and 223 us.
constexpr int kFewTotal = 40;

// launch_few, e4m3 pages: where the V scale bytes of keys that share a tile are further apart than this many
// powers of two, f16 no longer holds all of them well enough for a row in which the largest have little
// weight or none; such a tile's rows are taken key by key.  At 19 the values at the small end still meet
// weights of 2^-10 of the row's largest (2^15) in 11 bits.  Tokens of one sequence differ by far less.
constexpr int kWideRange = 19;

// Few query rows a KV head and sequence, groups of at most kFewRows: memory-bound, split over the keys.
void launch_few(const Args& a, int64_t max_q, int64_t max_len, cudaStream_t stream);

// Any number of rows, at most 128 query heads a KV head: tensor cores, split over the keys when
// there are few rows.
void launch_chunk(const Args& a, int64_t max_q, int64_t max_len, cudaStream_t stream);

}  // namespace paged
}  // namespace af3
