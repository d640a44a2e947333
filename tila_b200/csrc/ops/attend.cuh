// Attention over a paged cache with a shared prefix: what its kernels share.
//
//     out_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale q_i . k_j)
//
// over the shared prefix and the sequence's own tokens.  The keys are split
// into chunks that different blocks take; a block keeps the running maximum and
// sum of its chunk's softmax in 32 bits (base 2: scale carries log2 e) and
// leaves a normalised partial result with the log2 of its sum; the partial
// results of a row are joined by their weights 2^(lse_s - lse).  Prefix chunks
// hold the rows of the whole batch, so the prefix is read once for all of
// them; own chunks hold the rows of one sequence.
#pragma once

#include "ops_common.cuh"

namespace tila_ops {

struct AttendParams {
  const void *q, *k, *v;
  void *out;
  float *lse;
  float *partial;       // slots x tokens x heads x dim
  float *partial_lse;   // slots x tokens x heads
  i64 q_stride[2], out_stride[2], k_stride[3], v_stride[3];
  const i32 *table, *lengths, *offsets, *prefix_pages;
  i64 table_stride;
  i64 tokens;
  u32 *err;
  int batch, heads, kv_heads, group, dim;
  int page_size, page_shift;        // shift: log2 of page_size, -1 if it has none
  int table_width, num_pages, max_queries;
  int prefix;                       // tokens of the shared prefix
  float scale2;                     // scale * log2(e)
  // the split: chunks of keys, and the slots of their partial results
  int prefix_chunk, prefix_chunks;  // chunks = slots 0 .. prefix_chunks - 1
  int own_chunks, own_unit;         // slots prefix_chunks ..: a sequence's own tokens in equal parts of whole units,
  int own_least;                    // and of so many keys at least
  int direct;                       // one chunk in all: blocks write the result itself
  int prefix_inside;                // own tokens' blocks (wide, one chunk) take the prefix too
  int q_words, q_vectors;           // q can be read in 4-byte words, in 16-byte vectors
  int out_vectors;                  // out can be written in vectors of 4 elements
};

constexpr float kNegInf = -__builtin_huge_valf();

// First row of q of sequence b, and how many: offsets that run backwards or out
// of q are cut to it.
__device__ __forceinline__ void sequence_rows(const AttendParams &p, int b, i64 &first, int &count) {
  if (p.offsets == nullptr) {
    first = b;
    count = 1;
    return;
  }
  const i64 lo = p.offsets[b], hi = p.offsets[b + 1];
  first = min(max(lo, static_cast<i64>(0)), p.tokens);
  const i64 n = min(hi, p.tokens) - first;
  count = static_cast<int>(min(max(n, static_cast<i64>(0)), static_cast<i64>(p.max_queries)));
  if (lo < 0 || hi > p.tokens || hi < lo || hi - lo > p.max_queries) tila::report_error(p.err, kErrIndex, b);
}

// Own tokens of sequence b: a length beyond its table's pages is cut to them.
__device__ __forceinline__ int own_length(const AttendParams &p, int b) {
  const int n = p.lengths[b];
  const i64 most = static_cast<i64>(p.table_width) * p.page_size;
  if (n < 0 || n > most) tila::report_error(p.err, kErrIndex, b);
  return static_cast<int>(min(static_cast<i64>(max(n, 0)), most));
}

// Keys of each chunk of a sequence: by its own length, so that blocks share the
// work whatever the table's width.
__device__ __forceinline__ int own_chunk(const AttendParams &p, int length) {
  const int each = p.own_chunks > 1 ? (length + p.own_chunks - 1) / p.own_chunks : length;
  return max(p.own_least, (each + p.own_unit - 1) & ~(p.own_unit - 1));
}

// Whether any of 8 elements is infinite or not a number: its exponent bits are all
// ones, and adding their lowest carries into the sign's place.
template <typename T> __device__ __forceinline__ bool any_odd(uint4 x) {
  constexpr u32 kLowest = __is_same(T, __half) ? 0x04000400u : 0x00800080u, kExponent = 0x80008000u - kLowest;
  const u32 carried = ((x.x & kExponent) + kLowest) | ((x.y & kExponent) + kLowest) | ((x.z & kExponent) + kLowest) |
                      ((x.w & kExponent) + kLowest);
  return (carried & 0x80008000u) != 0;
}

__device__ __forceinline__ void split_key(const AttendParams &p, int key, int &page, int &row) {
  if (p.page_shift >= 0) {
    page = key >> p.page_shift;
    row = key & (p.page_size - 1);
  } else {
    page = key / p.page_size;
    row = key - page * p.page_size;
  }
}

}  // namespace tila_ops
