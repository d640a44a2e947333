// The wide form of the attention over a paged cache (attend_wide.cu).
#pragma once

#include "attend.cuh"

namespace tila_ops {

struct WideGrid {
  int pairs;         // blocks' shares of the rows: pairs of row tiles of 128 (prefix), or single ones
};

// Whether the caches' strides allow tensor maps; and whether pages and head size
// also fit the wide form: boxes of whole pages, or of 128 rows of one.
bool tma_possible(const tila_attend_args &a);
bool wide_possible(const tila_attend_args &a);
// Whether the compiler gave the wide form's kernel for these sizes the registers it
// needs (true also where that cannot be looked up).
bool wide_fits(const tila_attend_args &a, bool own);

// Tensor maps of both caches with boxes of 64 elements of `rows` rows, 128-byte
// swizzled.
int encode_caches(const tila_attend_args &a, int rows, tila::TensorMap *k, tila::TensorMap *v, char *log, size_t cap);

int launch_wide(const tila_attend_args &a, const AttendParams &p, bool prefix, bool after_previous, cudaStream_t stream,
                char *log, size_t cap);

}  // namespace tila_ops
