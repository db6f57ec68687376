// fz_grad_words.h -- which memory the int8 weight gradient reads of gradients whose rows do not lie on the 16-byte grid:
// plain index arithmetic, shared by the kernel and the host test of its bounds.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define ZF_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define ZF_HOST_DEVICE inline
#endif

namespace zf::int8_weight_grad {

// A CTA's columns of a row as the aligned 32-bit words that hold them: word i holds columns 2 i - odd and 2 i - odd + 1,
// odd = 1 where the row begins in the middle of a word.
ZF_HOST_DEVICE int word_column(const int word, const int odd) { return 2 * word - odd; }

// whether the word holds one of the CTA's columns (none do where it has none: a layer of up to 128 outputs leaves the second
// CTA of its pair without a column, and its first word begins before column 0 when odd)
ZF_HOST_DEVICE bool word_needed(const int word, const int odd, const int columns) { return columns > 0 && word_column(word, odd) < columns; }

// whether rows row0 .. row0 + rows - 1 of n may be read by whole words: such a word reaches at most one column past either
// end of the CTA's own, into the row before or the row behind, which the tensor has
ZF_HOST_DEVICE bool whole_words(const int64_t row0, const int rows, const int n) { return row0 > 0 && row0 + rows < n; }

}  // namespace zf::int8_weight_grad
