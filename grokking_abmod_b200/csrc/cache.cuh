// The 8-bit paged key/value cache as its kernels see it.
//
// A page holds `tokens` consecutive tokens of one sequence: per head,
// [tokens][width] signed codes c in -127..127 (width = head_dim rounded up to
// 32, the padding channels 0) and one scale; the stored value is c * scale.
//
// Scales are powers of two: the smallest 2^e >= 2^-126 with amax <= 127 2^e.
// Division and requantisation by them are exact, so c = rne(x / scale) has
// the same bits in any precision and any order of work, and attention takes
// the scales out of its products without rounding.  The price is a step of
// at most 2 amax / 127 instead of amax / 127.  When a token with a larger
// need joins a half-filled page the page's scale grows and its codes c move
// to rne(c scale / scale').  A page and head that was given an infinity or a
// NaN has scale NaN until its first token is written again.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace mb {
namespace cache {

constexpr int kMaxHeadDim = 128;
constexpr int kMaxLength = 1 << 30;  // tokens of a sequence: positions and their tiles stay in 32 bits

struct View {
  int8_t *k, *v;
  float *k_scale, *v_scale;
  int pages, heads, tokens, shift;  // tokens per page = 1 << shift
  int width;                        // channels a row takes
  __host__ __device__ size_t row(int page, int head, int slot) const {
    return (((size_t)page * heads + head) * tokens + slot) * width;
  }
  __host__ __device__ size_t scale_at(int page, int head) const { return (size_t)page * heads + head; }
};

// Where sequences are: their pages, their tokens with the new ones, and
// their rows in the packed arrays.
struct Batch {
  const int32_t* table;
  size_t table_stride;
  int table_pages;
  const int32_t* lengths;
  const int32_t* offsets;  // null: row b belongs to sequence b
  int count;
  size_t rows;
};

// Device status bits.
constexpr int kBadPage = 2;    // a page number outside the pool
constexpr int kBadLength = 4;  // a length below the new rows, or past the table
constexpr int kBadRows = 8;    // offsets outside the rows, or more new rows than announced
constexpr int kGaveUp = 1;     // a tensor-core wait ran out

struct Span {
  int length;  // tokens in the cache, the new ones among them
  size_t row;  // first new row
  int fresh;   // new rows
  int flags;   // not 0: the numbers do not fit; row and fresh are clamped to the rows there are
};

__device__ __forceinline__ Span span_of(const Batch& t, const View& c, int b) {
  Span s;
  s.flags = 0;
  long long lo = b, hi = (long long)b + 1;
  if (t.offsets) {
    lo = t.offsets[b];
    hi = t.offsets[b + 1];
  }
  const long long rows = (long long)t.rows;
  if (lo < 0 || hi < lo || hi > rows) {
    s.flags |= kBadRows;
    lo = lo < 0 ? 0 : (lo > rows ? rows : lo);
    hi = hi < lo ? lo : (hi > rows ? rows : hi);
  }
  s.row = (size_t)lo;
  s.fresh = (int)(hi - lo);
  const long long room = (long long)t.table_pages << c.shift;
  s.length = t.lengths[b];
  if (!s.flags && (s.length < s.fresh || s.length > room || s.length > kMaxLength)) s.flags |= kBadLength;
  return s;
}

// The page that holds token `pos` of sequence b, or -1.
__device__ __forceinline__ int page_of(const Batch& t, const View& c, int b, int index) {
  const int p = __ldg(t.table + (size_t)b * t.table_stride + index);
  return (unsigned)p < (unsigned)c.pages ? p : -1;
}

__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

// The scale for the largest magnitude `bits` (FP32 bits without the sign);
// NaN where that is not finite.  127 2^(E-6) = 1.984375 2^E for the exponent
// E of amax, so the mantissa decides between 2^(E-6) and 2^(E-5).
__device__ __forceinline__ float scale_for(uint32_t bits) {
  if (bits >= 0x7F800000u) return __int_as_float(0x7FC00000);
  const int e = (int)(bits >> 23) - 127 - 6 + ((bits & 0x7FFFFFu) > 0x7E0000u ? 1 : 0);
  return power_of_two(e < -126 ? -126 : e);
}

}  // namespace cache
}  // namespace mb
