// Rows of keys and values held in 4 bits, as every kernel over such pages reads and writes them.
//
// A row of `dim` values (one token, one KV head) is dim codes c of 4 bits and one 16-bit word: value = (c - zero) * step.  With
// lo = min(x, 0), hi = max(x, 0): step is the smallest number of four significant bits (at least 2^-126) with 15 step >= hi - lo,
// zero = -rint(lo / step), c = rint(x / step) + zero within 0 .. 15.  |c - zero| has at most four significant bits, the step
// four: every value is a bfloat16 number, so that what is computed from codes (products of small whole numbers, the step applied
// once per row) and what is computed from unpacked bfloat16 rows agree without a second rounding.  A step rounded up to four bits
// is 4 % too wide on average, 12.5 % at worst.  The word holds the step's bfloat16 bits, whose lowest four are zero, and
// there the zero.  A row with a NaN, an infinity or a magnitude above 2^120 reads back as NaN throughout.
//
// Eight codes are a 32-bit word, element i in bits 4i .. 4i + 3; rows start on 4-byte boundaries (dim a multiple of 8).
#pragma once

#include "common.cuh"

namespace {

constexpr float kPackedLargest = 1.329227995784916e36f;       // 2^120
constexpr float kPackedLeast = 1.1754943508222875e-38f;       // 2^-126

struct PackedPages {
  uint32_t* k;                 // [pages, g, page_size, dim / 8]
  uint32_t* v;
  uint32_t* words;             // [pages, g, page_size]: the key's word low, the value's high
  int num_pages, page_size, g, dim;
  int shift;                   // page_size is 2^shift, or -1
};

inline PackedPages packed_pages(void* k, void* v, void* words, int num_pages, int page_size, int g, int dim) {
  int shift = 0;
  while (1 << shift < page_size) ++shift;
  return {static_cast<uint32_t*>(k), static_cast<uint32_t*>(v), static_cast<uint32_t*>(words), num_pages, page_size, g, dim,
          1 << shift == page_size ? shift : -1};
}

__device__ __forceinline__ float step_of(uint32_t word16) { return __uint_as_float((word16 & 0xFFF0u) << 16); }
__device__ __forceinline__ float zero_of(uint32_t word16) { return (float)(word16 & 15u); }

// The page and row of cached token `at` of a request; page -1 where the table has none.
__device__ __forceinline__ int page_of(const PackedPages& c, const int32_t* table_row, int table_width, int at, int& row) {
  const int index = c.shift >= 0 ? at >> c.shift : at / c.page_size;
  row = at - index * c.page_size;
  const int page = index < table_width ? table_row[index] : -1;
  return page >= 0 && page < c.num_pages ? page : -1;
}
__device__ __forceinline__ size_t row_index(const PackedPages& c, int page, int kvh, int row) {
  return ((size_t)page * c.g + kvh) * c.page_size + row;
}

// The step of a row with the extremes -below <= 0 <= above, finite, at most 2^120.  A product with a little less than 1 / 15 is rounded
// up to four significant bits, and goes one further where 15 steps are still too few.  above + below was rounded before, which can
// only lose what stands above a number of four bits by less than a rounding: rounded + lost, the exact sum, is compared with 15 step,
// which is exact.
__device__ __forceinline__ float step_for(float below, float above) {
  const float range = above + below;
  const float a = range - below, lost = (above - a) + (below - (range - a));
  const uint32_t up = 0x000FFFFFu;
  float step = __uint_as_float((__float_as_uint(range * __uint_as_float(0x3D888888u)) + up) & ~up);
  const float most = 15.f * step;
  if (range > most || (range == most && lost > 0.f)) step = __uint_as_float(__float_as_uint(step) + up + 1u);
  return fmaxf(step, kPackedLeast);
}

// 2^22 + n + 2^23 for n = rint(x / step), the whole number in its lowest bits; `inverse` is 1 / step, nearly.  One step of
// refinement makes the product the rounded quotient (what it leaves is exact), so that ties are ties.  For bfloat16 values that is
// all: their quotients by four bits are ties or stand well apart from them.  A float32 quotient may round to a tie that the exact one
// misses by less; what is left over after the multiple is exact and says so.
template <bool EXACT>
__device__ __forceinline__ float multiple_of(float x, float step, float inverse) {
  constexpr float kWhole = 12582912.f;                        // 1.5 * 2^23: sums with it are whole numbers, ties to even
  const float near = x * inverse;
  float n = fmaf(fmaf(-near, step, x), inverse, near) + kWhole;
  if constexpr (EXACT) {
    const float left = fmaf(-(n - kWhole), step, x), half = 0.5f * step;
    if (left > half) n += 1.f;
    if (left < -half) n -= 1.f;
  }
  return n;
}

// The eight values of a word of codes as bfloat16, in order; exact.  Codes go into the middle bits of bytes 0x80 | c << 3, which under
// bytes 0x41 are the bfloat16 numbers 16 + c.
__device__ __forceinline__ uint4 unpack_bf16(uint32_t codes, uint32_t word16) {
  const uint32_t even = (codes << 3 & 0x78787878u) | 0x80808080u, odd = (codes >> 1 & 0x78787878u) | 0x80808080u;
  const uint32_t low = __byte_perm(even, odd, 0x5140), high = __byte_perm(even, odd, 0x7362);        // codes 0 .. 3, 4 .. 7
  const uint32_t zero = ((word16 & 15u) << 3 | 0x4180u) * 0x10001u, step = (word16 & 0xFFF0u) * 0x10001u;
  uint32_t pair[4] = {__byte_perm(low, 0x41414141u, 0x4140), __byte_perm(low, 0x41414141u, 0x4342), __byte_perm(high, 0x41414141u, 0x4140),
                      __byte_perm(high, 0x41414141u, 0x4342)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 v = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&pair[i]), *reinterpret_cast<const __nv_bfloat162*>(&zero)),
                                     *reinterpret_cast<const __nv_bfloat162*>(&step));
    pair[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(pair[0], pair[1], pair[2], pair[3]);
}

}  // namespace
