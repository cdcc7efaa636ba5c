// What the kernels over a paged e4m3 cache share: its layout, its scales, the 8-bit conversions.
//
// A layer's cache has pages of P tokens (a multiple of 64). Of one page and KV head the keys are [P / 64][D / 64][64 tokens][64 dimensions]
// and the values [P / 64][D][64], whose 64 bytes are the tokens 16 t + 4 g + i in the order (g, t, i): what lane (row, g) holds of two
// 16 x 16 x 32 matrix instructions' operands is then 16 bytes in a row, a wave's load is 1 KB in a row, and the probabilities of 64 keys, which the score
// products leave in the order (t, i) at lane group g, are the other operands as they are. Scales are powers of two, so that appending a louder token to
// a page moves the exponents of its codes (only what falls among e4m3's subnormals is rounded again), and what is multiplied by one loses nothing.
#pragma once

#include "hybrid.cuh"

namespace mui {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

struct PagedTable {
  const int32_t* table;    // [requests, pages], rows `stride` apart
  long stride;
  int pages;               // entries of a row
  const int64_t* lengths;  // [requests], the new tokens among them
  const int64_t* offsets;  // [requests + 1] rows of the new tokens, or null: one each
  int n_requests, n_rows, n_pages, page_shift;
};

// a request's new rows, whatever `offsets` holds: first row, how many, and the position of the first; the length cut to what the table can hold
struct PagedSpan { int row0, count; long start, length; };
__device__ __forceinline__ PagedSpan paged_span(const PagedTable& p, int b) {
  PagedSpan s;
  constexpr long kMost = 1L << 36;  // (tiles of 64 tokens are counted in 32 bits)
  long len = p.lengths[b];
  len = len < -kMost ? -kMost : (len > kMost ? kMost : len);
  const long cap = (long)p.pages << p.page_shift;
  long r0 = b, r1 = b + 1;
  if (p.offsets) { r0 = p.offsets[b]; r1 = p.offsets[b + 1]; }
  r0 = r0 < 0 ? 0 : (r0 > p.n_rows ? p.n_rows : r0);
  r1 = r1 < r0 ? r0 : (r1 > p.n_rows ? p.n_rows : r1);
  s.row0 = (int)r0;
  s.count = (int)(r1 - r0);
  s.start = len - s.count;  // may be negative: such tokens have no place
  s.length = len < 0 ? 0 : (len > cap ? cap : len);
  return s;
}

// the last request whose rows begin at or before `row`
__device__ __forceinline__ int request_of(const PagedTable& t, int row) {
  if (!t.offsets) return row;
  int lo = 0, hi = t.n_requests;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.offsets[mid] <= row) lo = mid; else hi = mid;
  }
  return lo;
}

// the same for a row that a whole wave asks for, 64 requests looked at at once
__device__ __forceinline__ int request_of_wave(const PagedTable& t, int row) {
  if (!t.offsets) return row;
  const int lane = threadIdx.x & 63;
  int lo = 0, len = t.n_requests;
  while (len > 1) {
    const int step = (len + kWave - 1) / kWave, at = lane * step;
    const unsigned long long in = __ballot(at < len && t.offsets[lo + (at < len ? at : 0)] <= row);
    const int k = in ? (63 - __clzll((long long)in)) * step : 0;
    lo += k;
    len = len - k < step ? len - k : step;
  }
  return lo;
}

// (what a request's numbers say is the same for a workgroup, which the compiler does not see where they come from memory: in scalar registers it costs the results no room)
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ long uniform(long x) {
  return (long)((unsigned long long)(uint32_t)uniform((int)(x >> 32)) << 32 | (uint32_t)uniform((int)(x & 0xffffffffL)));
}
__device__ __forceinline__ PagedSpan uniform(PagedSpan s) { return {uniform(s.row0), uniform(s.count), uniform(s.start), uniform(s.length)}; }

// the page of slot `slot` of request b's table, or -1 where that is none; in two steps, for those who have other work while the entry comes
__device__ __forceinline__ int paged_entry(const PagedTable& p, int b, int slot) { return slot < p.pages ? p.table[(long)b * p.stride + slot] : -1; }
__device__ __forceinline__ int page_of_entry(const PagedTable& p, int entry) { return entry >= 0 && entry < p.n_pages ? entry : -1; }
__device__ __forceinline__ int paged_page(const PagedTable& p, int b, int slot) { return page_of_entry(p, paged_entry(p, b, slot)); }

// 2^e, -126 <= e <= 127
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// smallest e >= -120 with a <= 448 * 2^e (448 = 0.875 * 2^9); a finite, >= 0
__device__ __forceinline__ int e4m3_exponent(float a) {
  const uint32_t u = __float_as_uint(a);
  const int x = (int)(u >> 23) - 126;  // a = m 2^x, 0.5 <= m < 1 (smaller for subnormal a: below the floor anyway)
  const int e = x - 9 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < -120 ? -120 : e;
}
__device__ __forceinline__ int scale_exponent(float s) { return (int)((__float_as_uint(s) >> 23) & 0xff) - 127; }

// four values -> four codes (nearest even; beyond 464, infinities and NaN: NaN)
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
// four codes times f, rounded to codes again
__device__ __forceinline__ uint32_t e4m3x4_times(uint32_t w, float f) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return to_e4m3x4(a[0] * f, a[1] * f, b[0] * f, b[1] * f);
}

}  // namespace mui
