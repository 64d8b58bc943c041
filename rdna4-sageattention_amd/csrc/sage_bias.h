// Relative position bias by buckets: what its own kernels and the attention for training share.
//
// The key `d` tokens ahead of its query (d < 0: behind) is in a bucket of a learned table [buckets, heads].  side = buckets / 2
// where the bias is two-sided, else buckets; n = |d|, or max(-d, 0) one-sided; near = side / 2.  n < near has bucket n, beyond
// them near + floor(ln(n / near) / ln(max_distance / near) * (side - near)), side - 1 at most; two-sided, keys ahead add side.
// The borders of the far buckets are whole numbers, borders[t] = the smallest n of bucket near + t, computed exactly by the
// host (n^m >= near^(m - t) max_distance^t with m = side - near), so no logarithm decides which side of a border a distance is on.
#pragma once

#include "sage_common.h"
#include "sage_host.h"

namespace sage {

constexpr int BIAS_BUCKETS = 256;                 // most buckets

struct BiasMap {
  int side, near, two_sided, buckets;
  int borders[BIAS_BUCKETS / 2];                  // side - near of them; borders[0] = near
  __host__ __device__ int reach() const { return borders[side - near - 1]; }   // from here on the bucket is the same
  // (at: the borders, or a copy of them where lanes that look for different ones are served faster)
  __device__ __forceinline__ int bucket(int64_t d, const int* at) const {
    const int64_t far = two_sided ? (d < 0 ? -d : d) : (d < 0 ? -d : 0);
    const int n = (int)(far < reach() ? far : reach());
    int b = n;
    if (n >= near) {                              // the last border at most n
      int lo = 0, hi = side - near - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (at[mid] <= n) lo = mid;
        else hi = mid - 1;
      }
      b = near + lo;
    }
    return two_sided && d > 0 ? b + side : b;
  }
  // The distances of bucket b as lo .. hi, the last ones standing for all that lie farther (+-reach); lo > hi: none
  __device__ __forceinline__ void range(int b, int& lo, int& hi) const {
    const bool ahead = two_sided && b >= side;
    if (ahead) b -= side;
    const int first = b < near ? b : borders[b - near];
    const int last = b < near ? b : b == side - 1 ? reach() : borders[b - near + 1] - 1;
    if (ahead) lo = first > 1 ? first : 1, hi = last;
    else lo = -last, hi = b == 0 && !two_sided ? reach() : -first;
  }
};

// float of a table's entry: dtype SAGE_DTYPE_BF16 / F16 / F32
__device__ __forceinline__ float bias_value(const void* table, int dtype, int64_t at) {
  if (dtype == SAGE_DTYPE_F32) return ((const float*)table)[at];
  const uint32_t u = ((const uint16_t*)table)[at];
  return dtype == SAGE_DTYPE_BF16 ? bf16_lo(u) : f16_lo(u);
}

// part[b] = 2^exponent times the sum over bucket b's distances of sums (LDS, n entries; entry x is of distance d0 + x), for a
// workgroup of THREADS: 16 lanes per bucket.  (A wave per bucket, one after another: 5 us more for 64 buckets of 2055
// diagonals.)
template <int THREADS>
__device__ __forceinline__ void bias_sum_buckets(const BiasMap& m, const float* sums, int64_t d0, int n, float* part, int exponent) {
  const int l = threadIdx.x & 15;
  for (int b = threadIdx.x >> 4; b < m.buckets; b += THREADS / 16) {
    int lo, hi, x0 = 0, x1 = 0;
    m.range(b, lo, hi);
    if (lo <= hi) {
      const int64_t y0 = lo <= -m.reach() ? 0 : lo - d0, y1 = hi >= m.reach() ? n : hi + 1 - d0;
      x0 = (int)max(min(y0, (int64_t)n), (int64_t)0);
      x1 = (int)max(min(y1, (int64_t)n), (int64_t)0);
    }
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    int x = x0 + l;
    for (; x + 48 < x1; x += 64)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] += sums[x + 16 * e];
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (x + 16 * e < x1) s[e] += sums[x + 16 * e];
    float t = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) t += __shfl_xor(t, o);
    if (l == 0) part[b] = __builtin_ldexpf(t, exponent);
  }
}

// vec [H, 2 reach + 1]: the bias by distance, times `mul`
int bias_expand_launch(const void* table, int table_dtype, int64_t tb, int64_t th, int H, const BiasMap& m, float mul, float* vec,
                       hipStream_t st);
// dtable[b, h] = the sum over t of part[(h * T + t) * buckets + b]
int bias_reduce_launch(const float* part, int64_t T, int H, const BiasMap& m, void* dtable, int table_dtype, int64_t tb, int64_t th,
                       hipStream_t st);
// checks a caller's buckets and borders
int bias_map(const char* who, int H, int buckets, int two_sided, const int* borders, int table_dtype, BiasMap* m);

}  // namespace sage
