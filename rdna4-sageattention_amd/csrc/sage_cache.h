// Shared by the cache's kernels: the codes' types, their conversion and the checks of a cache's tensors.
#pragma once

#include "sage_common.h"
#include "sage_host.h"

namespace sage {

enum { CACHE_INT8 = 0, CACHE_E4M3 = 1 };

// pages: a power of two of rows, so that the 16 keys of an MFMA operand never straddle two
inline bool cache_page_ok(int n) { return n >= 16 && n <= 1024 && (n & (n - 1)) == 0; }

int cache_check(const void* k8, const float* ks, const void* v8, const float* vs, int pages, int page_size, int Hkv,
                int D, int cache_dtype, const char* who);

// codes 2 half and 2 half + 1 of a word as floats
template <int CT> __device__ __forceinline__ void code_pair(uint32_t w, int half, float& lo, float& hi) {
  if (CT == CACHE_INT8) {
    const int s = 16 * half;
    lo = (float)(int8_t)(w >> s);
    hi = (float)(int8_t)(w >> (s + 8));
  } else if (half) {
    lo = __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
    hi = __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
  } else {
    lo = __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
    hi = __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
  }
}

}  // namespace sage
