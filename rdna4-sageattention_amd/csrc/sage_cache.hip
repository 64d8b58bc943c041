// The quantized key / value cache: rows of 8-bit codes with one float32 scale each, in pages.
//
//   codes  int8 or E4M3  [pages, Hkv, page_size, D]     scale  float32  [pages, Hkv, page_size]
//
// Row x of one (token, kv head): a = max |x|, scale = a / Q and code = round(Q x / a), to the nearest code, ties to
// even; Q is the largest code, 127 (int8) or 448 (E4M3).  A row of zeros has scale 0.  A row that holds an infinity or a
// NaN has scale NaN and codes 0: whatever reads it gets NaN, as from the row itself.  Q x is exact in float32 (Q has at
// most 7 bits, x at most 11) and the quotient is rounded once, so ties are met as in exact arithmetic; quotients that are
// no tie keep a relative distance of 2^-19 or more from one, so a code never depends on the arithmetic's width.
// Slot = page * page_size + row; slots outside the cache stand for tokens without one: the write leaves them out,
// the read gives zeros.
//
// Bound: HBM.  A row of 16-bit values is read (written) once, its codes written (read) once: 130000 tokens of 8 heads x 128
// written in 166 us (4.9 TB/s) and read in 195 us (4.1 TB/s, two thirds of it stores), a large copy moving 4.8.
//
// No counterpart in the reference, which quantizes K and V anew in every call (src/rdna4_sage/_attention.py:115-133).
#include "sage_cache.h"

namespace sage {

constexpr int CACHE_THREADS = 256;

// lanes of a row: 8 channels each (96 channels leave 4 of 16 idle)
template <int D> constexpr int row_lanes() { return D == 96 ? 16 : D / 8; }

template <int L> __device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp(v, DPP_QUAD_XOR1, 0xF, 0xF, false));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp(v, DPP_QUAD_XOR2, 0xF, 0xF, false));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, false));  // each 8 lanes mirrored
  if (L >= 16) v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp(v, DPP_ROW_ROR8, 0xF, 0xF, false));
  if (L >= 32) v = max(v, (uint32_t)__shfl_xor((int)v, 16));
  return v;
}

struct CacheRows {
  const uint16_t* x[2];          // write: k, v
  uint16_t* y[2];                // read: k, v
  int64_t sb[2], ss[2], sh[2];   // their (batch, token, head) element strides
  uint8_t* codes[2];
  float* scale[2];
  const void* slots;             // [B * S]
  int slots64, S, tokens, Hkv;
  int page_shift;
  int64_t capacity;              // pages * page_size
};

// slot -> row index within [pages, Hkv, page_size], or -1
__device__ __forceinline__ int64_t cache_row(const CacheRows& a, int tok, int h) {
  const int64_t slot = a.slots64 ? static_cast<const int64_t*>(a.slots)[tok] : static_cast<const int32_t*>(a.slots)[tok];
  if (slot < 0 || slot >= a.capacity) return -1;
  const int64_t page = slot >> a.page_shift;
  return ((page * a.Hkv + h) << a.page_shift) + (slot & ((1 << a.page_shift) - 1));
}

// One row per row_lanes lanes, neighbouring rows = neighbouring tokens of a head (their codes and scales are neighbours
// in a page); the heads of some tokens in neighbouring workgroups (read: 130000 tokens of 8 heads x 128 in 194 us, 214 with the
// heads far apart); blockIdx.y = k or v.  A thread takes U rows, a workgroup's rows apart, whose loads are in flight
// together.
template <int D, int U> struct RowsOf {
  static constexpr int L = row_lanes<D>(), PER = CACHE_THREADS / L;
  int tok[U], l;
  bool mine;  // (96 channels leave lanes without any)
  int64_t row[U], at[U];
  __device__ __forceinline__ RowsOf(const CacheRows& a, int h, int w) {
    l = threadIdx.x % L;
    mine = D != 96 || l < 12;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      tok[u] = (int)((blockIdx.x / a.Hkv * U + u) * PER) + threadIdx.x / L;
      row[u] = tok[u] < a.tokens ? cache_row(a, tok[u], h) : -1;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int t = min(tok[u], a.tokens - 1), b = t / a.S, s = t - b * a.S;
      at[u] = b * a.sb[w] + s * a.ss[w] + h * a.sh[w] + 8 * l;
    }
  }
};

template <int D, int DT, int CT, int U>
__global__ __launch_bounds__(CACHE_THREADS) void cache_write_kernel(const CacheRows a) {
  constexpr int L = row_lanes<D>();
  const int h = blockIdx.x % a.Hkv, w = blockIdx.y;
  const RowsOf<D, U> r(a, h, w);
  v4i in[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    in[u] = v4i{0, 0, 0, 0};
    if (r.mine && r.row[u] >= 0) in[u] = *reinterpret_cast<const v4i*>(a.x[w] + r.at[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const v4i x = in[u];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = (uint32_t)x[i] & 0x7FFF7FFFu;
      top = max(top, max(m & 0xFFFFu, m >> 16));
    }
    top = lanes_max<L>(top);
    const bool bad = top >= (DT == DT_BF16 ? 0x7F80u : 0x7C00u);
    const float amax = elem_lo<DT>(top);
    // rows near the ends of float32's range are brought inside it by a power of two, which changes no quotient
    const float fit = amax < 0x1p-60f ? 0x1p100f : amax > 0x1p60f ? 0x1p-100f : 1.0f;
    const float div = amax == 0.0f ? 1.0f : amax * fit, rec = 1.0f / div;
    constexpr float Q = CT == CACHE_INT8 ? 127.0f : 448.0f;
    float y[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (the correction of the quotient loses the sign of a zero)
      const float lo = elem_lo<DT>(x[i]), hi = elem_hi<DT>(x[i]);
      y[2 * i] = __builtin_copysignf(div_by_scale(lo * fit * Q, div, rec), lo);
      y[2 * i + 1] = __builtin_copysignf(div_by_scale(hi * fit * Q, div, rec), hi);
    }
    v2i codes;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float* z = y + 4 * i;
      int c;
      if (CT == CACHE_INT8) {
        c = (int)pack4_i8((int)__builtin_rintf(z[0]), (int)__builtin_rintf(z[1]), (int)__builtin_rintf(z[2]),
                          (int)__builtin_rintf(z[3]));
      } else {
        c = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
        c = __builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], c, true);
      }
      codes[i] = bad ? 0 : c;
    }
    if (r.row[u] >= 0) {
      if (r.mine) *reinterpret_cast<v2i*>(a.codes[w] + r.row[u] * D + 8 * r.l) = codes;
      if (r.l == 0) a.scale[w][r.row[u]] = bad ? __builtin_nanf("") : amax / Q;
    }
  }
}

template <int D, int DT, int CT, int U>
__global__ __launch_bounds__(CACHE_THREADS) void cache_read_kernel(const CacheRows a) {
  const int h = blockIdx.x % a.Hkv, w = blockIdx.y;
  const RowsOf<D, U> r(a, h, w);
  if (!r.mine) return;
  v2i c[U];
  float scale[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    c[u] = v2i{0, 0};
    scale[u] = 0.0f;
    if (r.row[u] >= 0) {
      c[u] = *reinterpret_cast<const v2i*>(a.codes[w] + r.row[u] * D + 8 * r.l);
      scale[u] = a.scale[w][r.row[u]];
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (r.tok[u] >= a.tokens) break;
    v4i out;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float lo, hi;
      code_pair<CT>((uint32_t)c[u][i / 2], i & 1, lo, hi);
      out[i] = (int)(f32_to_out_bits<DT>(lo * scale[u]) | (f32_to_out_bits<DT>(hi * scale[u]) << 16));
    }
    *reinterpret_cast<v4i*>(a.y[w] + r.at[u]) = out;
  }
}

template <int D, int DT, int CT> static void cache_rows_launch(const CacheRows& a, bool write, hipStream_t st) {
  const int per = CACHE_THREADS / row_lanes<D>();
  // four rows per thread where that leaves every CU some waves, us with four and with one (8 heads x 128): 130000 tokens written
  // 166 and 212, read 195 and 208; 18002 written 25 and 26, read 22 and 22; 9000 written 16.5 and 15.6, read 17.4 and 13.3
  const int u = (int64_t)a.tokens * a.Hkv * row_lanes<D>() >= 8 * 256 * 1024 ? 4 : 1;
  const dim3 grid((unsigned)((a.tokens + per * u - 1) / (per * u)) * a.Hkv, 2);
  if (u == 4) {
    if (write) cache_write_kernel<D, DT, CT, 4><<<grid, CACHE_THREADS, 0, st>>>(a);
    else cache_read_kernel<D, DT, CT, 4><<<grid, CACHE_THREADS, 0, st>>>(a);
  } else {
    if (write) cache_write_kernel<D, DT, CT, 1><<<grid, CACHE_THREADS, 0, st>>>(a);
    else cache_read_kernel<D, DT, CT, 1><<<grid, CACHE_THREADS, 0, st>>>(a);
  }
}
template <int D, int DT> static void cache_rows_codes(const CacheRows& a, int ct, bool write, hipStream_t st) {
  if (ct == CACHE_INT8) cache_rows_launch<D, DT, CACHE_INT8>(a, write, st);
  else cache_rows_launch<D, DT, CACHE_E4M3>(a, write, st);
}
template <int DT> static void cache_rows_dims(const CacheRows& a, int D, int ct, bool write, hipStream_t st) {
  if (D == 64) cache_rows_codes<64, DT>(a, ct, write, st);
  else if (D == 96) cache_rows_codes<96, DT>(a, ct, write, st);
  else if (D == 128) cache_rows_codes<128, DT>(a, ct, write, st);
  else cache_rows_codes<256, DT>(a, ct, write, st);
}

int cache_check(const void* k8, const float* ks, const void* v8, const float* vs, int pages, int page_size, int Hkv,
                int D, int cache_dtype, const char* who) {
  SAGE_REQUIRE(k8 && ks && v8 && vs, "%s: a cache tensor is NULL", who);
  SAGE_REQUIRE(aligned16(k8) && aligned16(v8) && aligned16(ks) && aligned16(vs),
               "%s: cache tensors must be 16-byte aligned", who);
  SAGE_REQUIRE(pages > 0 && Hkv > 0, "%s: sizes must be positive", who);
  if (!head_dim_ok(D)) return fail(SAGE_ERR_UNSUPPORTED, "%s: head_dim %d (supported 64, 96, 128, 256)", who, D);
  if (!cache_page_ok(page_size))
    return fail(SAGE_ERR_UNSUPPORTED, "%s: page_size %d (a power of two from 16 to 1024)", who, page_size);
  if (cache_dtype != SAGE_CACHE_INT8 && cache_dtype != SAGE_CACHE_E4M3)
    return fail(SAGE_ERR_UNSUPPORTED, "%s: cache dtype %d", who, cache_dtype);
  return SAGE_OK;
}

static int cache_rows(const void* k, int64_t ksb, int64_t kss, int64_t ksh, const void* v, int64_t vsb, int64_t vss,
                      int64_t vsh, int B, int S, int dtype, const void* slots, int slots64, void* k8, float* ks, void* v8,
                      float* vs, int pages, int page_size, int Hkv, int D, int cache_dtype, bool write, void* stream,
                      const char* who) {
  clear_error();
  int rc = cache_check(k8, ks, v8, vs, pages, page_size, Hkv, D, cache_dtype, who);
  if (rc) return rc;
  SAGE_REQUIRE(B > 0 && S > 0, "%s: sizes must be positive", who);
  SAGE_REQUIRE(k && v && slots, "%s: k, v or slots is NULL", who);
  SAGE_REQUIRE(aligned16(k) && aligned16(v), "%s: k and v must be 16-byte aligned", who);
  SAGE_REQUIRE(ksb % 8 == 0 && kss % 8 == 0 && ksh % 8 == 0 && vsb % 8 == 0 && vss % 8 == 0 && vsh % 8 == 0,
               "%s: strides must be multiples of 8 elements", who);
  SAGE_REQUIRE(((uintptr_t)slots & (slots64 ? 7u : 3u)) == 0, "%s: slots misaligned", who);
  if (dtype != SAGE_DTYPE_BF16 && dtype != SAGE_DTYPE_F16) return fail(SAGE_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  SAGE_REQUIRE((int64_t)B * S <= 0x3FFFFFFF && (int64_t)B * S * Hkv <= 0x7FFFFFFF, "%s: too many tokens or heads", who);
  CacheRows a = {};
  if (write) a.x[0] = (const uint16_t*)k, a.x[1] = (const uint16_t*)v;
  else a.y[0] = (uint16_t*)const_cast<void*>(k), a.y[1] = (uint16_t*)const_cast<void*>(v);
  a.sb[0] = ksb, a.ss[0] = kss, a.sh[0] = ksh, a.sb[1] = vsb, a.ss[1] = vss, a.sh[1] = vsh;
  a.codes[0] = (uint8_t*)k8, a.codes[1] = (uint8_t*)v8, a.scale[0] = ks, a.scale[1] = vs;
  a.slots = slots, a.slots64 = slots64, a.S = S, a.tokens = B * S, a.Hkv = Hkv;
  a.page_shift = __builtin_ctz((unsigned)page_size), a.capacity = (int64_t)pages * page_size;
  if (dtype == SAGE_DTYPE_BF16) cache_rows_dims<DT_BF16>(a, D, cache_dtype, write, (hipStream_t)stream);
  else cache_rows_dims<DT_F16>(a, D, cache_dtype, write, (hipStream_t)stream);
  return check_launch(who);
}

}  // namespace sage

extern "C" {

int sage_cache_write(const void* k, int64_t ksb, int64_t kss, int64_t ksh, const void* v, int64_t vsb, int64_t vss,
                     int64_t vsh, int B, int S, int dtype, const void* slots, int slots64, void* k8, float* k_scale,
                     void* v8, float* v_scale, int pages, int page_size, int Hkv, int D, int cache_dtype, void* stream) {
  return sage::cache_rows(k, ksb, kss, ksh, v, vsb, vss, vsh, B, S, dtype, slots, slots64, k8, k_scale, v8, v_scale,
                          pages, page_size, Hkv, D, cache_dtype, true, stream, "sage_cache_write");
}

int sage_cache_read(void* k, int64_t ksb, int64_t kss, int64_t ksh, void* v, int64_t vsb, int64_t vss, int64_t vsh,
                    int B, int S, int dtype, const void* slots, int slots64, const void* k8, const float* k_scale,
                    const void* v8, const float* v_scale, int pages, int page_size, int Hkv, int D, int cache_dtype,
                    void* stream) {
  return sage::cache_rows(k, ksb, kss, ksh, v, vsb, vss, vsh, B, S, dtype, slots, slots64, const_cast<void*>(k8),
                          const_cast<float*>(k_scale), const_cast<void*>(v8), const_cast<float*>(v_scale), pages,
                          page_size, Hkv, D, cache_dtype, false, stream, "sage_cache_read");
}

}  // extern "C"
