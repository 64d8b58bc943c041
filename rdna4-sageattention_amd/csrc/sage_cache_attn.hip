// Attention of new queries over the quantized, paged key / value cache (layouts: sage_cache.hip).
//
// Per sequence b with n_b cached keys, the T queries of one step are the last T of them: query i of head h attends the
// keys below n_b - T, and of the T new ones those up to its own (causal), those its row of the tree mask shows, or all.
// o_i = sum_j p_ij s^v_j V_j, p_ij = 2^(x_ij - m_i) / l_i, x_ij = (q_i . K_j) s^k_j c log2 e, over codes K_j, V_j with
// scales s^k_j, s^v_j.
//
// Mapping.  The T * G queries that share a kv head (G = H / Hkv) are the rows of a matrix; a workgroup takes 16 RT of
// them against a range of the keys, and its 4 waves take turns over tiles of 32 keys.  Each wave copies its own tiles
// to LDS ahead of their use (no barrier: a wave waits for its own loads only) and turns codes to float16 as it reads them:
// int8 and E4M3 codes are exact there, so both products run on v_mfma_f32_16x16x32_f16 with float32 accumulation.
//  * S^T = K Q^T: A = 16 keys x 32 channels.  Lane (m = l % 16, g = l / 16) reads the D/4 channels from g D/4 on of key
//    m, and MFMA i takes 8 of them from each g: any order of the channels will do that Q's operand has too.
//  * The accumulator gives lane (n, g) query n and keys 4g .. 4g + 3 of each 16: with the two 16-key blocks of a tile
//    that is, packed to float16, the B operand of O^T = V^T P^T for the key order k = 8g + 4t + i <-> key 16t + 4g + i.
//    V's operand takes that order too: lane (m, g) reads D/16 channels of each of those 8 keys, pairs of keys are
//    brought together by byte permutes.  Nothing crosses lanes but the row maxima.
//  * Q rows in bfloat16 are brought into float16's range by a power of two per row, which keeps all their bits.
//  * P in float16: 11 bits of p_ij s^v_j, p_ij = 2^(x_ij - m); in blocks of 16 rows a second number takes what the first leaves, 22
//    bits in all, and its product all but hides behind HBM (one token over 48 x 4100 keys 30.4 us with one number, 31.2 with two,
//    over 64 x 600 29.0 and 30.4, over 1000 11.6 and 11.7; 16 rows over 8 x 3000, 24 kv heads, 38 and 39).  Blocks of 32 and 48 rows take one: 132 rows over 16 x 4750 keys 107 us with one, 124
//    with two, a prompt of 4096 289 and 329, and a float16 output is off by 2.9e-4 of its size then where rounding alone gives
//    2.1e-4, a bfloat16 one by no more than its rounding.
//  * The running reference m of a row is set by its first product above 0, which it brings to 2^6, and raised when one of its own
//    products passes 2^15 (32 bits hold the sum l at any m).  The largest product so far lies between 2^6 and 2^15, so a product
//    keeps all 11 bits down to 2^-20 of the largest and an error of 2^-31 of it below.
// Bound: HBM for up to 16 rows, where a key costs 2 D + 8 bytes per kv head whatever T and G are (one token over 6 x 115000
// keys, 8 kv heads x 128: 254 us, 5.8 TB/s; over 48 x 4100, 4 kv heads x 64: 31 us in all, 3.5 TB/s), the turning of codes
// and the softmax's vector instructions beyond (132 rows over 16 x 4750 keys: 107 us, 0.38 PFLOP/s of products).
// Range: float32 holds K's scores and V's products on the way, for values of magnitude up to 2^100.
#include <cmath>

#include "sage_cache.h"

namespace sage {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

constexpr int CA_WAVES = 4;
constexpr int CA_THREADS = 64 * CA_WAVES;
constexpr int CA_TILE = 32;                      // keys per wave and step
constexpr int CA_STEP = CA_TILE * CA_WAVES;      // keys per workgroup and step

constexpr int MOST_CHOICES = 8;

struct CacheAttnArgs {
  const uint16_t* q;
  int64_t qsb, qss, qsh;
  uint16_t* out;
  int64_t osb, oss, osh;
  float* lse;                       // [B, H, T] or NULL
  const uint8_t *k8, *v8;
  const float *ks, *vs;
  const int* table;                 // [B] rows of max_pages entries, `tsb` apart
  const int* lengths;
  const uint8_t* tree;              // (b, i, j) at b * msb + i * msq + j * msk, or NULL
  int64_t tsb, msb;
  int msq, msk;
  int B, H, Hkv, G, T, dtype, causal;
  int pages, page_size, page_shift, max_pages;
  int row_blocks, workers;          // workers: the most ranges of keys
  int choose;                       // the lengths decide how many of 1 .. workers <= MOST_CHOICES there are:
  float step_time[MOST_CHOICES], fixed_time[MOST_CHOICES];  // n take steps * step_time[n - 1] + fixed_time[n - 1]
  int part_rows;                    // rows of a partial: 16 RT, or all of them where that is fewer
  float scale;                      // softmax scale * log2 e = scale 2^scale_exp, scale in [1/2, 1)
  int scale_exp;
  float* part_o;                    // [kv head][row block][worker][2][part_rows][D]
  float* part_lse;                  // the same without D, log2
};

// Work of one kv head and row block: the steps (CA_STEP keys) of all sequences in a row, at least one each, cut into
// ranges that differ by one step at most, the longer ones first, whatever the sequences' lengths.  A worker's
// range holds whole sequences, whose output it writes, and up to two parts: of the one it begins inside of (partial 0) and of the one that it begins
// but does not end (partial 1); a second kernel joins those.  The lengths stay on the device: every wave adds them up.
__device__ __forceinline__ int cache_keys(const CacheAttnArgs& a, int b) {
  return min(max(a.lengths[b], 0), a.max_pages * a.page_size);
}
// An entry of an input table at a wave-uniform index, by a scalar load (the compiler takes a vector load where it cannot
// rule out that the kernel's stores change the table, and waiting for one is waiting for all loads before it).
__device__ __forceinline__ int scalar_entry(const int* p, int64_t i) {
  return ((const __attribute__((address_space(4))) int*)p)[i];
}
__device__ __forceinline__ int uniform_keys(const CacheAttnArgs& a, int b) {
  return min(max(scalar_entry(a.lengths, b), 0), a.max_pages * a.page_size);
}
__device__ __forceinline__ int cache_steps(int keys) { return max((keys + CA_STEP - 1) / CA_STEP, 1); }

// sums of x over the lanes up to and with each
template <int CTRL, int ROWS_MASK> __device__ __forceinline__ int dpp_add(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS_MASK, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int x) {
  x = dpp_add<0x111, 0xF>(x);  // row_shr 1, 2, 4, 8: within 16 lanes
  x = dpp_add<0x112, 0xF>(x);
  x = dpp_add<0x114, 0xF>(x);
  x = dpp_add<0x118, 0xF>(x);
  x = dpp_add<0x142, 0xA>(x);  // the last lane of a row to the next: rows 1 and 3, then 2 and 3
  x = dpp_add<0x143, 0xC>(x);
  return x;
}
struct Shares {
  int workers, per, longer;  // ranges; steps of each; ranges with one more
  __device__ __forceinline__ Shares(const CacheAttnArgs& a, int total) {
    int most = a.workers;
    if (a.choose) {
      float best = __builtin_inff();
#pragma unroll
      for (int i = 0; i < MOST_CHOICES; ++i) {
        const float t = __builtin_fmaf((float)total, a.step_time[i], a.fixed_time[i]);
        if (i < a.workers && t < best) best = t, most = i + 1;
      }
      most = __builtin_amdgcn_readfirstlane(most);
    }
    workers = min(most, total);
    per = total / workers;
    longer = total - per * workers;
  }
  __device__ __forceinline__ int begin(int worker) const { return worker * per + min(worker, longer); }
  __device__ __forceinline__ int worker_of(int step) const {
    const int edge = longer * (per + 1);
    return step < edge ? step / (per + 1) : longer + (step - edge) / per;
  }
};
// steps of sequences [64 c, 64 c + 64), one per lane
__device__ __forceinline__ int lane_steps(const CacheAttnArgs& a, int c, int lane) {
  const int b = 64 * c + lane;
  return b < a.B ? cache_steps(cache_keys(a, b)) : 0;
}
// steps of all sequences; `before`: of those in front of sequence b_of
__device__ __forceinline__ int all_steps(const CacheAttnArgs& a, int lane, int b_of, int& before) {
  int total = 0;
  before = 0;
  for (int c = 0; 64 * c < a.B; ++c) {
    const int n = lane_steps(a, c, lane), scan = wave_scan(n);
    if (b_of / 64 == c) before = total + __builtin_amdgcn_readlane(scan, b_of % 64) - __builtin_amdgcn_readlane(n, b_of % 64);
    total += __builtin_amdgcn_readlane(scan, 63);
  }
  return total;
}

// Copies 16 (or 4) bytes per lane, from a wave-uniform base plus the lane's offset, straight to LDS, where the wave's lanes lie
// one after the other from `lds` on.  In assembly because the compiler would wait for every copy under way before each
// read of LDS; the kernel counts its copies itself (wait_loads).  No register is written but m0, and the addresses
// are read when the copy is issued.
template <int BYTES> __device__ __forceinline__ void copy_lds(const void* base, uint32_t offset, uint32_t lds) {
  if constexpr (BYTES == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
// the same from an address of each lane's own
__device__ __forceinline__ void copy_lds_from(const void* p, uint32_t lds, int bytes) {
  if (bytes == 16)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(p) : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}
template <int N> __device__ __forceinline__ void wait_loads() {
  static_assert(N >= 0 && N <= 63, "vmcnt immediate");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// bytes 0, 1 (half 0) or 2, 3 (half 1) of a word of codes as two float16; int8 codes come with their sign bit flipped
template <int CT> __device__ __forceinline__ f16x2 codes_f16(uint32_t w, bool half) {
  if constexpr (CT == CACHE_INT8) {
    // 0x64uu is 1024 + uu in float16
    const uint32_t u = __builtin_amdgcn_perm(0x64646464u, w, half ? 0x04030402u : 0x04010400u);
    return __builtin_bit_cast(f16x2, u) - f16x2{(_Float16)1152.0f, (_Float16)1152.0f};
  } else {
    return half ? __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true))
                : __builtin_bit_cast(f16x2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false));
  }
}

// a * b where 0 times anything, an infinity or a NaN among it, is 0
__device__ __forceinline__ float mul_zero(float a, float b) {
  float r;
  asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

__device__ __forceinline__ f16x8 join4(f16x2 a, f16x2 b, f16x2 c, f16x2 d) {
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// 2^(x / 2), a factor to be taken twice: weights between parts below float32's range still count for values far above 1
__device__ __forceinline__ float half_weight(float x) { return __builtin_amdgcn_exp2f(0.5f * x); }

// maximum / sum over the 4 lanes (n, 0..3) of a row, in all of them
__device__ __forceinline__ float row4_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return max_xor32_f32(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float row4_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return add_xor32_f32(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// channel of accumulator (m, tile ct): the lane's D/16 loaded channels in order (96: a word, then two bytes)
template <int D> __device__ __forceinline__ constexpr int v_channel(int m, int ct) {
  return D == 96 ? (ct < 4 ? 4 * m + ct : 64 + 2 * m + ct - 4) : m * (D / 16) + ct;
}

// One tile in LDS, private to its wave: 32 rows of K, 32 of V, then the 32 scales of each.  The 16-byte chunks of a row are
// swapped by the row's number so that the lanes that read one chunk of 8 rows together reach all banks (96 channels: in
// order).
template <int D> struct CacheTile {
  static constexpr int KV = 32 * D;              // bytes of K, of V
  static constexpr int BYTES = 2 * KV + 256;
  static constexpr int COPIES = KV / 1024;       // copies of 1 KiB for K, for V
  static constexpr int LOADS = 2 * COPIES + 1;   // vector loads per tile
  static constexpr int VW = D == 96 ? 2 : D / 64;  // words of V per lane and key
  __device__ static __forceinline__ int swap(int row) { return D == 96 ? 0 : D == 64 ? (row >> 1) & 3 : row & (D / 16 - 1); }
  // copy j: the lane's byte offset in its block of 16 rows, from copy 0's (96 channels: from the lane's number)
  __device__ static __forceinline__ uint32_t first(int lane) {
    return D == 96 ? lane : lane / (D / 16) * D + 16 * (lane % (D / 16) ^ swap(lane / (D / 16)));
  }
  __device__ static __forceinline__ uint32_t offset(int j, uint32_t from) {
    if (D == 96) {
      const int chunk = 64 * j + from, row = chunk / 6;
      return (row & 15) * 96 + 16 * (chunk - 6 * row);
    }
    return D == 256 ? (from ^ 64 * (j % 4)) + 1024 * (j % 4) : from + (D == 128 ? 1024 * (j % 2) : 0);
  }
};
// tiles of a wave in LDS (blocks of 16 rows): two workgroups then share a CU's 160 KiB, three at head dim 96, one at 256
template <int D> constexpr int ring_tiles() { return D == 64 ? 4 : 2; }

// rows in front of the first of 16 keys from k0 on; a page outside the cache hides its keys: page 0 is read in its place
struct CacheRow {
  int64_t row;
  bool usable;
};

// The rows of a wave against the keys it walks: softmax references and sums, output accumulators, Q's operand.
template <int D, int RT> struct Rows {
  static constexpr int NK = D / 32, NC = D / 16;
  static constexpr int PARTS = RT == 1 ? 2 : 1;  // float16 numbers per weight
  f16x8 qf[RT][NK];
  // Factor of the scores to log2 units, from one power of two, so that no step of it leaves float32's range.  Positive: a hidden
  // score stays -inf.  Below 2^-126 it has fewer bits, within 2^-150 of the exact factor: a score, which is below 2^124 before it,
  // is off by no more than 2^-26.
  float qs[RT];
  int row_t[RT];  // the row's new token
  float m[RT], l[RT];
  float limit[RT];  // of a product: 2^15, -1 while there was none above 0
  v4f acc[RT][NC];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m[rt] = -__builtin_inff();
      limit[rt] = -1.0f;
      l[rt] = 0.0f;
#pragma unroll
      for (int c = 0; c < NC; ++c) acc[rt][c] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
  }

  // rows first, first + 1, .. of sequence b and kv head h (past the last: the last again)
  __device__ __forceinline__ void load_q(const CacheAttnArgs& a, int b, int h, int first, int n, int g) {
    uint32_t qw[RT][D / 8];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int r = min(first + rt * 16 + n, a.T * a.G - 1);
      const int t = r / a.G, hq = h * a.G + r % a.G;
      row_t[rt] = t;
      const uint16_t* qp = a.q + b * a.qsb + t * a.qss + hq * a.qsh + g * (D / 4);
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const v4i x = *reinterpret_cast<const v4i*>(qp + 8 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) qw[rt][4 * i + j] = (uint32_t)x[j];
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const uint32_t(&w)[D / 8] = qw[rt];
      int power = a.scale_exp;
      bool endless;  // the row holds an infinity: each of its scores is one or NaN, and its weights are NaN whatever the signs
      if (a.dtype == DT_BF16) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) top = fmaxf(top, fmaxf(fabsf(bf16_lo(w[i])), fabsf(bf16_hi(w[i]))));
        const uint32_t e = max(__float_as_uint(row4_max(top)) >> 23, 15u);  // of the row's largest magnitude
        // largest magnitude to [2^14, 2^15): a value 2^-28 of it still keeps its 8 bits
        const float up = e == 255u ? 1.0f : __uint_as_float((268u - e) << 23);
        power += e == 255u ? 0 : (int)e - 141;
        endless = e == 255u;
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            qf[rt][i][2 * j] = (_Float16)(bf16_lo(w[4 * i + j]) * up);
            qf[rt][i][2 * j + 1] = (_Float16)(bf16_hi(w[4 * i + j]) * up);
          }
      } else {
        u16x2 top = {0, 0};
#pragma unroll
        for (int i = 0; i < D / 8; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, w[i] & 0x7FFF7FFFu));
        endless = row4_max((float)max(top[0], top[1])) >= (float)0x7C00;
#pragma unroll
        for (int i = 0; i < NK; ++i)
          qf[rt][i] = __builtin_bit_cast(f16x8, v4i{(int)w[4 * i], (int)w[4 * i + 1], (int)w[4 * i + 2], (int)w[4 * i + 3]});
      }
      // (scores of NaN: those of -inf would count as hidden)
      if (endless) qf[rt][0] = __builtin_bit_cast(f16x8, v4i{0x7E007E00, 0x7E007E00, 0x7E007E00, 0x7E007E00});
      qs[rt] = fminf(fmaxf(__builtin_ldexpf(a.scale, power), 0x1p-149f), 0x1.fffffep127f);
#pragma unroll
      for (int i = 0; i < NK; ++i) asm volatile("" : "+v"(qf[rt][i]));  // waited for here, not in the loop
    }
  }

  // Scores of hidden keys become -inf (tiles that hold one only).  gone: bit 4 t + i, key 16 t + 4 g + i of the tile is past the
  // sequence or on no page; node: the number of key 4 g among the new tokens.
  __device__ __forceinline__ void hide(const CacheAttnArgs& a, int b, int node, uint32_t gone, v4f (&s)[RT][2]) const {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      uint32_t hidden = gone;
      if (a.tree) {
        const auto* shown = (const __attribute__((address_space(1))) uint8_t*)(a.tree + b * a.msb);
        const int row = row_t[rt] * a.msq;  // (a mask's offsets fit 32 bits: checked on the host)
        uint8_t see[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) see[j] = shown[row + min(max(node + 16 * (j / 4) + j % 4, 0), a.T - 1) * a.msk];
#pragma unroll
        for (int j = 0; j < 8; ++j) hidden |= (uint32_t)(see[j] == 0 && node + 16 * (j / 4) + j % 4 >= 0) << j;
      } else if (a.causal) {
#pragma unroll
        for (int j = 0; j < 8; ++j) hidden |= (uint32_t)(node + 16 * (j / 4) + j % 4 > row_t[rt]) << j;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (hidden >> j & 1) s[rt][j / 4][j % 4] = -__builtin_inff();
    }
    asm volatile("" ::: "memory");  // (a block of its own: never turned into selects for every tile)
  }

  // Scores (with K's scales) to the weights' operand: sums and references brought up to date.  The terms are taken against the
  // references so far; where a product could pass 2^15, or a row has no reference from a product yet, the references are
  // looked at first.
  __device__ __forceinline__ void weights(const v4f (&s)[RT][2], const v4f (&vs)[2], f16x8 (&pf)[RT][PARTS]) {
    float vs_top = 0x1p-85f;  // (a weight stays within 2^100 whatever its scale is)
#pragma unroll
    for (int j = 0; j < 8; ++j) vs_top = fmaxf(vs_top, vs[j / 4][j % 4]);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float p[8], pv[8];
      float& M = m[rt];
      auto terms = [&](float ref) {
        float top = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rt][j / 4][j % 4], qs[rt], -ref));
          top = fmaxf(top, p[j]);
        }
        return top;
      };
      const float top = terms(M == -__builtin_inff() ? 0.0f : M);
      if (__any(!(top * vs_top <= limit[rt]))) {  // (a bound of the largest product, by two different keys)
        // Whether a reference is raised follows from the row's own products alone, or its last bits would depend on the scales of keys
        // that it does not see and on the other rows of the wave.
        bool raise = false;
        if (__any(limit[rt] > 0.0f)) {
          float now = 0.0f;  // (0 times the infinite scale of a hidden key: NaN, which fmaxf leaves out)
#pragma unroll
          for (int j = 0; j < 8; ++j) now = fmaxf(now, p[j] * fmaxf(vs[j / 4][j % 4], 0x1p-85f));
          raise = row4_max(now) > limit[rt];
        }
        float y = -__builtin_inff();
#pragma unroll
        for (int j = 0; j < 8; ++j) y = fmaxf(y, s[rt][j / 4][j % 4] * qs[rt]);
        y = row4_max(y);
        terms(y == -__builtin_inff() ? 0.0f : y);
        float most = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, mul_zero(p[j], vs[j / 4][j % 4]));
        most = row4_max(most);
        const bool first = limit[rt] < 0.0f, product = most > 0.0f && most < __builtin_inff();
        // the reference that brings the largest product to [2^6, 2^7), and no weight beyond 2^92
        float to = fmaxf(y - 92.0f, product ? y + (float)(__builtin_amdgcn_frexp_expf(most) - 7) : -__builtin_inff());
        if (first) to = product ? fmaxf(to, M - 92.0f) : fmaxf(M, y);
        if (first ? to > -__builtin_inff() : raise) {
          const float down = __builtin_amdgcn_exp2f(M - to);
          l[rt] *= down;
#pragma unroll
          for (int ct = 0; ct < NC; ++ct) acc[rt][ct] *= down;  // (zeros still, where down is large)
          M = to;
          if (product) limit[rt] = 0x1p15f;
        }
        terms(M == -__builtin_inff() ? 0.0f : M);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        l[rt] += p[j];
        pv[j] = mul_zero(p[j], vs[j / 4][j % 4]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) pf[rt][0][j] = (_Float16)pv[j];
      if constexpr (PARTS == 2) {
#pragma unroll
        for (int j = 0; j < 8; ++j) pf[rt][1][j] = (_Float16)(pv[j] - (float)pf[rt][0][j]);
      }
    }
  }
};

// A worker's place: kv head, row block and steps [s0, s1), the sequence of step s0 and the step's place in it.
struct Work {
  int h, rb, worker, s0, s1, b, first;
  int lane_keys;  // keys of sequence `lane`, where there are no more than 64
  __device__ __forceinline__ bool find(const CacheAttnArgs& a, int lane) {
    const bool few = a.B <= 64;  // the lengths are read once
    lane_keys = few && lane < a.B ? cache_keys(a, lane) : 0;
    int n = lane < a.B ? cache_steps(lane_keys) : 0, scan = few ? wave_scan(n) : 0, unused;
    const Shares shares(a, few ? __builtin_amdgcn_readlane(scan, 63) : all_steps(a, lane, -1, unused));
    // The row blocks of one range of keys on one XCD, next to each other: the ranges dealt to the XCDs one by one where that gives
    // each as many, the row blocks of all ranges in a row cut into eighths elsewhere (32-row blocks of 12 heads x 256, 36 ranges:
    // 547 us dealt, 387 cut; a prompt of 2048 of one head: 89 and 37).
    const int id = blockIdx.x, ranges = a.Hkv * shares.workers;
    int range;
    if (ranges % 8 == 0) {
      range = id / (8 * a.row_blocks) * 8 + id % 8;
      rb = id / 8 % a.row_blocks;
    } else {
      const int items = ranges * a.row_blocks, eighth = (items + 7) / 8;
      const int item = id / 8 < eighth ? id % 8 * eighth + id / 8 : items;
      range = item / a.row_blocks;
      rb = item - range * a.row_blocks;
    }
    if (range >= ranges) return false;
    h = range / shares.workers, worker = range - h * shares.workers;
    s0 = shares.begin(worker);
    s1 = shares.begin(worker + 1);
    b = first = 0;
    for (int c = 0, sum = 0; 64 * c < a.B; ++c) {
      if (!few) n = lane_steps(a, c, lane), scan = wave_scan(n) + sum;
      sum = __builtin_amdgcn_readlane(scan, 63);
      if (sum > s0) {
        const int at = __builtin_ctzll(__ballot(scan > s0));
        b = 64 * c + at;
        first = s0 - (__builtin_amdgcn_readlane(scan, at) - __builtin_amdgcn_readlane(n, at));
        break;
      }
    }
    return true;
  }
  __device__ __forceinline__ int keys(const CacheAttnArgs& a) const {
    return a.B <= 64 ? __builtin_amdgcn_readlane(lane_keys, b) : uniform_keys(a, b);
  }
};

// A wave's priority by how much of its workgroup's steps lies behind it.  Workgroups of equal work that share a CU would end far
// apart, the one that came first served first (6 x 115000 keys: 194 and 237 us; three 132-row workgroups: 87, 105 and
// 126 us), the last ones alone on their CUs; with those behind served first they end together.
struct Pace {
  int total, at, level;
  __device__ __forceinline__ explicit Pace(int steps) : total(steps), at(0), level(3) {
    __builtin_amdgcn_s_setprio(3);
    next();
  }
  __device__ __forceinline__ void next() {
    at = level == 3 ? total / 2 : level == 2 ? total - total / 5 : level == 1 ? total - total / 16 : 0x7FFFFFFF;
  }
  __device__ __forceinline__ void done(int steps) {
    if (steps < at) return;
    --level;
    if (level == 2) __builtin_amdgcn_s_setprio(2);
    else if (level == 1) __builtin_amdgcn_s_setprio(1);
    else __builtin_amdgcn_s_setprio(0);
    next();
  }
};

// A sequence's part of a worker's range: keys [k_begin, k_end) of its `len`.
struct Segment {
  int len, take, base, open, k_begin, k_end;
  bool whole;
  int64_t unit;      // rows in front of its partial
  const int* table;
  __device__ __forceinline__ Segment(const CacheAttnArgs& a, const Work& w, int block_rows) {
    len = w.keys(a);
    const int steps = cache_steps(len);
    take = max(min(steps - w.first, w.s1 - w.s0), 1);  // (1 and more, even if another stream rewrote the lengths by now)
    whole = take == steps;
    unit = ((((int64_t)w.h * a.row_blocks + w.rb) * a.workers + w.worker) * 2 + (w.first > 0 ? 0 : 1)) * a.part_rows;
    base = len - a.T;  // key of the first new token
    // keys below `open` are seen by every row of the block; its last row sees none from k_end on
    open = a.tree ? base : a.causal ? base + 1 + w.rb * block_rows / a.G : len;
    k_begin = w.first * CA_STEP, k_end = min(len, (w.first + take) * CA_STEP);
    if (a.causal && !a.tree) k_end = min(k_end, base + 1 + (min((w.rb + 1) * block_rows, a.T * a.G) - 1) / a.G);
    table = a.table + w.b * a.tsb;
  }
  __device__ __forceinline__ CacheRow rows_of(const CacheAttnArgs& a, int h, int key) const {
    const int page = scalar_entry(table, min(key >> a.page_shift, a.max_pages - 1));
    const bool usable = page >= 0 && page < a.pages;
    return CacheRow{((int64_t)(usable ? page : 0) * a.Hkv + h) * a.page_size + (key & (a.page_size - 1)), usable};
  }
  // bit 4 t + i: key k0 + 16 t + 4 g + i is past the sequence or (bit t of usable) on no page
  __device__ __forceinline__ uint32_t gone(int k0, int g, uint32_t usable) const {
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k0 + 4 * g + 16 * (j / 4) + j % 4 >= len || !(usable >> (j / 4) & 1)) bits |= 1u << j;
    return bits;
  }
};

template <int D, int CT, int RT>
__global__ __launch_bounds__(CA_THREADS, D == 64 && RT == 2 ? 3 : D == 256 && RT == 2 ? 1 : 2) void cache_attn_kernel(const CacheAttnArgs a) {
  constexpr int NK = D / 32, NC = D / 16;
  constexpr int ROWS = 16 * RT;
  constexpr int LD = D + 4;  // LDS row stride of the joining of the waves, in floats
  using Tile = CacheTile<D>;
  // LDS of a wave: NS whole tiles, a tile is replaced once it is done with (as many bytes under way as the LDS of the workgroups
  // that share a CU holds).  48 rows: K of one tile, V and the scales of two, the next tile is started once this one's scores are
  // there (132 rows over 16 x 4750 keys: 111 us, 112 with two whole tiles).  Blocks of 32 rows at head dim 128 in a third of a CU's
  // registers, with spills: 64 rows over 8 x 5000 keys 58 us, in half of them 45.
  constexpr bool EARLY = RT == 3;
  constexpr int NS = EARLY ? 1 : RT == 2 ? 2 : ring_tiles<D>();
  constexpr int PER_WAVE = EARLY ? 3 * Tile::KV + 512 : NS * Tile::BYTES;
  constexpr int JOIN = CA_WAVES * 16 * LD * 4, RING = CA_WAVES * PER_WAVE;
  __shared__ __attribute__((aligned(16))) uint8_t smem[JOIN > RING ? JOIN : RING];
  float (*so)[16][LD] = reinterpret_cast<float (*)[16][LD]>(smem);  // (the waves are joined after their last tile)
  __shared__ float sm[CA_WAVES][ROWS], sl[CA_WAVES][ROWS];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int rows = a.T * a.G;
  Work work;
  if (!work.find(a, lane)) return;
  Pace pace(work.s1 - work.s0);
  int done = 0;

  for (;; ++work.b, work.first = 0) {
  const int b = work.b, h = work.h, rb = work.rb;
  const Segment seg(a, work, ROWS);
  Rows<D, RT> r;
  r.clear();
  uint8_t* ring = smem + wave * PER_WAVE;
  const uint32_t ring_at = lds_address(ring);
  // place of tile `stage`'s K (kv 0), V (1), scales (2) in the wave's LDS
  auto place = [&](int stage, int kv) {
    return EARLY ? (kv == 0 ? 0 : kv == 1 ? (1 + stage) * Tile::KV : 3 * Tile::KV + 256 * stage) : stage * Tile::BYTES + kv * Tile::KV;
  };
  // where the lane's operands lie in a tile: K of key n, V and scales of key 4 g (keys and chunks further on differ by constants),
  // and what it copies
  const int k_at0 = n * D + (D == 96 ? 24 * g : 16 * ((D / 64 * g) ^ Tile::swap(n)));
  const int v_per = D == 96 ? 4 : D / 16;  // bytes of a key that the lane starts from
  const int v_at0 = 4 * g * D + (v_per * n & 15) + 16 * ((v_per * n >> 4) ^ (D == 96 ? 0 : Tile::swap(4 * g)));
  const uint32_t from0 = Tile::first(lane);
  // 32 rows and more leave no registers to keep what is derived from these through the loop
  auto afresh = [&](auto x) {
    if (RT >= 2) asm volatile("" : "+v"(x));
    return x;
  };
  auto issue = [&](CacheRow at0, CacheRow at1, int stage) {
    const uint32_t from = afresh(from0);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      const uint32_t to = __builtin_amdgcn_readfirstlane(ring_at + place(stage, kv));
      const uint8_t* codes = kv ? a.v8 : a.k8;
      const uint8_t *p0 = codes + at0.row * D, *p1 = codes + at1.row * D;
#pragma unroll
      for (int j = 0; j < Tile::COPIES; ++j) {
        const uint32_t dst = to + 1024 * j;
        if (D == 96 && j == 1) copy_lds_from((lane < 32 ? p0 : p1) + Tile::offset(j, from), dst, 16);  // half of it in each block
        else copy_lds<16>(2 * j / Tile::COPIES ? p1 : p0, Tile::offset(j, from), dst);
      }
    }
    const int64_t row = (lane & 16 ? at1.row : at0.row) + (lane & 15);
    copy_lds_from((lane < 32 ? a.ks : a.vs) + row, __builtin_amdgcn_readfirstlane(ring_at + place(stage, 2)), 4);
  };
  // NS tiles on their way or in use (the last one again where there are fewer)
  int k0 = seg.k_begin + wave * CA_TILE;
  const int tiles = k0 < seg.k_end ? (seg.k_end - k0 + CA_STEP - 1) / CA_STEP : 0;
  uint32_t usable = 0;  // bits 2 i, 2 i + 1: the two pages of tile i from the current one on
  if (tiles) {
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int k = k0 + min(i, tiles - 1) * CA_STEP;
      const CacheRow at0 = seg.rows_of(a, h, k), at1 = seg.rows_of(a, h, k + 16);
      usable |= ((uint32_t)at0.usable | (uint32_t)at1.usable << 1) << 2 * i;
      issue(at0, at1, i);
    }
  }

  r.load_q(a, b, h, rb * ROWS, n, g);

  if (tiles) {
    int stage = 0;
    for (int left = tiles;; --left, k0 += CA_STEP) {
      // the loads of the tiles behind this one may be outstanding
      if (left >= NS) wait_loads<(NS - 1) * Tile::LOADS>();
      else if (NS > 2 && left == 2) wait_loads<Tile::LOADS>();
      else wait_loads<0>();
      const int k_at = afresh(k_at0), v_at = afresh(v_at0);
      const uint8_t* const kt = ring + place(stage, 0);
      uint8_t* const vt = ring + place(stage, 1);
      const uint8_t* const st = ring + place(stage, 2);
      const bool more = left > NS;
      CacheRow next0 = {0, false}, next1 = {0, false};
      if (more) next0 = seg.rows_of(a, h, k0 + NS * CA_STEP), next1 = seg.rows_of(a, h, k0 + NS * CA_STEP + 16);
      const bool masked = k0 + CA_TILE > seg.open || (usable & 3) != 3;
      v4f s[RT][2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t kw[D / 16];
        if constexpr (D == 96) {
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            const v2i w = *reinterpret_cast<const v2i*>(kt + 16 * t * D + k_at + 8 * i);
            kw[2 * i] = w[0], kw[2 * i + 1] = w[1];
          }
        } else {
#pragma unroll
          for (int i = 0; i < D / 64; ++i) {
            const v4i w = *reinterpret_cast<const v4i*>(kt + 16 * t * D + (k_at ^ 16 * i));
#pragma unroll
            for (int j = 0; j < 4; ++j) kw[4 * i + j] = (uint32_t)w[j];
          }
        }
#pragma unroll
        for (int i = 0; i < NK; ++i) {
          uint32_t w0 = kw[2 * i], w1 = kw[2 * i + 1];
          if (CT == CACHE_INT8) w0 ^= 0x80808080u, w1 ^= 0x80808080u;
          const f16x8 ka = join4(codes_f16<CT>(w0, false), codes_f16<CT>(w0, true), codes_f16<CT>(w1, false),
                                 codes_f16<CT>(w1, true));
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[rt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ka, r.qf[rt][i], s[rt][t], 0, 0, 0);
        }
      }
      v4f ks[2], vs[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        ks[t] = *reinterpret_cast<const v4f*>(st + 64 * t + 16 * g);
        vs[t] = *reinterpret_cast<const v4f*>(st + 128 + 64 * t + 16 * g);
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int t = 0; t < 2; ++t) s[rt][t] *= ks[t];
      }
      if (EARLY && more) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K's reads are done: its place takes the next tile's
        issue(next0, next1, stage ^ 1);
      }
      // Tiles with hidden keys: their scores become -inf.  The rest needs no selects: a weight of 0 times whatever scale is 0
      // (mul_zero), and V codes of keys past the sequence or on no page, which may be NaN, become 0 where the lane reads them.
      if (masked) {
        const uint32_t gone = seg.gone(k0, g, usable);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (CT == CACHE_E4M3 && (gone >> j & 1)) {
            uint8_t* vp = vt + (16 * (j / 4) + j % 4) * D;
            if constexpr (D == 64) *reinterpret_cast<uint32_t*>(vp + (v_at ^ 16 * (j % 4 / 2))) = 0;
            else if constexpr (D == 128) *reinterpret_cast<v2i*>(vp + (v_at ^ 16 * (j % 4))) = v2i{0, 0};
            else if constexpr (D == 256) *reinterpret_cast<v4i*>(vp + (v_at ^ 16 * (j % 4))) = v4i{0, 0, 0, 0};
            else {
              *reinterpret_cast<uint32_t*>(vp + v_at) = 0;
              *reinterpret_cast<uint16_t*>(vp + 4 * g * D + 64 + 2 * n) = 0;
            }
          }
        }
        r.hide(a, b, k0 + 4 * g - seg.base, gone, s);
      }
      f16x8 pf[RT][r.PARTS];
      r.weights(s, vs, pf);
      // V operand: keys (0, 1), (2, 3) of each block side by side
      uint32_t vw[8][Tile::VW];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint8_t* vp = vt + (16 * (j / 4) + j % 4) * D;
        if constexpr (D == 64) {
          vw[j][0] = *reinterpret_cast<const uint32_t*>(vp + (v_at ^ 16 * (j % 4 / 2)));
        } else if constexpr (D == 96) {
          vw[j][0] = *reinterpret_cast<const uint32_t*>(vp + v_at);
          vw[j][1] = *reinterpret_cast<const uint16_t*>(vp + 4 * g * D + 64 + 2 * n);
        } else if constexpr (D == 128) {
          const v2i y = *reinterpret_cast<const v2i*>(vp + (v_at ^ 16 * (j % 4)));
          vw[j][0] = y[0], vw[j][1] = y[1];
        } else {
          const v4i y = *reinterpret_cast<const v4i*>(vp + (v_at ^ 16 * (j % 4)));
#pragma unroll
          for (int i = 0; i < 4; ++i) vw[j][i] = (uint32_t)y[i];
        }
      }
#pragma unroll
      for (int i = 0; i < Tile::VW; ++i) {
        if (CT == CACHE_INT8) {
#pragma unroll
          for (int j = 0; j < 8; ++j) vw[j][i] ^= 0x80808080u;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {  // channels 4 i + 2 u, + 1 of the lane
          if (D == 96 && i == 1 && u == 1) continue;
          uint32_t w[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)  // bytes (A_2u, B_2u, A_2u+1, B_2u+1)
            w[j] = __builtin_amdgcn_perm(vw[2 * j + 1][i], vw[2 * j][i], u ? 0x07030602u : 0x05010400u);
#pragma unroll
          for (int o = 0; o < 2; ++o) {
            const int c = 4 * i + 2 * u + o;
            const f16x8 va = join4(codes_f16<CT>(w[0], o), codes_f16<CT>(w[1], o), codes_f16<CT>(w[2], o), codes_f16<CT>(w[3], o));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
              for (int part = 0; part < r.PARTS; ++part)
                r.acc[rt][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pf[rt][part], r.acc[rt][c], 0, 0, 0);
            }
          }
        }
      }
      pace.done(++done);
      if (left == 1) break;
      usable >>= 2;
      if (more) {
        usable |= ((uint32_t)next0.usable | (uint32_t)next1.usable << 1) << 2 * (NS - 1);
        if (!EARLY) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile's reads are done: its place takes the one NS tiles on
          issue(next0, next1, stage);
        }
      }
      stage = EARLY ? stage ^ 1 : stage + 1 == NS ? 0 : stage + 1;
    }
  }

  // join the waves, 16 rows at a time
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float sum = row4_sum(r.l[rt]);
    if (g == 0) {
      sm[wave][rt * 16 + n] = r.m[rt];
      sl[wave][rt * 16 + n] = sum;
    }
  }
  __syncthreads();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int own = rt * 16 + n;
    float top = sm[0][own];
#pragma unroll
    for (int w = 1; w < CA_WAVES; ++w) top = fmaxf(top, sm[w][own]);
    const float down = r.m[rt] == -__builtin_inff() ? 1.0f : half_weight(r.m[rt] - top);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) so[wave][n][v_channel<D>(4 * g + i, c)] = r.acc[rt][c][i] * down * down;
    __syncthreads();
    // 16 threads per row
    const int row = threadIdx.x / 16, part = threadIdx.x % 16, rr = rt * 16 + row, R = rb * ROWS + rr;
    float M = sm[0][rr];
#pragma unroll
    for (int w = 1; w < CA_WAVES; ++w) M = fmaxf(M, sm[w][rr]);
    float L = 0.0f;
#pragma unroll
    for (int w = 0; w < CA_WAVES; ++w) {  // (a NaN sum stays one; references of one row lie up to some 190 apart by the sizes of values alone)
      const float down = sm[w][rr] == -__builtin_inff() ? 1.0f : half_weight(sm[w][rr] - M);
      L += sl[w][rr] * down * down;
    }
    // a row that sees no key: 0, logsumexp -inf
    const float fin = 1.0f / L;
    const float lse2 = L == 0.0f ? -__builtin_inff() : M + __builtin_log2f(L);
    constexpr int PER = D / 16;
    float o[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      float v = so[0][row][part * PER + i];
#pragma unroll
      for (int w = 1; w < CA_WAVES; ++w) v += so[w][row][part * PER + i];
      o[i] = L == 0.0f ? 0.0f : v * fin;
    }
    if (R < rows) {
      if (seg.whole) {
        const int t = R / a.G, hq = h * a.G + R % a.G;
        uint16_t* op = a.out + b * a.osb + t * a.oss + hq * a.osh + part * PER;
#pragma unroll
        for (int i = 0; i < PER; i += 2) {
          const uint32_t w = a.dtype == DT_BF16 ? f32_to_bf16_bits(o[i]) | (f32_to_bf16_bits(o[i + 1]) << 16)
                                                : f32_to_f16_bits(o[i]) | (f32_to_f16_bits(o[i + 1]) << 16);
          *reinterpret_cast<uint32_t*>(op + i) = w;
        }
        if (a.lse && part == 0) a.lse[((int64_t)b * a.H + hq) * a.T + t] = lse2 * 0.69314718055994530942f;
      } else {
        float* op = a.part_o + (seg.unit + rr) * D + part * PER;
#pragma unroll
        for (int i = 0; i < PER; i += 2) *reinterpret_cast<float2*>(op + i) = make_float2(o[i], o[i + 1]);
        if (part == 0) a.part_lse[seg.unit + rr] = lse2;
      }
    }
    if (rt + 1 < RT) __syncthreads();
  }
  work.s0 += seg.take;
  if (work.s0 >= work.s1 || work.b + 1 >= a.B) break;
  __syncthreads();  // the next sequence's rows go where these were read
  }
}

// Joins the parts of the rows of sequences that several workers shared: o = sum_i 2^(lse_i - M) o_i / sum_i 2^(lse_i - M).
// One row per group of `slices` waves, each of which adds up every slices-th part, in an order that the lengths alone
// decide; a wave that does it alone takes PER rows of one sequence and kv head.  Up to 8 parts
// per wave (4 of each of 4 rows) are all on their way before the first weight is known: 1000 keys of one sequence 11.1 us in all,
// 13.1 with the weights first.
constexpr int MERGE_SLICES = 16;
template <int D, int PER>
__global__ __launch_bounds__(PER > 1 ? 256 : 64 * MERGE_SLICES) void cache_merge_kernel(const CacheAttnArgs a, int block_rows, int slices) {
  constexpr int VEC = D <= 64 ? 1 : D <= 128 ? 2 : 4;  // channels per lane
  typedef float vec __attribute__((ext_vector_type(VEC)));
  __shared__ float so[MERGE_SLICES][D];
  __shared__ float sml[MERGE_SLICES][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = a.T * a.G;
  const bool alone = slices == 1;
  const int groups = (rows + PER - 1) / PER;
  const int at = alone ? blockIdx.x * (blockDim.x / 64) + wave : blockIdx.x;
  if (at >= groups * a.B * a.Hkv) return;
  const int slice = alone ? 0 : wave;
  const int pair = at / groups, group = at - pair * groups, b = pair / a.Hkv, h = pair - b * a.Hkv;
  int before;
  const int total = all_steps(a, lane, b, before), steps = cache_steps(uniform_keys(a, b));
  const Shares shares(a, total);
  const int w0 = shares.worker_of(before), parts = shares.worker_of(before + steps - 1) - w0 + 1;
  if (parts == 1) return;  // written whole
  const bool mine = lane * VEC < D;
  const int first = group * PER, last = min(first + PER, rows);
  auto place = [&](int R, int i) {  // part i of row R
    const int rb = R / block_rows, rr = R % block_rows;
    return (((((int64_t)h * a.row_blocks + rb) * a.workers + w0) + i) * 2 + (i == 0)) * a.part_rows + rr;
  };
  auto store = [&](int R, vec o, float M, float L) {
    if (L != 0.0f) o *= 1.0f / L;
    const int t = R / a.G, hq = h * a.G + R % a.G;
    if (mine) {
      uint16_t* op = a.out + b * a.osb + t * a.oss + hq * a.osh + lane * VEC;
      uint32_t w[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = a.dtype == DT_BF16 ? f32_to_bf16_bits(o[i]) : f32_to_f16_bits(o[i]);
      if constexpr (VEC == 1) *op = (uint16_t)w[0];
      else if constexpr (VEC == 2) *reinterpret_cast<uint32_t*>(op) = w[0] | (w[1] << 16);
      else *reinterpret_cast<v2i*>(op) = v2i{(int)(w[0] | (w[1] << 16)), (int)(w[2] | (w[3] << 16))};
    }
    if (a.lse && lane == 0)
      a.lse[((int64_t)b * a.H + hq) * a.T + t] = L == 0.0f ? -__builtin_inff() : (M + __builtin_log2f(L)) * 0.69314718055994530942f;
  };
  auto join = [&](int R, vec o, float M, float L) {  // the waves' sums
    if (slices > 1) {
      if (mine) *reinterpret_cast<vec*>(&so[wave][lane * VEC]) = o;
      if (lane == 0) sml[wave][0] = M, sml[wave][1] = L;
      __syncthreads();
      if (wave) return;
      float top = M;
      for (int i = 1; i < slices; ++i) top = fmaxf(top, sml[i][0]);
      const float down = M == -__builtin_inff() ? 1.0f : half_weight(M - top);
      o = o * down * down, L = L * down * down, M = top;
      for (int i = 1; i < slices; ++i) {
        const float w = sml[i][0] == -__builtin_inff() ? 1.0f : half_weight(sml[i][0] - top);
        L += sml[i][1] * w * w;
        if (mine) o += *reinterpret_cast<const vec*>(&so[i][lane * VEC]) * w * w;
      }
    }
    store(R, o, M, L);
  };

  constexpr int FEW = PER == 1 ? 8 : 4;
  if (parts <= FEW * slices) {
    // lane l: the wave's part l % FEW of row l / FEW (and so on all over); what is past the end is read again and weighs 0
    const int i_own = lane % FEW * slices + slice, r_own = lane / FEW % PER;
    const float read = a.part_lse[place(min(first + r_own, last - 1), min(i_own, parts - 1))];
    const int channel = mine ? lane * VEC : 0;
    vec v[PER][FEW];
#pragma unroll
    for (int r = 0; r < PER; ++r)
#pragma unroll
      for (int i = 0; i < FEW; ++i)
        v[r][i] = *reinterpret_cast<const vec*>(a.part_o + place(min(first + r, last - 1), min(i * slices + slice, parts - 1)) * D + channel);
    const float x = i_own < parts ? read : -__builtin_inff();
    auto over = [&](float y, auto with) {  // the parts of a row are neighbouring lanes
      y = with(y, __shfl_xor(y, 1));
      y = with(y, __shfl_xor(y, 2));
      return FEW == 8 ? with(y, __shfl_xor(y, 4)) : y;
    };
    const float M = over(x, [](float p, float q) { return fmaxf(p, q); });
    // (-inf: a part without a visible key; a NaN stays one)
    const float w = x == -__builtin_inff() ? 0.0f : half_weight(x - M);
    const float L = over(w * w, [](float p, float q) { return p + q; });
#pragma unroll
    for (int r = 0; r < PER; ++r) {
      if (first + r >= last) break;
      vec o = 0.0f;
#pragma unroll
      for (int i = 0; i < FEW; ++i) {
        const float wi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), r * FEW + i));
        if (i * slices + slice < parts) o += v[r][i] * wi * wi;
      }
      join(first + r, o, __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(M), r * FEW)),
            __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(L), r * FEW)));
    }
    return;
  }
  for (int R = first; R < last; ++R) {
  auto part = [&](int i) { return place(R, i); };

  float M = -__builtin_inff(), L = 0.0f;
  vec o = 0.0f;
  for (int i0 = 0; i0 < parts; i0 += 64 * slices) {  // part i0 + lane * slices + slice: one per lane
    const int i = i0 + lane * slices + slice;
    const float x = i < parts ? a.part_lse[part(i)] : -__builtin_inff();
    float top = x;
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float now = fmaxf(M, top);
    // (-inf: a part without a visible key; a NaN stays one)
    const float w = x == -__builtin_inff() ? 0.0f : half_weight(x - now);
    if (now > M) {
      const float down = M == -__builtin_inff() ? 0.0f : half_weight(M - now);
      o = o * down * down, L = L * down * down, M = now;
    }
    const int count = min(64, (parts - i0 - slice + slices - 1) / slices);
#pragma unroll 8
    for (int j = 0; j < count; ++j) {
      const float wj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), j));
      vec v = 0.0f;
      if (mine) v = *reinterpret_cast<const vec*>(a.part_o + part(i0 + j * slices + slice) * D + lane * VEC);
      L += wj * wj;
      o += v * wj * wj;  // (a part without a visible key holds zeros)
    }
  }
  join(R, o, M, L);
  }
}

// Rows per workgroup (16 rt) and the most workers per kv head and row block for a call.
struct CachePlan {
  int rt, row_blocks, workers, part_rows, choose;
  float step_time[MOST_CHOICES], fixed_time[MOST_CHOICES];
  int64_t o_bytes, bytes;
};

static CachePlan cache_plan(int B, int H, int Hkv, int T, int D, int max_keys, int cus) {
  CachePlan p;
  const int64_t rows = (int64_t)T * (H / Hkv);
  const int64_t most = (int64_t)B * ((max_keys + CA_STEP - 1) / CA_STEP);  // (the lengths are on the device: the table's width)
  auto units_of = [&](int rt) { return Hkv * ((rows + 16 * rt - 1) / (16 * rt)); };
  auto slots_of = [&](int rt) { return (int64_t)cus * (D == 256 ? 1 : D == 64 && rt == 2 ? 3 : 2); };
  // Time of a call in blocks of 16 rt rows, in steps of a workgroup of 32 rows, with n ranges: rounds of workgroups that run at
  // once, times a walk and what a workgroup costs beside it, which is 4 steps more where parts are written and joined
  // and 7 more in blocks of 48 rows (13 us).  A step of those takes 1.2 times one of 32 rows: turning codes to float16 costs as
  // much as the softmax and products of some 28 rows.
  auto time = [&](int rt, int64_t n, float& per_step, float& fixed) {
    const int64_t rounds = (units_of(rt) * n + slots_of(rt) - 1) / slots_of(rt);
    per_step = (float)rounds * (rt == 3 ? 1.2f : 1.0f) / (float)n;
    fixed = (float)rounds * ((n == 1 ? 3.0f : 7.0f) + (rt == 3 ? 7.0f : 0.0f));
    return __builtin_fmaf((float)most, per_step, fixed);
  };
  // the number w of ranges for it, of as many as are worth a look
  auto best = [&](int rt, int64_t& w) {
    const int64_t fill = slots_of(rt) / units_of(rt);
    float per_step, fixed;
    if (fill >= MOST_CHOICES) return w = fill, time(rt, fill, per_step, fixed);  // one round whatever w is
    float least = time(rt, w = 1, per_step, fixed);
    for (int64_t n = 2; n <= MOST_CHOICES; ++n) {
      const float t = time(rt, n, per_step, fixed);
      if (t < least) least = t, w = n;
    }
    return least;
  };
  int64_t w = 0, w3 = 0;
  p.rt = rows <= 16 ? 1 : 2;
  const float t = best(p.rt, w);
  // Blocks of 48 rows at head dims 96 and 128 (at 64 the turning is half as much, at 256 they do not fit the registers).  In us with
  // 32 and 48, 8 kv heads x 128: 132 rows over 16 sequences of up to 9001 keys 128 and 110, 96 rows over 16 of up to 16000 152
  // and 139, a prompt of 8192 962 and 834; 96 over 8 of up to 8000 54 and 58, 48 over 4 of up to 6000 33 and 40, four prompts of 512
  // 75 and 96.
  if (rows > 16 && (D == 96 || D == 128) && best(3, w3) < t) p.rt = 3, w = w3;
  p.row_blocks = (int)((rows + 16 * p.rt - 1) / (16 * p.rt));
  p.part_rows = (int)(rows < 16 * p.rt ? rows : 16 * p.rt);
  const int64_t units = units_of(p.rt);
  p.choose = slots_of(p.rt) / units < MOST_CHOICES;
  // one sequence of up to 512 keys: no parts to join (8 kv heads, 256 keys: 8.9 us, 10.9 with several workers and the joining
  // launch; 512: 10.4 and 11.0; 1000: 15 and 11.1)
  if (B == 1 && most <= 4) w = 1;
  // parts of 256 MiB at most: where they would take more there are rounds enough without
  const int64_t part_bytes = units * 2 * p.part_rows * (D + 1) * 4, fit = (256 << 20) / part_bytes;
  w = w > most ? most : w;
  p.workers = (int)(w > fit ? fit > 1 ? fit : 1 : w);
  // A table may be far wider than its sequences are long, so where w came from the estimate the device takes the best of up to w
  // ranges once more, by the lengths (a prompt of 2048, 32 / 8 heads x 128, with a table of 131072 keys: 250 us in 4 ranges, 100
  // in one).
  p.choose = p.choose && p.workers > 1;
  for (int i = 0; i < MOST_CHOICES; ++i) time(p.rt, i + 1, p.step_time[i], p.fixed_time[i]);
  const int64_t n = p.workers == 1 ? 0 : units * p.workers * 2 * p.part_rows;
  p.o_bytes = (n * D * 4 + 255) / 256 * 256;
  p.bytes = p.o_bytes + n * 4;
  return p;
}

template <int D, int CT> static void cache_attn_launch(const CacheAttnArgs& a, int rt, unsigned blocks, hipStream_t st) {
  if (rt == 1) cache_attn_kernel<D, CT, 1><<<blocks, CA_THREADS, 0, st>>>(a);
  else if (rt == 2) cache_attn_kernel<D, CT, 2><<<blocks, CA_THREADS, 0, st>>>(a);
  else if constexpr (D == 96 || D == 128) cache_attn_kernel<D, CT, 3><<<blocks, CA_THREADS, 0, st>>>(a);
}

template <int D> static void cache_attn_dims(const CacheAttnArgs& a, int ct, int rt, unsigned blocks, hipStream_t st) {
  if (ct == CACHE_INT8) cache_attn_launch<D, CACHE_INT8>(a, rt, blocks, st);
  else cache_attn_launch<D, CACHE_E4M3>(a, rt, blocks, st);
  if (a.workers > 1) {
    // the waves of a workgroup join a row together where a sequence comes in more parts than one wave holds at once
    // (one of 32760 keys in 64 parts: 23 us in all with 16 waves, 26 with 4, whose second round waits for the first)
    const int slices = a.workers <= 8 || a.workers <= 4 * a.B ? 1 : a.workers <= 32 * a.B ? 4 : MERGE_SLICES;
    // several rows per wave only where their number fills the GPU twice over (16896 rows: 12 us with one each, 8 with four)
    const int64_t rows = (int64_t)a.T * a.G * a.B * a.Hkv;
    const int per = slices == 1 && rows > 8192 ? 4 : 1;
    const int64_t merges = (int64_t)a.B * a.Hkv * ((a.T * a.G + per - 1) / per);
    const unsigned blocks = (unsigned)(slices == 1 ? (merges + 3) / 4 : merges);
    if (per == 4) cache_merge_kernel<D, 4><<<blocks, 256, 0, st>>>(a, 16 * rt, slices);
    else cache_merge_kernel<D, 1><<<blocks, 64 * (slices == 1 ? 4 : slices), 0, st>>>(a, 16 * rt, slices);
  }
}

static int cache_attn_sizes(int B, int H, int Hkv, int T, int D, int page_size, int max_pages, const char* who) {
  SAGE_REQUIRE(B > 0 && H > 0 && Hkv > 0 && T > 0 && max_pages > 0, "%s: sizes must be positive", who);
  SAGE_REQUIRE(H % Hkv == 0, "%s: heads %d not a multiple of kv heads %d", who, H, Hkv);
  if (!head_dim_ok(D)) return fail(SAGE_ERR_UNSUPPORTED, "%s: head_dim %d (supported 64, 96, 128, 256)", who, D);
  if (!cache_page_ok(page_size))
    return fail(SAGE_ERR_UNSUPPORTED, "%s: page_size %d (a power of two from 16 to 1024)", who, page_size);
  // keys of a sequence, steps of all of them and rows of all heads are counted in 32 bits, with room for a step past the end
  SAGE_REQUIRE((int64_t)B * (((int64_t)max_pages * page_size + CA_STEP - 1) / CA_STEP) <= 0x40000000,
               "%s: more than 2^37 keys", who);
  SAGE_REQUIRE((int64_t)max_pages * page_size <= 0x40000000, "%s: more than 2^30 keys per sequence", who);
  SAGE_REQUIRE((int64_t)B * H * T <= 0x01000000ll * 16, "%s: more than 2^28 query rows", who);
  return SAGE_OK;
}

}  // namespace sage

extern "C" {

int sage_cache_attn_workspace(int B, int H, int Hkv, int T, int D, int page_size, int max_pages,
                              int64_t* workspace_bytes) {
  using namespace sage;
  clear_error();
  SAGE_REQUIRE(workspace_bytes != nullptr, "sage_cache_attn_workspace: workspace_bytes is NULL");
  const int rc = cache_attn_sizes(B, H, Hkv, T, D, page_size, max_pages, "sage_cache_attn_workspace");
  if (rc) return rc;
  int cus = 0;
  if (const int e = device_cus(&cus)) return e;
  *workspace_bytes = cache_plan(B, H, Hkv, T, D, max_pages * page_size, cus).bytes;
  return SAGE_OK;
}

int sage_cache_attn(const void* q, int64_t qsb, int64_t qss, int64_t qsh, void* out, int64_t osb, int64_t oss,
                    int64_t osh, float* lse, const void* k8, const float* k_scale, const void* v8,
                    const float* v_scale, const int* block_table, int64_t table_stride, const int* lengths,
                    const void* tree_mask, int64_t msb, int64_t msq, int64_t msk, int B, int H, int Hkv, int T, int D,
                    int dtype, int cache_dtype, int pages, int page_size, int max_pages, int causal, float sm_scale,
                    void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace sage;
  clear_error();
  const char* who = "sage_cache_attn";
  int rc = cache_check(k8, k_scale, v8, v_scale, pages, page_size, Hkv, D, cache_dtype, who);
  if (rc) return rc;
  if ((rc = cache_attn_sizes(B, H, Hkv, T, D, page_size, max_pages, who))) return rc;
  SAGE_REQUIRE(q && out && block_table && lengths, "%s: q, out, block_table or lengths is NULL", who);
  SAGE_REQUIRE(aligned16(q) && aligned16(out), "%s: q and out must be 16-byte aligned", who);
  SAGE_REQUIRE(qsb % 8 == 0 && qss % 8 == 0 && qsh % 8 == 0 && osb % 8 == 0 && oss % 8 == 0 && osh % 8 == 0,
               "%s: strides must be multiples of 8 elements", who);
  SAGE_REQUIRE((((uintptr_t)block_table | (uintptr_t)lengths | (uintptr_t)lse) & 3u) == 0,
               "%s: block_table, lengths or lse misaligned", who);
  if (dtype != SAGE_DTYPE_BF16 && dtype != SAGE_DTYPE_F16) return fail(SAGE_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  SAGE_REQUIRE(sm_scale == 0.0f || (sm_scale >= 0x1p-126f && sm_scale <= 0x1.fffffep127f),
               "%s: sm_scale must be 0 or a positive normal number (got %g)", who, (double)sm_scale);
  if (tree_mask) {
    auto far = [&](int64_t stride) { return (stride < 0 ? -stride : stride) > 0x3FFFFFFF / (T > 1 ? T - 1 : 1); };
    SAGE_REQUIRE(!far(msq) && !far(msk), "%s: a tree mask's rows and columns must lie within 2^31 bytes", who);
  }
  int cus = 0;
  if ((rc = device_cus(&cus))) return rc;
  const CachePlan p = cache_plan(B, H, Hkv, T, D, max_pages * page_size, cus);
  SAGE_REQUIRE(p.bytes == 0 || (workspace && ((uintptr_t)workspace & 255u) == 0 && workspace_bytes >= p.bytes),
               "%s: workspace of %lld bytes (256-byte aligned), the plan needs %lld", who, (long long)workspace_bytes,
               (long long)p.bytes);
  CacheAttnArgs a = {};
  a.q = (const uint16_t*)q, a.qsb = qsb, a.qss = qss, a.qsh = qsh;
  a.out = (uint16_t*)out, a.osb = osb, a.oss = oss, a.osh = osh, a.lse = lse;
  a.k8 = (const uint8_t*)k8, a.v8 = (const uint8_t*)v8, a.ks = k_scale, a.vs = v_scale;
  a.table = block_table, a.tsb = table_stride, a.lengths = lengths;
  a.tree = (const uint8_t*)tree_mask, a.msb = msb, a.msq = (int)msq, a.msk = (int)msk;
  a.B = B, a.H = H, a.Hkv = Hkv, a.G = H / Hkv, a.T = T, a.dtype = dtype, a.causal = causal;
  a.pages = pages, a.page_size = page_size, a.max_pages = max_pages;
  a.page_shift = __builtin_ctz((unsigned)page_size);
  a.row_blocks = p.row_blocks, a.workers = p.workers, a.part_rows = p.part_rows, a.choose = p.choose;
  for (int i = 0; i < MOST_CHOICES; ++i) a.step_time[i] = p.step_time[i], a.fixed_time[i] = p.fixed_time[i];
  const double scale = sm_scale > 0.0f ? (double)sm_scale : 1.0 / __builtin_sqrt((double)D);
  a.scale = (float)std::frexp(scale * 1.44269504088896340736, &a.scale_exp);
  a.part_o = (float*)workspace;
  a.part_lse = (float*)((char*)workspace + p.o_bytes);
  const int64_t blocks = ((int64_t)Hkv * p.workers * p.row_blocks + 7) / 8 * 8;
  SAGE_REQUIRE(blocks <= 0x7FFFFFFF, "%s: too many workgroups", who);
  hipStream_t st = (hipStream_t)stream;
  if (D == 64) cache_attn_dims<64>(a, cache_dtype, p.rt, (unsigned)blocks, st);
  else if (D == 96) cache_attn_dims<96>(a, cache_dtype, p.rt, (unsigned)blocks, st);
  else if (D == 128) cache_attn_dims<128>(a, cache_dtype, p.rt, (unsigned)blocks, st);
  else cache_attn_dims<256>(a, cache_dtype, p.rt, (unsigned)blocks, st);
  return check_launch(who);
}

}  // extern "C"
