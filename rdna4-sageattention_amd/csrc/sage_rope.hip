// Rotary positions of Q and K in one launch (no counterpart in the reference, whose callers rotate with torch).
//
// The first R channels of every head are R/2 pairs (a, b), channels (i, i + R/2) or, interleaved, (2i, 2i + 1); at
// position p pair i turns by the angle p f_i: (a, b) -> c (a cos - b sin, b cos + a sin), with a common factor c.  The
// other channels are copied.  The transpose, which the gradient needs, turns back (`inverse`).
//
// Angles: a float32 product p f_i is wrong in its turns from p ~ 10^5 on (a relative error of 2^-24 of 10^5 radians is
// 0.006), so the turns p f_i / 2 pi are taken in float64, their whole part is dropped there, and the rest, within half
// a turn, is exact to 2^-25 in float32, where sine and cosine are evaluated.
//
// Bound: HBM where there is much to turn, 4 bytes per element: 2 x 8192 tokens of 32 + 8 heads x 128 in 69 us, 4.9 TB/s, the
// rate of a large copy.  A thread takes 8 or 16 elements of each of its heads as 16-byte vectors (angles once for all of them, while
// the loads are under way).
#include "sage_common.h"
#include "sage_host.h"

namespace sage {

constexpr int ROPE_THREADS = 256;
enum { ROPE_HALF8 = 0, ROPE_HALF4 = 1, ROPE_PAIRS = 2 };  // pairs of halves, 8 or 4 per thread; neighbouring channels

struct RopeArgs {
  const uint16_t* x[2];           // q, k
  uint16_t* y[2];
  int64_t xb[2], xs[2], xh[2];    // (batch, token, head) element strides
  int64_t yb[2], ys[2], yh[2];
  const void* pos;                // NULL: the token's index
  int64_t pb, ps;                 // its (batch, token) element strides
  const double* freqs;
  int pos64, inverse;
  float factor;
  int H, heads;                   // heads of q, of q and k together
  int S, tokens, D, R;
  int chunks;                     // threads per token and head
  int slots;                      // threads side by side over the heads: thread slot s takes heads s, s + slots, ..
  int token_inner;                // neighbouring threads take neighbouring tokens (not heads) of a chunk's row
};

template <int DT, int N> struct Elems {
  float v[N];
  __device__ __forceinline__ void load(const uint16_t* p) {
    if constexpr (N == 8) {
      const v4i w = *reinterpret_cast<const v4i*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[2 * i] = elem_lo<DT>(w[i]), v[2 * i + 1] = elem_hi<DT>(w[i]);
    } else {
      const v2i w = *reinterpret_cast<const v2i*>(p);
#pragma unroll
      for (int i = 0; i < 2; ++i) v[2 * i] = elem_lo<DT>(w[i]), v[2 * i + 1] = elem_hi<DT>(w[i]);
    }
  }
  __device__ __forceinline__ void store(uint16_t* p) const {
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = f32_to_out_bits<DT>(v[2 * i]) | (f32_to_out_bits<DT>(v[2 * i + 1]) << 16);
    if constexpr (N == 8) *reinterpret_cast<v4i*>(p) = v4i{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
    else *reinterpret_cast<v2i*>(p) = v2i{(int)w[0], (int)w[1]};
  }
};

// HP heads per thread: the angles of a thread's pairs serve them all, and their loads are in flight while the angles
// are computed.
template <int DT, int MODE, int HP> __global__ __launch_bounds__(ROPE_THREADS) void rope_kernel(const RopeArgs a) {
  constexpr int NP = MODE == ROPE_HALF8 ? 8 : 4;  // pairs of a thread
  constexpr int NE = MODE == ROPE_HALF4 ? 4 : 8;  // elements per load
  const int64_t id = (int64_t)blockIdx.x * ROPE_THREADS + threadIdx.x;
  if (id >= (int64_t)a.tokens * a.slots * a.chunks) return;
  const int c = (int)(id % a.chunks);
  const int64_t rest = id / a.chunks;
  int tok, slot;
  if (a.token_inner) {
    tok = (int)(rest % a.tokens);
    slot = (int)(rest / a.tokens);
  } else {
    tok = (int)(rest / a.slots);
    slot = (int)(rest % a.slots);
  }
  const int b = tok / a.S, s = tok - b * a.S;
  const int half = a.R / 2;
  const int turning = MODE == ROPE_PAIRS ? a.R / 8 : half / NP;  // chunks with pairs; the others are copied
  const bool copy = c >= turning;
  const int e0 = copy ? a.R + 8 * (c - turning) : MODE == ROPE_PAIRS ? 8 * c : NP * c;

  const uint16_t* xp[HP];
  uint16_t* yp[HP];
#pragma unroll
  for (int i = 0; i < HP; ++i) {
    int h = slot + i * a.slots;
    if (h >= a.heads) h = slot;  // (not stored)
    const int w = h >= a.H, hh = w ? h - a.H : h;
    xp[i] = a.x[w] + b * a.xb[w] + s * a.xs[w] + hh * a.xh[w] + e0;
    yp[i] = a.y[w] + b * a.yb[w] + s * a.ys[w] + hh * a.yh[w] + e0;
  }
  if (copy) {
#pragma unroll
    for (int i = 0; i < HP; ++i)
      if (slot + i * a.slots < a.heads) *reinterpret_cast<v4i*>(yp[i]) = *reinterpret_cast<const v4i*>(xp[i]);
    return;
  }
  Elems<DT, NE> lo[HP], hi[HP];
#pragma unroll
  for (int i = 0; i < HP; ++i) {
    lo[i].load(xp[i]);
    if (MODE != ROPE_PAIRS) hi[i].load(xp[i] + half);
  }

  int64_t p = s;
  if (a.pos) {
    const int64_t o = b * a.pb + s * a.ps;
    p = a.pos64 ? static_cast<const int64_t*>(a.pos)[o] : static_cast<const int32_t*>(a.pos)[o];
  }
  const double turns_per_radian = 0.15915494309189533577;
  const double pd = (double)p * turns_per_radian;
  float cs[NP], sn[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    double t = pd * a.freqs[(MODE == ROPE_PAIRS ? 4 : NP) * c + i];
    t -= __builtin_rint(t);
    float si, co;
    sincospif(2.0f * (float)t, &si, &co);
    cs[i] = co * a.factor;
    sn[i] = (a.inverse ? -si : si) * a.factor;
  }
#pragma unroll
  for (int i = 0; i < HP; ++i) {
    if (slot + i * a.slots >= a.heads) break;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      float& u = MODE == ROPE_PAIRS ? lo[i].v[2 * j] : lo[i].v[j];
      float& v = MODE == ROPE_PAIRS ? lo[i].v[2 * j + 1] : hi[i].v[j];
      const float x = u, y = v;
      u = __builtin_fmaf(x, cs[j], -(y * sn[j]));
      v = __builtin_fmaf(y, cs[j], x * sn[j]);
    }
    lo[i].store(yp[i]);
    if (MODE != ROPE_PAIRS) hi[i].store(yp[i] + half);
  }
}

template <int DT, int MODE> static void rope_launch(const RopeArgs& a, int hp, unsigned blocks, hipStream_t st) {
  if (hp == 1) rope_kernel<DT, MODE, 1><<<blocks, ROPE_THREADS, 0, st>>>(a);
  else rope_kernel<DT, MODE, 4><<<blocks, ROPE_THREADS, 0, st>>>(a);
}

}  // namespace sage

extern "C" int sage_rope(const void* q, int64_t qsb, int64_t qss, int64_t qsh, void* q_out, int64_t qob, int64_t qos,
                         int64_t qoh, int H, const void* k, int64_t ksb, int64_t kss, int64_t ksh, void* k_out,
                         int64_t kob, int64_t kos, int64_t koh, int Hk, int B, int S, int D, int dtype,
                         const void* positions, int positions64, int64_t psb, int64_t pss, const double* freqs,
                         int rot_dim, int interleaved, float factor, int inverse, void* stream) {
  using namespace sage;
  clear_error();
  SAGE_REQUIRE(B > 0 && S > 0 && H > 0 && Hk >= 0, "sage_rope: sizes must be positive");
  SAGE_REQUIRE(q && q_out && freqs, "sage_rope: q, q_out or freqs is NULL");
  SAGE_REQUIRE(Hk == 0 || (k && k_out), "sage_rope: k or k_out is NULL");
  if (dtype != SAGE_DTYPE_BF16 && dtype != SAGE_DTYPE_F16) return fail(SAGE_ERR_UNSUPPORTED, "sage_rope: dtype %d", dtype);
  if (!head_dim_ok(D)) return fail(SAGE_ERR_UNSUPPORTED, "sage_rope: head_dim %d (supported 64, 96, 128, 256)", D);
  if (rot_dim <= 0 || rot_dim > D || rot_dim % 8)
    return fail(SAGE_ERR_UNSUPPORTED, "sage_rope: rotated channels %d (a positive multiple of 8 up to head_dim %d)",
                rot_dim, D);
  const void* ptrs[] = {q, q_out, Hk ? k : q, Hk ? k_out : q_out};
  const int64_t strides[] = {qsb, qss, qsh, qob, qos, qoh, ksb, kss, ksh, kob, kos, koh};
  for (const void* p : ptrs) SAGE_REQUIRE(aligned16(p), "sage_rope: pointers must be 16-byte aligned");
  for (int i = 0; i < (Hk ? 12 : 6); ++i)
    SAGE_REQUIRE(strides[i] % 8 == 0, "sage_rope: strides must be multiples of 8 elements");
  SAGE_REQUIRE(((uintptr_t)freqs & 7u) == 0 && ((uintptr_t)positions & (positions64 ? 7u : 3u)) == 0,
               "sage_rope: freqs or positions misaligned");
  SAGE_REQUIRE((int64_t)B * S <= 0x3FFFFFFF && (int64_t)H + Hk <= 0x7FFFFFFF, "sage_rope: too many tokens or heads");

  RopeArgs a = {};
  a.x[0] = (const uint16_t*)q, a.y[0] = (uint16_t*)q_out;
  a.x[1] = (const uint16_t*)k, a.y[1] = (uint16_t*)k_out;
  a.xb[0] = qsb, a.xs[0] = qss, a.xh[0] = qsh, a.yb[0] = qob, a.ys[0] = qos, a.yh[0] = qoh;
  a.xb[1] = ksb, a.xs[1] = kss, a.xh[1] = ksh, a.yb[1] = kob, a.ys[1] = kos, a.yh[1] = koh;
  a.pos = positions, a.pos64 = positions64, a.pb = psb, a.ps = pss;
  a.freqs = freqs, a.factor = factor, a.inverse = inverse;
  a.H = H, a.heads = H + Hk, a.S = S, a.tokens = B * S, a.D = D, a.R = rot_dim;
  const int mode = interleaved ? ROPE_PAIRS : rot_dim % 16 == 0 ? ROPE_HALF8 : ROPE_HALF4;
  a.chunks = (mode == ROPE_PAIRS ? rot_dim / 8 : mode == ROPE_HALF8 ? rot_dim / 16 : rot_dim / 8) + (D - rot_dim) / 8;
  // four heads per thread share its angles, one where that leaves too few threads (16384 tokens of 40 heads x 128: 68.5 us with
  // four, 96 with one; 6141 of 20 x 64: 11.7 and 13.9; 1000 of 40 x 128, 320000 threads with one: 9.4 and 8.9)
  const int hp = (int64_t)a.tokens * a.chunks * a.heads >= 512 * 1024 ? 4 : 1;
  a.slots = (a.heads + hp - 1) / hp;
  a.token_inner = qss < qsh;
  const int64_t blocks = ((int64_t)a.tokens * a.slots * a.chunks + ROPE_THREADS - 1) / ROPE_THREADS;
  SAGE_REQUIRE(blocks <= 0x7FFFFFFF, "sage_rope: too large");
  hipStream_t st = (hipStream_t)stream;
  const unsigned n = (unsigned)blocks;
  if (dtype == SAGE_DTYPE_BF16) {
    if (mode == ROPE_PAIRS) rope_launch<DT_BF16, ROPE_PAIRS>(a, hp, n, st);
    else if (mode == ROPE_HALF8) rope_launch<DT_BF16, ROPE_HALF8>(a, hp, n, st);
    else rope_launch<DT_BF16, ROPE_HALF4>(a, hp, n, st);
  } else {
    if (mode == ROPE_PAIRS) rope_launch<DT_F16, ROPE_PAIRS>(a, hp, n, st);
    else if (mode == ROPE_HALF8) rope_launch<DT_F16, ROPE_HALF8>(a, hp, n, st);
    else rope_launch<DT_F16, ROPE_HALF4>(a, hp, n, st);
  }
  return check_launch("rope_kernel");
}
