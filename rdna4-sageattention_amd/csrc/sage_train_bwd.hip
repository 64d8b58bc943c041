// Backward pass of the attention for training: see sage_train.h for the form.
//
// Two kernels, each of which recomputes the scores and the gradient of the probabilities: one owns queries and streams keys
// (dq), one owns keys and streams queries (dk, dv).  That is seven products for the five of the formulas, and it needs neither
// atomics nor partial results in memory: every gradient is one sum in a fixed order, so equal inputs give equal bits.  A single
// kernel would have to add dq over its workgroups: 4 bytes written and read for every 2 * 128 keys' products of a channel.
#include "sage_train.h"

namespace sage {

// fp16 holds ds only in a window of 2^30.  |do_i . v_j - D_i| <= 2 max |do| max |v|, so ds times this power of two stays below
// 2^15, and full precision reaches down to 2^-29 of the bound.  (bf16 has float32's exponents: 0.)
__device__ __forceinline__ int tr_exponent(const uint32_t* norms) {
  const float n = __uint_as_float(norms[0]) * __uint_as_float(norms[1]);   // the squared bound / 4
  if (!(n > 0.0f && n < INFINITY)) return 0;
  int e;
  (void)frexpf(n, &e);                       // n < 2^e, so the bound is below 2^(e / 2 + 1)
  return min(max(13 - ((e + 1) >> 1), -100), 100);
}
// P is at most 1 and is taken times 2^15 in fp16 where it is an operand
template <int DT> constexpr float BWD_SHIFT = DT == DT_F16 ? 15.0f : 0.0f;

// ---- preparation: -lse / sm_scale and -D of every row; the norms of fp16 inputs -----------------------------------------------

template <int D, int DT> __global__ __launch_bounds__(TR_THREADS) void train_prep(TrainArgs a, int row_blocks, int norm_blocks) {
  constexpr int LPR = D == 96 ? 16 : D / 8;       // lanes per row (12 of the 16 at head dim 96)
  constexpr int ROWS = TR_THREADS / LPR;
  const int tid = threadIdx.x, r = tid / LPR, l = tid % LPR;
  const bool has = l * 8 < D;
  float top = 0.0f;                               // largest squared norm of this thread's rows
  auto row_sum = [&](float x) {
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) x += __shfl_xor(x, o);
    return x;
  };
  if ((int)blockIdx.x >= row_blocks) {            // fp16: the rows of v
    const int64_t n = (int64_t)(a.cu_q ? 1 : a.B) * a.Hkv * a.Skv;
    for (int64_t x = (int64_t)(blockIdx.x - row_blocks) * ROWS + r; x < n; x += (int64_t)norm_blocks * ROWS) {
      const int64_t h = x % a.Hkv, t = x / a.Hkv, j = t % a.Skv, b = t / a.Skv;
      float s = 0.0f;
      if (has) {
        const v4i w = *reinterpret_cast<const v4i*>(a.v + b * a.vb + j * a.vs + h * a.vh + l * 8);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x0 = elem_lo<DT>(w[e]), x1 = elem_hi<DT>(w[e]);
          s = __builtin_fmaf(x0, x0, __builtin_fmaf(x1, x1, s));
        }
      }
      s = row_sum(s);
      if (s < INFINITY) top = fmaxf(top, s);
    }
  } else {
    // 128 rows of one head
    const int tiles = a.q_tiles, bh = blockIdx.x / tiles, t = blockIdx.x % tiles;
    TrSeq s;
    s.b = bh / a.H, s.h = bh % a.H, s.c0 = t * TR_COLS, s.q_len = a.Sq, s.qr = 0, s.lr = 0;
    if (a.cu_q) {
      const int2 e = a.q_tab[t];
      if (e.x < 0) return;
      const int q0 = a.cu_q[e.x];
      s.b = e.x, s.c0 = e.y * TR_COLS, s.q_len = a.cu_q[e.x + 1] - q0, s.qr = q0, s.lr = q0 / 64 * 64 + (int64_t)64 * e.x;
    }
    const int64_t at = tr_stat_row(a, s, s.h);
    const int64_t lse_at = a.cu_q ? (int64_t)s.h * a.Sq + s.qr : ((int64_t)s.b * a.H + s.h) * a.Sq;
    const int end = min(s.c0 + TR_COLS, (s.q_len + 63) / 64 * 64);
    const uint16_t* op = a.o + (a.cu_q ? 0 : s.b * a.ob) + s.qr * a.os + s.h * a.oh + l * 8;
    const uint16_t* gp = a.dout + (a.cu_q ? 0 : s.b * a.gb) + s.qr * a.gs + s.h * a.gh + l * 8;
    for (int i = s.c0 + r; i < end; i += ROWS) {
      float d = 0.0f, g2 = 0.0f;
      if (i < s.q_len && has) {
        const v4i x = *reinterpret_cast<const v4i*>(op + i * a.os), g = *reinterpret_cast<const v4i*>(gp + i * a.gs);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float g0 = elem_lo<DT>(g[e]), g1 = elem_hi<DT>(g[e]);
          d = __builtin_fmaf(elem_lo<DT>(x[e]), g0, __builtin_fmaf(elem_hi<DT>(x[e]), g1, d));
          if (DT == DT_F16) g2 = __builtin_fmaf(g0, g0, __builtin_fmaf(g1, g1, g2));
        }
      }
      d = row_sum(d);
      if (DT == DT_F16) {
        g2 = row_sum(g2);
        if (g2 < INFINITY) top = fmaxf(top, g2);
      }
      if (l == 0) {
        // a row that sees nothing: p = 0; one with an infinity or a NaN in it: p = NaN wherever it sees a key
        const float lse = i < s.q_len ? a.lse[lse_at + i] : -INFINITY;
        float nl = -(lse / a.scale), nd = -d;
        if (lse == -INFINITY) nl = -INFINITY, nd = 0.0f;
        else if (!(fabsf(lse) < INFINITY) || !(fabsf(d) < INFINITY)) nl = NAN;
        a.nl[at + i] = nl;
        a.nd[at + i] = nd;
      }
    }
  }
  if (DT == DT_F16) {
    top = wave_max_pos(top);
    if ((tid & 63) == 0 && top > 0.0f) atomicMax(a.norms + ((int)blockIdx.x >= row_blocks ? 1 : 0), __float_as_uint(top));
  }
}

__global__ void train_norms_zero(uint32_t* norms) {
  if (threadIdx.x < 2) norms[threadIdx.x] = 0;
}

// ---- dq (and the bias' gradient by distance) ---------------------------------------------------------------------------------

template <int D, int DT, bool EX>
__global__ __launch_bounds__(TR_THREADS, D == 256 ? 1 : 2) void train_dq(TrainArgs a, BiasMap map) {
  using G = TrGeo<D>;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2][2][G::TILE];
  __shared__ float bl[EX ? 2 * TR_REACH + 1 : 1];
  extern __shared__ float by_distance[];   // EX with bias_part: 4 waves x (2 reach + 1)

  TrSeq s;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool biased = EX && a.bias, want_part = EX && a.bias_part;
  const int R = 2 * a.reach + 1;
  if (!tr_tile<false>(a, blockIdx.x, s)) {
    if (want_part)   // (only packed batches have unused tiles)
      for (int x = tid; x < map.buckets; x += TR_THREADS) a.bias_part[(s.h * a.parts + s.part) * map.buckets + x] = 0.0f;
    return;
  }
  const int ln = lane & 31, hf = lane >> 5;
  const int hk = s.h / (a.H / a.Hkv);
  const int off = s.k_len - s.q_len;
  const int w0 = s.c0 + wave * 32, i = w0 + ln;
  const bool on = i < s.q_len;
  const int ir = on ? i : s.q_len - 1;

  const uint16_t* kp = a.k + (a.cu_q ? 0 : s.b * a.kb) + s.kr * a.ks + hk * a.kh;
  const uint16_t* vp = a.v + (a.cu_q ? 0 : s.b * a.vb) + s.kr * a.vs + hk * a.vh;
  const int64_t at_row = tr_stat_row(a, s, s.h);
  float nl = on ? a.nl[at_row + i] : -INFINITY;
  const float nd = on ? a.nd[at_row + i] : 0.0f;
  const bool empty = nl == -INFINITY;   // sees nothing: its q and dout may hold anything

  v4i qf[G::NK], gf[G::NK];
  {
    const uint16_t* p = a.q + (a.cu_q ? 0 : s.b * a.qb) + (s.qr + ir) * a.qs + s.h * a.qh + 8 * hf;
    const uint16_t* g = a.dout + (a.cu_q ? 0 : s.b * a.gb) + (s.qr + ir) * a.gs + s.h * a.gh + 8 * hf;
#pragma unroll
    for (int x = 0; x < G::NK; ++x) {
      qf[x] = *reinterpret_cast<const v4i*>(p + 16 * x);
      gf[x] = *reinterpret_cast<const v4i*>(g + 16 * x);
      if (empty) qf[x] = v4i{0, 0, 0, 0}, gf[x] = v4i{0, 0, 0, 0};
    }
  }
  const int ex = DT == DT_F16 ? tr_exponent(a.norms) : 0;
  nl = __builtin_fmaf(nl, a.c, (float)ex);

  TrLoader<D> lk, lv;
  lk.init(a.ks, wave, lane);
  lv.init(a.vs, wave, lane);
  TrAddr<D> at;
  at.init(lane);
  tr_arrived(qf);
  tr_arrived(gf);

  int kv_end = s.k_len;
  if (a.causal) kv_end = min(kv_end, min(s.c0 + TR_COLS, s.q_len) + off);
  const int ntiles = kv_end > 0 ? (kv_end + TR_ROWS - 1) / TR_ROWS : 0;
  const int lim = a.causal ? min(s.k_len - 1, ir + off) : s.k_len - 1;
  int t_mask = s.k_len / TR_ROWS, t_end = ntiles;
  if (a.causal) {
    t_mask = min(t_mask, max(0, w0 + off + 1) / TR_ROWS);
    t_end = min(t_end, (max(0, min(w0 + 31, s.q_len - 1) + off + 1) + TR_ROWS - 1) / TR_ROWS);
  }
  if (w0 >= s.q_len) t_end = 0;
  t_mask = min(t_mask, t_end);
  const uint32_t* bits = nullptr;
  if (EX && a.bits) {
    bits = a.bits + s.b * a.mb + s.h * a.mh + (int64_t)ir * a.mi;
    t_mask = 0;
  }
  float* mine = by_distance + wave * R;
  if (biased)
    for (int x = tid; x < R; x += TR_THREADS) bl[x] = a.bias[(int64_t)s.h * R + x];

  v16f dq[G::NDB];
  // the bias' gradient: the lane's sums of ds and p over the keys at distance -reach and farther behind, reach and farther ahead,
  // and of ds over the others
  float flo = 0.0f, fhi = 0.0f, plo = 0.0f, phi = 0.0f, fnear = 0.0f;

  auto issue = [&](int t) {
    lk.issue(kp, a.ks, t * TR_ROWS, s.k_len, smem[t & 1][0], wave, lane);
    lv.issue(vp, a.vs, t * TR_ROWS, s.k_len, smem[t & 1][1], wave, lane);
  };
  auto tile = [&](int t, auto masked_) {
    constexpr bool masked = decltype(masked_)::value;
    const TrAddr<D> kt = at.in(smem[t & 1][0]), vt = at.in(smem[t & 1][1]);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      v16f x = {}, dp;
#pragma unroll
      for (int v = 0; v < 16; ++v) dp[v] = nd;
#pragma unroll
      for (int kk = 0; kk < G::NK; ++kk) {
        x = tr_mfma<DT>(kt.rows(kb, kk), qf[kk], x);
        dp = tr_mfma<DT>(vt.rows(kb, kk), gf[kk], dp);
      }
      const int key0 = t * TR_ROWS + 32 * kb;
      const int d0 = key0 + 4 * hf - (ir + off);
      const int wlo = key0 - (min(w0 + 31, s.q_len - 1) + off), whi = key0 + 31 - (w0 + off);
      const bool near = biased && !(whi <= -a.reach || wlo >= a.reach);
      if (EX) {
        if (near) {
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int d = min(max(d0 + 8 * (v >> 2) + (v & 3), -a.reach), a.reach);
            x[v] = __builtin_fmaf(x[v], a.c, bl[a.reach + d]);
          }
        } else {
          const float far = biased ? bl[whi <= -a.reach ? 0 : 2 * a.reach] : 0.0f;
#pragma unroll
          for (int v = 0; v < 16; ++v) x[v] = __builtin_fmaf(x[v], a.c, far);
        }
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) x[v] = __builtin_amdgcn_exp2f(EX ? x[v] + nl : __builtin_fmaf(x[v], a.c, nl));
      if (masked) {
        uint32_t w = ~0u;
        if (EX && bits && key0 < s.k_len) w = bits[(int64_t)(key0 >> 5) * a.mw];
        const int room = lim - key0 - 4 * hf;
        w >>= 4 * hf;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int r = 8 * (v >> 2) + (v & 3);
          if (r > room || !((w >> r) & 1u)) x[v] = 0.0f, dp[v] = 0.0f;
        }
      }
      if (want_part) {
        // d[v]: of ds; every lane of a half wave has a distance of its own, so one half at a time adds without conflicts and in
        // one order
        float all = 0.0f, ps = 0.0f;
        if (near) {
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int d = d0 + 8 * (v >> 2) + (v & 3);
            const float y = x[v] * dp[v];
            if (d <= -a.reach) flo += y, plo += x[v];
            else if (d >= a.reach) fhi += y, phi += x[v];
            else {
              fnear += y;
              __attribute__((address_space(3))) float* slot = (__attribute__((address_space(3))) float*)(mine + a.reach + d);
              if (hf == 0) {
                __builtin_amdgcn_ds_faddf(slot, y, 0, 0, false);
                asm volatile("; the lower half's" ::: "memory");   // (keeps the two from becoming one)
              } else {
                __builtin_amdgcn_ds_faddf(slot, y, 0, 0, false);
                asm volatile("; the upper half's" ::: "memory");
              }
            }
          }
        } else {
#pragma unroll
          for (int v = 0; v < 16; ++v) all += x[v] * dp[v], ps += x[v];
          if (whi <= -a.reach) flo += all, plo += ps;
          else fhi += all, phi += ps;
        }
      }
      v4i ds[2];
#pragma unroll
      for (int v = 0; v < 16; v += 2) ds[v >> 3][(v & 7) >> 1] = tr_pack<DT>(x[v] * dp[v], x[v + 1] * dp[v + 1]);
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int db = 0; db < G::NDB; ++db) dq[db] = tr_mfma<DT>(kt.cols(2 * kb + st, db), ds[st], dq[db]);
    }
  };

  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int db = 0; db < G::NDB; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) dq[db][v] = 0.0f;
    if (want_part) {
      flo = fhi = plo = phi = fnear = 0.0f;
      for (int x = lane; x < R; x += 64) mine[x] = 0.0f;
    }
    if (ntiles > 0) issue(0);
    int t = 0;
    auto next = [&]() {   // tile t has arrived, the one before is read: the one after goes there
      wait_vmcnt<0>();
      tile_barrier();
      if (t + 1 < ntiles) issue(t + 1);
    };
    for (; t < t_mask; ++t) {
      next();
      tile(t, std::false_type{});
    }
    for (; t < ntiles; ++t) {
      next();
      if (pass) {
        tr_clean<D, DT>(smem[t & 1][0], nullptr, tid);
        tr_clean<D, DT>(smem[t & 1][1], nullptr, tid);
        __syncthreads();
      }
      if (t < t_end) tile(t, std::true_type{});
      if (pass) __syncthreads();
    }
    const bool bad = !(tr_nonfinite(dq) == 0.0f);
    if (!__syncthreads_or(on && bad)) break;
    t_mask = 0;   // every tile cleaned, hidden keys taken out
  }

  const float f = __builtin_ldexpf(a.scale, -ex);
  uint16_t* op = a.dq + (a.cu_q ? 0 : s.b * a.dqb) + (s.qr + ir) * a.dqs + s.h * a.dqh;
#pragma unroll
  for (int db = 0; db < G::NDB; ++db) tr_store<DT>(dq[db], f, op + 32 * db, hf, on);

  if (want_part) {
    // The row sums of ds are 0, but D holds the rounding of o to 16 bits and of its weights: sum_j ds = D' - D, exactly the error of
    // D.  In a far bucket, which holds most of a long row's weight, it would not average out: it is taken from there.
    const float delta = add_xor32_f32(fnear + flo + fhi);
    flo -= delta * __builtin_ldexpf(plo, -ex);
    fhi -= delta * __builtin_ldexpf(phi, -ex);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) flo += __shfl_xor(flo, o), fhi += __shfl_xor(fhi, o);
    if (lane == 0) mine[0] += flo, mine[2 * a.reach] += fhi;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __syncthreads();
    for (int x = tid; x < R; x += TR_THREADS)
      by_distance[x] = (by_distance[x] + by_distance[R + x]) + (by_distance[2 * R + x] + by_distance[3 * R + x]);
    __syncthreads();
    float* part = a.bias_part + (s.h * a.parts + s.part) * map.buckets;
    for (int b = wave; b < map.buckets; b += TR_THREADS / 64) {
      int lo, hi;
      map.range(b, lo, hi);
      float y = 0.0f;
      for (int x = lo + lane; x <= hi; x += 64) y += by_distance[a.reach + x];
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) y += __shfl_xor(y, o);
      if (lane == 0) part[b] = __builtin_ldexpf(y, -ex);
    }
  }
}

// ---- dk, dv --------------------------------------------------------------------------------------------------------------------
//
// A wave's keys and values (D / 2 registers) and the sums of its dk and dv (2 D) leave room for one wave per SIMD, so a wave has to
// keep the matrix unit busy by itself: a tile is a stream of products in an order of its own, the operands of product n + AHEAD read
// from LDS when product n is issued, into the next tile too, and the weights of one block of 32 queries made beside the products
// of the other.  (Two waves per SIMD with half of the registers each, four operands ahead: 625 us at 1 x 24 x 4608 x 128.)
template <int D> struct DkvGeo {
  static constexpr int ROWS = 64;                  // queries per tile
  static constexpr int SLOTS = 3;                  // tiles in LDS: one at work, one arrived, one on its way
  static constexpr int AHEAD = D == 64 ? 4 : 8;    // products between an operand's read and its use
  static constexpr int OCC = D == 64 ? 2 : 1;      // waves per SIMD
};

template <int D, int DT, bool EX>
__global__ __launch_bounds__(TR_THREADS, DkvGeo<D>::OCC) void train_dkv(TrainArgs a) {
  using P = DkvGeo<D>;
  using G = TrGeo<D, P::ROWS>;
  constexpr int ROWS = P::ROWS;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[P::SLOTS][2][G::TILE];
  __shared__ __attribute__((aligned(256))) float stat[P::SLOTS][2][ROWS];
  __shared__ float bl[EX ? 2 * TR_REACH + 1 : 1];

  TrSeq s;
  if (!tr_tile<true>(a, blockIdx.x, s)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 31, hf = lane >> 5;
  const int group = a.H / a.Hkv;
  const int off = s.k_len - s.q_len;
  const int w0 = s.c0 + wave * 32, j = w0 + ln;   // the wave's first key, the lane's
  const bool on = j < s.k_len;
  const int jr = on ? j : s.k_len - 1;

  TrAddr<D> at;
  at.init(lane);
  v4i kf[G::NK], vf[G::NK];
  {
    const uint16_t* kp = a.k + (a.cu_q ? 0 : s.b * a.kb) + (s.kr + jr) * a.ks + s.h * a.kh + 8 * hf;
    const uint16_t* vp = a.v + (a.cu_q ? 0 : s.b * a.vb) + (s.kr + jr) * a.vs + s.h * a.vh + 8 * hf;
#pragma unroll
    for (int x = 0; x < G::NK; ++x) {
      kf[x] = *reinterpret_cast<const v4i*>(kp + 16 * x);
      vf[x] = *reinterpret_cast<const v4i*>(vp + 16 * x);
    }
  }
  const int ex = DT == DT_F16 ? tr_exponent(a.norms) : 0;
  const float ds_mul = __builtin_ldexpf(1.0f, ex - (int)BWD_SHIFT<DT>);

  const int t_all = (s.q_len + ROWS - 1) / ROWS;
  int t0 = 0;                                     // the first tile that sees one of the workgroup's keys
  if (a.causal) t0 = min(t_all, max(0, s.c0 - off) / ROWS);
  const int nt = t_all - t0;
  const int steps = nt * group;
  int t_full = 0;                                 // from this tile on every query sees every key of the wave
  if (a.causal) t_full = (max(0, w0 + 31 - off) + ROWS - 1) / ROWS;
  if (EX && a.bits) t_full = t_all;
  t_full = min(max(t_full, t0), t_all);

  // Loads, from the last tile back to the diagonal: workgroups of one head that start together stream the same tiles together.
  TrLoader<D, ROWS> lq, lg;
  lq.init(a.qs, wave, lane);
  lg.init(a.gs, wave, lane);
  const uint16_t* qp = a.q + (a.cu_q ? 0 : s.b * a.qb) + s.qr * a.qs + s.h * group * a.qh;
  const uint16_t* gp = a.dout + (a.cu_q ? 0 : s.b * a.gb) + s.qr * a.gs + s.h * group * a.gh;
  const float* sp = (wave ? a.nd : a.nl) + tr_stat_row(a, s, s.h * group);
  int tn = t_all - 1, un = 0, sn = 0;             // of the tile that is loaded next: its number, the step, the slot
  auto issue = [&]() {
    if (un < steps) {
      lq.issue(qp, a.qs, tn * ROWS, s.q_len, smem[sn][0], wave, lane);
      lg.issue(gp, a.gs, tn * ROWS, s.q_len, smem[sn][1], wave, lane);
      if (wave < 2) tr_copy4(sp + tn * ROWS + lane, stat[sn][wave]);
      if (--tn < t0) tn = t_all - 1, qp += a.qh, gp += a.gh, sp += a.pad;
      ++un;
      sn = sn + 1 == P::SLOTS ? 0 : sn + 1;
    }
  };

  v16f dk[G::NDB], dv[G::NDB], x[2], dp[2];
  v4i ring[P::AHEAD];
  auto begin = [&](int slot, int qb) __attribute__((always_inline)) {   // the first products' sums begin at the rows' numbers
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const v4f y = *reinterpret_cast<const v4f*>(&stat[slot][0][32 * qb + 8 * g + 4 * hf]);
      const v4f z = *reinterpret_cast<const v4f*>(&stat[slot][1][32 * qb + 8 * g + 4 * hf]);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[qb][4 * g + e] = y[e], dp[qb][4 * g + e] = z[e];
    }
  };
  constexpr int N = 2 * G::NK;                     // products per quarter of a tile
  auto operand = [&](const TrAddr<D>& qt, const TrAddr<D>& gt, auto n_) __attribute__((always_inline)) {
    constexpr int n = decltype(n_)::value, part = n / N, y = n % N;
    if constexpr (part < 2) return (y & 1) ? gt.rows(part, y >> 1) : qt.rows(part, y >> 1);
    else return (y & 1) ? qt.cols(2 * (part - 2) + y / (2 * G::NDB), y % (2 * G::NDB) >> 1)
                        : gt.cols(2 * (part - 2) + y / (2 * G::NDB), y % (2 * G::NDB) >> 1);
  };
  // One tile: the products of block 0's scores and weights' gradients, those of block 1's while block 0's weights are made, block
  // 0's parts of dv and dk while block 1's weights are made, block 1's parts.
  auto tile = [&](int slot, int next, int t, int h, auto masked_) __attribute__((always_inline)) {
    constexpr bool masked = decltype(masked_)::value;
    constexpr int AHEAD = P::AHEAD;
    const TrAddr<D> qt = at.in(smem[slot][0]), gt = at.in(smem[slot][1]);
    const TrAddr<D> qn = at.in(smem[next][0]), gn = at.in(smem[next][1]);
    v4i p[2][2], ds[2][2];
    // the weights of elements v0 .. v1 (in pairs) of a block
    auto weights = [&](int qb, int v0, int v1) __attribute__((always_inline)) {
      const int q0 = t * ROWS + 32 * qb;
      const int d0 = jr - off - q0 - 4 * hf;      // key - query of register 0; a row further is 1 less
      const int whi = w0 + 31 - off - q0, wlo = w0 - off - q0 - 31;
      const bool near = EX && a.bias && !(whi <= -a.reach || wlo >= a.reach);
      const float far = (EX && a.bias && !near ? bl[whi <= -a.reach ? 0 : 2 * a.reach] : 0.0f) + BWD_SHIFT<DT>;
#pragma unroll
      for (int v = v0; v < v1; ++v) {
        float y = x[qb][v];
        if (EX) {
          float more = far;
          if (near) more = bl[a.reach + min(max(d0 - 8 * (v >> 2) - (v & 3), -a.reach), a.reach)] + BWD_SHIFT<DT>;
          y = __builtin_fmaf(y, a.c, more);
        } else {
          y = DT == DT_F16 ? __builtin_fmaf(y, a.c, BWD_SHIFT<DT>) : y * a.c;
        }
        y = __builtin_amdgcn_exp2f(y);
        if (masked) {
          const int r = 8 * (v >> 2) + (v & 3), room = q0 + 4 * hf - (jr - off);   // row r sees the key where r + room >= 0
          bool hidden = a.causal && r + room < 0;
          if (EX && a.bits && w0 < s.k_len) {
            const uint32_t* w = a.bits + s.b * a.mb + h * a.mh + (int64_t)(w0 >> 5) * a.mw;
            hidden |= !((w[a.mi ? q0 + r + 4 * hf : 0] >> ln) & 1u);
          }
          if (hidden) y = 0.0f, dp[qb][v] = 0.0f;
        }
        x[qb][v] = y;
      }
#pragma unroll
      for (int v = v0; v < v1; v += 2) {
        p[qb][v >> 3][(v & 7) >> 1] = tr_pack<DT>(x[qb][v], x[qb][v + 1]);
        float e0 = x[qb][v] * dp[qb][v], e1 = x[qb][v + 1] * dp[qb][v + 1];
        if (DT == DT_F16) e0 *= ds_mul, e1 *= ds_mul;
        ds[qb][v >> 3][(v & 7) >> 1] = tr_pack<DT>(e0, e1);
      }
    };
    begin(slot, 1);
    tr_unroll<4 * N>([&](auto n_) __attribute__((always_inline)) {
      constexpr int n = decltype(n_)::value, part = n / N, y = n % N;
      const v4i f = ring[n % AHEAD];
      if constexpr (part < 2) {
        if constexpr (y & 1) dp[part] = tr_mfma<DT>(f, vf[y >> 1], dp[part]);
        else x[part] = tr_mfma<DT>(f, kf[y >> 1], x[part]);
      } else {
        constexpr int st = y / (2 * G::NDB), db = y % (2 * G::NDB) >> 1;
        if constexpr (y & 1) dk[db] = tr_mfma<DT>(f, ds[part - 2][st], dk[db]);
        else dv[db] = tr_mfma<DT>(f, p[part - 2][st], dv[db]);
      }
      if constexpr (n + AHEAD < 4 * N) ring[n % AHEAD] = operand(qt, gt, std::integral_constant<int, n + AHEAD>{});
      else ring[n % AHEAD] = operand(qn, gn, std::integral_constant<int, n + AHEAD - 4 * N>{});
      // 8 pairs over the quarter's products but the first
      if constexpr (part == 1 || part == 2) {
        constexpr int e0 = y < 1 ? 0 : (y - 1) * 8 / (N - 1) * 2, e1 = y * 8 / (N - 1) * 2;
        if constexpr (e1 > e0) weights(part - 1, e0, e1);
      }
      if constexpr (n == 3 * N + N / 2) begin(next, 0);
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int db = 0; db < G::NDB; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) dk[db][v] = 0.0f, dv[db][v] = 0.0f;
    if (pass) qp -= group * a.qh, gp -= group * a.gh, sp -= group * a.pad;   // (the loads begin anew)
    un = sn = 0;
    int slot = 0, u = 0;
    // The tile after u has arrived, the one before u is read and its place free
    auto top = [&]() __attribute__((always_inline)) {
      wait_vmcnt<0>();
      tile_barrier();
      issue();
      if (pass) {   // a tile is cleaned when it has arrived, one step before anything of it is read
        const int c = slot + 1 == P::SLOTS ? 0 : slot + 1;
        if (u == 0) tr_clean<D, DT, ROWS>(smem[0][0], nullptr, tid), tr_clean<D, DT, ROWS>(smem[0][1], nullptr, tid);
        if (u + 1 < steps) tr_clean<D, DT, ROWS>(smem[c][0], nullptr, tid), tr_clean<D, DT, ROWS>(smem[c][1], nullptr, tid);
        __syncthreads();
      }
    };
    issue();
    issue();
    tr_arrived(kf);
    tr_arrived(vf);
    if (steps > 0) {
      top();
      begin(0, 0);
      const TrAddr<D> qt = at.in(smem[0][0]), gt = at.in(smem[0][1]);
      tr_unroll<P::AHEAD>([&](auto n_) __attribute__((always_inline)) { ring[decltype(n_)::value] = operand(qt, gt, n_); });
    }
    int h = s.h * group;
    for (int g = 0; g < group && nt > 0; ++g, ++h) {
      if (EX && a.bias) {
        __syncthreads();
        for (int y = tid; y <= 2 * a.reach; y += TR_THREADS) bl[y] = a.bias[(int64_t)h * (2 * a.reach + 1) + y];
        __syncthreads();
      }
      // first the tiles that hide no keys of the wave, then, in a loop of their own, those that do
      int t = t_all - 1;
      auto one = [&](auto masked_) __attribute__((always_inline)) {
        const int next = slot + 1 == P::SLOTS ? 0 : slot + 1;
        tile(slot, next, t, h, masked_);
        slot = next, ++u;
        if (u < steps) top();
      };
      const int full = pass ? t_all : t_full;      // (a second pass takes hidden keys out of every tile)
      for (; t >= full; --t) one(std::false_type{});
      for (; t >= t0; --t) one(std::true_type{});
    }
    const bool bad = !(tr_nonfinite(dk) + tr_nonfinite(dv) == 0.0f);
    if (!__syncthreads_or(on && bad)) break;   // (a second time with every tile cleaned)
    tn = t_all - 1;
  }

  const float fk = __builtin_ldexpf(a.scale, -ex), fv = DT == DT_F16 ? 1.0f / 32768.0f : 1.0f;
  uint16_t* kp = a.dk + (a.cu_q ? 0 : s.b * a.dkb) + (s.kr + jr) * a.dks + s.h * a.dkh;
  uint16_t* vp = a.dv + (a.cu_q ? 0 : s.b * a.dvb) + (s.kr + jr) * a.dvs + s.h * a.dvh;
#pragma unroll
  for (int db = 0; db < G::NDB; ++db) {
    tr_store<DT>(dk[db], fk, kp + 32 * db, hf, on);
    tr_store<DT>(dv[db], fv, vp + 32 * db, hf, on);
  }
}

// Two waves share each 32 keys: the first recomputes the scores, makes the weights and sums dv, the second recomputes the gradient
// of the weights, multiplies it by the weights, which it gets in fp32 through LDS one tile later, and sums dk.  Each has half of the
// accumulators and half of the operands, so both fit a SIMD's registers together with operands read far ahead, and one's exponentials
// run beside the other's products.  (One wave with everything: 695 us at 1 x 24 x 4608 x 128 with one wave per SIMD, 636 with
// two, whose registers left four operands ahead.)
//
// Step u: the first waves work on tile u of 32 queries, the second ones on tile u - 1, and both read the first operands of their next
// tile ahead; tiles u + 2 and u + 3 are on their way.  One barrier a step.  (Head dim 256, for whose tiles there is less room: the
// next tile's operands are read after the barrier, one tile on its way.)
template <int D> struct DkvPairGeo {
  static constexpr int ROWS = 32;                  // queries per tile
  static constexpr int WAVES = 8;
  static constexpr bool CROSS = D != 256;          // reads ahead into the next tile
  static constexpr int SLOTS = CROSS ? 5 : 3;      // tiles in LDS
  static constexpr int AHEAD = D == 128 ? 8 : 4;   // products between an operand's read and its use
  static constexpr int PER_WAVE = D == 64 ? 1 : D == 256 ? 4 : 2;   // 1 KiB loads of a wave per step, of q or of dout
  static constexpr int PER_TENSOR = D * ROWS * 2 / 1024;            // (96: 6, so that the last two waves repeat some)
  static constexpr int OCC = D == 64 ? 4 : 2;      // waves per SIMD
};

template <int D, int DT, bool EX>
__global__ __launch_bounds__(512, DkvPairGeo<D>::OCC) void train_dkv_pair(TrainArgs a) {
  using P = DkvPairGeo<D>;
  using G = TrGeo<D, P::ROWS>;
  constexpr int ROWS = P::ROWS;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[P::SLOTS][2][G::TILE];
  __shared__ __attribute__((aligned(16))) v4f pmem[2][4][4][64];   // the weights of a tile: slot, pair of waves, quarter, lane
  __shared__ __attribute__((aligned(256))) float stat[P::SLOTS][2][ROWS];
  __shared__ float bl[EX ? 2 * TR_REACH + 1 : 1];

  TrSeq s;
  if (!tr_tile<true>(a, blockIdx.x, s)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 31, hf = lane >> 5;
  const int pair = wave & 3, second = wave >> 2;
  const int group = a.H / a.Hkv;
  const int off = s.k_len - s.q_len;
  const int w0 = s.c0 + pair * 32, j = w0 + ln;   // the pair's first key, the lane's
  const bool on = j < s.k_len;
  const int jr = on ? j : s.k_len - 1;

  TrAddr<D> at;
  at.init(lane);
  v4i of[G::NK];                                  // keys or values
  {
    const uint16_t* p = second ? a.v + (a.cu_q ? 0 : s.b * a.vb) + (s.kr + jr) * a.vs + s.h * a.vh
                               : a.k + (a.cu_q ? 0 : s.b * a.kb) + (s.kr + jr) * a.ks + s.h * a.kh;
#pragma unroll
    for (int x = 0; x < G::NK; ++x) of[x] = *reinterpret_cast<const v4i*>(p + 8 * hf + 16 * x);
  }
  const int ex = DT == DT_F16 ? tr_exponent(a.norms) : 0;
  const float ds_mul = __builtin_ldexpf(1.0f, ex - (int)BWD_SHIFT<DT>);

  const int t_all = (s.q_len + ROWS - 1) / ROWS;
  int t0 = 0;                                     // the first tile that sees one of the workgroup's keys
  if (a.causal) t0 = min(t_all, max(0, s.c0 - off) / ROWS);
  const int nt = t_all - t0;
  const int steps = nt * group;

  // Loads: a wave's are all of q or all of dout.  From the last tile back to the diagonal: workgroups of one head that start
  // together stream the same tiles together.
  const int l0 = wave * P::PER_WAVE % (2 * P::PER_TENSOR), side = l0 / P::PER_TENSOR;
  const int64_t ls = side ? a.gs : a.qs, lh = side ? a.gh : a.qh;
  const uint16_t* lsrc = (side ? a.dout + (a.cu_q ? 0 : s.b * a.gb) : a.q + (a.cu_q ? 0 : s.b * a.qb)) + s.qr * ls + s.h * group * lh;
  const float* stat_src = (wave ? a.nd : a.nl) + tr_stat_row(a, s, s.h * group);
  const int row_l = (l0 - side * P::PER_TENSOR) * 64 + lane;   // the lane's chunk of the wave's first load
  const bool fits = ls >= 0 && ls < (1 << 24);
  uint32_t loff[D == 96 ? P::PER_WAVE : 1], lchunk = 0;
#pragma unroll
  for (int x = 0; x < (D == 96 ? P::PER_WAVE : 1); ++x) {
    const int L = row_l + 64 * x, row = L / G::KCH, c = tr_swz<D>(row, L % G::KCH);
    loff[x] = (uint32_t)((row * ls + (D == 96 ? c * 8 : 0)) * 2);
    lchunk = c * 16;
  }
  int tn = t_all - 1, un = 0;                     // of the step that is loaded
  auto issue = [&]() {
    if (un < steps) {
      const int slot = un % P::SLOTS;
      uint8_t* dst = &smem[slot][side][0] + (l0 - side * P::PER_TENSOR) * 1024;
      if ((tn + 1) * ROWS <= s.q_len && fits) {
        const uint8_t* p = reinterpret_cast<const uint8_t*>(lsrc + (int64_t)(tn * ROWS) * ls);
        asm volatile("" : "+s"(p));
#pragma unroll
        for (int x = 0; x < P::PER_WAVE; ++x) {
          constexpr int RPL = 64 / G::KCH;
          uint32_t o = D == 96 ? loff[D == 96 ? x : 0] : loff[0] + (lchunk ^ (uint32_t)(tr_swz<D>(RPL * x, 0) * 16));
          tr_copy16(p + (D == 96 ? 0 : x * RPL * ls * 2), o, dst + x * 1024);
        }
      } else {
#pragma unroll 1
        for (int x = 0; x < P::PER_WAVE; ++x) {
          const int L = row_l + 64 * x, row = L / G::KCH;
          tr_copy16(lsrc + min(tn * ROWS + row, s.q_len - 1) * ls + tr_swz<D>(row, L % G::KCH) * 8, dst + x * 1024);
        }
      }
      if (wave < 2 && lane < ROWS) tr_copy4(stat_src + tn * ROWS + lane, stat[slot][wave]);
    }
    ++un;
    if (--tn < t0) tn = t_all - 1, lsrc += lh, stat_src += a.pad;
  };

  v16f acc[G::NDB], x;
  v4i ring[P::AHEAD], w[2];
  constexpr int N = G::NK;                         // products of either kind per tile
  TrAddr<D> rt, ct;                                // operands of the tile: by rows, transposed
  auto fetch = [&](const TrAddr<D>& r, const TrAddr<D>& c, auto n_) __attribute__((always_inline)) {
    constexpr int n = decltype(n_)::value, z = n - N;
    if constexpr (n < N) ring[n % P::AHEAD] = r.rows(0, n);
    else ring[n % P::AHEAD] = c.cols(z / G::NDB, z % G::NDB);
  };
  auto begin = [&](const float* st) __attribute__((always_inline)) {   // the sums of the first products begin at the rows' numbers
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const v4f y = *reinterpret_cast<const v4f*>(st + 8 * g + 4 * hf);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * g + e] = y[e];
    }
  };
  // The products of the tile in rt, ct: first those over the channels into x, then `middle` makes of x (elements v0 .. v1) the
  // operand w, then those over the tile's rows into acc.
  auto stream = [&](int next, auto middle) __attribute__((always_inline)) {
    const TrAddr<D> rn = at.in(smem[next][second]);
    tr_unroll<2 * N>([&](auto n_) __attribute__((always_inline)) {
      constexpr int n = decltype(n_)::value;
      const v4i f = ring[n % P::AHEAD];
      if constexpr (n < N) {
        x = tr_mfma<DT>(f, of[n], x);
      } else {
        constexpr int z = n - N;
        acc[z % G::NDB] = tr_mfma<DT>(f, w[z / G::NDB], acc[z % G::NDB]);
      }
      if constexpr (n + P::AHEAD < 2 * N) fetch(rt, ct, std::integral_constant<int, n + P::AHEAD>{});
      else if constexpr (P::CROSS) ring[n % P::AHEAD] = rn.rows(0, n + P::AHEAD - 2 * N);
      if constexpr (n == N - 1) middle(0, 8);
      if constexpr (n >= N && n < N + N / 2) {
        constexpr int e0 = (n - N) * 4 / (N / 2) * 2, e1 = (n - N + 1) * 4 / (N / 2) * 2;
        if constexpr (e1 > e0) middle(8 + e0, 8 + e1);
      }
      if constexpr (P::CROSS && n == 2 * N - 1) begin(stat[next][second]);
      __builtin_amdgcn_sched_barrier(0);
    });
    rt = rn;
  };
  auto enter = [&](int slot) __attribute__((always_inline)) {   // without reads ahead: before a tile
    rt = at.in(smem[slot][second]);
    begin(stat[slot][second]);
    tr_unroll<P::AHEAD>([&](auto n_) __attribute__((always_inline)) { fetch(rt, ct, n_); });
  };

  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int db = 0; db < G::NDB; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[db][v] = 0.0f;
    // (a second pass begins its loads anew)
    if (pass) lsrc -= group * lh, stat_src -= group * a.pad;
    un = 0, tn = t_all - 1;
    int u = 0, slot = 0;
    auto next_slot = [&](int x) { return x + 1 == P::SLOTS ? 0 : x + 1; };
    // The loads of the tile after u (without reads ahead: of u) have arrived, what step u - 1 read may be overwritten
    auto top = [&]() __attribute__((always_inline)) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (P::CROSS && u + 2 < steps && !pass) {
        if (wave < 2) wait_vmcnt<P::PER_WAVE + 1>();
        else wait_vmcnt<P::PER_WAVE>();
      } else {
        wait_vmcnt<0>();
      }
      tile_barrier();
      issue();
      if (pass) {   // tiles are cleaned one step before anything of them is read
        const int c = P::CROSS ? next_slot(slot) : slot;
        auto clean = [&](int y) {
          tr_clean<D, DT, ROWS, 512>(smem[y][0], nullptr, tid);
          tr_clean<D, DT, ROWS, 512>(smem[y][1], nullptr, tid);
        };
        if (P::CROSS && u == 0 && steps > 0) clean(0);
        if (P::CROSS ? u + 1 < steps : u < steps) clean(c);
        __syncthreads();
      }
    };
    if (steps > 0) {
      issue();
      if (P::CROSS) issue(), issue();
    }
    tr_arrived(of);
    // a head's bias, when the first waves come to its first tile
    auto bias = [&]() __attribute__((always_inline)) {
      if (EX && a.bias && u < steps && u % nt == 0) {
        __syncthreads();
        const float* b = a.bias + (int64_t)(s.h * group + u / nt) * (2 * a.reach + 1);
        for (int y = tid; y <= 2 * a.reach; y += 512) bl[y] = b[y];
        __syncthreads();
      }
    };
    bias();
    top();
    if (second == 0) {
      int t = t_all - 1, h = s.h * group;
      if (P::CROSS && steps > 0) enter(slot);
      while (u < steps) {
        if (!P::CROSS) enter(slot);
        ct = at.in(smem[slot][1]);
        const int q0 = t * ROWS, nx = next_slot(slot);
        int room = a.causal ? q0 + 4 * hf - (jr - off) : 0;   // row r sees the key where r + room >= 0
        asm volatile("" : "+v"(room));                        // (16 comparisons' operands are not to be kept for all tiles)
        const int d0 = jr - off - q0 - 4 * hf;                // key - query of register 0; a row further is 1 less
        const int whi = w0 + 31 - off - q0, wlo = w0 - off - q0 - 31;
        const bool near = EX && a.bias && !(whi <= -a.reach || wlo >= a.reach);
        const float far = (EX && a.bias && !near ? bl[whi <= -a.reach ? 0 : 2 * a.reach] : 0.0f) + BWD_SHIFT<DT>;
        const bool masked = EX && a.bits && w0 < s.k_len;
        const uint32_t* bits = a.bits + s.b * a.mb + h * a.mh + (int64_t)(w0 >> 5) * a.mw + (a.mi ? q0 + 4 * hf : 0);
        stream(nx, [&](int v0, int v1) __attribute__((always_inline)) {
#pragma unroll
          for (int v = v0; v < v1; ++v) {
            const int r = 8 * (v >> 2) + (v & 3);
            float y = x[v];
            if (EX) {
              float more = far;
              if (near) more = bl[a.reach + min(max(d0 - r, -a.reach), a.reach)] + BWD_SHIFT<DT>;
              y = __builtin_fmaf(y, a.c, more);
            } else {
              y = DT == DT_F16 ? __builtin_fmaf(y, a.c, BWD_SHIFT<DT>) : y * a.c;
            }
            y = __builtin_amdgcn_exp2f(y);
            y = r + room < 0 ? 0.0f : y;
            if (masked) y = (bits[a.mi ? r : 0] >> ln) & 1u ? y : 0.0f;
            x[v] = y;
          }
#pragma unroll
          for (int v = v0; v < v1; v += 2) w[v >> 3][(v & 7) >> 1] = tr_pack<DT>(x[v], x[v + 1]);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (v1 >= 4 * q + 4 && v0 < 4 * q + 4)
              pmem[u & 1][pair][q][lane] = v4f{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
        });
        if (--t < t0) t = t_all - 1, ++h;
        slot = nx, ++u;
        bias();
        top();
      }
    } else if (steps > 0) {
      slot = next_slot(slot), ++u;
      bias();
      top();
      int mine = 0;                                            // the slot of tile u - 1
      if (P::CROSS) enter(mine);
      for (;;) {
        if (!P::CROSS) enter(mine);
        ct = at.in(smem[mine][0]);
        v4f pw[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) pw[q] = pmem[(u - 1) & 1][pair][q][lane];
        stream(slot, [&](int v0, int v1) __attribute__((always_inline)) {
          // (0 where the weight is, whatever its key or query holds)
#pragma unroll
          for (int v = v0; v < v1; ++v) {
            const float y = pw[v >> 2][v & 3];
            x[v] = y == 0.0f ? 0.0f : x[v] * (DT == DT_F16 ? y * ds_mul : y);
          }
#pragma unroll
          for (int v = v0; v < v1; v += 2) w[v >> 3][(v & 7) >> 1] = tr_pack<DT>(x[v], x[v + 1]);
        });
        if (u == steps) break;
        mine = slot, slot = next_slot(slot), ++u;
        bias();
        top();
      }
    }
    const bool bad = !(tr_nonfinite(acc) == 0.0f);
    if (!__syncthreads_or(on && bad)) break;   // (a second time with every tile cleaned)
  }

  const float f = second ? __builtin_ldexpf(a.scale, -ex) : DT == DT_F16 ? 1.0f / 32768.0f : 1.0f;
  uint16_t* p = second ? a.dk + (a.cu_q ? 0 : s.b * a.dkb) + (s.kr + jr) * a.dks + s.h * a.dkh
                       : a.dv + (a.cu_q ? 0 : s.b * a.dvb) + (s.kr + jr) * a.dvs + s.h * a.dvh;
#pragma unroll
  for (int db = 0; db < G::NDB; ++db) tr_store<DT>(acc[db], f, p + 32 * db, hf, on);
}

template <int D, int DT> int train_bwd_launch(const TrainArgs& a, const BiasMap& m, hipStream_t st) {
  const int B = a.cu_q ? 1 : a.B;
  const unsigned rows = (unsigned)((int64_t)B * a.H * a.q_tiles);
  int norm_blocks = 0;
  if (DT == DT_F16) {
    train_norms_zero<<<1, 64, 0, st>>>(a.norms);
    const int64_t need = ((int64_t)B * a.Hkv * a.Skv * (D == 96 ? 16 : D / 8) + TR_THREADS - 1) / TR_THREADS;
    norm_blocks = (int)(need < 1024 ? need : 1024);
  }
  train_prep<D, DT><<<rows + norm_blocks, TR_THREADS, 0, st>>>(a, (int)rows, norm_blocks);
  const unsigned keys = (unsigned)((int64_t)B * a.Hkv * a.k_tiles);
  if (a.bits || a.bias) {
    const unsigned lds = a.bias_part ? 4u * 4u * (2u * a.reach + 1u) : 0u;
    if (a.dk) {
      if constexpr (D == 256) train_dkv_pair<D, DT, true><<<keys, 512, 0, st>>>(a);
      else train_dkv<D, DT, true><<<keys, TR_THREADS, 0, st>>>(a);
    }
    if (a.dq) train_dq<D, DT, true><<<rows, TR_THREADS, lds, st>>>(a, m);
  } else {
    if (a.dk) {
      if constexpr (D == 256) train_dkv_pair<D, DT, false><<<keys, 512, 0, st>>>(a);
      else train_dkv<D, DT, false><<<keys, TR_THREADS, 0, st>>>(a);
    }
    if (a.dq) train_dq<D, DT, false><<<rows, TR_THREADS, 0, st>>>(a, m);
  }
  return check_launch("train_bwd");
}

#define SAGE_BWD(D) template int train_bwd_launch<D, DT_BF16>(const TrainArgs&, const BiasMap&, hipStream_t); \
                    template int train_bwd_launch<D, DT_F16>(const TrainArgs&, const BiasMap&, hipStream_t);
SAGE_BWD(64) SAGE_BWD(96) SAGE_BWD(128) SAGE_BWD(256)

}  // namespace sage
