// Backward pass of the attention for training, dk and dv: see sage_train.h for the form and sage_train_bwd.hip for the split.
// (Compiled with the results of matrix products in ordinary registers where they are read again: else the compiler moves every
// score to and from the accumulation registers.)
#include "sage_train.h"

namespace sage {

// ---- dk, dv --------------------------------------------------------------------------------------------------------------------
//
// A wave's keys and values (D / 2 registers) and the sums of its dk and dv (2 D) leave room for one wave per SIMD, so a wave has to
// keep the matrix unit busy by itself.  It walks blocks of 32 queries, two a tile, as one stream of products: those of block b + 1's
// scores and weights' gradients in turn with block b - 1's parts of dv and dk, and beside them the weights of block b.  The operands
// of product n + AHEAD are read from LDS when product n is issued, whatever tile they are of.  (Two waves per SIMD with half of the
// registers each, four operands ahead: 625 us at 1 x 24 x 4608 x 128; the weights beside half of the products only: 606; this
// 543, 0.96 PFLOP/s, the matrix unit busy for 51%, and 2000 at 2 x 32 on 8 x 8192 x 128 causal, 1.10 PFLOP/s.)  What bounds it is
// issue: one wave has to issue 64 products and some 400 other instructions a tile.
template <int D> struct DkvGeo {
  static constexpr int ROWS = 64;                  // queries per tile
  static constexpr int SLOTS = 4;                  // tiles in LDS: one still read, one at work, one arrived, one on its way
  static constexpr int AHEAD = 4;                  // products between an operand's read and its use (a power of two)
  static constexpr int OCC = D == 64 ? 2 : 1;      // waves per SIMD
};

template <int D, int DT, bool EX>
__global__ __launch_bounds__(TR_THREADS, DkvGeo<D>::OCC) void train_dkv(TrainArgs a) {
  using P = DkvGeo<D>;
  using G = TrGeo<D, P::ROWS>;
  constexpr int ROWS = P::ROWS, AHEAD = P::AHEAD;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[P::SLOTS][2][G::TILE];
  __shared__ __attribute__((aligned(256))) float stat[P::SLOTS][2][ROWS];
  __shared__ float bl[EX ? 2 * TR_REACH + 1 : 1];
  __shared__ __attribute__((aligned(256))) uint32_t wl[P::SLOTS][4][EX ? ROWS : 1];   // a mask's words of the tiles, for each wave's keys

  TrSeq s;
  if (!tr_tile<true>(a, blockIdx.x, s)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 31, hf = lane >> 5;
  const int group = s.hn;
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
  const int steps = EX ? tr_steps<0>(a, s, group, t0, t_all) : (t_all - t0) * group;
  int t_full = 0;                                 // from this tile on every query sees every key of the wave
  if (a.causal) t_full = (max(0, w0 + 31 - off) + ROWS - 1) / ROWS;
  if (EX && a.bits) t_full = t_all;
  t_full = min(max(t_full, t0), t_all);

  // Loads, from the last tile back to the diagonal: workgroups of one head that start together stream the same tiles together.
  TrLoader<D, ROWS> lq, lg;
  lq.init(a.qs, wave, lane);
  lg.init(a.gs, wave, lane);
  const uint16_t* qp = a.q + (a.cu_q ? 0 : s.b * a.qb) + s.qr * a.qs + s.h0 * a.qh;
  const uint16_t* gp = a.dout + (a.cu_q ? 0 : s.b * a.gb) + s.qr * a.gs + s.h0 * a.gh;
  const float* sp = (wave & 1 ? a.nd : a.nl) + tr_stat_row(a, s, s.h0) + lane;
  const uint32_t* mp = EX && a.bits ? a.bits + s.b * a.mb + s.h0 * a.mh + (int64_t)(min(w0, s.k_len - 1) >> 5) * a.mw : nullptr;
  TrWalk<0, EX> ld;                               // the tile that is loaded next
  int un = 0;
  auto shift = [&](int heads) { qp += heads * a.qh, gp += heads * a.gh, sp += heads * a.pad, mp += heads * a.mh; };
  auto issue = [&]() __attribute__((always_inline)) {
    if (un >= steps) return;
    const int slot = un & (P::SLOTS - 1), row = ld.t * ROWS;
    uint8_t* dst = smem[slot][0];
    if (row + ROWS <= s.q_len && lq.fits && lg.fits) {
      lq.whole(qp + row * a.qs, dst, wave);
      lg.whole(gp + row * a.gs, dst + G::TILE, wave);
    } else {
      lq.part(qp, a.qs, row, s.q_len, dst, wave, lane);
      lg.part(gp, a.gs, row, s.q_len, dst + G::TILE, wave, lane);
    }
    if (wave < 2) tr_copy4(sp + row, stat[slot][wave]);
    if (EX && a.bits) tr_copy4(mp + (a.mi ? row + lane : 0), wl[slot][wave]);
    ++un;
    shift(ld.advance(a, s, group, t0, t_all));
  };

  constexpr int N = 2 * G::NK;                     // products of either kind per block
  v16f dk[G::NDB], dv[G::NDB], x[2], dp[2];        // (x, dp, p, ds: of even and odd blocks)
  v4i ring[AHEAD], p[2][2], ds[2][2];
  TrAddr<D> prev, cur, next;                       // the tiles of steps u - 1, u, u + 1 (q's; dout's lie behind them)
  auto slot_of = [&](int u) __attribute__((always_inline)) { return at.in(smem[u & (P::SLOTS - 1)][0]); };
  auto begin = [&](int u, auto qb_) __attribute__((always_inline)) {   // the first products' sums begin at the rows' numbers
    constexpr int qb = decltype(qb_)::value;
    const float(&st)[2][ROWS] = stat[u & (P::SLOTS - 1)];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const v4f y = *reinterpret_cast<const v4f*>(&st[0][32 * qb + 8 * g + 4 * hf]);
      const v4f z = *reinterpret_cast<const v4f*>(&st[1][32 * qb + 8 * g + 4 * hf]);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[qb][4 * g + e] = y[e], dp[qb][4 * g + e] = z[e];
    }
  };
  // Product y of a block's first kind (over the channels) and of its second (over its 32 queries): operand and product
  auto first_op = [&](const TrAddr<D>& tile, int qb, int y) __attribute__((always_inline)) {
    return tile.rows(qb, y >> 1, y & 1 ? G::TILE : 0);
  };
  auto second_op = [&](const TrAddr<D>& tile, int qb, int y) __attribute__((always_inline)) {
    return tile.cols(2 * qb + y / (2 * G::NDB), y % (2 * G::NDB) >> 1, y & 1 ? 0 : G::TILE);
  };
  auto first = [&](const v4i& f, auto qb_, auto y_) __attribute__((always_inline)) {
    constexpr int qb = decltype(qb_)::value, y = decltype(y_)::value;
    if constexpr (y & 1) dp[qb] = tr_mfma<DT>(f, vf[y >> 1], dp[qb]);
    else x[qb] = tr_mfma<DT>(f, kf[y >> 1], x[qb]);
  };
  auto second = [&](const v4i& f, auto qb_, auto y_) __attribute__((always_inline)) {
    constexpr int qb = decltype(qb_)::value, y = decltype(y_)::value, st = y / (2 * G::NDB), db = y % (2 * G::NDB) >> 1;
    if constexpr (y & 1) dk[db] = tr_mfma<DT>(f, ds[qb][st], dk[db]);
    else dv[db] = tr_mfma<DT>(f, p[qb][st], dv[db]);
  };
  // The products beside the weights of block `par` of tile u: first ones of the block after it, second ones of the block before it
  // (both of the other parity), in turn.
  auto operand = [&](auto par_, auto n_) __attribute__((always_inline)) {
    constexpr int par = decltype(par_)::value, n = decltype(n_)::value;
    if constexpr (n & 1) return second_op(par ? cur : prev, 1 - par, n >> 1);
    else return first_op(par ? next : cur, 1 - par, n >> 1);
  };
  auto half = [&](int u, int t, auto par_, auto masked_) __attribute__((always_inline)) {
    constexpr int par = decltype(par_)::value;
    constexpr bool masked = decltype(masked_)::value;
    using Other = std::integral_constant<int, 1 - par>;
    const int q0 = t * ROWS + 32 * par;
    const int d0 = jr - off - q0 - 4 * hf;        // key - query of register 0; a row further is 1 less
    const int whi = w0 + 31 - off - q0, wlo = w0 - off - q0 - 31;
    const bool near = EX && a.bias && !(whi <= -a.reach || wlo >= a.reach);
    const float far = (EX && a.bias && !near ? bl[whi <= -a.reach ? 0 : 2 * a.reach] : 0.0f) + BWD_SHIFT<DT>;
    int room = masked && a.causal ? q0 + 4 * hf - (jr - off) : 0;   // row r sees the key where r + room >= 0
    if (masked) asm volatile("" : "+v"(room));                      // (16 comparisons' operands are not to be kept for all tiles)
    const bool hiding = masked && EX && a.bits;
    const uint32_t* bits = &wl[u & (P::SLOTS - 1)][wave][EX ? 32 * par + 4 * hf : 0];
    v4i seen;                                                       // the words of four rows
    // Elements v, v + 1 in four slices of about as many instructions as there is time for beside a product; where a quarter of
    // the block's numbers has been used up, those of the block after the next take its place.
    float w0_ = 0.0f, w1_ = 0.0f, e0_ = 0.0f, e1_ = 0.0f;
    const float(&st)[2][ROWS] = stat[(u + 1) & (P::SLOTS - 1)];
    auto score = [&](int v) __attribute__((always_inline)) {
      const int r = 8 * (v >> 2) + (v & 3);
      if (EX) {
        float more = far;
        if (near) more = bl[a.reach + min(max(d0 - r, -a.reach), a.reach)] + BWD_SHIFT<DT>;
        return __builtin_fmaf(x[par][v], a.c, more);
      }
      return DT == DT_F16 ? __builtin_fmaf(x[par][v], a.c, BWD_SHIFT<DT>) : x[par][v] * a.c;
    };
    auto shown = [&](int v, float& w) __attribute__((always_inline)) {
      if (masked) {
        const int r = 8 * (v >> 2) + (v & 3);
        bool hidden = r + room < 0;
        if (hiding) hidden |= !(((uint32_t)seen[v & 3] >> ln) & 1u);
        if (hidden) w = 0.0f, dp[par][v] = 0.0f;
      }
    };
    auto slice = [&](auto m_) __attribute__((always_inline)) {
      constexpr int m = decltype(m_)::value, v = m / 4 * 2;
      if constexpr (m % 4 == 0) {
        if (hiding && (v & 3) == 0) seen = *reinterpret_cast<const v4i*>(bits + 8 * (v >> 2));
        w0_ = score(v), w1_ = score(v + 1);
        w0_ = __builtin_amdgcn_exp2f(w0_);
      } else if constexpr (m % 4 == 1) {
        w1_ = __builtin_amdgcn_exp2f(w1_);
        shown(v, w0_);
        e0_ = w0_ * dp[par][v];
      } else if constexpr (m % 4 == 2) {
        shown(v + 1, w1_);
        e1_ = w1_ * dp[par][v + 1];
        int pw = tr_pack<DT>(w0_, w1_);
        asm volatile("" : "+v"(pw));              // (here, not where the next tile's products use it)
        p[par][v >> 3][(v & 7) >> 1] = pw;
      } else {
        if (DT == DT_F16) e0_ *= ds_mul, e1_ *= ds_mul;
        int dw = tr_pack<DT>(e0_, e1_);
        asm volatile("" : "+v"(dw));
        ds[par][v >> 3][(v & 7) >> 1] = dw;
        if constexpr ((v & 3) == 2) {
          constexpr int g = v >> 2;
          const v4f y = *reinterpret_cast<const v4f*>(&st[0][32 * par + 8 * g + 4 * hf]);
          const v4f z = *reinterpret_cast<const v4f*>(&st[1][32 * par + 8 * g + 4 * hf]);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[par][4 * g + e] = y[e], dp[par][4 * g + e] = z[e];
        }
      }
    };
    tr_unroll<2 * N>([&](auto n_) __attribute__((always_inline)) {
      constexpr int n = decltype(n_)::value;
      const v4i f = ring[n % AHEAD];
      if constexpr (n & 1) second(f, Other{}, std::integral_constant<int, (n >> 1)>{});
      else first(f, Other{}, std::integral_constant<int, (n >> 1)>{});
      if constexpr (n + AHEAD < 2 * N) {
        ring[n % AHEAD] = operand(par_, std::integral_constant<int, n + AHEAD>{});
      } else {
        // of the half after this one: (next, 0) and (cur, 0) of the same tile, or (cur, 1) and (prev, 1) of the tile after it
        constexpr int m = n + AHEAD - 2 * N;
        if constexpr (m & 1) ring[n % AHEAD] = second_op(cur, par, m >> 1);
        else ring[n % AHEAD] = first_op(next, par, m >> 1);
      }
      // 32 slices over the products but the first and the last three
      if constexpr (n >= 1 && n < 2 * N - 3) {
        constexpr int m0 = (n - 1) * 32 / (2 * N - 4), m1 = n * 32 / (2 * N - 4);
        tr_unroll<m1 - m0>([&](auto m_) __attribute__((always_inline)) { slice(std::integral_constant<int, m0 + decltype(m_)::value>{}); });
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int db = 0; db < G::NDB; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) dk[db][v] = 0.0f, dv[db][v] = 0.0f;
    p[1][0] = p[1][1] = ds[1][0] = ds[1][1] = v4i{0, 0, 0, 0};   // (before the first block there is none)
    // The tile after u has arrived, the one two before u is read and its place free
    auto top = [&](int u) __attribute__((always_inline)) {
      wait_vmcnt<0>();
      tile_barrier();
      issue();
      if (pass) {   // a tile is cleaned when it has arrived, one step before anything of it is read
        for (int y = u ? 1 : 0; y < 2; ++y) {
          if (u + y >= steps) break;
          uint8_t* tile = smem[(u + y) & (P::SLOTS - 1)][0];
          tr_clean<D, DT, ROWS>(tile, nullptr, tid);
          tr_clean<D, DT, ROWS>(tile + G::TILE, nullptr, tid);
        }
        __syncthreads();
      }
    };
    shift(ld.start(a, s, group, t0, t_all));
    issue();
    issue();
    tr_arrived(kf);
    tr_arrived(vf);
    if (steps > 0) {
      using Zero = std::integral_constant<int, 0>;
      using One = std::integral_constant<int, 1>;
      top(0);
      prev = cur = slot_of(0), next = slot_of(1);
      begin(0, Zero{});
      begin(0, One{});
      tr_unroll<N>([&](auto y_) __attribute__((always_inline)) { first(first_op(cur, 0, decltype(y_)::value), Zero{}, y_); });
      tr_unroll<AHEAD>([&](auto n_) __attribute__((always_inline)) { ring[decltype(n_)::value] = operand(Zero{}, n_); });
      TrWalk<0, EX> at_work;
      at_work.start(a, s, group, t0, t_all);
      int u = 0;
      while (u < steps) {
        const int h = s.h0 + at_work.g;
        if (EX && a.bias) {
          __syncthreads();
          for (int y = tid; y <= 2 * a.reach; y += TR_THREADS) bl[y] = a.bias[(int64_t)h * (2 * a.reach + 1) + y];
          __syncthreads();
        }
        // a head: first the tiles that hide no keys of the wave, then, in a loop of their own, those that do
        bool same = true;
        auto one = [&](auto masked_) __attribute__((always_inline)) {
          half(u, at_work.t, Zero{}, masked_);
          half(u, at_work.t, One{}, masked_);
          prev = cur, cur = next, next = slot_of(u + 2), ++u;
          same = at_work.advance(a, s, group, t0, t_all) == 0 && u < steps;
          if (u < steps) top(u);
        };
        const int full = pass ? t_all : t_full;      // (a second pass takes hidden keys out of every tile)
        while (same && at_work.t >= full) one(std::false_type{});
        while (same) one(std::true_type{});
      }
      tr_unroll<N>([&](auto y_) __attribute__((always_inline)) { second(second_op(prev, 1, decltype(y_)::value), One{}, y_); });
    }
    const bool bad = !(tr_nonfinite(dk) + tr_nonfinite(dv) == 0.0f);
    if (!__syncthreads_or(on && bad)) break;   // (a second time with every tile cleaned: the loads begin anew)
    shift(-ld.g);
    un = 0;
  }

  const float fk = __builtin_ldexpf(a.scale, -ex), fv = DT == DT_F16 ? 1.0f / 32768.0f : 1.0f;
  if (a.split > 1) {
    float *kp = tr_kv_part<D>(a, s, 0, jr), *vp = tr_kv_part<D>(a, s, 1, jr);
#pragma unroll
    for (int db = 0; db < G::NDB; ++db) {
      tr_store_f32(dk[db], fk, kp + 32 * db, hf, on);
      tr_store_f32(dv[db], fv, vp + 32 * db, hf, on);
    }
    return;
  }
  uint16_t* kp = a.dk + (a.cu_q ? 0 : s.b * a.dkb) + (s.kr + jr) * a.dks + s.h * a.dkh;
  uint16_t* vp = a.dv + (a.cu_q ? 0 : s.b * a.dvb) + (s.kr + jr) * a.dvs + s.h * a.dvh;
#pragma unroll
  for (int db = 0; db < G::NDB; ++db) {
    tr_store<DT>(dk[db], fk, kp + 32 * db, hf, on);
    tr_store<DT>(dv[db], fv, vp + 32 * db, hf, on);
  }
}

// Head dim 256, where one wave's operands and sums pass its 512 registers: two waves share each 32 keys.  The first recomputes the
// scores, makes the weights and sums dv; the second recomputes the gradient of the weights, multiplies it by the weights, which it
// gets in fp32 through LDS one tile later, and sums dk.  Each has half of the operands and sums, so two waves fit a SIMD, and one's
// exponentials run beside the other's products.  Step u: the first waves work on tile u of 32 queries, the second ones on tile
// u - 1, tile u + 1 is on its way.  (2 x 12 x 2180 x 256: 648 us in one wave, whose registers spill, 400 like this; at head dim
// 128 one wave is faster, 702 and 567 us at 1 x 24 x 4608 when they were compared.)
template <int D> struct DkvPairGeo {
  static constexpr int ROWS = 32;                  // queries per tile
  static constexpr int SLOTS = 3;                  // tiles in LDS
  static constexpr int AHEAD = 4;                  // products between an operand's read and its use
  static constexpr int PER_WAVE = D * ROWS * 4 / 1024 / 8;    // 1 KiB loads of a wave per step, of q or of dout
  static constexpr int PER_TENSOR = D * ROWS * 2 / 1024;
};

template <int D, int DT, bool EX>
__global__ __launch_bounds__(512, 2) void train_dkv_pair(TrainArgs a) {
  using P = DkvPairGeo<D>;
  using G = TrGeo<D, P::ROWS>;
  constexpr int ROWS = P::ROWS;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[P::SLOTS][2][G::TILE];
  __shared__ __attribute__((aligned(16))) v4f pmem[2][4][4][64];   // the weights of a tile: slot, pair of waves, quarter, lane
  __shared__ __attribute__((aligned(256))) float stat[P::SLOTS][2][ROWS];
  __shared__ float bl[EX ? 2 * TR_REACH + 1 : 1];
  __shared__ __attribute__((aligned(256))) uint32_t wl[P::SLOTS][4][EX ? ROWS : 1];   // a mask's words of the tiles, for each pair's keys

  TrSeq s;
  if (!tr_tile<true>(a, blockIdx.x, s)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 31, hf = lane >> 5;
  const int pair = wave & 3, second = wave >> 2;
  const int group = s.hn;
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
  const int steps = EX ? tr_steps<1>(a, s, group, t0, t_all) : (t_all - t0) * group;

  // Loads: a wave's are all of q or all of dout.  From the last tile back to the diagonal: workgroups of one head that start
  // together stream the same tiles together.
  const int l0 = wave * P::PER_WAVE, side = l0 / P::PER_TENSOR;
  const int64_t ls = side ? a.gs : a.qs, lh = side ? a.gh : a.qh;
  const uint16_t* lsrc = (side ? a.dout + (a.cu_q ? 0 : s.b * a.gb) : a.q + (a.cu_q ? 0 : s.b * a.qb)) + s.qr * ls + s.h0 * lh;
  const float* stat_src = (wave ? a.nd : a.nl) + tr_stat_row(a, s, s.h0);
  const int row_l = (l0 - side * P::PER_TENSOR) * 64 + lane;   // the lane's chunk of the wave's first load
  const bool fits = ls >= 0 && ls < (1 << 24);
  uint32_t loff[P::PER_WAVE];
#pragma unroll
  for (int x = 0; x < P::PER_WAVE; ++x) {
    const int L = row_l + 64 * x, row = L / G::KCH;
    loff[x] = (uint32_t)((row * ls + tr_swz<D>(row, L % G::KCH) * 8) * 2);
  }
  const uint32_t* mp = EX && a.bits ? a.bits + s.b * a.mb + s.h0 * a.mh + (int64_t)(min(w0, s.k_len - 1) >> 5) * a.mw : nullptr;
  TrWalk<1, EX> ld;                               // the tile that is loaded next
  int un = 0;
  auto shift = [&](int heads) { lsrc += heads * lh, stat_src += heads * a.pad, mp += heads * a.mh; };
  auto issue = [&]() {
    if (un < steps) {
      const int slot = un % P::SLOTS, tn = ld.t;
      uint8_t* dst = &smem[slot][side][0] + (l0 - side * P::PER_TENSOR) * 1024;
      if ((tn + 1) * ROWS <= s.q_len && fits) {
        const uint16_t* p = lsrc + (int64_t)(tn * ROWS) * ls;
#pragma unroll
        for (int x = 0; x < P::PER_WAVE; ++x) tr_copy16(p, loff[x], dst + x * 1024);
      } else {
#pragma unroll 1
        for (int x = 0; x < P::PER_WAVE; ++x) {
          const int L = row_l + 64 * x, row = L / G::KCH;
          tr_copy16(lsrc + min(tn * ROWS + row, s.q_len - 1) * ls + tr_swz<D>(row, L % G::KCH) * 8, dst + x * 1024);
        }
      }
      if (wave < 2 && lane < ROWS) tr_copy4(stat_src + tn * ROWS + lane, stat[slot][wave]);
      if (EX && a.bits && !second && lane < ROWS) tr_copy4(mp + (a.mi ? tn * ROWS + lane : 0), wl[slot][pair]);
      shift(ld.advance(a, s, group, t0, t_all));
    }
    ++un;
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
  auto stream = [&](auto middle) __attribute__((always_inline)) {
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
      if constexpr (n == N - 1) middle(0, 8);
      if constexpr (n >= N && n < N + N / 2) {
        constexpr int e0 = (n - N) * 4 / (N / 2) * 2, e1 = (n - N + 1) * 4 / (N / 2) * 2;
        if constexpr (e1 > e0) middle(8 + e0, 8 + e1);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  auto enter = [&](int slot) __attribute__((always_inline)) {   // before a tile
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
    if (pass) shift(-ld.g);
    shift(ld.start(a, s, group, t0, t_all));
    un = 0;
    int u = 0, slot = 0;
    auto next_slot = [&](int x) { return x + 1 == P::SLOTS ? 0 : x + 1; };
    // Tile u has arrived, what step u - 1 read last may be overwritten
    auto top = [&]() __attribute__((always_inline)) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      wait_vmcnt<0>();
      tile_barrier();
      issue();
      if (pass) {   // a tile is cleaned when it has arrived
        if (u < steps) {
          tr_clean<D, DT, ROWS, 512>(smem[slot][0], nullptr, tid);
          tr_clean<D, DT, ROWS, 512>(smem[slot][1], nullptr, tid);
        }
        __syncthreads();
      }
    };
    issue();
    tr_arrived(of);
    TrWalk<1, EX> at_work;                         // tile u
    at_work.start(a, s, group, t0, t_all);
    bool entered = true;                           // tile u is the first of its head
    // a head's bias, when the first waves come to its first tile
    auto bias = [&]() __attribute__((always_inline)) {
      if (EX && a.bias && u < steps && entered) {
        __syncthreads();
        const float* b = a.bias + (int64_t)(s.h0 + at_work.g) * (2 * a.reach + 1);
        for (int y = tid; y <= 2 * a.reach; y += 512) bl[y] = b[y];
        __syncthreads();
      }
    };
    auto step = [&]() __attribute__((always_inline)) { entered = at_work.advance(a, s, group, t0, t_all) != 0, ++u; };
    bias();
    top();
    if (second == 0) {
      while (u < steps) {
        enter(slot);
        ct = at.in(smem[slot][1]);
        const int q0 = at_work.t * ROWS, nx = next_slot(slot);
        int room = a.causal ? q0 + 4 * hf - (jr - off) : 0;   // row r sees the key where r + room >= 0
        asm volatile("" : "+v"(room));                        // (16 comparisons' operands are not to be kept for all tiles)
        const int d0 = jr - off - q0 - 4 * hf;                // key - query of register 0; a row further is 1 less
        const int whi = w0 + 31 - off - q0, wlo = w0 - off - q0 - 31;
        const bool near = EX && a.bias && !(whi <= -a.reach || wlo >= a.reach);
        const float far = (EX && a.bias && !near ? bl[whi <= -a.reach ? 0 : 2 * a.reach] : 0.0f) + BWD_SHIFT<DT>;
        const bool masked = EX && a.bits;
        const uint32_t* bits = &wl[slot][pair][EX ? 4 * hf : 0];
        stream([&](int v0, int v1) __attribute__((always_inline)) {
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
            if (masked) y = (bits[r] >> ln) & 1u ? y : 0.0f;
            x[v] = y;
          }
#pragma unroll
          for (int v = v0; v < v1; v += 2) w[v >> 3][(v & 7) >> 1] = tr_pack<DT>(x[v], x[v + 1]);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (v1 >= 4 * q + 4 && v0 < 4 * q + 4)
              pmem[u & 1][pair][q][lane] = v4f{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
        });
        slot = nx;
        step();
        bias();
        top();
      }
    } else if (steps > 0) {
      slot = next_slot(slot);
      step();
      bias();
      top();
      int mine = 0;                                            // the slot of tile u - 1
      for (;;) {
        enter(mine);
        ct = at.in(smem[mine][0]);
        v4f pw[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) pw[q] = pmem[(u - 1) & 1][pair][q][lane];
        stream([&](int v0, int v1) __attribute__((always_inline)) {
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
        mine = slot, slot = next_slot(slot);
        step();
        bias();
        top();
      }
    }
    const bool bad = !(tr_nonfinite(acc) == 0.0f);
    if (!__syncthreads_or(on && bad)) break;   // (a second time with every tile cleaned)
  }

  const float f = second ? __builtin_ldexpf(a.scale, -ex) : DT == DT_F16 ? 1.0f / 32768.0f : 1.0f;
  if (a.split > 1) {
    float* p = tr_kv_part<D>(a, s, 1 - second, jr);
#pragma unroll
    for (int db = 0; db < G::NDB; ++db) tr_store_f32(acc[db], f, p + 32 * db, hf, on);
    return;
  }
  uint16_t* p = second ? a.dk + (a.cu_q ? 0 : s.b * a.dkb) + (s.kr + jr) * a.dks + s.h * a.dkh
                       : a.dv + (a.cu_q ? 0 : s.b * a.dvb) + (s.kr + jr) * a.dvs + s.h * a.dvh;
#pragma unroll
  for (int db = 0; db < G::NDB; ++db) tr_store<DT>(acc[db], f, p + 32 * db, hf, on);
}

// dk and dv where several workgroups share a kv head's query heads: their sums in the order of the heads, one thread per 8 channels
template <int D, int DT> __global__ __launch_bounds__(TR_THREADS) void train_kv_join(TrainArgs a) {
  const int64_t rows = (int64_t)(a.cu_q ? 1 : a.B) * a.Skv, n = rows * a.Hkv * (D / 8);
  const int which = blockIdx.y;
  for (int64_t x = (int64_t)blockIdx.x * TR_THREADS + threadIdx.x; x < n; x += (int64_t)gridDim.x * TR_THREADS) {
    const int64_t rh = x / (D / 8), row = rh / a.Hkv;
    const int ch = (int)(x % (D / 8)) * 8, h = (int)(rh % a.Hkv);
    if (a.cu_q && (row < a.bounds[2] || row >= a.bounds[3])) continue;   // (zeros already)
    const float* p = a.kv_part + (which * rows * a.Hkv + rh) * D + ch;
    v4f lo = *reinterpret_cast<const v4f*>(p), hi = *reinterpret_cast<const v4f*>(p + 4);
    for (int z = 1; z < a.split; ++z) {
      p += 2 * rows * a.Hkv * D;
      const v4f y = *reinterpret_cast<const v4f*>(p), w = *reinterpret_cast<const v4f*>(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) lo[e] += y[e], hi[e] += w[e];
    }
    const int64_t b = a.cu_q ? 0 : row / a.Skv, r = a.cu_q ? row : row % a.Skv;
    uint16_t* o = which ? a.dv + b * a.dvb + r * a.dvs + h * a.dvh : a.dk + b * a.dkb + r * a.dks + h * a.dkh;
    *reinterpret_cast<v4i*>(o + ch) = v4i{tr_pack<DT>(lo[0], lo[1]), tr_pack<DT>(lo[2], lo[3]), tr_pack<DT>(hi[0], hi[1]),
                                          tr_pack<DT>(hi[2], hi[3])};
  }
}

template <int D, int DT> int train_dkv_launch(const TrainArgs& a, hipStream_t st) {
  const unsigned n = (unsigned)((int64_t)(a.cu_q ? 1 : a.B) * a.Hkv * a.split * a.k_tiles);
  if constexpr (D == 256) {
    if (a.bits || a.bias) train_dkv_pair<D, DT, true><<<n, 512, 0, st>>>(a);
    else train_dkv_pair<D, DT, false><<<n, 512, 0, st>>>(a);
  } else {
    if (a.bits || a.bias) train_dkv<D, DT, true><<<n, TR_THREADS, 0, st>>>(a);
    else train_dkv<D, DT, false><<<n, TR_THREADS, 0, st>>>(a);
  }
  if (a.split > 1) {
    const int64_t need = ((int64_t)(a.cu_q ? 1 : a.B) * a.Skv * a.Hkv * (D / 8) + TR_THREADS - 1) / TR_THREADS;
    train_kv_join<D, DT><<<dim3((unsigned)(need < 65536 ? need : 65536), 2), TR_THREADS, 0, st>>>(a);
  }
  return check_launch("train_dkv");
}

#define SAGE_DKV(D) template int train_dkv_launch<D, DT_BF16>(const TrainArgs&, hipStream_t); \
                    template int train_dkv_launch<D, DT_F16>(const TrainArgs&, hipStream_t);
SAGE_DKV(64) SAGE_DKV(96) SAGE_DKV(128) SAGE_DKV(256)

}  // namespace sage
