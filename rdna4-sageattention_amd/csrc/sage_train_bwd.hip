// Backward pass of the attention for training: see sage_train.h for the form.
//
// Two kernels, each of which recomputes the scores and the gradient of the probabilities: one owns queries and streams keys
// (dq), one owns keys and streams queries (dk, dv).  That is seven products for the five of the formulas, and it needs neither
// atomics nor (but for few tiles of shared heads, train_split) partial results in memory: every gradient is one sum in a fixed
// order, so equal inputs give equal bits.  A single kernel would have to add dq over its workgroups: 4 bytes written and read for
// every 2 * 128 keys' products of a channel.
#include "sage_train.h"

namespace sage {

// ---- preparation: -lse / sm_scale and -D of every row; the norms of fp16 inputs -----------------------------------------------
//
// Bound by its reads of out, its remainder and dout: 75 us for 2 x 32 x 8192 x 128 (402 MB, 5.4 TB/s).

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
  if ((int)blockIdx.x >= row_blocks) {            // fp16: the rows of v that a query sees (what others hold is not to matter)
    const uint32_t len = a.cu_q ? a.k_tiles * TR_COLS : a.Skv, n = (a.cu_q ? 1 : a.B) * a.Hkv * len;
    for (uint32_t x = (blockIdx.x - row_blocks) * ROWS + r; x < n; x += norm_blocks * ROWS) {
      const uint32_t t = x / a.Hkv;
      const int64_t h = x % a.Hkv, b = t / len;
      int64_t j = t % len;
      bool seen = true;
      if (a.cu_q) {                               // (the last query of a sequence sees all of its keys)
        const int2 e = a.k_tab[j / TR_COLS];
        const int k0 = e.x < 0 ? 0 : a.cu_k[e.x], i = e.y * TR_COLS + (int)(j % TR_COLS);
        seen = e.x >= 0 && k0 + i < a.cu_k[e.x + 1] && a.cu_q[e.x] < a.cu_q[e.x + 1];
        j = k0 + i;
      } else if (a.keys_seen) {
        uint64_t w = 0;
        const int heads = a.th ? a.H / a.Hkv : 1;
        for (int g = 0; g < heads; ++g)
          for (int y = 0; y < a.tw; ++y) w |= a.keys_seen[b * a.tb + (h * heads + g) * a.th + (j >> 6) * a.tw + y];
        seen = w >> (j & 63) & 1;
      }
      float s = 0.0f;
      if (has && seen) {
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
    const uint16_t* lp = a.lo + lse_at * D + l * 8;
    for (int i = s.c0 + r; i < end; i += ROWS) {
      const float lse = i < s.q_len ? a.lse[lse_at + i] : -INFINITY;
      float d = 0.0f, g2 = 0.0f;
      if (i < s.q_len && has) {
        const v4i x = *reinterpret_cast<const v4i*>(op + i * a.os), g = *reinterpret_cast<const v4i*>(gp + i * a.gs);
        const v4i y = *reinterpret_cast<const v4i*>(lp + (int64_t)i * D);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float g0 = elem_lo<DT>(g[e]), g1 = elem_hi<DT>(g[e]);
          d = __builtin_fmaf(elem_lo<DT>(x[e]) + elem_lo<DT>(y[e]), g0, __builtin_fmaf(elem_hi<DT>(x[e]) + elem_hi<DT>(y[e]), g1, d));
          if (DT == DT_F16) g2 = __builtin_fmaf(g0, g0, __builtin_fmaf(g1, g1, g2));
        }
      }
      d = row_sum(d);
      if (DT == DT_F16) {
        g2 = row_sum(g2);
        if (g2 < INFINITY && lse != -INFINITY) top = fmaxf(top, g2);
      }
      if (l == 0) {
        // a row that sees nothing: p = 0; one with an infinity or a NaN in it: p = NaN wherever it sees a key
        float nl = -(lse / a.scale), nd = -d;
        if (lse == -INFINITY) nl = -INFINITY, nd = 0.0f;
        else if (!(fabsf(nl) < INFINITY) || !(fabsf(d) < INFINITY)) nl = NAN;
        a.nl[at + i] = nl;
        a.nd[at + i] = nd;
      }
    }
  }
  if (DT == DT_F16) {
    // (a maximum does not depend on the order; few workgroups are the first to see a larger one)
    __shared__ float tops[TR_THREADS / 64];
    top = wave_max_pos(top);
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
    if (tid == 0) {
      uint32_t* norm = a.norms + ((int)blockIdx.x >= row_blocks ? 1 : 0);
      const uint32_t m = __float_as_uint(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
      if (m > __atomic_load_n(norm, __ATOMIC_RELAXED)) atomicMax(norm, m);
    }
  }
}

__global__ void train_norms_zero(uint32_t* norms) {
  if (threadIdx.x < 2) norms[threadIdx.x] = 0;
}

// ---- dq (and the bias' gradient by distance) ---------------------------------------------------------------------------------
//
// A wave per 32 queries, 12 D / 32 products per 32 keys and two workgroups per unit: 356 us at 1 x 24 x 4608 x 128 bf16 (1.10 PFLOP/s;
// the matrix unit busy for 62%), 1360 at 2 x 32 x 8192 x 128 causal (1.21).  With a table's gradient a block near the diagonal
// costs 28 LDS accesses more: 55 us at 4 x 16 x 1024 x 64, reach 128, where an atomic per pair took 99.

template <int D, int DT, bool EX>
__global__ __launch_bounds__(TR_THREADS, D == 256 ? 1 : 2) void train_dq(TrainArgs a, BiasMap map) {
  using G = TrGeo<D>;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2][2][G::TILE];
  __shared__ __attribute__((aligned(256))) uint32_t wl[2][4][EX ? 64 : 1];   // a mask's words of the tiles, for each wave's queries
  // With bias_part: 16 x 32 sums of each wave, unless D is 256, and 4 waves' sums by distance, 2 reach + 1 each; then the bias.  (As
  // much as the reach needs: up to 128, two workgroups of 128 channels fit a unit.)
  extern __shared__ __attribute__((aligned(16))) float diag[];

  TrSeq s;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const bool biased = EX && a.bias, want_part = EX && a.bias_part;
  const int R = 2 * a.reach + 1;
  float *by_distance = diag + (D < 256 ? 4 * 16 * 32 : 0), *bl = want_part ? by_distance + 4 * R : diag;
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
    // lane l brings word l / 32 of the tile's two for row l % 32
    bits = a.bits + s.b * a.mb + s.h * a.mh + hf * a.mw + (a.mi ? min((int64_t)i, a.mw - 1) : 0);
    t_mask = 0;
  }
  float* mine = by_distance + wave * R;
  if (biased) {
    for (int x = tid; x < R; x += TR_THREADS) bl[x] = a.bias[(int64_t)s.h * R + x];
    __syncthreads();   // (the tiles' barriers wait for no stores to LDS)
  }

  v16f dq[G::NDB];
  // the bias' gradient: the lane's sums of ds (of any rows of the wave's) and p (of its own row) over the keys at distance -reach and
  // farther behind, reach and farther ahead, and its row's sum of ds over all keys
  float flo = 0.0f, fhi = 0.0f, plo = 0.0f, phi = 0.0f, frow = 0.0f;

  const TrBlocks blocks = EX ? tr_key_blocks(a, s) : TrBlocks();
  auto issue = [&](int t, int slot) {
    lk.issue(kp, a.ks, t * TR_ROWS, s.k_len, smem[slot][0], wave, lane);
    lv.issue(vp, a.vs, t * TR_ROWS, s.k_len, smem[slot][1], wave, lane);
    if (EX && bits) tr_copy4(bits + (int64_t)(2 * t) * a.mw, wl[slot][wave]);
  };
  auto tile = [&](int t, int slot, auto masked_) {
    constexpr bool masked = decltype(masked_)::value;
    const TrAddr<D> kt = at.in(smem[slot][0]), vt = at.in(smem[slot][1]);
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
        if (EX && bits) w = wl[slot][wave][32 * kb + ln];
        const int room = lim - key0 - 4 * hf;
        w >>= 4 * hf;
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int r = 8 * (v >> 2) + (v & 3);
          if (r > room || !((w >> r) & 1u)) x[v] = 0.0f, dp[v] = 0.0f;
        }
      }
      if (want_part) {
        float all = 0.0f, ps = 0.0f;
        if (near && D < 256) {
          // Sums along the block's diagonals: 16 queries at a time go through LDS, from where lane c of a half wave takes key
          // (q + c) % 32 of query q, of 8 queries each: distance c where that is q + c, c - 32 where it began anew.
          float* y = diag + wave * 16 * 32;
          float s0 = 0.0f, s1 = 0.0f;
          int c = ln + 8 * hf;
          asm volatile("" : "+v"(c));            // (16 addresses are not to be kept for all tiles)
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            if ((ln >> 4) == part) {
#pragma unroll
              for (int g = 0; g < 4; ++g)
                *reinterpret_cast<v4f*>(y + (ln & 15) * 32 + (((2 * g + hf) ^ (ln & 7)) << 2)) =
                    v4f{x[4 * g] * dp[4 * g], x[4 * g + 1] * dp[4 * g + 1], x[4 * g + 2] * dp[4 * g + 2], x[4 * g + 3] * dp[4 * g + 3]};
            }
            asm volatile("" ::: "memory");       // (a wave's LDS accesses stay in order)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int r = c + 16 * part + k;
              const float z = y[8 * 32 * hf + 32 * k + ((r & 31) ^ (k << 2))];
              s0 += r < 32 ? z : 0.0f;
              s1 += r < 32 ? 0.0f : z;
            }
            asm volatile("" ::: "memory");       // (a wave's LDS accesses stay in order)
          }
          s0 = add_xor32_f32(s0), s1 = add_xor32_f32(s1);
          const float z = hf ? s1 : s0;
          const int d = key0 - (w0 + off) + ln - 32 * hf;
          if (d <= -a.reach) flo += z;
          else if (d >= a.reach) fhi += z;
          else mine[a.reach + d] += z;
#pragma unroll
          for (int v = 0; v < 16; ++v) frow = __builtin_fmaf(x[v], dp[v], frow);
          if (wlo <= -a.reach || whi >= a.reach) {
#pragma unroll
            for (int v = 0; v < 16; ++v) {
              const int e = d0 + 8 * (v >> 2) + (v & 3);
              plo += e <= -a.reach ? x[v] : 0.0f;
              phi += e >= a.reach ? x[v] : 0.0f;
            }
          }
        } else if (near) {
          // Every lane of a half wave has a distance of its own, so one half at a time adds without conflicts and in one order.
          // (256 channels leave no LDS for a block.)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int d = d0 + 8 * (v >> 2) + (v & 3);
            const float y = x[v] * dp[v];
            frow += y;
            if (d <= -a.reach) flo += y, plo += x[v];
            else if (d >= a.reach) fhi += y, phi += x[v];
            else {
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
          frow += all;
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
      flo = fhi = plo = phi = frow = 0.0f;
      for (int x = lane; x < R; x += 64) mine[x] = 0.0f;
    }
    int t = EX ? blocks.next(-1, ntiles) : 0, slot = 0, tn = 0;
    if (t < ntiles) issue(t, 0);
    auto next = [&]() {   // tile t has arrived, the one before is read: the one after goes there
      wait_vmcnt<0>();
      tile_barrier();
      tn = EX ? blocks.next(t, ntiles) : t + 1;
      if (tn < ntiles) issue(tn, slot ^ 1);
    };
    for (; t < t_mask; t = tn, slot ^= 1) {
      next();
      tile(t, slot, std::false_type{});
    }
    for (; t < ntiles; t = tn, slot ^= 1) {
      next();
      if (pass) {
        tr_clean<D, DT>(smem[slot][0], nullptr, tid);
        tr_clean<D, DT>(smem[slot][1], nullptr, tid);
        __syncthreads();
      }
      if (t < t_end) tile(t, slot, std::true_type{});
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
    // The row sums of ds are 0, but D holds the rounding of o's weights to 16 bits: sum_j ds = D' - D, exactly the error of D.  In a
    // far bucket, which holds most of a long row's weight, it would not average out: it is taken from there.
    const float delta = add_xor32_f32(frow);
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
    bias_sum_buckets<TR_THREADS>(map, by_distance, -a.reach, R, part, -ex);
  }
}

template <int D, int DT> int train_bwd_launch(const TrainArgs& a, const BiasMap& m, hipStream_t st) {
  const int B = a.cu_q ? 1 : a.B;
  const unsigned rows = (unsigned)((int64_t)B * a.H * a.q_tiles);
  int norm_blocks = 0;
  if (DT == DT_F16) {
    train_norms_zero<<<1, 64, 0, st>>>(a.norms);
    const int64_t len = a.cu_q ? (int64_t)a.k_tiles * TR_COLS : a.Skv;
    const int64_t need = (B * a.Hkv * len * (D == 96 ? 16 : D / 8) + TR_THREADS - 1) / TR_THREADS;
    norm_blocks = (int)(need < 1024 ? need : 1024);
  }
  train_prep<D, DT><<<rows + norm_blocks, TR_THREADS, 0, st>>>(a, (int)rows, norm_blocks);
  if (a.dk)
    if (int rc = train_dkv_launch<D, DT>(a, st)) return rc;
  if (!a.dq) return check_launch("train_prep");
  if (a.bits || a.bias) {
    const unsigned R = 2u * a.reach + 1u, lds = a.bias ? 4u * (R + (a.bias_part ? (D < 256 ? 4u * 16u * 32u : 0u) + 4u * R : 0u)) : 0u;
    train_dq<D, DT, true><<<rows, TR_THREADS, lds, st>>>(a, m);
  } else {
    train_dq<D, DT, false><<<rows, TR_THREADS, 0, st>>>(a, m);
  }
  return check_launch("train_bwd");
}

#define SAGE_BWD(D) template int train_bwd_launch<D, DT_BF16>(const TrainArgs&, const BiasMap&, hipStream_t); \
                    template int train_bwd_launch<D, DT_F16>(const TrainArgs&, const BiasMap&, hipStream_t);
SAGE_BWD(64) SAGE_BWD(96) SAGE_BWD(128) SAGE_BWD(256)

}  // namespace sage
