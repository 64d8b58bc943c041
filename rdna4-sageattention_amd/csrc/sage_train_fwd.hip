// Forward pass of the attention for training: see sage_train.h for the form.
//
// A wave per 32 queries, four in a workgroup, streams its keys once with a running reference and sum per row (online softmax); the
// weights go from the score registers straight into the second product.  Two workgroups per unit, so that one wave's exponentials
// run beside the other's products: 283 us at 1 x 24 x 4608 x 128 bf16 (0.92 PFLOP/s; the matrix unit busy for 50% of it, 17% of
// the places empty while the last of 864 workgroups run) and 1050 at 2 x 32 x 8192 x 128 causal (1.05 PFLOP/s).  What bounds it is
// the issue of both: 32 products and some 165 vector instructions a tile of 64 keys and wave, 16 of which look for scores of -inf
// (276, 1040, at 256 channels 196 for 202 and with a bias at 64 35 for 39 us without).  One stream of products, scores a tile
// ahead of the weights' products and the exponentials in slices beside them: 286 for 278 and 1100 us then, 186 for 197 at 256
// channels, 41 for 35 with a bias at 64; higher wave priority around the products: within 1%, 228 for 196 us at 256 channels.
#include "sage_train.h"

namespace sage {

// P is rounded to 16 bits for its product with V.  fp16: weights are taken times 2^6 against a running reference that trails the
// maximum by at most 2^8, so they stay below 2^15 and keep full precision down to 2^-20 of the reference.
template <int DT> constexpr float FWD_SHIFT = DT == DT_F16 ? 6.0f : 0.0f;
constexpr float FWD_LAG = 8.0f;

template <int D, int DT, bool EX>
__global__ __launch_bounds__(TR_THREADS, D == 256 ? 1 : 2) void train_fwd(TrainArgs a) {
  using G = TrGeo<D>;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[2][2][G::TILE];
  __shared__ float bl[EX ? 2 * TR_REACH + 1 : 1];
  __shared__ __attribute__((aligned(256))) uint32_t wl[2][4][EX ? 64 : 1];   // a mask's words of the tiles, for each wave's queries
  __shared__ int poison[TR_ROWS];

  TrSeq s;
  if (!tr_tile<false>(a, blockIdx.x, s)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int ln = lane & 31, hf = lane >> 5;
  const int hk = s.h / (a.H / a.Hkv);
  const int off = s.k_len - s.q_len;
  const int w0 = s.c0 + wave * 32, i = w0 + ln;   // the wave's first query, the lane's
  const bool on = i < s.q_len;
  const int ir = on ? i : s.q_len - 1;

  const uint16_t* kp = a.k + s.b * (a.cu_q ? 0 : a.kb) + s.kr * a.ks + hk * a.kh;
  const uint16_t* vp = a.v + s.b * (a.cu_q ? 0 : a.vb) + s.kr * a.vs + hk * a.vh;

  v4i qf[G::NK];
  {
    const uint16_t* p = a.q + s.b * (a.cu_q ? 0 : a.qb) + (s.qr + ir) * a.qs + s.h * a.qh + 8 * hf;
#pragma unroll
    for (int x = 0; x < G::NK; ++x) qf[x] = *reinterpret_cast<const v4i*>(p + 16 * x);
  }
  TrLoader<D> lk, lv;
  lk.init(a.ks, wave, lane);
  lv.init(a.vs, wave, lane);
  TrAddr<D> at;
  at.init(lane);

  int kv_end = s.k_len;
  if (a.causal) kv_end = min(kv_end, min(s.c0 + TR_COLS, s.q_len) + off);
  const int ntiles = kv_end > 0 ? (kv_end + TR_ROWS - 1) / TR_ROWS : 0;
  const int lim = a.causal ? min(s.k_len - 1, ir + off) : s.k_len - 1;           // the lane's last visible key
  // tiles before t_mask show every key to every query of the wave, from t_end on none
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
  const bool biased = EX && a.bias;
  if (biased) {
    for (int x = tid; x <= 2 * a.reach; x += TR_THREADS) bl[x] = a.bias[(int64_t)s.h * (2 * a.reach + 1) + x];
    __syncthreads();   // (the tiles' barriers wait for no stores to LDS)
  }

  float m = -INFINITY, negm = FWD_SHIFT<DT>, l = 0.0f;
  // A score of -inf has weight 0 as a hidden one does, and leaves the sums finite.  The smallest score before bias and mask tells that
  // there may be one (as the largest of the bits, one instruction for two scores: floats' minimum takes three), and the second pass
  // whose it is: an infinite query's or key's, whose rows are NaN, or an overflow.
  uint32_t low = 0;
  bool qbad = false, sees = lim >= 0;   // the lane's query is non-finite (known in the second pass); it sees a key
  v16f o[G::NDB];
  const TrBlocks blocks = EX ? tr_key_blocks(a, s) : TrBlocks();
  auto issue = [&](int t, int slot) {
    lk.issue(kp, a.ks, t * TR_ROWS, s.k_len, smem[slot][0], wave, lane);
    lv.issue(vp, a.vs, t * TR_ROWS, s.k_len, smem[slot][1], wave, lane);
    if (EX && bits) tr_copy4(bits + (int64_t)(2 * t) * a.mw, wl[slot][wave]);
  };

  auto tile = [&](int t, int slot, auto masked_, bool slow) {
    constexpr bool masked = decltype(masked_)::value;
    const TrAddr<D> kt = at.in(smem[slot][0]), vt = at.in(smem[slot][1]);
    v16f x[2] = {};
#pragma unroll
    for (int kk = 0; kk < G::NK; ++kk) {
      x[0] = tr_mfma<DT>(kt.rows(0, kk), qf[kk], x[0]);
      x[1] = tr_mfma<DT>(kt.rows(1, kk), qf[kk], x[1]);
    }
    if (masked && slow) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (qbad || poison[32 * kb + 8 * (v >> 2) + 4 * hf + (v & 3)]) x[kb][v] = NAN;
    }
    if (EX || masked) {   // (elsewhere beside the exponentials: at 256 channels the scores would be moved about, 915 for 870 us a step)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int v = 0; v < 16; ++v) low = max(low, __float_as_uint(x[kb][v]));
    }
    if (EX) {
      // scores in the log2 domain, with the bias
      const int d0 = t * TR_ROWS + 4 * hf - (ir + off);
      const int wlo = t * TR_ROWS - (min(w0 + 31, s.q_len - 1) + off), whi = t * TR_ROWS + TR_ROWS - 1 - (w0 + off);
      if (biased && !(whi <= -a.reach || wlo >= a.reach)) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int v = 0; v < 16; ++v) {
            const int d = min(max(d0 + 32 * kb + 8 * (v >> 2) + (v & 3), -a.reach), a.reach);
            x[kb][v] = __builtin_fmaf(x[kb][v], a.c, bl[a.reach + d]);
          }
      } else {
        const float far = biased ? bl[whi <= -a.reach ? 0 : 2 * a.reach] : 0.0f;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int v = 0; v < 16; ++v) x[kb][v] = __builtin_fmaf(x[kb][v], a.c, far);
      }
    }
    if (masked) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int key0 = t * TR_ROWS + 32 * kb;
        uint32_t w = ~0u;
        if (EX && bits) {
          w = wl[slot][wave][32 * kb + ln];
          sees |= key0 <= lim && (w << max(0, 31 - (lim - key0))) != 0;
        }
        tr_hide_keys(x[kb], key0, lim, w, hf);
      }
    }
    float mx = x[0][0];
#pragma unroll
    for (int v = 1; v < 16; ++v) mx = fmaxf(mx, x[0][v]);
#pragma unroll
    for (int v = 0; v < 16; ++v) mx = fmaxf(mx, x[1][v]);
    mx = max_xor32_f32(mx);
    if (!EX) mx *= a.c;
    if (__ballot(mx > m + FWD_LAG) != 0) {
      const float m_new = mx > m + FWD_LAG ? mx : m;   // (each row by itself: its bits follow from what it sees alone)
      const float corr = m == m_new ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
      l *= corr;
#pragma unroll
      for (int db = 0; db < G::NDB; ++db)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[db][v] *= corr;
      m = m_new;
      negm = m == -INFINITY ? FWD_SHIFT<DT> : FWD_SHIFT<DT> - m;
    }
    v4i p[4];
    float ps[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int v = 0; v < 16; v += 2) {
        if (!EX && !masked) low = max(max(low, __float_as_uint(x[kb][v])), __float_as_uint(x[kb][v + 1]));
        const float e0 = __builtin_amdgcn_exp2f(EX ? x[kb][v] + negm : __builtin_fmaf(x[kb][v], a.c, negm));
        const float e1 = __builtin_amdgcn_exp2f(EX ? x[kb][v + 1] + negm : __builtin_fmaf(x[kb][v + 1], a.c, negm));
        ps[v & 2] += e0;
        ps[(v & 2) + 1] += e1;
        p[2 * kb + (v >> 3)][(v & 7) >> 1] = tr_pack<DT>(e0, e1);
      }
    l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
#pragma unroll
    for (int st = 0; st < 4; ++st)
#pragma unroll
      for (int db = 0; db < G::NDB; ++db) o[db] = tr_mfma<DT>(vt.cols(st, db), p[st], o[db]);
  };

  for (int pass = 0; pass < 2; ++pass) {
    m = -INFINITY, negm = FWD_SHIFT<DT>, l = 0.0f, low = 0;
    if (EX && bits) sees = false;
#pragma unroll
    for (int db = 0; db < G::NDB; ++db)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[db][v] = 0.0f;
    int t = EX ? blocks.next(-1, ntiles) : 0, slot = 0, tn = 0;
    if (t < ntiles) issue(t, 0);
    auto next = [&]() {   // tile t has arrived, the one before is read: the one after goes there
      wait_vmcnt<0>();
      tile_barrier();
      tn = EX ? blocks.next(t, ntiles) : t + 1;
      if (tn < ntiles) issue(tn, slot ^ 1);
    };
    // the tiles without hidden keys for the wave, in a loop of their own
    for (; t < t_mask; t = tn, slot ^= 1) {
      next();
      tile(t, slot, std::false_type{}, false);
    }
    for (; t < ntiles; t = tn, slot ^= 1) {
      next();
      if (pass) {
        if (tid < TR_ROWS) poison[tid] = 0;
        __syncthreads();
        tr_clean<D, DT>(smem[slot][0], poison, tid);
        tr_clean<D, DT>(smem[slot][1], poison, tid);
        __syncthreads();
      }
      if (t < t_end) tile(t, slot, std::true_type{}, pass != 0);
      if (pass) __syncthreads();
    }
    const bool bad = !(tr_nonfinite(o) == 0.0f) || (sees && !(__uint_as_float(low) * a.c > -INFINITY));
    if (!__syncthreads_or(on && bad)) break;
    t_mask = 0;   // every tile cleaned, hidden keys taken out
    qbad = tr_nonfinite_operand<DT>(qf);
    qbad |= __shfl_xor((int)qbad, 32) != 0;
  }

  l = add_xor32_f32(l);
  low = max(low, (uint32_t)__shfl_xor((int)low, 32));
  if (l == 0.0f && sees && !(__uint_as_float(low) * a.c > -INFINITY)) l = NAN;   // (nothing but overflows: no row that sees nothing)
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* op = a.out + s.b * (a.cu_q ? 0 : a.ob) + (s.qr + ir) * a.os + s.h * a.oh;
#pragma unroll
  for (int db = 0; db < G::NDB; ++db) tr_store<DT>(o[db], inv, op + 32 * db, hf, on);
  if (a.lo) {
    // the same channels' remainders: as many as there are, in 16 bits again
    uint16_t* lp = a.lo + ((a.cu_q ? (int64_t)s.h * a.Sq + s.qr : ((int64_t)s.b * a.H + s.h) * a.Sq) + ir) * D;
#pragma unroll
    for (int db = 0; db < G::NDB; ++db) {
#pragma unroll
      for (int v = 0; v < 16; v += 2) {
        const int w = tr_pack<DT>(o[db][v] * inv, o[db][v + 1] * inv);
        o[db][v] = __builtin_fmaf(o[db][v], inv, -elem_lo<DT>((uint32_t)w));
        o[db][v + 1] = __builtin_fmaf(o[db][v + 1], inv, -elem_hi<DT>((uint32_t)w));
      }
      tr_store<DT>(o[db], 1.0f, lp + 32 * db, hf, on);
    }
  }
  if (on && hf == 0) {
    const float lse = l == 0.0f ? -INFINITY : (m - FWD_SHIFT<DT> + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
    a.lse[(a.cu_q ? (int64_t)s.h * a.Sq + s.qr : ((int64_t)s.b * a.H + s.h) * a.Sq) + i] = lse;
  }
}

template <int D, int DT> int train_fwd_launch(const TrainArgs& a, hipStream_t st) {
  const unsigned n = (unsigned)((int64_t)(a.cu_q ? 1 : a.B) * a.H * a.q_tiles);
  if (a.bits || a.bias) train_fwd<D, DT, true><<<n, TR_THREADS, 0, st>>>(a);
  else train_fwd<D, DT, false><<<n, TR_THREADS, 0, st>>>(a);
  return check_launch("train_fwd");
}

#define SAGE_FWD(D) template int train_fwd_launch<D, DT_BF16>(const TrainArgs&, hipStream_t); \
                    template int train_fwd_launch<D, DT_F16>(const TrainArgs&, hipStream_t);
SAGE_FWD(64) SAGE_FWD(96) SAGE_FWD(128) SAGE_FWD(256)

}  // namespace sage
