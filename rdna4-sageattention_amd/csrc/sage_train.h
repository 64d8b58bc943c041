// Attention on 16-bit inputs for training: what its forward and backward kernels share.
//
// x_ij = (q_i . k_j) * sm_scale + bias(j - i), hidden pairs at -inf; lse_i = ln sum_j e^x_ij; p_ij = e^(x_ij - lse_i);
// o_i = sum_j p_ij v_j.  Backward: D_i = do_i . o_i; ds_ij = p_ij (do_i . v_j - D_i); dv_j = sum_i p_ij do_i;
// dq_i = sm_scale sum_j ds_ij k_j; dk_j = sm_scale sum_i ds_ij q_i.  All sums, statistics and scores in fp32; p and ds are
// rounded to the inputs' 16 bits where they become an operand of the next product.
//
// One form serves the three kernels.  A wave owns 32 columns (queries in the forward and dq kernels, keys in the dk / dv
// kernel), one per lane of a half wave, their operands in registers, and the workgroup streams 64-row tiles of the other side
// through LDS.  v_mfma_f32_32x32x16 with A = 32 rows x 16 channels of the tile and B = the columns gives the accumulator in
// which lane l holds column l % 32 and, in register v, row 8 (v / 4) + 4 (l / 32) + v % 4 of the block: row statistics of a
// query are per lane there.  The second product of each score tile (p v, ds k, p^T do, ds^T q) sums over the tile's rows, and a
// sum may take its terms in any order: registers 8 s .. 8 s + 7 of the scores, rounded, are already its B operand for the 16
// rows 16 s .. 16 s + 15, when the A operand (the tile, transposed) takes the rows in that order too.  The transposed operand
// comes from the same LDS tile by ds_read_b64_tr_b16: of four rows x 16 channels that a group of 16 lanes addresses, lane i gets
// channel i's four rows.  No score goes through LDS and nothing is transposed in memory.
#pragma once

#include <type_traits>
#include <utility>

#include "sage_bias.h"
#include "sage_common.h"
#include "sage_host.h"

namespace sage {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr int TR_COLS = 128;     // columns per workgroup, 4 waves x 32
constexpr int TR_ROWS = 64;      // rows per streamed tile
constexpr int TR_THREADS = 256;
constexpr float TR_LOG2E = 1.4426950408889634f;
// Smallest sm_scale with a backward pass, which takes -lse / sm_scale as a score: below 2^128 for every |lse| below 2^28.
constexpr float TR_LEAST_SCALE = 0x1p-100f;

// Arguments of the three kernels and the preparation.  Strides in elements: b (batch), s (token), h (head).
struct TrainArgs {
  const uint16_t *q, *k, *v, *o, *dout;
  uint16_t *out, *dq, *dk, *dv;
  int64_t qb, qs, qh, kb, ks, kh, vb, vs, vh, ob, os, oh, gb, gs, gh;   // o and out: o*, dout: g*
  int64_t dqb, dqs, dqh, dkb, dks, dkh, dvb, dvs, dvh;
  int B, H, Hkv, Sq, Skv;          // packed: B sequences, Sq / Skv the totals of tokens
  int q_tiles, k_tiles;            // 128-column tiles of a batch entry (packed: of the whole batch, an upper bound)
  int causal;                      // bottom-right: query i of a sequence sees keys j <= i + (kv_len - q_len)
  float scale, c;                  // sm_scale, sm_scale * log2(e)
  float* lse;                      // fp32 [B, H, Sq] (packed [H, Sq]), natural log
  // what the rounding of out to 16 bits took away, in 16 bits, [B, H, Sq, D] (packed [H, Sq, D]); NULL where no backward pass comes.
  // D_i is the sum of do_i . o_i, whose terms' roundings would be the largest part of ds' error in rows of few keys.
  uint16_t* lo;
  // backward: -lse / sm_scale and -D of every row, where the sums of the scores and of dout . v begin; -inf and 0 in the padding: rows
  // of `pad` entries per (b, h) (packed: per h, sequence s at floor(cu_q[s] / 64) * 64 + 64 s)
  float *nl, *nd;
  int64_t pad;
  uint32_t* norms;                 // fp16: the largest squared norms of dout's and v's rows that take part, as bits
  // packed batches: offsets and the (sequence, tile) of each tile id, sequence -1 for none
  const int *cu_q, *cu_k;
  const int* bounds;               // the rows of q, [0] .. [1] - 1, and of k, [2] .. [3] - 1, that the sequences cover
  const int2 *q_tab, *k_tab;
  // boolean masks as bits: word w of row i holds keys 32 w ..; word w of row i at bits + b*mb + h*mh + w*mw + i*mi
  const uint32_t* bits;
  int64_t mb, mh, mw, mi;
  // which blocks of 64 rows x 64 keys of it show anything: for each row block a bit for every key block, at any + b*ab + h*ah +
  // block*aw (64-bit words), and for each key block a bit for every row block, at any_t + ..
  const uint64_t *any, *any_t;
  int64_t ab, ah, aw, tb, th, tw;
  // fp16 with a backward pass: the keys of each key block that a row of 64 row blocks sees, at keys_seen + b*tb + h*th + block*tw + ..
  const uint64_t* keys_seen;
  // bias by distance: [H, 2 reach + 1] fp32 times log2(e); entry reach + d for key - query = d, clamped to +-reach
  const float* bias;
  int reach;
  float* bias_part;                // backward: [H][parts][buckets] sums of ds, a part for every tile of queries
  int64_t parts;
  // dk, dv: the query heads of a kv head in `split` workgroups, whose fp32 sums [split][2][B, Skv (packed: Skv)][Hkv][D] are added up
  int split;
  float* kv_part;
};

// f(0), f(1), .. f(N - 1) with constants for arguments
template <class F, int... I> __device__ __forceinline__ void tr_unrolled(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F> __device__ __forceinline__ void tr_unroll(F&& f) { tr_unrolled(f, std::make_integer_sequence<int, N>{}); }

template <int D, int ROWS_ = TR_ROWS> struct TrGeo {
  static constexpr int ROWS = ROWS_;                    // rows per tile
  static constexpr int ROWB = 2 * D;                    // bytes per LDS row
  static constexpr int KCH = D / 8;                     // 16-byte chunks per row
  static constexpr int TILE = ROWS * ROWB;              // bytes per tile
  static constexpr int LOADS = TILE / 1024 / 4;         // 1 KiB direct loads per wave and tile
  static constexpr int NK = D / 16;                     // products over the channels per 32 x 32 block
  static constexpr int NDB = D / 32;                    // 32-channel blocks
};

// Position of 16-byte chunk c in LDS row `row` (an involution).  Two kinds of reads have to spread over the 64 banks: 16 rows'
// same chunk (row operands) and 4 consecutive rows' 4 neighbouring chunks (transposed operands).
template <int D> __device__ __forceinline__ int tr_swz(int row, int c) {
  if (D == 64) return c ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3));  // (two rows per 256 bytes)
  if (D == 96) return c ^ ((row >> 2) & 3);                              // (192-byte rows turn by 64 bytes each)
  return c ^ (((row & 3) << 2) | ((row >> 2) & 3));
}

template <int DT> __device__ __forceinline__ v16f tr_mfma(v4i a, v4i b, v16f c) {
  if constexpr (DT == DT_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// two floats to 16 bits each, to nearest even, one instruction
template <int DT> __device__ __forceinline__ int tr_pack(float a, float b) {
  if constexpr (DT == DT_BF16) return __builtin_bit_cast(int, __builtin_convertvector(f32x2{a, b}, bf16x2));
  else return __builtin_bit_cast(int, __builtin_convertvector(f32x2{a, b}, f16x2));
}

// Direct loads from memory to LDS: lane l's 16 (4) bytes go to lds + 16 l (4 l).  As assembly, which has no result register: behind
// the builtin the compiler, which cannot tell tiles apart, waits for every load in flight before each transposed LDS read (dk and dv
// at 1 x 24 x 4608 x 128: 636 us with such waits).  The kernels wait for their tiles themselves, by vmcnt; a wait that the
// compiler places for a load of its own counts these too, and so waits for more than it needs, never less.
__device__ __forceinline__ uint32_t tr_lds(const void* p) {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p);
}
__device__ __forceinline__ void tr_copy16(const void* g, const void* lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(tr_lds(lds)), "v"(g) : "memory", "m0");
}
__device__ __forceinline__ void tr_copy16(const void* base, uint32_t off, const void* lds) {   // base: the same in every lane
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(tr_lds(lds)), "v"(off), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void tr_copy4(const void* g, const void* lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(tr_lds(lds)), "v"(g) : "memory", "m0");
}

// A workgroup's loads of tiles of one tensor: load j of wave w fills chunks (w * LOADS + j) * 64 + lane of the tile.  Whole
// tiles: the tile's address in scalar registers and a lane's 32-bit offsets.
template <int D, int ROWS = TR_ROWS> struct TrLoader {
  using G = TrGeo<D, ROWS>;
  uint32_t off[G::LOADS];
  bool fits;               // a tile's offsets pass 32 bits otherwise
  __device__ __forceinline__ void init(int64_t stride, int wave, int lane) {
    fits = stride >= 0 && stride < (1 << 24);
#pragma unroll
    for (int j = 0; j < G::LOADS; ++j) {
      const int L = (wave * G::LOADS + j) * 64 + lane, row = L / G::KCH;
      off[j] = (uint32_t)((row * stride + tr_swz<D>(row, L % G::KCH) * 8) * 2);
    }
  }
  __device__ __forceinline__ void whole(const void* tile, uint8_t* lds, int wave) const {
#pragma unroll
    for (int j = 0; j < G::LOADS; ++j) tr_copy16(tile, off[j], lds + (wave * G::LOADS + j) * 1024);
  }
  // rows row0 .. of a sequence of `len` (>= 1) rows; rows behind it repeat its last one
  __device__ __forceinline__ void part(const uint16_t* base, int64_t stride, int row0, int len, uint8_t* lds, int wave, int lane) const {
#pragma unroll 1
    for (int j = 0; j < G::LOADS; ++j) {
      const int L = (wave * G::LOADS + j) * 64 + lane, row = L / G::KCH;
      tr_copy16(base + min(row0 + row, len - 1) * stride + tr_swz<D>(row, L % G::KCH) * 8, lds + (wave * G::LOADS + j) * 1024);
    }
  }
  __device__ __forceinline__ void issue(const uint16_t* base, int64_t stride, int row0, int len, uint8_t* lds, int wave, int lane) const {
    if (row0 + ROWS <= len && fits) whole(base + row0 * stride, lds, wave);
    else part(base, stride, row0, len, lds, wave, lane);
  }
};

// Byte offsets of a lane's operands in a tile.  Row operands: row l % 32 (a block of 32 rows adds 32 * ROWB), chunk 2 i + half.
// Transposed operands: rows 16 s + 8 e + 4 half + (l % 16) / 4, channels 32 db + 16 ((l / 16) % 2) + 4 (l % 4) ..; s adds
// 16 * ROWB.  The swizzle is an exclusive or, so the operands of i and of db follow from the first one's offset by one (head dim
// 96, whose swizzle leaves the chunk's upper bits alone, by an addition where those are concerned).
template <int D> struct TrAddr {
  using G = TrGeo<D>;
  int row, col[2];
  __device__ __forceinline__ void init(int lane) {
    const int ln = lane & 31, hf = lane >> 5, r = (lane & 15) >> 2, c = lane & 3, g = (lane >> 4) & 1;
    row = ln * G::ROWB + tr_swz<D>(ln, hf) * 16;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int rw = 8 * e + 4 * hf + r;
      col[e] = rw * G::ROWB + tr_swz<D>(rw, 2 * g + (c >> 1)) * 16 + (c & 1) * 8;
    }
  }
  // the same in the tile at `lds` (a multiple of 1 KiB, above every bit that the swizzles touch)
  __device__ __forceinline__ TrAddr in(const uint8_t* lds) const {
    const int base = (int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)lds;
    TrAddr r;
    r.row = row + base;
    r.col[0] = col[0] + base;
    r.col[1] = col[1] + base;
    return r;
  }
  // (more: bytes to another tile)
  __device__ __forceinline__ v4i rows(int blk, int i, int more = 0) const {
    const int at = D == 96 ? (row ^ ((i & 1) * 32)) + (i >> 1) * 64 : row ^ (32 * i);
    return *(__attribute__((address_space(3))) const v4i*)(uintptr_t)(uint32_t)(at + blk * 32 * G::ROWB + more);
  }
  __device__ __forceinline__ v4i cols(int s, int db, int more = 0) const {
    v4i r;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int at = D == 96 ? col[e] + 64 * db : col[e] ^ (64 * db);
      const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(uintptr_t)(uint32_t)(at + s * 16 * G::ROWB + more));
      const v2i y = __builtin_bit_cast(v2i, x);
      r[2 * e] = y[0];
      r[2 * e + 1] = y[1];
    }
    return r;
  }
};

// The operands that a wave keeps have arrived from here on (so that no wait for them lands in a loop, where it would be one for the
// tiles on their way)
template <int N> __device__ __forceinline__ void tr_arrived(v4i (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// Channels 32 db .. of column l % 32, held as acc registers (row 8 (v / 4) + 4 half + v % 4 = channel), times f, to 16 bits at p:
// one exchange between the halves makes 16-byte stores.
template <int DT> __device__ __forceinline__ void tr_store(const v16f& acc, float f, uint16_t* p, int hf, bool on) {
#pragma unroll
  for (int gp = 0; gp < 2; ++gp) {
    v4i w;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int lo = tr_pack<DT>(acc[8 * gp + 2 * e] * f, acc[8 * gp + 2 * e + 1] * f);
      const int hi = tr_pack<DT>(acc[8 * gp + 4 + 2 * e] * f, acc[8 * gp + 4 + 2 * e + 1] * f);
      const auto r = __builtin_amdgcn_permlane32_swap((unsigned)lo, (unsigned)hi, false, false);
      w[e] = (int)r[0];
      w[2 + e] = (int)r[1];
    }
    if (on) *reinterpret_cast<v4i*>(p + 16 * gp + 8 * hf) = w;
  }
}

// The same in 32 bits
__device__ __forceinline__ void tr_store_f32(const v16f& acc, float f, float* p, int hf, bool on) {
#pragma unroll
  for (int g = 0; g < 4; ++g)
    if (on) *reinterpret_cast<v4f*>(p + 8 * g + 4 * hf) = v4f{acc[4 * g] * f, acc[4 * g + 1] * f, acc[4 * g + 2] * f, acc[4 * g + 3] * f};
}

// Blocks of a mask, by the words of two neighbouring blocks that a workgroup's columns are in (m0 NULL: no mask).
struct TrBlocks {
  const uint64_t *m0 = nullptr, *m1 = nullptr;
  __device__ __forceinline__ uint64_t word(int i) const { return m0[i] | m1[i]; }
  // the first block behind t that shows anything, `end` where none before it does
  __device__ __forceinline__ int next(int t, int end) const {
    if (++t >= end || !m0) return min(t, end);
    for (;;) {
      const uint64_t w = word(t >> 6) >> (t & 63);
      if (w) return min(t + __builtin_ctzll(w), end);
      t = (t | 63) + 1;
      if (t >= end) return end;
    }
  }
  // The same backwards for tiles of 64 >> S rows: the last one before t, t0 - 1 where there is none
  template <int S> __device__ __forceinline__ int prev(int t, int t0) const {
    if (--t < t0 || !m0) return max(t, t0 - 1);
    for (;;) {
      const int b = t >> S;
      const uint64_t w = word(b >> 6) << (63 - (b & 63));
      if (w) {
        const int skip = __builtin_clzll(w);
        if (skip) t = ((b - skip) << S) + (1 << S) - 1;
        return max(t, t0 - 1);
      }
      t = ((b & ~63) << S) - 1;
      if (t < t0) return t0 - 1;
    }
  }
  // how many tiles t0 .. t1 - 1 of 64 >> S rows show anything
  template <int S> __device__ __forceinline__ int count(int t0, int t1) const {
    if (t1 <= t0) return 0;
    if (!m0) return t1 - t0;
    const int b0 = t0 >> S, b1 = (t1 - 1) >> S;
    int n = 0;
    for (int i = b0 >> 6; i <= b1 >> 6; ++i) {
      uint64_t w = word(i);
      if (i == b0 >> 6) w &= ~0ull << (b0 & 63);
      if (i == b1 >> 6) w &= ~0ull >> (63 - (b1 & 63));
      n += __builtin_popcountll(w);
    }
    n <<= S;
    if (S) {   // halves of blocks that lie outside
      if (t0 & 1) n -= (int)(word(b0 >> 6) >> (b0 & 63) & 1);
      if (t1 & 1) n -= (int)(word(b1 >> 6) >> (b1 & 63) & 1);
    }
    return n;
  }
};

// What a workgroup works on: a 128-column tile of one head of one sequence.
struct TrSeq {
  int b, h;                // batch entry (packed: sequence) and head
  int c0;                  // first column of the tile in the sequence
  int q_len, k_len;
  int64_t qr, kr;          // first row of the sequence in q and k (packed), 0 otherwise
  int64_t lr;              // its row 0 in nl / nd
  int part;                // the tile's number among all of a head
  int h0, hn, z;           // keys: the query heads that the workgroup takes, and which of the `split` workgroups it is
};

// The tile of workgroup `id`; false where there is none.  keys: column tiles of keys (heads are kv heads).  Heads of one batch
// entry that share the streamed side follow each other on one XCD; causal launches take long tiles first, over all pairs (in turn over
// the XCDs where the pairs do not divide over them: dq at 3 x 10 x 1777 x 2049 x 96 53 us, 56 with each XCD's pairs to itself).
template <bool KEYS> __device__ __forceinline__ bool tr_tile(const TrainArgs& a, int id, TrSeq& s) {
  const int heads = KEYS ? a.Hkv * a.split : a.H, tiles = KEYS ? a.k_tiles : a.q_tiles;
  const int pairs = a.cu_q ? heads : a.B * heads;
  int bh, t;
  if (a.causal || (KEYS && a.cu_q)) {
    if (pairs % 8) bh = id % pairs, t = tiles - 1 - id / pairs;
    else causal_tile(id, pairs, tiles, bh, t);
    if (KEYS) t = tiles - 1 - t;   // (the first keys are seen by the most queries; packed: train_order's order)
  } else {
    const int lg = xcd_remap(id, pairs * tiles);
    bh = lg / tiles;
    t = lg % tiles;
  }
  s.part = a.cu_q ? t : bh / heads * tiles + t;
  s.h = a.cu_q ? bh : bh % heads;
  if (KEYS) {
    s.z = s.h % a.split;
    s.h /= a.split;
    s.hn = a.H / a.Hkv / a.split;
    s.h0 = (s.h * a.split + s.z) * s.hn;
  }
  if (a.cu_q) {
    const int2 e = (KEYS ? a.k_tab : a.q_tab)[t];
    if (e.x < 0) return false;
    s.b = e.x;
    s.c0 = e.y * TR_COLS;
    const int q0 = a.cu_q[e.x], k0 = a.cu_k[e.x];
    s.q_len = a.cu_q[e.x + 1] - q0;
    s.k_len = a.cu_k[e.x + 1] - k0;
    s.qr = q0;
    s.kr = k0;
    s.lr = q0 / 64 * 64 + (int64_t)64 * e.x;
  } else {
    s.b = bh / heads;
    s.c0 = t * TR_COLS;
    s.q_len = a.Sq;
    s.k_len = a.Skv;
    s.qr = s.kr = 0;
    s.lr = 0;
  }
  return true;
}

// The blocks that a column tile's queries see / a column tile's keys are seen by
__device__ __forceinline__ TrBlocks tr_key_blocks(const TrainArgs& a, const TrSeq& s) {
  TrBlocks r;
  if (!a.bits) return r;
  r.m0 = r.m1 = a.any + s.b * a.ab + s.h * a.ah + (a.mi ? s.c0 / 64 * a.aw : 0);
  if (a.mi && s.c0 + 64 < s.q_len) r.m1 += a.aw;
  return r;
}
__device__ __forceinline__ TrBlocks tr_row_blocks(const TrainArgs& a, const TrSeq& s, int h, bool& none) {
  TrBlocks r;
  none = false;
  if (!a.bits) return r;
  r.m0 = r.m1 = a.any_t + s.b * a.tb + h * a.th + s.c0 / 64 * a.tw;
  if (s.c0 + 64 < s.k_len) r.m1 += a.tw;
  if (!a.mi) {   // the same for every row
    none = r.word(0) == 0;
    r.m0 = r.m1 = nullptr;
  }
  return r;
}

// The tiles of a head's queries that see a key tile: from the last one before `end` to first
struct TrRows {
  TrBlocks m;
  int first;
};
__device__ __forceinline__ TrRows tr_rows(const TrainArgs& a, const TrSeq& s, int h, int first, int end) {
  bool none;
  TrRows r;
  r.m = tr_row_blocks(a, s, h, none);
  r.first = none ? end : first;
  return r;
}
// How many tiles a workgroup of keys walks, over the heads that share them
template <int S> __device__ __forceinline__ int tr_steps(const TrainArgs& a, const TrSeq& s, int group, int first, int end) {
  if (!a.bits) return (end - first) * group;
  int n = 0;
  for (int g = 0; g < group; ++g) {
    const TrRows r = tr_rows(a, s, s.h0 + g, first, end);
    n += r.m.template count<S>(r.first, end);
  }
  return n;
}
// A walk over them: tile t of head g
template <int S, bool MASKS> struct TrWalk {
  int g, t;
  TrRows rows;
  __device__ __forceinline__ void head(const TrainArgs& a, const TrSeq& s, int group, int first, int end) {
    if constexpr (MASKS) rows = tr_rows(a, s, s.h0 + g, first, end);
    else rows.first = first;
    t = MASKS ? rows.m.template prev<S>(end, rows.first) : end - 1;
  }
  // to the next tile; the number of heads that were passed (the last one's end: t stays below its first)
  __device__ __forceinline__ int advance(const TrainArgs& a, const TrSeq& s, int group, int first, int end) {
    t = MASKS ? rows.m.template prev<S>(t, rows.first) : t - 1;
    int passed = 0;
    while (t < rows.first && g + 1 < group) ++g, ++passed, head(a, s, group, first, end);
    return passed;
  }
  __device__ __forceinline__ int start(const TrainArgs& a, const TrSeq& s, int group, int first, int end) {
    g = 0;
    head(a, s, group, first, end);
    int passed = 0;
    while (t < rows.first && g + 1 < group) ++g, ++passed, head(a, s, group, first, end);
    return passed;
  }
};

// Row `r` of the workgroup's sums for dk (which 0) or dv (1) among those that are added up
template <int D> __device__ __forceinline__ float* tr_kv_part(const TrainArgs& a, const TrSeq& s, int which, int r) {
  const int64_t rows = (int64_t)(a.cu_q ? 1 : a.B) * a.Skv, row = a.cu_q ? s.kr + r : (int64_t)s.b * a.Skv + r;
  return a.kv_part + (((2 * s.z + which) * rows + row) * a.Hkv + s.h) * D;
}

__device__ __forceinline__ int64_t tr_stat_row(const TrainArgs& a, const TrSeq& s, int h) {
  return a.cu_q ? h * a.pad + s.lr : ((int64_t)s.b * a.H + h) * a.pad;
}

// Largest distance of a bias inside the kernels: it and four waves' sums by distance have to fit the LDS that tiles of 256
// channels leave.
constexpr int TR_REACH = 760;

// Hidden pairs and the bias of one 32 x 32 block of scores whose columns are queries: register v of lane l is key
// key0 + 8 (v / 4) + 4 (l / 32) + v % 4.  Values at the keys of `bits` (the word of the lane's query and these 32 keys) that are 0,
// and behind `lim`, become -inf.
__device__ __forceinline__ void tr_hide_keys(v16f& x, int key0, int lim, uint32_t bits, int hf) {
  const int room = lim - key0 - 4 * hf;
  const uint32_t w = bits >> (4 * hf);
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const int r = 8 * (v >> 2) + (v & 3);
    if (r > room || !((w >> r) & 1u)) x[v] = -INFINITY;
  }
}

// Whether a wave's 16-bit vector of finite sums is finite: 0 or NaN
template <int N> __device__ __forceinline__ float tr_nonfinite(const v16f (&a)[N]) {
  float t = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int v = 0; v < 16; ++v) t = __builtin_fmaf(a[i][v], 0.0f, t);
  return t;
}

// Whether any of a lane's 16-bit operands is an infinity or a NaN
template <int DT, int N> __device__ __forceinline__ bool tr_nonfinite_operand(const v4i (&f)[N]) {
  constexpr uint32_t E = DT == DT_BF16 ? 0x7F80u : 0x7C00u;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) bad |= ((uint32_t)f[i][e] & E) == E || ((uint32_t)f[i][e] & (E << 16)) == (E << 16);
  return bad;
}

// The infinities and NaN of a tile become 0; poison[r] is set where row r had one.  A hidden pair has weight 0, but 0 times an
// infinity is NaN: results that come out non-finite are computed a second time from tiles cleaned like this, in which the rows
// that see a poisoned one get NaN by their scores.  Two barriers are the caller's.
template <int D, int DT, int ROWS = TR_ROWS, int THREADS = TR_THREADS> __device__ __forceinline__ void tr_clean(uint8_t* tile, int* poison, int tid) {
  using G = TrGeo<D, ROWS>;
  constexpr uint32_t E = DT == DT_BF16 ? 0x7F80u : 0x7C00u;
  for (int i = tid; i < G::TILE / 16; i += THREADS) {
    v4i* p = reinterpret_cast<v4i*>(tile) + i;
    v4i w = *p;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t u = (uint32_t)w[e];
      if ((u & E) == E) u &= 0xFFFF0000u, bad = true;
      if ((u & (E << 16)) == (E << 16)) u &= 0x0000FFFFu, bad = true;
      w[e] = (int)u;
    }
    if (bad) {
      *p = w;
      if (poison) poison[i / G::KCH] = 1;
    }
  }
}

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

template <int D, int DT> int train_fwd_launch(const TrainArgs& a, hipStream_t st);
template <int D, int DT> int train_bwd_launch(const TrainArgs& a, const BiasMap& m, hipStream_t st);
template <int D, int DT> int train_dkv_launch(const TrainArgs& a, hipStream_t st);

}  // namespace sage
