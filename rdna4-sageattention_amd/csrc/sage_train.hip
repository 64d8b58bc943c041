// The attention for training: tables, masks as bits and the C entry points (kernels in sage_train_fwd.hip, sage_train_bwd.hip).
#include "sage_train.h"

namespace sage {

// Packed batches: the (sequence, tile) of every tile id, on the device.  Offsets that fall or pass the totals make no tiles at all.
// bounds: the rows of q and of k that sequences cover, [q0, q1), [k0, k1).
__global__ __launch_bounds__(TR_THREADS) void train_plan(const int* cu_q, const int* cu_k, int batch, int total_q, int total_k,
                                                         int2* q_tab, int q_tiles, int2* k_tab, int k_tiles, int* bounds) {
  __shared__ int scan[2][TR_THREADS];
  const int tid = threadIdx.x;
  int bad = 0;
  for (int x = tid; x <= batch; x += TR_THREADS) {
    bad |= cu_q[x] < 0 || cu_q[x] > total_q || cu_k[x] < 0 || cu_k[x] > total_k;
    if (x) bad |= cu_q[x] < cu_q[x - 1] || cu_k[x] < cu_k[x - 1];
  }
  bad = __syncthreads_or(bad);
  if (tid == 0) {
    bounds[0] = bad ? 0 : cu_q[0], bounds[1] = bad ? 0 : cu_q[batch];
    bounds[2] = bad ? 0 : cu_k[0], bounds[3] = bad ? 0 : cu_k[batch];
  }
  int at_q = 0, at_k = 0;
  for (int x0 = 0; x0 < batch && !bad; x0 += TR_THREADS) {
    const int x = x0 + tid;
    const int nq = x < batch ? (cu_q[x + 1] - cu_q[x] + TR_COLS - 1) / TR_COLS : 0;
    const int nk = x < batch ? (cu_k[x + 1] - cu_k[x] + TR_COLS - 1) / TR_COLS : 0;
    scan[0][tid] = nq;
    scan[1][tid] = nk;
    __syncthreads();
    for (int o = 1; o < TR_THREADS; o <<= 1) {
      const int p = tid >= o ? scan[0][tid - o] : 0, r = tid >= o ? scan[1][tid - o] : 0;
      __syncthreads();
      scan[0][tid] += p;
      scan[1][tid] += r;
      __syncthreads();
    }
    const int fq = at_q + scan[0][tid] - nq, fk = at_k + scan[1][tid] - nk;
    for (int i = 0; i < nq; ++i) q_tab[fq + i] = make_int2(x, i);
    for (int i = 0; i < nk; ++i) k_tab[fk + i] = make_int2(x, i);
    at_q += scan[0][TR_THREADS - 1];
    at_k += scan[1][TR_THREADS - 1];
    __syncthreads();
  }
  for (int i = at_q + tid; i < q_tiles; i += TR_THREADS) q_tab[i] = make_int2(-1, 0);
  for (int i = at_k + tid; i < k_tiles; i += TR_THREADS) k_tab[i] = make_int2(-1, 0);
}

// The tiles of keys from the one that the most queries see to the one that the fewest do, those of about the same number in their
// order: so the units end at about the same time, with short tiles.  One workgroup, a counting sort by 256 lengths.  (14 sequences of
// 77 to 3001, causal, 32 heads on 8 x 128: dk and dv 10% faster for the 15 us that this takes; q's tiles, four times as many
// workgroups on twice as many places, are no faster sorted.)
__global__ __launch_bounds__(TR_THREADS) void train_order(const int* cu_q, const int* cu_k, int causal, const int2* from, int2* to,
                                                          int tiles) {
  const int tid = threadIdx.x;
  __shared__ __attribute__((aligned(16))) uint8_t bin[TR_THREADS];
  __shared__ int scan[TR_THREADS], most;   // of every length: how many tiles there are, then where the next one goes
  auto length = [&](int i) -> int {        // queries; -1 where there is no tile
    const int2 e = i < tiles ? from[i] : make_int2(-1, 0);
    if (e.x < 0) return -1;
    const int c0 = e.y * TR_COLS, nq = cu_q[e.x + 1] - cu_q[e.x], nk = cu_k[e.x + 1] - cu_k[e.x];
    return causal ? nq - min(nq, max(0, c0 - (nk - nq))) : nq;
  };
  if (tid == 0) most = 1;
  scan[tid] = 0;
  __syncthreads();
  const int own = length(tid);
  int mine = own;
  for (int i = tid + TR_THREADS; i < tiles; i += TR_THREADS) mine = max(mine, length(i));
  atomicMax(&most, mine);
  __syncthreads();
  const int top = most;
  auto bin_of = [&](int i) {               // (the longest first, none at the end)
    const int n = i == tid ? own : length(i);
    return n < 0 ? 255 : 254 - (int)((int64_t)n * 254 / top);
  };
  for (int i = tid; i < tiles; i += TR_THREADS) atomicAdd(&scan[bin_of(i)], 1);
  __syncthreads();
  const int many = scan[tid];
  for (int o = 1; o < TR_THREADS; o <<= 1) {
    const int x = tid >= o ? scan[tid - o] : 0;
    __syncthreads();
    scan[tid] += x;
    __syncthreads();
  }
  const int first = scan[tid] - many;
  __syncthreads();
  scan[tid] = first;
  for (int i0 = 0; i0 < tiles; i0 += TR_THREADS) {
    const int i = i0 + tid, b = bin_of(i);
    bin[tid] = (uint8_t)b;
    __syncthreads();
    int rank = 0;                          // among the 256 tiles
    for (int x = 0; x < TR_THREADS; x += 16) {
      const v4i w = *reinterpret_cast<const v4i*>(bin + x);
#pragma unroll
      for (int y = 0; y < 16; ++y) rank += ((uint32_t)w[y >> 2] >> (8 * (y & 3)) & 255u) == (uint32_t)b && x + y < tid;
    }
    if (i < tiles) to[scan[b] + rank] = from[i];
    __syncthreads();
    if (i < tiles) atomicAdd(&scan[b], 1);
    __syncthreads();
  }
}

// Packed batches: zeros in the rows that no sequence covers, of up to three tensors [rows, heads, D].
struct TrainGaps {
  uint16_t* p[3];
  int64_t s[3], h[3];
  int heads[3], rows[3], chunks;   // 16-byte chunks per head
  int side[3];                     // 0: q's rows, 1: k's
};
__global__ __launch_bounds__(TR_THREADS) void train_gaps(TrainGaps a, const int* bounds) {
  const int z = blockIdx.y;
  if (!a.p[z]) return;
  const int b0 = bounds[2 * a.side[z]], b1 = bounds[2 * a.side[z] + 1];
  for (int r = blockIdx.x; r < a.rows[z]; r += gridDim.x) {
    if (r >= b0 && r < b1) continue;
    for (int x = threadIdx.x; x < a.heads[z] * a.chunks; x += TR_THREADS)
      *reinterpret_cast<v4i*>(a.p[z] + r * a.s[z] + x / a.chunks * a.h[z] + x % a.chunks * 8) = v4i{0, 0, 0, 0};
  }
}

__device__ __forceinline__ uint64_t wave_or(uint64_t w) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) w |= (uint64_t)__shfl_xor((unsigned long long)w, o);
  return w;
}

// Four bytes' truth as four bits: each byte's bits folded onto its lowest, and those gathered by a product
__device__ __forceinline__ uint32_t truth4(uint32_t w) {
  w |= w >> 4;
  w |= w >> 2;
  w |= w >> 1;
  return ((w & 0x01010101u) * 0x01020408u) >> 24 & 15u;
}
typedef uint32_t v4u_a1 __attribute__((ext_vector_type(4), aligned(1)));

// A boolean mask as bits, word-major: word w (keys 32 w ..) of 64 consecutive rows side by side.  A wave makes the words of 64
// keys of 64 rows: lane r reads row r's 64 bytes, or, at the last keys and where keys are not contiguous, the wave reads a byte per
// lane of row after row and lane r keeps row r's ballot.  (1250 x 1250 x 6: 25 us with the latter alone.)  seen (or NULL): a block's
// keys that one of its rows sees, of which row i, under a causal mask, those up to i + first (without: first is the last key).
__global__ __launch_bounds__(TR_THREADS) void train_mask_bits(const uint8_t* __restrict__ mask, int64_t msb, int64_t msh, int64_t msq,
                                                              int64_t msk, int heads, int rows, int row_pad, int keys, int chunks,
                                                              int blocks, int64_t units, uint32_t* __restrict__ bits,
                                                              uint8_t* __restrict__ shows, uint64_t* __restrict__ seen, int first) {
  const int lane = threadIdx.x & 63;
  const int64_t u = (int64_t)blockIdx.x * (TR_THREADS / 64) + (threadIdx.x >> 6);
  if (u >= units) return;
  const int c = (int)(u % chunks);
  const int64_t y = u / chunks;
  const int rb = (int)(y % blocks);
  const int64_t bh = y / blocks;
  const uint8_t* p = mask + bh / heads * msb + bh % heads * msh;
  const int key = c * 64 + lane;
  const bool in = key < keys;
  const int r0 = rb * 64, n = min(64, rows - r0);
  uint32_t lo = 0, hi = 0;
  if (msk == 1 && c * 64 + 64 <= keys) {
    if (lane < n) {
      const v4u_a1* q = (const v4u_a1*)(p + (r0 + lane) * msq + c * 64);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const v4u_a1 w = q[x];
        const uint32_t b = truth4(w[0]) | truth4(w[1]) << 4 | truth4(w[2]) << 8 | truth4(w[3]) << 12;
        if (x < 2) lo |= b << (16 * x);
        else hi |= b << (16 * x - 32);
      }
    }
  } else {
    p += (int64_t)(in ? key : 0) * msk;
    auto one = [&](int r) {
      const uint64_t w = __ballot(in && p[(r0 + r) * msq] != 0);
      if (lane == r) lo = (uint32_t)w, hi = (uint32_t)(w >> 32);
    };
    if (n == 64) {
#pragma unroll 16
      for (int r = 0; r < 64; ++r) one(r);
    } else {
      for (int r = 0; r < n; ++r) one(r);
    }
  }
  if (r0 + lane < row_pad) {
    uint32_t* o = bits + (bh * chunks * 2 + 2 * c) * row_pad + r0 + lane;
    o[0] = lo;
    o[row_pad] = hi;
  }
  const bool any = __ballot(lo | hi) != 0;
  if (lane == 0) shows[u] = any;   // [batch x head][block of 64 rows][block of 64 keys]
  if (seen) {
    const int64_t last = (int64_t)r0 + lane + first - c * 64;   // of the 64 keys
    uint64_t w = last < 0 ? 0 : ((uint64_t)hi << 32 | lo) & (last < 63 ? (2ull << last) - 1 : ~0ull);
    w = wave_or(w);
    if (lane == 0) seen[u] = w;
  }
}

// What blocks show, as bits both ways: a wave for 64 key blocks of a row block, or for 64 row blocks of a key block, which also
// joins what those see of its keys
__global__ __launch_bounds__(TR_THREADS) void train_mask_any(const uint8_t* __restrict__ shows, int blocks, int chunks, int aw, int tw,
                                                             int64_t units, int64_t units_t, uint64_t* __restrict__ any,
                                                             uint64_t* __restrict__ any_t, const uint64_t* __restrict__ seen,
                                                             uint64_t* __restrict__ keys_seen) {
  const int lane = threadIdx.x & 63;
  int64_t u = (int64_t)blockIdx.x * (TR_THREADS / 64) + (threadIdx.x >> 6);
  if (u < units) {
    const int w = (int)(u % aw), c = 64 * w + lane;
    const uint64_t m = __ballot(c < chunks && shows[u / aw * chunks + c] != 0);
    if (lane == 0) any[u] = m;
  } else if ((u -= units) < units_t) {
    const int w = (int)(u % tw), b = 64 * w + lane, c = (int)(u / tw % chunks);
    const int64_t bh = u / tw / chunks;
    const uint64_t m = __ballot(b < blocks && shows[(bh * blocks + b) * chunks + c] != 0);
    if (lane == 0) any_t[u] = m;
    if (seen) {
      const uint64_t k = wave_or(b < blocks ? seen[(bh * blocks + b) * chunks + c] : 0);
      if (lane == 0) keys_seen[u] = k;
    }
  }
}

// Where everything lies in the state that the forward pass leaves to the backward pass, and in its workspace.
struct TrainLayout {
  int q_tiles, k_tiles, mask_b, mask_h, row_pad, words, blocks, chunks, aw, tw;
  int64_t q_tab, k_tab, bits, shows, any, any_t, seen, keys_seen, vec, lo, state;      // byte offsets; bounds at 0
  int64_t pad, nl, nd, norms, parts, part, kv_part, k_order, work;
};

// In how many workgroups the query heads of a kv head go for dk and dv, where there are tiles of keys for half of the places at most.
// Tiles that see different numbers of queries, under causal or a mask or packed, are twice as many as places then, so that the long
// ones do not last alone.  The sums that are added up afterwards are 8 D bytes a key and workgroup.  (6 x 16 heads on 4 x 1250 x 64,
// masked, 240 tiles for 512 places: 145 us whole, 89 + 8 in two, 77 + 12 in four.  3 x 10 heads on 5 x 1777 x 2049 x 96, causal, 255
// tiles for 256 places: 85 us whole, 75 + 10 in two.)
static int train_split(bool packed, bool uneven, int B, int H, int Hkv, int k_tiles, int D) {
  const int64_t places = D == 64 ? 512 : 256, n = (int64_t)(packed ? 1 : B) * Hkv * k_tiles;   // (256 units, DkvGeo::OCC workgroups each)
  const int group = H / Hkv;
  int s = 1;
  for (int x = 2; x <= group && 2 * n <= places && n * x <= (uneven ? 2 : 1) * places; ++x)
    if (group % x == 0) s = x;
  return s;
}

static TrainLayout train_layout(bool packed, int B, int H, int Hkv, int Sq, int Skv, int D, bool mask, bool mb, bool mh, bool mq,
                                int reach, int buckets, bool keep) {   // keep: a backward pass comes
  TrainLayout l = {};
  auto take = [](int64_t& at, int64_t n) {
    const int64_t r = at;
    at += (n + 255) / 256 * 256;
    return r;
  };
  l.q_tiles = packed ? Sq / TR_COLS + B : (Sq + TR_COLS - 1) / TR_COLS;
  l.k_tiles = packed ? Skv / TR_COLS + B : (Skv + TR_COLS - 1) / TR_COLS;
  int64_t at = 0;
  if (packed) {
    take(at, 16);
    l.q_tab = take(at, (int64_t)l.q_tiles * 8);
    l.k_tab = take(at, (int64_t)l.k_tiles * 8);
  }
  if (mask) {
    l.mask_b = mb ? B : 1, l.mask_h = mh ? H : 1, l.row_pad = mq ? (Sq + 63) / 64 * 64 : 1, l.words = (Skv + 63) / 64 * 2;
    l.blocks = mq ? (Sq + 63) / 64 : 1, l.chunks = l.words / 2, l.aw = (l.chunks + 63) / 64, l.tw = (l.blocks + 63) / 64;
    const int64_t bh = (int64_t)l.mask_b * l.mask_h;
    l.bits = take(at, bh * l.row_pad * l.words * 4);
    l.shows = take(at, bh * l.blocks * l.chunks);
    l.any = take(at, bh * l.blocks * l.aw * 8);
    l.any_t = take(at, bh * l.chunks * l.tw * 8);
    l.seen = take(at, keep ? bh * l.blocks * l.chunks * 8 : 0);       // (bf16 leaves them as they are)
    l.keys_seen = take(at, keep ? bh * l.chunks * l.tw * 8 : 0);
  }
  if (reach) l.vec = take(at, (int64_t)H * (2 * reach + 1) * 4);
  if (keep) l.lo = take(at, (int64_t)(packed ? 1 : B) * H * Sq * D * 2);
  l.state = at;
  at = 0;
  l.pad = packed ? (int64_t)Sq / 64 * 64 + 64 * ((int64_t)B + 1) : ((int64_t)Sq + 63) / 64 * 64;
  const int64_t rows = l.pad * H * (packed ? 1 : B);
  l.nl = take(at, rows * 4);
  l.nd = take(at, rows * 4);
  l.norms = take(at, 8);
  l.parts = (int64_t)l.q_tiles * (packed ? 1 : B);
  l.part = take(at, reach ? l.parts * H * buckets * 4 : 0);
  const int split = train_split(packed, true, B, H, Hkv, l.k_tiles, D);
  l.kv_part = take(at, split > 1 ? (int64_t)split * 2 * (packed ? 1 : B) * Skv * Hkv * D * 4 : 0);
  l.k_order = take(at, packed ? (int64_t)l.k_tiles * 8 : 0);
  l.work = at;
  return l;
}

// A launch holds fewer than 2^32 threads, so fewer than 2^24 workgroups of 256 (dk and dv at 256 channels: 2^23 of 512), one for each
// tile and head; the preparation adds 1024.  A tensor's rows and heads then fit 31 bits.
static int train_sizes(const char* who, bool packed, int B, int H, int Hkv, int Sq, int Skv, int D, int dtype) {
  SAGE_REQUIRE(B > 0 && H > 0 && Hkv > 0 && Sq > 0 && Skv > 0, "%s: sizes must be positive", who);
  SAGE_REQUIRE(H % Hkv == 0, "%s: %d heads are no multiple of %d kv heads", who, H, Hkv);
  if (dtype != SAGE_DTYPE_BF16 && dtype != SAGE_DTYPE_F16) return fail(SAGE_ERR_UNSUPPORTED, "%s: dtype %d", who, dtype);
  if (!head_dim_ok(D)) return fail(SAGE_ERR_UNSUPPORTED, "%s: head_dim %d (supported 64, 96, 128, 256)", who, D);
  SAGE_REQUIRE(Sq <= 0x3FFFFFFF && Skv <= 0x3FFFFFFF && H <= 65535 && B <= 0xFFFFFF, "%s: too large", who);
  const int64_t rows = Sq > Skv ? Sq : Skv;
  const int64_t tiles = packed ? (rows / TR_COLS + B) * H : (rows + TR_COLS - 1) / TR_COLS * B * H;
  SAGE_REQUIRE(tiles < (D == 256 ? 1 << 23 : (1 << 24) - 1024), "%s: %lld tiles of 128 rows are too many", who, (long long)tiles);
  return SAGE_OK;
}

// (a wave for each block of 64 rows x 64 keys of a mask, and one or two for its bits)
static int train_mask_size(const char* who, const TrainLayout& l) {
  SAGE_REQUIRE((int64_t)l.mask_b * l.mask_h * l.blocks * l.chunks < 1 << 25, "%s: mask too large", who);
  return SAGE_OK;
}

struct TrainTensor { const void* p; int64_t b, s, h; const char* name; };
static int train_tensors(const char* who, const TrainTensor* t, int n) {
  for (int i = 0; i < n; ++i) {
    SAGE_REQUIRE(t[i].p, "%s: %s is NULL", who, t[i].name);
    SAGE_REQUIRE(aligned16(t[i].p) && t[i].b % 8 == 0 && t[i].s % 8 == 0 && t[i].h % 8 == 0,
                 "%s: %s must be 16-byte aligned, its strides multiples of 8 elements", who, t[i].name);
  }
  return SAGE_OK;
}

static int train_dispatch(bool bwd, const TrainArgs& a, const BiasMap& m, int D, int dtype, hipStream_t st) {
  const bool bf = dtype == SAGE_DTYPE_BF16;
#define SAGE_TRAIN(X)                                                                                                   \
  if (D == X) return bwd ? (bf ? train_bwd_launch<X, DT_BF16>(a, m, st) : train_bwd_launch<X, DT_F16>(a, m, st))       \
                         : (bf ? train_fwd_launch<X, DT_BF16>(a, st) : train_fwd_launch<X, DT_F16>(a, st));
  SAGE_TRAIN(64) SAGE_TRAIN(96) SAGE_TRAIN(128) SAGE_TRAIN(256)
  return SAGE_ERR_UNSUPPORTED;
}

// What both passes check and fill in alike
static int train_common(const char* who, TrainArgs& a, TrainLayout& l, BiasMap& m, int B, int H, int Hkv, int Sq, int Skv, int D,
                        int dtype, int causal, float sm_scale, const int* cu_q, const int* cu_k, bool mask, int64_t msb,
                        int64_t msh, int64_t msq, int buckets, int two_sided, const int* borders, int table_dtype, int keep, void* state,
                        int64_t state_bytes) {
  if (int rc = train_sizes(who, cu_q != nullptr, B, H, Hkv, Sq, Skv, D, dtype)) return rc;
  SAGE_REQUIRE((cu_q != nullptr) == (cu_k != nullptr), "%s: cu_q and cu_k go together", who);
  SAGE_REQUIRE(!(cu_q && mask), "%s: packed batches take no mask", who);
  SAGE_REQUIRE(sm_scale >= 0.0f && sm_scale <= 0x1p127f, "%s: sm_scale %g", who, (double)sm_scale);   // (log2(e) times it is finite)
  if (keep && sm_scale > 0.0f && sm_scale < TR_LEAST_SCALE)
    return fail(SAGE_ERR_UNSUPPORTED, "%s: sm_scale %g (with a backward pass at least 2^-100)", who, (double)sm_scale);
  int reach = 0;
  if (buckets) {
    if (int rc = bias_map(who, H, buckets, two_sided, borders, table_dtype, &m)) return rc;
    reach = m.reach();
    if (reach > TR_REACH)
      return fail(SAGE_ERR_UNSUPPORTED, "%s: the last bucket begins at distance %d (at most %d)", who, reach, TR_REACH);
  }
  l = train_layout(cu_q != nullptr, B, H, Hkv, Sq, Skv, D, mask, msb != 0, msh != 0, msq != 0, reach, buckets, keep != 0);
  if (int rc = train_mask_size(who, l)) return rc;
  SAGE_REQUIRE(l.state == 0 || (state && ((uintptr_t)state & 255u) == 0 && state_bytes >= l.state),
               "%s: a state of %lld bytes, 256-byte aligned, is needed (got %lld)", who, (long long)l.state, (long long)state_bytes);
  a.B = B, a.H = H, a.Hkv = Hkv, a.Sq = Sq, a.Skv = Skv, a.q_tiles = l.q_tiles, a.k_tiles = l.k_tiles, a.causal = causal != 0;
  a.scale = sm_scale > 0.0f ? sm_scale : 1.0f / __builtin_sqrtf((float)D);
  a.c = (float)((double)a.scale * 1.4426950408889634);
  char* base = (char*)state;
  if (keep) a.lo = (uint16_t*)(base + l.lo);
  if (cu_q) a.cu_q = cu_q, a.cu_k = cu_k, a.q_tab = (const int2*)(base + l.q_tab), a.k_tab = (const int2*)(base + l.k_tab), a.bounds = (const int*)base;
  if (mask) {
    const int64_t per = (int64_t)l.row_pad * l.words;
    a.bits = (const uint32_t*)(base + l.bits);
    a.mb = msb ? per * l.mask_h : 0, a.mh = msh ? per : 0, a.mw = l.row_pad, a.mi = msq ? 1 : 0;
    const int64_t na = (int64_t)l.blocks * l.aw, nt = (int64_t)l.chunks * l.tw;
    a.any = (const uint64_t*)(base + l.any), a.any_t = (const uint64_t*)(base + l.any_t);
    if (keep && dtype == SAGE_DTYPE_F16) a.keys_seen = (const uint64_t*)(base + l.keys_seen);
    a.ab = msb ? na * l.mask_h : 0, a.ah = msh ? na : 0, a.aw = l.aw;
    a.tb = msb ? nt * l.mask_h : 0, a.th = msh ? nt : 0, a.tw = l.tw;
  }
  if (buckets) a.bias = (const float*)(base + l.vec), a.reach = reach;
  return SAGE_OK;
}

}  // namespace sage

extern "C" int sage_train_workspace(int packed, int B, int H, int Hkv, int Sq, int Skv, int D, int has_mask, int64_t msb,
                                    int64_t msh, int64_t msq, int buckets, int two_sided, const int* borders, int keep,
                                    int64_t* state_bytes, int64_t* workspace_bytes) {
  using namespace sage;
  clear_error();
  SAGE_REQUIRE(state_bytes && workspace_bytes, "sage_train_workspace: a result is NULL");
  if (int rc = train_sizes("sage_train_workspace", packed != 0, B, H, Hkv, Sq, Skv, D, SAGE_DTYPE_BF16)) return rc;
  int reach = 0;
  if (buckets) {
    BiasMap m;
    if (int rc = bias_map("sage_train_workspace", H, buckets, two_sided, borders, SAGE_DTYPE_F32, &m)) return rc;
    reach = m.reach();
    if (reach > TR_REACH)
      return fail(SAGE_ERR_UNSUPPORTED, "sage_train_workspace: the last bucket begins at distance %d (at most %d)", reach, TR_REACH);
  }
  const TrainLayout l = train_layout(packed != 0, B, H, Hkv, Sq, Skv, D, has_mask != 0, msb != 0, msh != 0, msq != 0, reach, buckets,
                                     keep != 0);
  if (int rc = train_mask_size("sage_train_workspace", l)) return rc;
  *state_bytes = l.state;
  *workspace_bytes = l.work;
  return SAGE_OK;
}

extern "C" int sage_train_fwd(const void* q, int64_t qsb, int64_t qss, int64_t qsh, const void* k, int64_t ksb, int64_t kss,
                              int64_t ksh, const void* v, int64_t vsb, int64_t vss, int64_t vsh, void* out, int64_t osb,
                              int64_t oss, int64_t osh, float* lse, int B, int H, int Hkv, int Sq, int Skv, int D, int dtype,
                              int causal, float sm_scale, const int* cu_q, const int* cu_k, const void* mask, int64_t msb,
                              int64_t msh, int64_t msq, int64_t msk, const void* table, int table_dtype, int64_t tb, int64_t th,
                              int buckets, int two_sided, const int* borders, int keep, void* state, int64_t state_bytes, void* stream) {
  using namespace sage;
  clear_error();
  TrainArgs a = {};
  TrainLayout l;
  BiasMap m = {};
  if (int rc = train_common("sage_train_fwd", a, l, m, B, H, Hkv, Sq, Skv, D, dtype, causal, sm_scale, cu_q, cu_k, mask != nullptr,
                            msb, msh, msq, buckets, two_sided, borders, table_dtype, keep, state, state_bytes))
    return rc;
  const TrainTensor ts[] = {{q, qsb, qss, qsh, "q"}, {k, ksb, kss, ksh, "k"}, {v, vsb, vss, vsh, "v"}, {out, osb, oss, osh, "out"}};
  if (int rc = train_tensors("sage_train_fwd", ts, 4)) return rc;
  SAGE_REQUIRE(lse && ((uintptr_t)lse & 3u) == 0, "sage_train_fwd: lse is NULL or misaligned");
  SAGE_REQUIRE(!buckets || table, "sage_train_fwd: table is NULL");
  a.q = (const uint16_t*)q, a.qb = qsb, a.qs = qss, a.qh = qsh;
  a.k = (const uint16_t*)k, a.kb = ksb, a.ks = kss, a.kh = ksh;
  a.v = (const uint16_t*)v, a.vb = vsb, a.vs = vss, a.vh = vsh;
  a.out = (uint16_t*)out, a.ob = osb, a.os = oss, a.oh = osh;
  a.lse = lse;
  hipStream_t st = (hipStream_t)stream;
  if (cu_q) {
    train_plan<<<1, TR_THREADS, 0, st>>>(cu_q, cu_k, B, Sq, Skv, (int2*)a.q_tab, l.q_tiles, (int2*)a.k_tab, l.k_tiles, (int*)state);
    TrainGaps g = {};
    g.p[0] = a.out, g.s[0] = oss, g.h[0] = osh, g.heads[0] = H, g.rows[0] = Sq, g.chunks = D / 8;
    train_gaps<<<dim3(Sq < 1024 ? Sq : 1024, 1), TR_THREADS, 0, st>>>(g, (const int*)state);
  }
  if (mask) {
    const int64_t bh = (int64_t)l.mask_b * l.mask_h, units = bh * l.blocks * l.chunks;
    uint8_t* shows = (uint8_t*)state + l.shows;
    uint64_t* seen = a.keys_seen ? (uint64_t*)((char*)state + l.seen) : nullptr;
    train_mask_bits<<<(unsigned)((units + 3) / 4), TR_THREADS, 0, st>>>((const uint8_t*)mask, msb, msh, msq, msk, l.mask_h,
                                                                        msq ? Sq : 1, l.row_pad, Skv, l.chunks, l.blocks, units,
                                                                        (uint32_t*)a.bits, shows, seen, causal && msq ? Skv - Sq : Skv - 1);
    const int64_t n = bh * l.blocks * l.aw, nt = bh * l.chunks * l.tw;
    train_mask_any<<<(unsigned)((n + nt + 3) / 4), TR_THREADS, 0, st>>>(shows, l.blocks, l.chunks, l.aw, l.tw, n, nt, (uint64_t*)a.any,
                                                                        (uint64_t*)a.any_t, seen, (uint64_t*)a.keys_seen);
  }
  if (buckets)
    if (int rc = bias_expand_launch(table, table_dtype, tb, th, H, m, TR_LOG2E, (float*)a.bias, st)) return rc;
  return train_dispatch(false, a, m, D, dtype, st);
}

extern "C" int sage_train_bwd(const void* dout, int64_t gsb, int64_t gss, int64_t gsh, const void* q, int64_t qsb, int64_t qss,
                              int64_t qsh, const void* k, int64_t ksb, int64_t kss, int64_t ksh, const void* v, int64_t vsb,
                              int64_t vss, int64_t vsh, const void* out, int64_t osb, int64_t oss, int64_t osh, const float* lse,
                              void* dq, int64_t dqb, int64_t dqs, int64_t dqh, void* dk, int64_t dkb, int64_t dks, int64_t dkh,
                              void* dv, int64_t dvb, int64_t dvs, int64_t dvh, int B, int H, int Hkv, int Sq, int Skv, int D,
                              int dtype, int causal, float sm_scale, const int* cu_q, const int* cu_k, int has_mask, int64_t msb,
                              int64_t msh, int64_t msq, void* dtable, int table_dtype, int64_t tb, int64_t th, int buckets,
                              int two_sided, const int* borders, const void* state, int64_t state_bytes, void* workspace,
                              int64_t workspace_bytes, void* stream) {
  using namespace sage;
  clear_error();
  TrainArgs a = {};
  TrainLayout l;
  BiasMap m = {};
  if (int rc = train_common("sage_train_bwd", a, l, m, B, H, Hkv, Sq, Skv, D, dtype, causal, sm_scale, cu_q, cu_k, has_mask != 0,
                            msb, msh, msq, buckets, two_sided, borders, table_dtype, 1, (void*)state, state_bytes))
    return rc;
  const TrainTensor ts[] = {{q, qsb, qss, qsh, "q"},    {k, ksb, kss, ksh, "k"},       {v, vsb, vss, vsh, "v"},
                            {out, osb, oss, osh, "out"}, {dout, gsb, gss, gsh, "dout"}, {dq, dqb, dqs, dqh, "dq"},
                            {dk, dkb, dks, dkh, "dk"},   {dv, dvb, dvs, dvh, "dv"}};
  SAGE_REQUIRE((dk != nullptr) == (dv != nullptr), "sage_train_bwd: dk and dv go together");
  SAGE_REQUIRE(dq || !dtable, "sage_train_bwd: dtable comes with dq");
  SAGE_REQUIRE(dq || dk, "sage_train_bwd: no gradient asked for");
  if (int rc = train_tensors("sage_train_bwd", ts, dq ? 6 : 5)) return rc;
  if (dk)
    if (int rc = train_tensors("sage_train_bwd", ts + 6, 2)) return rc;
  SAGE_REQUIRE(lse && ((uintptr_t)lse & 3u) == 0, "sage_train_bwd: lse is NULL or misaligned");
  SAGE_REQUIRE(workspace && ((uintptr_t)workspace & 255u) == 0 && workspace_bytes >= l.work,
               "sage_train_bwd: a workspace of %lld bytes, 256-byte aligned, is needed (got %lld)", (long long)l.work,
               (long long)workspace_bytes);
  a.q = (const uint16_t*)q, a.qb = qsb, a.qs = qss, a.qh = qsh;
  a.k = (const uint16_t*)k, a.kb = ksb, a.ks = kss, a.kh = ksh;
  a.v = (const uint16_t*)v, a.vb = vsb, a.vs = vss, a.vh = vsh;
  a.o = (const uint16_t*)out, a.ob = osb, a.os = oss, a.oh = osh;
  a.dout = (const uint16_t*)dout, a.gb = gsb, a.gs = gss, a.gh = gsh;
  a.dq = (uint16_t*)dq, a.dqb = dqb, a.dqs = dqs, a.dqh = dqh;
  a.dk = (uint16_t*)dk, a.dkb = dkb, a.dks = dks, a.dkh = dkh;
  a.dv = (uint16_t*)dv, a.dvb = dvb, a.dvs = dvs, a.dvh = dvh;
  a.lse = (float*)lse;
  char* w = (char*)workspace;
  a.nl = (float*)(w + l.nl), a.nd = (float*)(w + l.nd), a.pad = l.pad, a.norms = (uint32_t*)(w + l.norms);
  a.split = train_split(cu_q != nullptr, causal || has_mask || cu_q, B, H, Hkv, l.k_tiles, D), a.kv_part = (float*)(w + l.kv_part);
  if (buckets && dtable) a.bias_part = (float*)(w + l.part), a.parts = l.parts;
  hipStream_t st = (hipStream_t)stream;
  if (cu_q) {
    TrainGaps g = {};
    g.chunks = D / 8;
    g.p[0] = a.dq, g.s[0] = dqs, g.h[0] = dqh, g.heads[0] = H, g.rows[0] = Sq;
    g.p[1] = a.dk, g.s[1] = dks, g.h[1] = dkh, g.heads[1] = Hkv, g.rows[1] = Skv, g.side[1] = 1;
    g.p[2] = a.dv, g.s[2] = dvs, g.h[2] = dvh, g.heads[2] = Hkv, g.rows[2] = Skv, g.side[2] = 1;
    const int rows = Sq > Skv ? Sq : Skv;
    train_gaps<<<dim3(rows < 1024 ? rows : 1024, 3), TR_THREADS, 0, st>>>(g, (const int*)state);
    if (dk) {
      train_order<<<1, TR_THREADS, 0, st>>>(cu_q, cu_k, a.causal, a.k_tab, (int2*)(w + l.k_order), l.k_tiles);
      a.k_tab = (const int2*)(w + l.k_order);
    }
  }
  if (int rc = train_dispatch(true, a, m, D, dtype, st)) return rc;
  if (a.bias_part) return bias_reduce_launch(a.bias_part, l.parts, H, m, dtable, table_dtype, tb, th, st);
  return SAGE_OK;
}
