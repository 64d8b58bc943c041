// Relative position bias by buckets (sage_bias.h) as a tensor [H, q_len, kv_len], and its table's gradient.
#include <vector>

#include "sage_bias.h"

namespace sage {

constexpr int BIAS_THREADS = 256;

__global__ __launch_bounds__(BIAS_THREADS) void bias_expand(const void* __restrict__ table, int dtype, int64_t tb, int64_t th, int H,
                                                            BiasMap m, float mul, float* __restrict__ vec) {
  const int R = 2 * m.reach() + 1;
  const int64_t x = (int64_t)blockIdx.x * BIAS_THREADS + threadIdx.x;
  if (x >= (int64_t)H * R) return;
  const int h = (int)(x / R), d = (int)(x % R) - m.reach();
  vec[x] = bias_value(table, dtype, m.bucket(d, m.borders) * tb + h * th) * mul;
}

int bias_expand_launch(const void* table, int table_dtype, int64_t tb, int64_t th, int H, const BiasMap& m, float mul, float* vec,
                       hipStream_t st) {
  const int64_t n = (int64_t)H * (2 * m.reach() + 1);
  bias_expand<<<(unsigned)((n + BIAS_THREADS - 1) / BIAS_THREADS), BIAS_THREADS, 0, st>>>(table, table_dtype, tb, th, H, m, mul, vec);
  return check_launch("bias_expand");
}

// ---- the tensor ------------------------------------------------------------------------------------------------------------------
//
// A row's values follow from key - query alone: a workgroup looks the buckets of its rows' and columns' distances up once and
// keeps their values in LDS, in the output's type, as `16 / size` copies, each shifted by one value, so that any run of 16
// bytes is one aligned LDS read, ready to be stored.  Bound by the stores: 24 x 4352 x 4352 in 16 bits at 5.1 TB/s (non-temporal
// ones: 4.0), odd rows of 16 x 2047 x 2511 at 4.7.

struct BiasOut {
  const void* table;
  int table_dtype;
  int64_t tb, th;
  void* out;               // contiguous [H, q_len, kv_len]
  int q_len, kv_len;
  int64_t offset;          // position of query 0; key j is at position j
  const void* offset_at;   // where it is in device memory instead, int64 or int32
  int offset64;
  int rows;                // per workgroup
  int segs, seg;           // column segments, columns of each
};
constexpr int BIAS_SEG = 2048;   // columns per workgroup, at most
constexpr int BIAS_ROWS = 64;    // rows per workgroup, at most

template <int DT> struct BiasElem { using T = uint16_t; };
template <> struct BiasElem<SAGE_DTYPE_F32> { using T = uint32_t; };
template <int DT> __device__ __forceinline__ typename BiasElem<DT>::T bias_bits(float f) {
  if constexpr (DT == SAGE_DTYPE_F32) return __float_as_uint(f);
  else return (uint16_t)f32_to_out_bits<DT>(f);
}

template <int DT> __global__ __launch_bounds__(BIAS_THREADS) void bias_write(BiasOut a, BiasMap m) {
  using T = typename BiasElem<DT>::T;
  constexpr int N = 16 / sizeof(T);                      // values per store, and copies
  constexpr int W = BIAS_SEG + BIAS_ROWS + 4 * N;        // values per copy (a multiple of N)
  __shared__ __attribute__((aligned(16))) T tab[N][W];
  __shared__ int borders[BIAS_BUCKETS / 2];
  __shared__ T learned[BIAS_BUCKETS];
  const int seg = blockIdx.x % a.segs, h = blockIdx.y;
  const int i0 = blockIdx.x / a.segs * a.rows, i1 = min(i0 + a.rows, a.q_len);
  const int c0 = seg * a.seg, c1 = min(c0 + a.seg, a.kv_len);
  int64_t off = a.offset;
  if (a.offset_at) off = a.offset64 ? *(const int64_t*)a.offset_at : (int64_t)*(const int*)a.offset_at;
  for (int x = threadIdx.x; x < m.buckets; x += BIAS_THREADS) {
    learned[x] = bias_bits<DT>(bias_value(a.table, a.table_dtype, x * a.tb + h * a.th));
    if (x < m.side - m.near) borders[x] = m.borders[x];
  }
  __syncthreads();
  // value x of the table is that of (row, column) with column - row = x + c0 - N - (i1 - 1)
  const int used = (c1 - c0) + (i1 - i0) + 2 * N;
  for (int x = threadIdx.x; x < used + N; x += BIAS_THREADS) {
    const int64_t d = (int64_t)x + c0 - N - (i1 - 1) - off;
    const T y = learned[m.bucket(d, borders)];
#pragma unroll
    for (int c = 0; c < N; ++c)
      if (x >= c) tab[c][x - c] = y;
  }
  __syncthreads();
  // the threads side by side over the rows' chunks, a row's at 16-byte boundaries: up to two more than fit it
  const int chunks = (c1 - c0) / N + 2;
  int i = i0 + (int)threadIdx.x / chunks, k = (int)threadIdx.x % chunks;
  const int di = BIAS_THREADS / chunks, dk = BIAS_THREADS % chunks;
  while (i < i1) {
    T* row = (T*)a.out + ((int64_t)h * a.q_len + i) * a.kv_len;
    const int skew = (int)(((uintptr_t)(row + c0) & 15u) / sizeof(T));
    const int j = c0 - skew + k * N;
    if (j < c1) {
      const int x = j - i - c0 + N + (i1 - 1), c = x & (N - 1);
      if (j >= c0 && j + N <= c1) {
        *reinterpret_cast<v4i*>(row + j) = *reinterpret_cast<const v4i*>(&tab[c][x - c]);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
          if (j + e >= c0 && j + e < c1) row[j + e] = tab[0][x + e];
      }
    }
    i += di, k += dk;
    if (k >= chunks) k -= chunks, ++i;
  }
}

// ---- the table's gradient -----------------------------------------------------------------------------------------------------------
//
// Every diagonal (key - query) is in one bucket.  A thread walks down a chunk of rows N = 16 / size at a time, N columns further
// right each time: its N x N squares all lie on the same 2 N - 1 diagonals, whose sums it keeps, and its loads are 16 bytes, aligned
// where rows are.  Neighbours share N - 1 diagonals, which are added in LDS; there the workgroup's diagonals are summed by bucket and
// written as one part; the parts are summed in a second launch.  No atomics: one order.  Bound by the loads, of
// which odd rows' are unaligned: 59 us for 16 x 2047 x 2511 fp16 (2.8 TB/s), 33 for 16 x 2048 x 2048 out of the last-level cache.  (With
// each place at the tensor's edges tested and loaded by itself 10 us more; with the next square's loads on their way 5 to 15 more.)

constexpr int BIAS_CHUNK = 64;        // rows per workgroup
constexpr int BIAS_GRAD_THREADS = 256;

struct BiasIn {
  const void* d;
  int64_t sh, sq;          // element strides of heads and rows; keys contiguous
  int q_len, kv_len;
  int64_t offset;
  const void* offset_at;
  int offset64;
  int segs, chunks;
  float* part;             // [H][chunks * segs][buckets]
};

// rows of a chunk and columns as the squares cover them: the first diagonal of chunk rows i0 .. i1 - 1, and how many
__host__ __device__ inline int64_t bias_first(int i1, int n) { return -(int64_t)((i1 - 1 + n - 1) / n * n); }

template <int DT> __global__ __launch_bounds__(BIAS_GRAD_THREADS) void bias_grad(BiasIn a, BiasMap m) {
  using T = typename BiasElem<DT>::T;
  constexpr int N = 16 / sizeof(T);
  constexpr int SEG = BIAS_GRAD_THREADS * N;
  __shared__ float sums[SEG + N - 1];
  const int seg = blockIdx.x % a.segs, chunk = blockIdx.x / a.segs, h = blockIdx.y;
  const int i0 = chunk * BIAS_CHUNK, i1 = min(i0 + BIAS_CHUNK, a.q_len);
  const int64_t g0 = bias_first(i1, N) + (int64_t)seg * SEG;   // key - query index of the first thread's middle diagonal
  const int64_t g = g0 + (int64_t)threadIdx.x * N;
  float acc[2 * N - 1];
#pragma unroll
  for (int e = 0; e < 2 * N - 1; ++e) acc[e] = 0.0f;
  const T* base = (const T*)a.d + h * a.sh;
  typedef uint32_t v4u_a4 __attribute__((ext_vector_type(4), aligned(4)));
  // (i0 and g are multiples of N, so columns are.)
  auto inside = [&](int i) { return i + N <= i1 && i + g >= 0 && i + g + N <= a.kv_len; };
  auto bring = [&](int i, v4i(&w)[N]) {
    const T* p = base + i * a.sq + (i + g);
#pragma unroll
    for (int r = 0; r < N; ++r) {
      if constexpr (DT == SAGE_DTYPE_F32) w[r] = __builtin_bit_cast(v4i, *(const v4u_a4*)(p + r * a.sq));
      else w[r] = load16_2aligned(p + r * a.sq);
    }
  };
  auto add = [&](int i, const v4i(&w)[N]) {
    const int64_t j = i + g;
    if (inside(i)) {
#pragma unroll
      for (int r = 0; r < N; ++r)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (DT == SAGE_DTYPE_F32) {
            acc[e - r + N - 1] += __int_as_float(w[r][e]);
          } else {
            acc[2 * e - r + N - 1] += elem_lo<DT>((uint32_t)w[r][e]);
            acc[2 * e + 1 - r + N - 1] += elem_hi<DT>((uint32_t)w[r][e]);
          }
        }
    } else if (j + N > 0 && j < a.kv_len && i < i1) {
      // rows or columns that end inside the square (none begins inside): columns from the last one that there is, so that no load
      // waits for another
      const int c = (int)j;
#pragma unroll
      for (int r = 0; r < N; ++r)
        if (i + r < i1) {
          const T* row = base + (i + r) * a.sq;
          T x[N];
#pragma unroll
          for (int e = 0; e < N; ++e) x[e] = row[min(c + e, a.kv_len - 1)];
#pragma unroll
          for (int e = 0; e < N; ++e) {
            float y;
            if constexpr (DT == SAGE_DTYPE_F32) y = __uint_as_float(x[e]);
            else y = elem_lo<DT>(x[e]);
            acc[e - r + N - 1] += c + e < a.kv_len ? y : 0.0f;
          }
        }
    }
  };
  v4i w[N];
#pragma unroll 1
  for (int i = i0; i < i1; i += N) {
    if (inside(i)) bring(i, w);
    add(i, w);
  }
  // sums[x]: of diagonal g0 - (N - 1) + x
  if (threadIdx.x == 0)
#pragma unroll
    for (int e = 0; e < N - 1; ++e) sums[e] = 0.0f;
#pragma unroll
  for (int e = N - 1; e < 2 * N - 1; ++e) sums[threadIdx.x * N + e] = acc[e];
  __syncthreads();
#pragma unroll
  for (int e = 0; e < N - 1; ++e) sums[threadIdx.x * N + e] += acc[e];
  __syncthreads();

  int64_t off = a.offset;
  if (a.offset_at) off = a.offset64 ? *(const int64_t*)a.offset_at : (int64_t)*(const int*)a.offset_at;
  float* part = a.part + ((int64_t)h * (a.chunks * a.segs) + blockIdx.x) * m.buckets;
  bias_sum_buckets<BIAS_GRAD_THREADS>(m, sums, g0 - (N - 1) - off, SEG + N - 1, part, 0);
}

// One workgroup per head and 64 buckets: four waves each sum a quarter of the parts in fp64.
__global__ __launch_bounds__(BIAS_THREADS) void bias_reduce(const float* __restrict__ part, int64_t T, int buckets, void* dtable,
                                                            int dtype, int64_t tb, int64_t th) {
  __shared__ double s[4][64];
  const int h = blockIdx.x, l = threadIdx.x & 63, w = threadIdx.x >> 6, b = blockIdx.y * 64 + l;
  double x = 0.0;
  if (b < buckets) {
    const float* p = part + (int64_t)h * T * buckets + b;
#pragma unroll 4
    for (int64_t t = w; t < T; t += 4) x += p[t * buckets];
  }
  s[w][l] = x;
  __syncthreads();
  if (w == 0 && b < buckets) {
    const float y = (float)((s[0][l] + s[1][l]) + (s[2][l] + s[3][l]));
    const int64_t at = b * tb + h * th;
    if (dtype == SAGE_DTYPE_F32) ((float*)dtable)[at] = y;
    else ((uint16_t*)dtable)[at] = (uint16_t)(dtype == SAGE_DTYPE_BF16 ? f32_to_bf16_bits(y) : f32_to_f16_bits(y));
  }
}

int bias_reduce_launch(const float* part, int64_t T, int H, const BiasMap& m, void* dtable, int table_dtype, int64_t tb, int64_t th,
                       hipStream_t st) {
  bias_reduce<<<dim3(H, (m.buckets + 63) / 64), BIAS_THREADS, 0, st>>>(part, T, m.buckets, dtable, table_dtype, tb, th);
  return check_launch("bias_reduce");
}

int bias_map(const char* who, int H, int buckets, int two_sided, const int* borders, int table_dtype, BiasMap* m) {
  SAGE_REQUIRE(table_dtype == SAGE_DTYPE_BF16 || table_dtype == SAGE_DTYPE_F16 || table_dtype == SAGE_DTYPE_F32,
               "%s: table dtype %d", who, table_dtype);
  SAGE_REQUIRE(buckets >= 2 && buckets <= BIAS_BUCKETS && !(two_sided && (buckets % 2 || buckets < 4)),
               "%s: %d buckets (2 to %d, two-sided an even number from 4)", who, buckets, BIAS_BUCKETS);
  SAGE_REQUIRE(H > 0 && H <= 65535, "%s: %d heads", who, H);
  SAGE_REQUIRE(borders, "%s: borders is NULL", who);
  m->buckets = buckets;
  m->two_sided = two_sided != 0;
  m->side = two_sided ? buckets / 2 : buckets;
  m->near = m->side / 2;
  for (int t = 0; t < m->side - m->near; ++t) {
    SAGE_REQUIRE(borders[t] >= (t ? borders[t - 1] : m->near) && borders[t] <= 0x3FFFFFFF, "%s: borders must not fall", who);
    m->borders[t] = borders[t];
  }
  SAGE_REQUIRE(borders[0] == m->near, "%s: borders[0] must be %d", who, m->near);
  return SAGE_OK;
}

}  // namespace sage

namespace {

// whole numbers of any size, 32 bits a word, lowest first
typedef std::vector<uint32_t> Big;
Big power(uint32_t base, int n) {
  Big r = {1};
  for (int i = 0; i < n; ++i) {
    uint64_t carry = 0;
    for (uint32_t& w : r) {
      carry += (uint64_t)w * base;
      w = (uint32_t)carry;
      carry >>= 32;
    }
    if (carry) r.push_back((uint32_t)carry);
  }
  return r;
}
Big times(Big r, uint32_t base, int n) {
  for (int i = 0; i < n; ++i) {
    uint64_t carry = 0;
    for (uint32_t& w : r) {
      carry += (uint64_t)w * base;
      w = (uint32_t)carry;
      carry >>= 32;
    }
    if (carry) r.push_back((uint32_t)carry);
  }
  return r;
}
bool at_least(const Big& a, const Big& b) {
  if (a.size() != b.size()) return a.size() > b.size();
  for (size_t i = a.size(); i-- > 0;)
    if (a[i] != b[i]) return a[i] > b[i];
  return true;
}

}  // namespace

extern "C" int sage_bias_borders(int buckets, int two_sided, int max_distance, int* borders) {
  using namespace sage;
  clear_error();
  SAGE_REQUIRE(borders, "sage_bias_borders: borders is NULL");
  SAGE_REQUIRE(buckets >= 2 && buckets <= BIAS_BUCKETS && !(two_sided && (buckets % 2 || buckets < 4)),
               "sage_bias_borders: %d buckets (2 to %d, two-sided an even number from 4)", buckets, BIAS_BUCKETS);
  const int side = two_sided ? buckets / 2 : buckets, near = side / 2, m = side - near;
  SAGE_REQUIRE(max_distance > near && max_distance <= 0x3FFFFFFF, "sage_bias_borders: max_distance %d (more than %d)", max_distance, near);
  try {
    for (int t = 0; t < m; ++t) {
      // the smallest n with n^m >= near^(m - t) max_distance^t: from an estimate, compared in whole numbers
      const Big want = times(power((uint32_t)near, m - t), (uint32_t)max_distance, t);
      int64_t n = (int64_t)(near * __builtin_pow((double)max_distance / near, (double)t / m));
      if (n < 1) n = 1;
      while (!at_least(power((uint32_t)n, m), want)) ++n;
      while (n > 1 && at_least(power((uint32_t)(n - 1), m), want)) --n;
      borders[t] = (int)n;
    }
  } catch (...) {
    return fail(SAGE_ERR_INVALID, "sage_bias_borders: out of memory");
  }
  return SAGE_OK;
}

namespace sage {
static int bias_sizes(const char* who, int q_len, int kv_len, const void* offset_at, int offset64) {
  SAGE_REQUIRE(q_len > 0 && kv_len > 0 && q_len <= 0x3FFFFFFF && kv_len <= 0x3FFFFFFF, "%s: lengths must be positive", who);
  SAGE_REQUIRE(((uintptr_t)offset_at & (offset64 ? 7u : 3u)) == 0, "%s: offset misaligned", who);
  return SAGE_OK;
}
}  // namespace sage

extern "C" int sage_relative_bias(const void* table, int table_dtype, int64_t tb, int64_t th, int H, int buckets, int two_sided,
                                  const int* borders, int q_len, int kv_len, int64_t offset, const void* offset_at, int offset64,
                                  void* out, int dtype, void* stream) {
  using namespace sage;
  clear_error();
  BiasMap m;
  if (int rc = bias_map("sage_relative_bias", H, buckets, two_sided, borders, table_dtype, &m)) return rc;
  if (int rc = bias_sizes("sage_relative_bias", q_len, kv_len, offset_at, offset64)) return rc;
  SAGE_REQUIRE(table && out, "sage_relative_bias: table or out is NULL");
  SAGE_REQUIRE(dtype == SAGE_DTYPE_BF16 || dtype == SAGE_DTYPE_F16 || dtype == SAGE_DTYPE_F32, "sage_relative_bias: dtype %d", dtype);
  SAGE_REQUIRE(((uintptr_t)out & (dtype == SAGE_DTYPE_F32 ? 3u : 1u)) == 0, "sage_relative_bias: out misaligned");
  BiasOut a = {};
  a.table = table, a.table_dtype = table_dtype, a.tb = tb, a.th = th, a.out = out, a.q_len = q_len, a.kv_len = kv_len;
  a.offset = offset, a.offset_at = offset_at, a.offset64 = offset64;
  a.segs = (kv_len + BIAS_SEG - 1) / BIAS_SEG;
  a.seg = ((kv_len + a.segs - 1) / a.segs + 127) / 128 * 128;   // (equal ones: 2511 columns as 2048 and 463 take 72 us for 16 x 2047 rows)
  a.rows = q_len < BIAS_ROWS ? q_len : BIAS_ROWS;
  const int64_t blocks = (int64_t)((q_len + a.rows - 1) / a.rows) * a.segs;
  SAGE_REQUIRE(blocks <= 0x7FFFFFFF, "sage_relative_bias: too large");
  const dim3 grid((unsigned)blocks, H);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SAGE_DTYPE_BF16) bias_write<SAGE_DTYPE_BF16><<<grid, BIAS_THREADS, 0, st>>>(a, m);
  else if (dtype == SAGE_DTYPE_F16) bias_write<SAGE_DTYPE_F16><<<grid, BIAS_THREADS, 0, st>>>(a, m);
  else bias_write<SAGE_DTYPE_F32><<<grid, BIAS_THREADS, 0, st>>>(a, m);
  return check_launch("bias_write");
}

namespace sage {
// workgroups side by side for a chunk's diagonals (the first chunk's are the most)
static int bias_segs(int q_len, int kv_len, int dtype) {
  const int n = dtype == SAGE_DTYPE_F32 ? 4 : 8, seg = BIAS_GRAD_THREADS * n;
  const int64_t width = -bias_first(q_len < BIAS_CHUNK ? q_len : BIAS_CHUNK, n) + kv_len;
  return (int)((width + seg - 1) / seg);
}
}  // namespace sage

extern "C" int sage_relative_bias_grad_workspace(int H, int buckets, int q_len, int kv_len, int dtype, int64_t* workspace_bytes) {
  using namespace sage;
  clear_error();
  SAGE_REQUIRE(workspace_bytes, "sage_relative_bias_grad_workspace: workspace_bytes is NULL");
  SAGE_REQUIRE(H > 0 && buckets > 0 && q_len > 0 && kv_len > 0, "sage_relative_bias_grad_workspace: sizes must be positive");
  const int64_t chunks = ((int64_t)q_len + BIAS_CHUNK - 1) / BIAS_CHUNK;
  *workspace_bytes = 4 * (int64_t)bias_segs(q_len, kv_len, dtype) * chunks * H * buckets;
  return SAGE_OK;
}

extern "C" int sage_relative_bias_grad(const void* dbias, int64_t sh, int64_t sq, int dtype, int H, int buckets, int two_sided,
                                       const int* borders, int q_len, int kv_len, int64_t offset, const void* offset_at,
                                       int offset64, void* dtable, int table_dtype, int64_t tb, int64_t th, void* workspace,
                                       int64_t workspace_bytes, void* stream) {
  using namespace sage;
  clear_error();
  BiasMap m;
  if (int rc = bias_map("sage_relative_bias_grad", H, buckets, two_sided, borders, table_dtype, &m)) return rc;
  if (int rc = bias_sizes("sage_relative_bias_grad", q_len, kv_len, offset_at, offset64)) return rc;
  SAGE_REQUIRE(dbias && dtable && workspace, "sage_relative_bias_grad: a pointer is NULL");
  SAGE_REQUIRE(dtype == SAGE_DTYPE_BF16 || dtype == SAGE_DTYPE_F16 || dtype == SAGE_DTYPE_F32, "sage_relative_bias_grad: dtype %d", dtype);
  SAGE_REQUIRE(((uintptr_t)dbias & (dtype == SAGE_DTYPE_F32 ? 3u : 1u)) == 0 && aligned16(workspace), "sage_relative_bias_grad: misaligned");
  int64_t need = 0;
  if (int rc = sage_relative_bias_grad_workspace(H, buckets, q_len, kv_len, dtype, &need)) return rc;
  SAGE_REQUIRE(workspace_bytes >= need, "sage_relative_bias_grad: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
               (long long)need);
  BiasIn a = {};
  a.d = dbias, a.sh = sh, a.sq = sq, a.q_len = q_len, a.kv_len = kv_len;
  a.offset = offset, a.offset_at = offset_at, a.offset64 = offset64;
  a.segs = bias_segs(q_len, kv_len, dtype);
  a.chunks = (q_len + BIAS_CHUNK - 1) / BIAS_CHUNK;
  a.part = (float*)workspace;
  SAGE_REQUIRE((int64_t)a.segs * a.chunks <= 0x7FFFFFFF, "sage_relative_bias_grad: too large");
  const dim3 grid(a.segs * a.chunks, H);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SAGE_DTYPE_BF16) bias_grad<SAGE_DTYPE_BF16><<<grid, BIAS_GRAD_THREADS, 0, st>>>(a, m);
  else if (dtype == SAGE_DTYPE_F16) bias_grad<SAGE_DTYPE_F16><<<grid, BIAS_GRAD_THREADS, 0, st>>>(a, m);
  else bias_grad<SAGE_DTYPE_F32><<<grid, BIAS_GRAD_THREADS, 0, st>>>(a, m);
  if (int rc = check_launch("bias_grad")) return rc;
  return bias_reduce_launch(a.part, (int64_t)a.segs * a.chunks, H, m, dtable, table_dtype, tb, th, st);
}
