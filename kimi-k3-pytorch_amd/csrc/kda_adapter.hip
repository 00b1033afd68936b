// Low-rank adapters of many requests beside a shared projection:
//   y_m = W x_m + bias + c_a B_a (A_a x_m),  a = the adapter of row m, or none.
// Row m's adapter is ids[m / span]: a negative id has none, an id past the stack
// gives a row of NaN (the host cannot see it without waiting for the GPU).
//
// First s_m = A_a x_m in f32 (down), then c_a B_a s_m (up).  Rows that share an
// adapter share its reading; whose rows they are is found by the kernels
// themselves, so a call needs no sorted batch and no plan:
//  - runs (a prompt's tokens): a workgroup owns 16 or 32 neighbouring rows and goes through
//    the adapters it meets in them, mostly one, both steps in one kernel; the
//    shared projection is a library GEMM's f32 product, which the second step adds;
//  - up to 512 rows in any order (decode): the workgroup of row i counts the earlier
//    rows with row i's adapter; where their number is a multiple of 16 it owns
//    the next 16 such rows, otherwise it has nothing to do.  A launch for each
//    step; of up to 32 rows the projection is formed beside the first.
// Measured, bf16: 8195 rows 2048 -> 2048 rank 16, 41 us beside a GEMM of 76 us (its
// floor is x and the product read and y written, 22 us; the GEMM's adding to a 16-bit
// bias + c B s would need 11, but rounds that sum and loses one past f16's range);
// 200 rows 4096 -> 4096 rank 32 of 48 adapters, 10 + 11 us beside 20 to 24 us; one
// row 2048 -> 2048, 7.8 + 6 us.
#include <type_traits>

#include "kda_launch.h"

namespace kda {

typedef float ad_f32x4 __attribute__((ext_vector_type(4)));

template <class T>
struct Frag {
  typedef T type __attribute__((ext_vector_type(8), aligned(16)));
  typedef T loose __attribute__((ext_vector_type(8), aligned(sizeof(T))));
};

// D[n][m] += sum over 32 columns: lane l holds row l % 16 of either operand, its
// columns 8 (l / 16) .. + 7; the result has column m = l % 16, rows 4 (l / 16) .. + 3.
__device__ __forceinline__ ad_f32x4 mma(Frag<bf16>::type a, Frag<bf16>::type b, ad_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ ad_f32x4 mma(Frag<f16>::type a, Frag<f16>::type b, ad_f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ ad_f32x4 mma(Frag<float>::type a, Frag<float>::type b, ad_f32x4 c) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// EVEN calls: widths of whole 64-column slices, a rank of whole vectors and aligned
// addresses, with code for nothing else: these kernels run for some ten
// microseconds, and reading instructions that are skipped took a third of them.
// Other calls load vectors at element alignment, which the hardware takes, and
// the columns at a row's end one by one.

// Eight columns, c to c + 7, of a row of `len`; zeros past it.
template <class T, bool EVEN>
__device__ __forceinline__ typename Frag<T>::type load8(const T* row, int c, int len) {
  typename Frag<T>::type v{};
  if constexpr (EVEN) {
    if (c < len) v = *reinterpret_cast<const typename Frag<T>::type*>(row + c);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const T x = row[c + e < len ? c + e : len - 1];
      v[e] = c + e < len ? x : static_cast<T>(0.f);
    }
  }
  return v;
}

// Sixteen columns from c of a row of `len`; zeros past it.
template <class T, bool EVEN>
__device__ __forceinline__ void load16(const T* row, int c, int len, typename Frag<T>::type (&v)[2]) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if constexpr (EVEN)
      v[u] = *reinterpret_cast<const typename Frag<T>::type*>(row + c + 8 * u);
    else
      v[u] = load8<T, false>(row, c + 8 * u, len);
  }
}

template <class T>
struct Adapters {
  const T *x, *a, *b, *bias;  // x [rows, in], a [n, rank, in], b [n, out, rank], bias [out] or null
  const float* scaling;       // [n] or null (1)
  const void* ids;            // int32 or int64
  int ids64;
  int64_t rows;
  int span, in, out, rank, n, splits, parts;
  T* y;         // [rows, out]
  float* s;     // [splits, rows, rank]: sums over a part of the columns each
  const T* weight;  // [out, in]
  float* wide;  // [parts, rows, out]: x W^T, over a part of the columns each (the caller's
                // product: one part); parts 0 without
};

constexpr int kNone = -1, kMissing = -2, kNoRow = -3;

// the row's adapter, kNone or kMissing
template <class T>
__device__ __forceinline__ int adapter_of(const Adapters<T>& a, int64_t row) {
  if (a.n == 0) return kNone;
  unsigned i = static_cast<unsigned>(row);  // rows < 2^31
  if (a.span != 1) i /= static_cast<unsigned>(a.span);
  const int64_t id = a.ids64 != 0 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
  return id < 0 ? kNone : (id < a.n ? static_cast<int>(id) : kMissing);
}

__device__ __forceinline__ int below(uint64_t mask, int lane) {  // set bits under the lane's
  return __popcll(mask & ((uint64_t{1} << lane) - 1));
}

constexpr int kAnyOrder = 512;  // rows in any order, at most

// The rows that the workgroup of `row` owns among the rows with its id, in rowS;
// their number, none where an earlier row's workgroup owns it.
template <int R, class T>
__device__ __forceinline__ int gather_rows(const Adapters<T>& a, int row, int id, int* rowS) {
  const int lane = threadIdx.x & 63;
  int of[kAnyOrder / 64];
#pragma unroll
  for (int u = 0; u < kAnyOrder / 64; ++u) {
    of[u] = kNoRow;
    if (64 * u < a.rows && 64 * u + lane < a.rows) of[u] = adapter_of(a, 64 * u + lane);
  }
  int before = 0;
#pragma unroll
  for (int u = 0; u < kAnyOrder / 64; ++u) before += __popcll(__ballot(of[u] == id && 64 * u + lane < row));
  if (before % R != 0) return 0;  // the same in every wave
  int count = 0;
#pragma unroll
  for (int u = 0; u < kAnyOrder / 64; ++u) {
    const bool same = of[u] == id && 64 * u + lane >= row;
    const uint64_t mask = __ballot(same);
    const int at = count + below(mask, lane);
    if (same && at < R && threadIdx.x < 64) rowS[at] = 64 * u + lane;
    count += __popcll(mask);
  }
  __syncthreads();
  return count < R ? count : R;
}

// ---- matrix products of a workgroup ---------------------------------------------
constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kSlice64 = 64;

template <int TILES>
struct Meet {  // partial tiles of the waves
  __attribute__((aligned(16))) float red[kWaves / 2][TILES][256];
};

// The sum of the eight waves' 16 x 16 tiles, in two steps: the upper four waves'
// tiles are added to the lower four's, which then meet.  `take(tile, n, m, sum)`
// gets each element, row n and column m of its tile.
template <int TILES, int ROOM, class F>
__device__ __forceinline__ void meet_tiles(Meet<ROOM>& lds, ad_f32x4 (&acc)[TILES], F take) {
  static_assert(TILES <= ROOM, "the tiles fit");
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  if (w >= kWaves / 2) {
#pragma unroll
    for (int t = 0; t < TILES; ++t) *reinterpret_cast<ad_f32x4*>(&lds.red[w - kWaves / 2][t][4 * lane]) = acc[t];
  }
  __syncthreads();
  if (w < kWaves / 2) {
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      ad_f32x4* p = reinterpret_cast<ad_f32x4*>(&lds.red[w][t][4 * lane]);
      *p = *p + acc[t];
    }
  }
  __syncthreads();
  for (int i = tid; i < TILES * 256; i += kThreads) {
    const int tile = i >> 8, n = i & 15, m = (i >> 4) & 15, at = 4 * (m + 16 * (n >> 2)) + (n & 3);
    take(tile, n, m, (lds.red[0][tile][at] + lds.red[1][tile][at]) + (lds.red[2][tile][at] + lds.red[3][tile][at]));
  }
}

// 16 NT rows of an adapter's A from row j0 times 16 MT rows of x (a lane's of each
// tile at xp), over the slices first.. < last of 64 columns, the waves every
// eighth of them, E half slices in flight.  acc[t * MT + m]: tile (t, m), this
// wave's part.
template <class T, bool EVEN, int MT, int NT, int E>
__device__ __forceinline__ void down_product(const Adapters<T>& a, int id, int j0, const T* const (&xp)[MT], int first,
                                             int last, ad_f32x4 (&acc)[NT * MT]) {
  using v8 = typename Frag<T>::type;
  using vec = typename std::conditional<EVEN, v8, typename Frag<T>::loose>::type;
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T* ap[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {  // rows past the rank repeat its last one; their sums are dropped
    const int j = j0 + 16 * t + li;
    ap[t] = a.a + (static_cast<int64_t>(id) * a.rank + (j < a.rank ? j : a.rank - 1)) * a.in;
  }
#pragma unroll
  for (int t = 0; t < NT * MT; ++t) acc[t] = ad_f32x4{0.f, 0.f, 0.f, 0.f};
  const int whole = EVEN || last * kSlice64 <= a.in ? last : last - 1;  // slices of 64 columns
  for (int c = first + w; c < whole; c += kWaves * E / 2) {
    v8 av[NT][E], xv[MT][E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int slice = c + kWaves * (e / 2);
      const int k = (slice < whole ? slice : c) * kSlice64 + 32 * (e & 1) + 8 * g;  // past the part: read, not used
#pragma unroll
      for (int m = 0; m < MT; ++m) xv[m][e] = *reinterpret_cast<const vec*>(xp[m] + k);
#pragma unroll
      for (int t = 0; t < NT; ++t) av[t][e] = *reinterpret_cast<const vec*>(ap[t] + k);
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (c + kWaves * (e / 2) < whole) {  // uniform
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int t = 0; t < NT; ++t) acc[t * MT + m] = mma(av[t][e], xv[m][e], acc[t * MT + m]);
      }
  }
  if (!EVEN && first < last && whole < last && (whole - first) % kWaves == w) {  // the slice that a row ends in
#pragma unroll 1
    for (int k = whole * kSlice64; k < a.in; k += 32) {
      v8 av[NT], xv[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) xv[m] = load8<T, false>(xp[m], k + 8 * g, a.in);
#pragma unroll
      for (int t = 0; t < NT; ++t) av[t] = load8<T, false>(ap[t], k + 8 * g, a.in);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t * MT + m] = mma(av[t], xv[m], acc[t * MT + m]);
    }
  }
}

// How B's products hold s.  bf16: as two bf16 values (2^-17 of it is left) on bf16
// products; f16 and f32: f32 products (f16 has not the range of s).
template <class T>
struct UpType {
  using type = float;
  static constexpr int P = 1;
};
template <>
struct UpType<bf16> {
  using type = bf16;
  static constexpr int P = 2;
};

template <class T, int R, int RANK>
struct LowRows {  // s of R rows, RANK of the rank
  using U = typename UpType<T>::type;
  static constexpr int P = UpType<T>::P;
  __attribute__((aligned(16))) U s[P][R][RANK + 8];

  __device__ __forceinline__ void put(int r, int j, float v) {
    const U hi = static_cast<U>(v);
    s[0][r][j] = hi;
    const float f = static_cast<float>(hi);
    if constexpr (P == 2) s[P - 1][r][j] = static_cast<U>(v == f ? 0.f : v - f);  // nothing is left of an infinity
  }
};

// What 64 columns from c0 need of B (the first 32 of the rank) and of the bias, for
// a wave: asked for ahead of the sums they meet.  Row i of tile t is column
// 16 (i / 4) + 4 t + i % 4, so a lane's results over the four tiles are sixteen
// neighbouring columns of a row.
template <class T, bool EVEN>
struct UpLoads {
  typename Frag<T>::type b[4];
  typename Frag<T>::type bias[2];

  __device__ __forceinline__ static const T* row(const Adapters<T>& a, int id, int c0, int t) {
    const int li = threadIdx.x & 15, col = c0 + 16 * (li >> 2) + 4 * t + (li & 3);
    return a.b + (static_cast<int64_t>(id) * a.out + (EVEN || col < a.out ? col : a.out - 1)) * a.rank;
  }
  __device__ __forceinline__ void ask(const Adapters<T>& a, int id, int c0) {
    const int g = (threadIdx.x & 63) >> 4;
    if (c0 >= a.out) return;
    if (id >= 0) {
#pragma unroll
      for (int t = 0; t < 4; ++t) b[t] = load8<T, EVEN>(row(a, id, c0, t), 8 * g, a.rank);
    }
    bias[0] = bias[1] = typename Frag<T>::type{};
    if (a.bias != nullptr) load16<T, EVEN>(a.bias, c0 + 16 * g, a.out, bias);
  }
};

// y = bias + c B s + x W^T of 64 columns from c0, a wave, rounded once: s of 16 MT rows
// in LDS.  rows[m]: the lane's row of tile m, or -1.
template <class T, bool EVEN, int MT, int R, int RANK>
__device__ __forceinline__ void up_columns(const Adapters<T>& a, int id, float c, const UpLoads<T, EVEN>& in,
                                           const LowRows<T, R, RANK>& low, const int (&rows)[MT], int c0) {
  using U = typename UpType<T>::type;
  using v8 = typename Frag<U>::type;
  constexpr int P = UpType<T>::P;
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4, mycol = c0 + 16 * g;
  ad_f32x4 d[P][4][MT];
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m) d[p][t][m] = ad_f32x4{0.f, 0.f, 0.f, 0.f};
  if (id >= 0) {
    typename Frag<T>::type raw[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) raw[t] = in.b[t];
    for (int k = 0; k < a.rank; k += 32) {
      if (k != 0) {
#pragma unroll
        for (int t = 0; t < 4; ++t) raw[t] = load8<T, EVEN>(UpLoads<T, EVEN>::row(a, id, c0, t), k + 8 * g, a.rank);
      }
      v8 bv[4];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e) bv[t][e] = static_cast<U>(raw[t][e]);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int p = 0; p < P; ++p) {
          const v8 sv = *reinterpret_cast<const v8*>(&low.s[p][16 * m + li][k + 8 * g]);
#pragma unroll
          for (int t = 0; t < 4; ++t) d[p][t][m] = mma(bv[t], sv, d[p][t][m]);
        }
    }
  }
  if (id == kMissing) c = __builtin_nanf("");  // times zero
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    if (rows[m] < 0) continue;
    const int64_t row = rows[m];
    float y[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      float bs = d[0][e >> 2][m][e & 3];
      // of an infinity the larger part decides: times what is left of s, zero or of the
      // other sign, it would make the sum NaN
      if constexpr (P == 2) bs = fabsf(bs) < __builtin_inff() ? bs + d[P - 1][e >> 2][m][e & 3] : bs;
      y[e] = c * bs + to_float(static_cast<T>(in.bias[e / 8][e % 8]));
    }
    for (int u = 0; u < a.parts; ++u) {
      Frag<float>::type part[2];
      load16<float, EVEN>(a.wide + (u * a.rows + row) * a.out, mycol, a.out, part);
#pragma unroll
      for (int e = 0; e < 16; ++e) y[e] += part[e / 8][e % 8];
    }
    T* out = a.y + row * a.out + mycol;
    constexpr int N = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(N), aligned(EVEN ? 16 : sizeof(T))));
    if (EVEN || mycol + 16 <= a.out) {
#pragma unroll
      for (int u = 0; u < 16 / N; ++u) {
        vec v;
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = from_compute<T>(y[u * N + e]);
        *reinterpret_cast<vec*>(out + u * N) = v;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (mycol + e < a.out) out[e] = from_compute<T>(y[e]);
    }
  }
}

// All columns from c0 in steps, the next ones' loads ahead of the products (two
// sets in turn: copying one to the other would wait for it).
template <class T, bool EVEN, int MT, int R, int RANK>
__device__ __forceinline__ void up_all(const Adapters<T>& a, int id, float c, UpLoads<T, EVEN>& in,
                                       const LowRows<T, R, RANK>& low, const int (&rows)[MT], int c0, int step) {
  UpLoads<T, EVEN> next;
  while (c0 < a.out) {
    next.ask(a, id, c0 + step);
    up_columns<T, EVEN, MT>(a, id, c, in, low, rows, c0);
    c0 += step;
    if (c0 >= a.out) break;
    in.ask(a, id, c0 + step);
    up_columns<T, EVEN, MT>(a, id, c, next, low, rows, c0);
    c0 += step;
  }
}

template <class T>
__device__ __forceinline__ float factor(const Adapters<T>& a, int id) {
  return id >= 0 && a.scaling != nullptr ? a.scaling[id] : 1.f;
}

// ---- runs of rows ---------------------------------------------------------------
// y = x W^T + bias + c B (A x) of 16 MT neighbouring rows a workgroup of eight waves, adapter
// by adapter (every row's products are formed, the adapter's own rows are kept):
// s by 16 NT of the rank into LDS, then all columns, 64 a wave in turn.  Two
// workgroups share the adapters of the rows where a run ends in them (the second
// has nothing to do elsewhere).
constexpr int kMaxRank = 256;
constexpr int kRunTurns = 2;

template <class T, bool EVEN, int MT, int NT>
__global__ __launch_bounds__(kThreads) void adapter_run_kernel(const Adapters<T> a) {
  constexpr int R = 16 * MT;
  __shared__ Meet<2 * MT> meet;
  __shared__ LowRows<T, R, kMaxRank> low;
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, w = tid >> 6;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * R;
  int mine = kNoRow;  // the adapter of the lane's row
  if (lane < R && row0 + lane < a.rows) mine = adapter_of(a, row0 + lane);
  const T* xp[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t row = row0 + 16 * m + li;
    xp[m] = a.x + (row < a.rows ? row : a.rows - 1) * a.in;
  }
  const int slices = (a.in + kSlice64 - 1) / kSlice64;
  int turn = 0;
  for (uint64_t pending = __ballot(mine != kNoRow); pending != 0;) {
    const int id = __shfl(mine, __ffsll(static_cast<unsigned long long>(pending)) - 1);
    pending &= ~__ballot(mine == id);
    if (turn++ % gridDim.y != blockIdx.y) continue;  // another workgroup's; the same in every wave
    int rows[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
      rows[m] = __shfl(mine, 16 * m + li) == id ? static_cast<int>(row0) + 16 * m + li : -1;
    UpLoads<T, EVEN> first;
    first.ask(a, id, 64 * w);
    const float c = factor(a, id);
    if (id >= 0) {
      for (int j0 = 0; j0 < a.rank; j0 += 16 * NT) {
        ad_f32x4 acc[NT * MT];
        down_product<T, EVEN, MT, NT, NT == 1 ? 8 : 4>(a, id, j0, xp, 0, slices, acc);
#pragma unroll
        for (int t0 = 0; t0 < NT; t0 += 2) {  // two rank tiles at a time
          constexpr int N = NT < 2 ? 1 : 2;
          ad_f32x4 some[N * MT];
#pragma unroll
          for (int t = 0; t < N * MT; ++t) some[t] = acc[t0 * MT + t];
          if (t0 != 0) __syncthreads();
          meet_tiles<N * MT>(meet, some, [&](int tile, int n, int m, float sum) {
            const int j = j0 + 16 * (t0 + tile / MT) + n;
            if (j < kMaxRank) low.put(16 * (tile % MT) + m, j, j < a.rank ? sum : 0.f);
            if (NT == 1) low.put(16 * (tile % MT) + m, j + 16, 0.f);  // products take 32 of the rank
          });
        }
        __syncthreads();
      }
    }
    up_all<T, EVEN, MT>(a, id, c, first, low, rows, 64 * w, 64 * kWaves);
    __syncthreads();  // before the next adapter's sums
  }
}

// ---- few rows in any order --------------------------------------------------------
// s of 16 rows of one adapter over a part of the columns: 16 NT of the rank from
// block `ranks` on, every `step`th of them.
template <class T, bool EVEN, int NT>
__device__ __forceinline__ void down_body(const Adapters<T>& a, int row, int part, int ranks, int step, Meet<NT>& meet,
                                          int* rowS) {
  const int id = adapter_of(a, row);
  if (id < 0) return;
  const int count = gather_rows<16>(a, row, id, rowS);
  if (count == 0) return;
  const int slices = (a.in + kSlice64 - 1) / kSlice64, per = (slices + a.splits - 1) / a.splits;
  const int first = part * per, last = first + per < slices ? first + per : slices;
  float* s = a.s + static_cast<int64_t>(part) * a.rows * a.rank;
  const int li = threadIdx.x & 15;
  const T* xp[1] = {a.x + static_cast<int64_t>(rowS[li < count ? li : count - 1]) * a.in};
  for (int j0 = 16 * NT * ranks; j0 < a.rank; j0 += 16 * NT * step) {
    ad_f32x4 acc[NT];
    down_product<T, EVEN, 1, NT, 4>(a, id, j0, xp, first, last, acc);
    meet_tiles<NT>(meet, acc, [&](int tile, int n, int m, float sum) {
      const int j = j0 + 16 * tile + n;
      if (m < count && j < a.rank) s[static_cast<int64_t>(rowS[m]) * a.rank + j] = sum;
    });
    __syncthreads();  // before the next block's tiles
  }
}

template <class T, bool EVEN, int NT>
__global__ __launch_bounds__(kThreads) void adapter_down_kernel(const Adapters<T> a) {
  __shared__ Meet<NT> meet;
  __shared__ int rowS[16];
  down_body<T, EVEN, NT>(a, blockIdx.x, blockIdx.y, blockIdx.z, gridDim.z, meet, rowS);
}

// x W^T of 16 NT weight rows and 16 MT rows of x over a part of the columns, in f32.
template <class T, int MT, int NT>
__device__ __forceinline__ void wide_body(const Adapters<T>& a, int block, Meet<NT * MT>& meet) {
  using v8 = typename Frag<T>::type;
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int across = (a.out + 16 * NT - 1) / (16 * NT);
  const int n0 = (block % across) * 16 * NT, part = block / across;
  const T *wp[NT], *xp[MT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {  // rows past the weight repeat its last one; their results are dropped
    const int row = n0 + 16 * t + li;
    wp[t] = a.weight + static_cast<int64_t>(row < a.out ? row : a.out - 1) * a.in + 8 * g;
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int64_t row = 16 * t + li;
    xp[t] = a.x + (row < a.rows ? row : a.rows - 1) * a.in + 8 * g;
  }
  ad_f32x4 acc[NT * MT];
#pragma unroll
  for (int t = 0; t < NT * MT; ++t) acc[t] = ad_f32x4{0.f, 0.f, 0.f, 0.f};
  const int all = a.in / kSlice64, per = (all + a.parts - 1) / a.parts;
  const int slices = part * per + per < all ? part * per + per : all;
  constexpr int U = 4;  // slices in flight
  for (int s0 = part * per + w; s0 < slices; s0 += kWaves * U) {
    v8 wv[U][NT][2], xv[U][MT][2];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = s0 + u * kWaves;
      const int k = (c < slices ? c : s0) * kSlice64;  // past the end: a slice already read, not used
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) wv[u][t][e] = *reinterpret_cast<const v8*>(wp[t] + k + 32 * e);
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e) xv[u][m][e] = *reinterpret_cast<const v8*>(xp[m] + k + 32 * e);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u * kWaves < slices) {  // uniform
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int e = 0; e < 2; ++e) acc[t * MT + m] = mma(wv[u][t][e], xv[u][m][e], acc[t * MT + m]);
      }
    }
  }
  meet_tiles<NT * MT>(meet, acc, [&](int tile, int n, int m, float sum) {
    const int col = n0 + 16 * (tile / MT) + n, row = 16 * (tile % MT) + m;
    if (col < a.out && row < a.rows) a.wide[(part * a.rows + row) * a.out + col] = sum;
  });
}

// Several projections of few rows (one, or those of a layer's decode step).
constexpr int kMaxSet = 6;

template <class T>
struct AdapterSet {
  Adapters<T> p[kMaxSet];
  int first[kMaxSet + 1];  // workgroups of projection j
  int wide[kMaxSet];       // of them those that form x W^T
  int ranks[kMaxSet];      // blocks of 32 of the rank
  bool even[kMaxSet];
  int count;
};

// Both in one launch, for up to 16 MT rows: workgroups that form s and workgroups
// that form x W^T.  Neither waits for the other, and the weights, whose bytes
// bound the call, are read while s is formed.
template <class T, int MT>
__global__ __launch_bounds__(kThreads) void adapter_both_kernel(const AdapterSet<T> set) {
  constexpr int NT = 2;
  __shared__ union {
    Meet<NT * MT> wide;
    struct {
      Meet<NT> meet;
      int rows[16];
    } down;
  } lds;
  const int block = static_cast<int>(blockIdx.x);
  int j = 0;
  while (j + 1 < set.count && block >= set.first[j + 1]) ++j;
  const Adapters<T>& a = set.p[j];
  const int b = block - set.first[j];
  if (b < set.wide[j]) {
    wide_body<T, MT, NT>(a, b, lds.wide);
    return;
  }
  const int d = b - set.wide[j], part = d % a.splits, ranks = d / a.splits % set.ranks[j];
  const int row = d / a.splits / set.ranks[j];
  if (set.even[j])
    down_body<T, true, NT>(a, row, part, ranks, set.ranks[j], lds.down.meet, lds.down.rows);
  else
    down_body<T, false, NT>(a, row, part, ranks, set.ranks[j], lds.down.meet, lds.down.rows);
}

// y of 16 rows with one id (an adapter, none, or a missing one), the workgroup's four
// waves 64 columns each in turn.
template <class T, bool EVEN>
__device__ __forceinline__ void up_body(const Adapters<T>& a, LowRows<T, 16, kMaxRank>& low, int* rowS) {
  const int id = adapter_of(a, blockIdx.x), count = gather_rows<16>(a, blockIdx.x, id, rowS);
  if (count == 0) return;
  const int c0 = 64 * (4 * blockIdx.y + (threadIdx.x >> 6));
  UpLoads<T, EVEN> first;
  first.ask(a, id, c0);
  const float c = factor(a, id);
  if (id >= 0) {
    const int quads = (a.rank + 31) / 32 * 8;
    for (int i = threadIdx.x; i < 16 * quads; i += 256) {
      const int r = i / quads, j = i % quads * 4;
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      if (r < count) {
        const float* p = a.s + static_cast<int64_t>(rowS[r]) * a.rank + j;
        for (int u = 0; u < a.splits; ++u, p += a.rows * a.rank) {
          if constexpr (EVEN) {
            if (j < a.rank) {
              const ad_f32x4 v = *reinterpret_cast<const ad_f32x4*>(p);
#pragma unroll
              for (int e = 0; e < 4; ++e) sum[e] += v[e];
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (j + e < a.rank) sum[e] += p[e];
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) low.put(r, j + e, sum[e]);
    }
    __syncthreads();
  }
  const int li = threadIdx.x & 15;
  const int rows[1] = {li < count ? rowS[li] : -1};
  up_all<T, EVEN, 1>(a, id, c, first, low, rows, c0, 256 * gridDim.y);
}

template <class T, bool EVEN>
__global__ __launch_bounds__(256) void adapter_up_kernel(const Adapters<T> a) {
  __shared__ LowRows<T, 16, kMaxRank> low;
  __shared__ int rowS[16];
  up_body<T, EVEN>(a, low, rowS);
}

template <class T>
__global__ __launch_bounds__(256) void adapter_up_set_kernel(const AdapterSet<T> set) {
  __shared__ LowRows<T, 16, kMaxRank> low;
  __shared__ int rowS[16];
  const Adapters<T>& a = set.p[blockIdx.z];
  if (256 * static_cast<int>(blockIdx.y) >= a.out) return;
  if (set.even[blockIdx.z])
    up_body<T, true>(a, low, rowS);
  else
    up_body<T, false>(a, low, rowS);
}

}  // namespace kda

namespace kda_host {

using namespace kda;

// A launch has fewer than 2^32 threads along its rows: 512 for 32 of them.
constexpr int64_t kRowsLimit = (int64_t{1} << 32) / kThreads * 32;
int64_t adapter_rows_limit() { return kRowsLimit; }

// Few rows whose ids may lie in any order go by adapter, the rest by runs.
static bool by_adapter(const kda_adapter_args& d) { return d.rows <= kAnyOrder && d.span < 16; }

// Parts of the columns of A x: of 1024, so that a wave has two slices, up to eight.
static int column_splits(const kda_adapter_args& d) {
  const int64_t n = (d.d_in + 1023) / 1024;
  return static_cast<int>(n < 8 ? n : 8);
}

// Parts of the columns of x W^T: four slices a wave at most (one round of loads),
// and 256 workgroups where a wave keeps two slices.
static int wide_parts(const kda_adapter_args& d) {
  const int64_t slices = d.d_in / 64, across = (d.d_out + 31) / 32;
  const int64_t fit = (slices + 31) / 32, fill = (255 + across) / across, most = slices / 16;
  const int64_t n = fill < most ? fill : most;
  return static_cast<int>(n > fit ? n : fit);
}

// The projection of few rows beside the adapters, in this library's own kernel.
bool adapter_takes_projection(const kda_adapter_args& d) {
  const uintptr_t bits = reinterpret_cast<uintptr_t>(d.x) | reinterpret_cast<uintptr_t>(d.a) |
                         reinterpret_cast<uintptr_t>(d.weight);
  return d.dtype != KDA_DTYPE_F32 && by_adapter(d) && d.rows <= 32 && d.d_in % 64 == 0 && bits % 16 == 0;
}

static int64_t s_floats(const kda_adapter_args& d) {
  return by_adapter(d) && d.adapters > 0 ? (static_cast<int64_t>(column_splits(d)) * d.rows * d.rank + 7) / 8 * 8 : 0;
}

size_t adapter_workspace_bytes(const kda_adapter_args& d) {
  const int64_t wide = d.weight != nullptr ? wide_parts(d) * d.rows * d.d_out : 0;
  return static_cast<size_t>(s_floats(d) + wide) * 4;
}

template <class T>
static Adapters<T> adapters_of(const kda_adapter_args& d) {
  Adapters<T> a{};
  a.x = static_cast<const T*>(d.x), a.a = static_cast<const T*>(d.a), a.b = static_cast<const T*>(d.b);
  a.bias = static_cast<const T*>(d.bias), a.scaling = d.scaling, a.ids = d.ids, a.ids64 = d.ids_are_int64;
  a.span = static_cast<int>(d.span < d.rows ? d.span : d.rows), a.rows = d.rows;
  a.in = static_cast<int>(d.d_in), a.out = static_cast<int>(d.d_out);
  a.rank = static_cast<int>(d.rank), a.n = static_cast<int>(d.adapters), a.splits = column_splits(d);
  a.y = static_cast<T*>(d.y), a.s = static_cast<float*>(d.workspace);
  return a;
}

static bool even_call(const kda_adapter_args& d) {
  const void* ptrs[] = {d.x, d.a, d.b, d.y, d.bias};
  uintptr_t bits = 0;
  for (const void* p : ptrs) bits |= reinterpret_cast<uintptr_t>(p);
  return d.d_in % kSlice64 == 0 && d.d_out % 64 == 0 && d.rank % 8 == 0 && bits % 16 == 0;
}

// Workgroups along the columns: about a thousand in all, whose rows are found once.
static unsigned up_blocks(int64_t out, int64_t rows) {
  const int64_t blocks = (out + 255) / 256, fill = (1023 + rows) / rows;
  return static_cast<unsigned>(blocks < fill ? blocks : fill);
}

template <class T, bool EVEN>
static void launch_delta(const Adapters<T>& a, bool any_order, hipStream_t s) {
  if (!any_order) {
    // 16 rows a workgroup while 32 would leave CUs empty (2048 -> 2048 rank 16, the whole
    // call on inputs from HBM: 2000 rows 42 us against 49 with 32, 4096 rows 70 against 63,
    // 8195 rows 121 against 124)
    auto go = [&](auto kernel, int rows) {
      const dim3 grid(static_cast<unsigned>((a.rows + rows - 1) / rows), kRunTurns);
      hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, s, a);
    };
    if (a.rows <= 2048) {
      if (a.rank <= 16) go(adapter_run_kernel<T, EVEN, 1, 1>, 16);
      else if (a.rank <= 32) go(adapter_run_kernel<T, EVEN, 1, 2>, 16);
      else go(adapter_run_kernel<T, EVEN, 1, 4>, 16);
    } else {
      if (a.rank <= 16) go(adapter_run_kernel<T, EVEN, 2, 1>, 32);
      else if (a.rank <= 32) go(adapter_run_kernel<T, EVEN, 2, 2>, 32);
      else go(adapter_run_kernel<T, EVEN, 2, 4>, 32);
    }
    return;
  }
  // 32 of the rank a workgroup while all of them run at once: most of many rows'
  // workgroups have nothing to do, and a second round of them waits
  const int64_t ranks = (a.rank + 31) / 32, fill = 1024 / (a.rows * a.splits);
  const dim3 grid(static_cast<unsigned>(a.rows), a.splits, static_cast<unsigned>(fill < 1 ? 1 : fill < ranks ? fill : ranks));
  if (a.rank <= 16)
    hipLaunchKernelGGL((adapter_down_kernel<T, EVEN, 1>), grid, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((adapter_down_kernel<T, EVEN, 2>), grid, dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL((adapter_up_kernel<T, EVEN>), dim3(static_cast<unsigned>(a.rows), up_blocks(a.out, a.rows)),
                     dim3(256), 0, s, a);
}

template <class T>
static int run_adapter_delta(const kda_adapter_args& d, const float* product, hipStream_t s) {
  Adapters<T> a = adapters_of<T>(d);
  if (product != nullptr) a.wide = const_cast<float*>(product), a.parts = 1;  // read only
  if (even_call(d) && reinterpret_cast<uintptr_t>(product) % 16 == 0)
    launch_delta<T, true>(a, by_adapter(d), s);
  else
    launch_delta<T, false>(a, by_adapter(d), s);
  return check_launch("adapter_delta");
}

int launch_adapter_delta(const kda_adapter_args& d, const float* product, hipStream_t s) {
  switch (d.dtype) {
    case KDA_DTYPE_BF16: return run_adapter_delta<bf16>(d, product, s);
    case KDA_DTYPE_F16: return run_adapter_delta<f16>(d, product, s);
    default: return run_adapter_delta<float>(d, product, s);
  }
}

template <class T>
static int run_adapter_set(const kda_adapter_args* calls, int count, hipStream_t s) {
  AdapterSet<T> set{};
  set.count = count;
  int64_t blocks = 0;
  unsigned columns = 1;
  for (int j = 0; j < count; ++j) {
    const kda_adapter_args& d = calls[j];
    Adapters<T>& a = set.p[j];
    a = adapters_of<T>(d);
    a.weight = static_cast<const T*>(d.weight), a.wide = a.s + s_floats(d), a.parts = wide_parts(d);
    set.even[j] = even_call(d);
    set.first[j] = static_cast<int>(blocks);
    set.wide[j] = a.parts * ((a.out + 31) / 32);  // 2^30 at most
    set.ranks[j] = (a.rank + 31) / 32;
    blocks += set.wide[j] + (a.n != 0 ? a.rows * a.splits * set.ranks[j] : 0);
    if (blocks > 0x7fffffffLL) {
      set_detail("adapter_linear: grid too large");
      return KDA_ERR_UNSUPPORTED;
    }
    const unsigned n = up_blocks(a.out, a.rows * count);
    columns = n > columns ? n : columns;
  }
  set.first[count] = static_cast<int>(blocks);
  const int64_t rows = calls[0].rows;
  if (rows <= 16)
    hipLaunchKernelGGL((adapter_both_kernel<T, 1>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, s, set);
  else
    hipLaunchKernelGGL((adapter_both_kernel<T, 2>), dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, s, set);
  hipLaunchKernelGGL((adapter_up_set_kernel<T>), dim3(static_cast<unsigned>(rows), columns, count), dim3(256), 0, s, set);
  return check_launch("adapter_linear");
}

int launch_adapter_set(const kda_adapter_args* calls, int count, hipStream_t s) {
  if (count > kMaxSet) {
    set_detail("adapter_linear: %d projections at once", count);
    return KDA_ERR_UNSUPPORTED;
  }
  return calls[0].dtype == KDA_DTYPE_BF16 ? run_adapter_set<bf16>(calls, count, s)
                                          : run_adapter_set<f16>(calls, count, s);
}

}  // namespace kda_host
