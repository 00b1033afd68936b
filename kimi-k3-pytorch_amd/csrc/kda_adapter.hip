// Low-rank adapters of many requests beside a shared projection:
//   y_m = W x_m + bias + c_a B_a (A_a x_m),  a = the adapter of row m, or none.
// Row m's adapter is ids[m / span]: a negative id has none, an id past the stack
// gives a row of NaN (the host cannot see it without waiting for the GPU).
//
// Two passes: s_m = A_a x_m in f32 (down), then c_a B_a s_m (up).  Rows that share
// an adapter share its reading; whose rows they are is found by the kernels
// themselves, so a call needs no sorted batch and no plan:
//  - long runs (a prompt's tokens): a workgroup owns 64 neighbouring rows and goes
//    through the adapters it meets in them, mostly one;
//  - few rows in any order (decode): the workgroup of row i counts the earlier rows
//    with row i's adapter; where their number is a multiple of 16 it owns the next
//    16 such rows, otherwise it has nothing to do.
#include "kda_launch.h"

namespace kda {

typedef float ad_f32x4 __attribute__((ext_vector_type(4)));

template <class T>
struct Frag {
  typedef T type __attribute__((ext_vector_type(8)));
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

// Eight columns from k of a row of `len`; FULL: rows of whole vectors at aligned
// addresses.  Columns past the row are zeros.
template <class T, bool FULL>
__device__ __forceinline__ typename Frag<T>::type load8(const T* row, int k, int len) {
  typename Frag<T>::type v{};
  if constexpr (FULL) {
    if (k < len) v = *reinterpret_cast<const typename Frag<T>::type*>(row + k);
  } else if (k + 8 <= len) {
    v = *reinterpret_cast<const typename Frag<T>::loose*>(row + k);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < len) v[e] = row[k + e];
  }
  return v;
}

template <class T>
struct Adapters {
  const T *x, *a, *b, *bias;  // x [rows, in], a [n, rank, in], b [n, out, rank], bias [out] or null
  const float* scaling;       // [n] or null (1)
  const void* ids;            // int32 or int64
  int ids64;
  int64_t rows;
  int span, in, out, rank, n, splits;
  T* y;      // [rows, out]
  float* s;  // [splits, rows, rank]: sums over a part of the columns each
};

constexpr int kNone = -1, kMissing = -2;

// the row's adapter, kNone or kMissing
template <class T>
__device__ __forceinline__ int adapter_of(const Adapters<T>& a, int64_t row) {
  const unsigned i = static_cast<unsigned>(row) / static_cast<unsigned>(a.span);  // rows < 2^31
  const int64_t id = a.ids64 != 0 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
  return id < 0 ? kNone : (id < a.n ? static_cast<int>(id) : kMissing);
}

__device__ __forceinline__ int below(uint64_t mask, int lane) {  // set bits under the lane's
  return __popcll(mask & ((uint64_t{1} << lane) - 1));
}

// ---- s = A x -------------------------------------------------------------------
// A workgroup of four waves: 16 MT rows of one adapter, 16 NT of its rank, a part
// of the columns, the waves every fourth 64-column slice of it; their sums meet
// in LDS.  RUNS: 64 neighbouring rows, adapter by adapter.
constexpr int kDownWaves = 4;
constexpr int kAnyOrder = 512;  // rows in any order, at most
constexpr int kSlice64 = 64;

template <class T, bool FULL, int MT, int NT, bool RUNS>
__global__ __launch_bounds__(64 * kDownWaves) void adapter_down_kernel(const Adapters<T> a) {
  using v8 = typename Frag<T>::type;
  constexpr int R = 16 * MT;
  __shared__ int rowS[R];
  __shared__ __attribute__((aligned(16))) float red[kDownWaves][NT * MT][256];
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j0 = blockIdx.z * 16 * NT;
  const int slices = (a.in + kSlice64 - 1) / kSlice64, per = (slices + a.splits - 1) / a.splits;
  const int first = blockIdx.y * per, last = first + per < slices ? first + per : slices;
  float* s = a.s + static_cast<int64_t>(blockIdx.y) * a.rows * a.rank;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (RUNS ? R : 1);

  int id, count;
  uint64_t pending = 0;
  int mine = kNone;  // RUNS: the adapter of the lane's row
  if constexpr (RUNS) {
    static_assert(R <= 64, "a lane per row");
    if (lane < R && row0 + lane < a.rows) mine = adapter_of(a, row0 + lane);
    pending = __ballot(mine >= 0);
    if (pending == 0) return;
  } else {
    id = adapter_of(a, row0);
    if (id < 0) return;
    int of[kAnyOrder / 64];
#pragma unroll
    for (int u = 0; u < kAnyOrder / 64; ++u) of[u] = 64 * u + lane < a.rows ? adapter_of(a, 64 * u + lane) : kNone;
    const int self = static_cast<int>(row0);
    int before = 0;
#pragma unroll
    for (int u = 0; u < kAnyOrder / 64; ++u) before += __popcll(__ballot(of[u] == id && 64 * u + lane < self));
    if (before % R != 0) return;
    count = 0;
#pragma unroll
    for (int u = 0; u < kAnyOrder / 64; ++u) {
      const bool same = of[u] == id && 64 * u + lane >= self;
      const uint64_t mask = __ballot(same);
      const int at = count + below(mask, lane);
      if (same && at < R && w == 0) rowS[at] = 64 * u + lane;
      count += __popcll(mask);
    }
    count = count < R ? count : R;
    __syncthreads();
  }
  do {
    if constexpr (RUNS) {
      id = __shfl(mine, __ffsll(static_cast<unsigned long long>(pending)) - 1);
      const uint64_t mask = __ballot(mine == id);
      pending &= ~mask;
      count = __popcll(mask);
      if (w == 0 && mine == id) rowS[below(mask, lane)] = static_cast<int>(row0) + lane;
      __syncthreads();
    }
    const T *ap[NT], *xp[MT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {  // rows past the rank repeat its last one; their sums are dropped
      const int j = j0 + 16 * t + li;
      ap[t] = a.a + (static_cast<int64_t>(id) * a.rank + (j < a.rank ? j : a.rank - 1)) * a.in;
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int r = 16 * t + li;
      xp[t] = a.x + static_cast<int64_t>(rowS[r < count ? r : count - 1]) * a.in;
    }
    ad_f32x4 acc[NT][MT];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[t][m] = ad_f32x4{0.f, 0.f, 0.f, 0.f};
    // E half slices in flight: of one slice with four row tiles, of two with one
    constexpr int E = MT == 1 ? 4 : 2;
    for (int c = first + w; c < last; c += kDownWaves * E / 2) {
      v8 av[NT][E], xv[MT][E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int slice = c + kDownWaves * (e / 2);
        const int k = slice < last ? slice * kSlice64 + 32 * (e & 1) + 8 * g : a.in;  // past the part: zeros
#pragma unroll
        for (int t = 0; t < NT; ++t) av[t][e] = load8<T, FULL>(ap[t], k, a.in);
#pragma unroll
        for (int m = 0; m < MT; ++m)
          if (16 * m < count) xv[m][e] = load8<T, FULL>(xp[m], k, a.in);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
        if (16 * m < count) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < E; ++e) acc[t][m] = mma(av[t][e], xv[m][e], acc[t][m]);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m) *reinterpret_cast<ad_f32x4*>(&red[w][t * MT + m][4 * lane]) = acc[t][m];
    __syncthreads();
    for (int i = tid; i < NT * MT * 256; i += 64 * kDownWaves) {
      const int jl = i % (16 * NT), rl = i / (16 * NT), j = j0 + jl;
      const int at = 4 * ((rl & 15) + 16 * ((jl & 15) >> 2)) + (jl & 3), tile = (jl >> 4) * MT + (rl >> 4);
      if (rl < count && j < a.rank) {
        float sum = red[0][tile][at];
#pragma unroll
        for (int v = 1; v < kDownWaves; ++v) sum += red[v][tile][at];
        s[static_cast<int64_t>(rowS[rl]) * a.rank + j] = sum;
      }
    }
    if constexpr (RUNS) __syncthreads();  // before the next adapter's rows
  } while (RUNS && pending != 0);
}

// ---- y = bias + c B s, 64 neighbouring rows -----------------------------------
// A workgroup of four waves: 64 rows, 64 columns a wave.  The sums s meet in LDS,
// 64 of the rank at a time.  bf16: s as two bf16 values (2^-17 of it is left) on
// bf16 products; f16 and f32: f32 products (f16 has not the range of s).
template <class T>
struct UpType {
  using type = float;
};
template <>
struct UpType<bf16> {
  using type = bf16;
};

constexpr int kUpRows = 64, kUpCols = 256, kUpRank = 64;

template <class T>
__global__ __launch_bounds__(256) void adapter_up_tile_kernel(const Adapters<T> a) {
  using U = typename UpType<T>::type;
  using v8 = typename Frag<U>::type;
  constexpr int P = sizeof(U) == 2 ? 2 : 1;  // parts of s
  constexpr int LD = kUpRank + 8;
  __shared__ __attribute__((aligned(16))) U sS[P][kUpRows][LD];
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, g = lane >> 4, w = tid >> 6;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kUpRows;
  const int c0 = blockIdx.y * kUpCols + 64 * w;
  int mine = kNone;  // adapter of row `lane`
  if (row0 + lane < a.rows) mine = adapter_of(a, row0 + lane);
  int of[4];  // adapters of the four rows the lane's results belong to
#pragma unroll
  for (int m = 0; m < 4; ++m) of[m] = __shfl(mine, 16 * m + li);
  ad_f32x4 y[4][4];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const float start = of[m] == kMissing ? __builtin_nanf("") : 0.f;
      y[t][m] = ad_f32x4{start, start, start, start};
    }
  const uint64_t some = __ballot(mine >= 0);
  for (int r0 = 0; some != 0 && r0 < a.rank; r0 += kUpRank) {
    if (r0 != 0) __syncthreads();
    for (int i = tid; i < kUpRows * kUpRank; i += 256) {
      const int r = i / kUpRank, j = i % kUpRank;
      float s = 0.f;
      if (r0 + j < a.rank && row0 + r < a.rows) {
        const float* p = a.s + (row0 + r) * a.rank + r0 + j;
        for (int u = 0; u < a.splits; ++u) s += p[static_cast<int64_t>(u) * a.rows * a.rank];
      }
      const U hi = static_cast<U>(s);
      sS[0][r][j] = hi;
      if constexpr (P == 2) sS[1][r][j] = static_cast<U>(s - static_cast<float>(hi));
    }
    __syncthreads();
    const int left = a.rank - r0 < kUpRank ? a.rank - r0 : kUpRank;
    for (uint64_t pending = some; pending != 0;) {
      const int id = __shfl(mine, __ffsll(static_cast<unsigned long long>(pending)) - 1);
      pending &= ~__ballot(mine == id);
      const float c = a.scaling != nullptr ? a.scaling[id] : 1.f;
      const T* b = a.b + static_cast<int64_t>(id) * a.out * a.rank + r0;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int col = c0 + 16 * t + li;
        const T* row = b + static_cast<int64_t>(col < a.out ? col : a.out - 1) * a.rank;
        ad_f32x4 d[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) d[m] = ad_f32x4{0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < left; k += 32) {
          const auto raw = load8<T, false>(row, k + 8 * g, left);
          v8 bv;
#pragma unroll
          for (int e = 0; e < 8; ++e) bv[e] = static_cast<U>(raw[e]);
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int p = 0; p < P; ++p)
              d[m] = mma(bv, *reinterpret_cast<const v8*>(&sS[p][16 * m + li][k + 8 * g]), d[m]);
        }
#pragma unroll
        for (int m = 0; m < 4; ++m)
          if (of[m] == id) y[t][m] += c * d[m];  // rows of other adapters: dropped, not weighted by zero
      }
    }
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int col = c0 + 16 * t + 4 * g;
    float bias[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = a.bias != nullptr && col + e < a.out ? to_float(a.bias[col + e]) : 0.f;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int64_t row = row0 + 16 * m + li;
      if (row >= a.rows) continue;
      T* out = a.y + row * a.out + col;
      typedef T o4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
      if (col + 4 <= a.out) {
        o4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = from_compute<T>(y[t][m][e] + bias[e]);
        *reinterpret_cast<o4*>(out) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < a.out) out[e] = from_compute<T>(y[t][m][e] + bias[e]);
      }
    }
  }
}

// ---- y = bias + c B s, a row a workgroup (few rows in any order) ----------------
constexpr int kUpRowCols = 256;

template <class T>
__global__ __launch_bounds__(256) void adapter_up_row_kernel(const Adapters<T> a) {
  __shared__ float sS[256];
  const int64_t row = blockIdx.x;
  const int id = adapter_of(a, row), col = blockIdx.y * kUpRowCols + threadIdx.x;
  if (id >= 0) {
    if (static_cast<int>(threadIdx.x) < a.rank) {
      float s = 0.f;
      for (int u = 0; u < a.splits; ++u) s += a.s[(u * a.rows + row) * a.rank + threadIdx.x];
      sS[threadIdx.x] = s;
    }
    __syncthreads();
  }
  if (col >= a.out) return;
  float y = id == kMissing ? __builtin_nanf("") : 0.f;
  if (id >= 0) {
    const T* b = a.b + (static_cast<int64_t>(id) * a.out + col) * a.rank;
    for (int j = 0; j < a.rank; j += 8) {
      const auto v = load8<T, false>(b, j, a.rank);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (j + e < a.rank) y += sS[j + e] * to_float(static_cast<T>(v[e]));
    }
    if (a.scaling != nullptr) y *= a.scaling[id];
  }
  if (a.bias != nullptr) y += to_float(a.bias[col]);
  a.y[row * a.out + col] = from_compute<T>(y);
}

}  // namespace kda

namespace kda_host {

using namespace kda;

// Few rows whose ids may lie in any order go by adapter, the rest by runs.
static bool by_adapter(const kda_adapter_args& d) { return d.rows <= kAnyOrder && d.span < 16; }

// Parts of the columns: of 512, so that a wave has two slices, up to eight parts
// and, of runs, as many as make a thousand workgroups.
static int column_splits(const kda_adapter_args& d) {
  const int64_t n = (d.d_in + 511) / 512, tiles = (d.rows + 63) / 64;
  const int64_t most = by_adapter(d) ? 8 : (1023 + tiles) / tiles < 8 ? (1023 + tiles) / tiles : 8;
  return static_cast<int>(n < most ? n : most);
}

size_t adapter_delta_workspace_bytes(const kda_adapter_args& d) {
  return static_cast<size_t>(column_splits(d)) * d.rows * d.rank * 4;
}

template <class T, bool FULL, int MT, bool RUNS>
static void launch_down(const Adapters<T>& a, int64_t blocks, hipStream_t s) {
  auto go = [&](auto kernel, int ranks) {
    const dim3 grid(static_cast<unsigned>(blocks), a.splits, static_cast<unsigned>((a.rank + ranks - 1) / ranks));
    hipLaunchKernelGGL(kernel, grid, dim3(64 * kDownWaves), 0, s, a);
  };
  if (a.rank <= 16)
    go(adapter_down_kernel<T, FULL, MT, 1, RUNS>, 16);
  else
    go(adapter_down_kernel<T, FULL, MT, 2, RUNS>, 32);
}

template <class T>
static int run_adapter_delta(const kda_adapter_args& d, hipStream_t s) {
  Adapters<T> a{};
  a.x = static_cast<const T*>(d.x), a.a = static_cast<const T*>(d.a), a.b = static_cast<const T*>(d.b);
  a.bias = static_cast<const T*>(d.bias), a.scaling = d.scaling, a.ids = d.ids, a.ids64 = d.ids_are_int64;
  a.span = static_cast<int>(d.span < d.rows ? d.span : d.rows), a.rows = d.rows, a.in = static_cast<int>(d.d_in), a.out = static_cast<int>(d.d_out);
  a.rank = static_cast<int>(d.rank), a.n = static_cast<int>(d.adapters), a.splits = column_splits(d);
  a.y = static_cast<T*>(d.y), a.s = static_cast<float*>(d.workspace);
  const bool full = d.d_in % 8 == 0 &&
                    (reinterpret_cast<uintptr_t>(d.x) | reinterpret_cast<uintptr_t>(d.a)) % (8 * sizeof(T)) == 0;
  if (by_adapter(d)) {
    if (full)
      launch_down<T, true, 1, false>(a, a.rows, s);
    else
      launch_down<T, false, 1, false>(a, a.rows, s);
    hipLaunchKernelGGL((adapter_up_row_kernel<T>),
                       dim3(static_cast<unsigned>(a.rows), static_cast<unsigned>((a.out + kUpRowCols - 1) / kUpRowCols)),
                       dim3(256), 0, s, a);
  } else {
    const int64_t tiles = (a.rows + 63) / 64;
    if (full)
      launch_down<T, true, 4, true>(a, tiles, s);
    else
      launch_down<T, false, 4, true>(a, tiles, s);
    hipLaunchKernelGGL((adapter_up_tile_kernel<T>),
                       dim3(static_cast<unsigned>(tiles), static_cast<unsigned>((a.out + kUpCols - 1) / kUpCols)),
                       dim3(256), 0, s, a);
  }
  return check_launch("adapter_delta");
}

int launch_adapter_delta(const kda_adapter_args& d, hipStream_t s) {
  switch (d.dtype) {
    case KDA_DTYPE_BF16: return run_adapter_delta<bf16>(d, s);
    case KDA_DTYPE_F16: return run_adapter_delta<f16>(d, s);
    default: return run_adapter_delta<float>(d, s);
  }
}

}  // namespace kda_host
