// RMSNorm with the residual's addition, its backward, and its 8-bit output.
//
//   h = round(x + r);  s = 1 / sqrt(mean(h^2) + eps);  y = h s w
// over rows of `width` elements; the norm reads the stored (rounded) sum, so
// the backward, which has h alone, differentiates the function that ran.  With
// 8-bit output, over each group of a row (or the row):
//   scale = max|y| / 448,  q = e4m3(y / scale)   (448: e4m3's largest value; y, scale
//                                                 and quotient in f32)
// and a group whose largest magnitude is under 2^-100 has scale 0 and zeros:
// its quotients would leave f32.
// Backward, with the gradients dy and dh of the two outputs:
//   dx = dr = dh + s (w dy - h s^2 mean(w dy h)),  dw = sum over rows of dy h s.
#include <initializer_list>

#include "kda_launch.h"

namespace kda {

template <class T>
struct NormCompute {
  using type = float;
};
template <>
struct NormCompute<double> {
  using type = double;
};

constexpr float kTinyGroup = 0x1p-100f;
constexpr float kE4m3Max = 448.f;

// The larger one, a NaN if either is.
template <class C>
__device__ __forceinline__ C nan_max(C a, C b) {
  return (a > b || a != a) ? a : b;
}

template <class T>
struct AddNorm {
  const T *x, *r;      // r: may be null
  const void* w;       // null, or of T, or (wide_w) f32
  bool wide_w;
  T *h, *y;            // h: null without a residual (h is x)
  uint8_t* q;          // e4m3, in place of y
  float* scales;       // [rows, width / group]
  int64_t rows, width, group;
  typename NormCompute<T>::type eps;
};

template <class T>
__device__ __forceinline__ typename NormCompute<T>::type norm_weight(const void* w, bool wide, int64_t c) {
  if (wide) return static_cast<const float*>(w)[c];
  return to_compute<typename NormCompute<T>::type>(static_cast<const T*>(w)[c]);
}

template <class C>
__device__ __forceinline__ C block_sum(C v, C* part) {  // over a workgroup of four waves
  v = group_sum<64>(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
  __syncthreads();
  return (part[0] + part[1]) + (part[2] + part[3]);
}

__device__ __forceinline__ uint8_t to_e4m3(float v) {
  return static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xff);
}

// The scale of a group's largest magnitude, zero for a tiny one, and y over it: the f32
// quotient itself, as the definition has it (a product with the rounded 448 / m
// falls to the other side of some ties).
__device__ __forceinline__ float group_scale(float m) { return m < kTinyGroup ? 0.f : m / kE4m3Max; }
__device__ __forceinline__ float scaled(float y, float scale) { return scale == 0.f ? 0.f : y / scale; }

// Any width, one workgroup a row, the sum kept in h (in x without a residual)
// between the passes.  Where a row has several groups, a wave reads back sums that
// other waves wrote: the barriers in block_sum order them.
template <class T, bool Q>
__global__ __launch_bounds__(256) void add_norm_row_kernel(const AddNorm<T> a) {
  using C = typename NormCompute<T>::type;
  __shared__ C part[4];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x, D = a.width, at = row * D;
  const T* src = a.r != nullptr ? a.h : a.x;
  C ss = C(0);
  for (int64_t c = tid; c < D; c += 256) {
    T h = a.x[at + c];
    if (a.r != nullptr) {
      h = from_compute<T>(to_compute<C>(h) + to_compute<C>(a.r[at + c]));
      a.h[at + c] = h;
    }
    ss += to_compute<C>(h) * to_compute<C>(h);
  }
  const C s = frsqrt(block_sum(ss, part) / C(D) + a.eps);
  auto value = [&](int64_t c) -> C {
    const C v = to_compute<C>(src[at + c]) * s;
    return a.w != nullptr ? v * norm_weight<T>(a.w, a.wide_w, c) : v;
  };
  if constexpr (!Q) {
    for (int64_t c = tid; c < D; c += 256) a.y[at + c] = from_compute<T>(value(c));
  } else {
    // a wave per group in turn; a single group is shared by the four waves
    __shared__ float top[4];
    const int lane = tid & 63, wave = tid >> 6;
    const bool whole = a.group == D;
    const int64_t step = whole ? 256 : 64, first = whole ? tid : lane;
    for (int64_t g = whole ? 0 : wave; g < D / a.group; g += whole ? 1 : 4) {
      float m = 0.f;
      for (int64_t c = first; c < a.group; c += step) m = nan_max(fabsf(static_cast<float>(value(g * a.group + c))), m);
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) m = nan_max(__shfl_xor(m, off), m);
      if (whole) {  // uniform: every thread of the workgroup is here
        if (lane == 0) top[wave] = m;
        __syncthreads();
        m = nan_max(nan_max(top[0], top[1]), nan_max(top[2], top[3]));
      }
      const float scale = group_scale(m);
      for (int64_t c = first; c < a.group; c += step)
        a.q[at + g * a.group + c] = to_e4m3(scaled(static_cast<float>(value(g * a.group + c)), scale));
      if (first == 0) a.scales[row * (D / a.group) + g] = scale;
    }
  }
}

// Bound: the rows' bytes, each read and written once.  8192 x 7168 bf16 (470 MB)
// 79 us, 5.9 TB/s; with e4m3 output 8192 x 4096 (236 MB) 41.4 us, 5.7 TB/s (39 with a
// product by 448 / m in place of the division); one workgroup a row through memory
// (add_norm_row_kernel) took 169 us for the latter.
// Rows in registers: TPR threads a row (a wave with four rows a workgroup, or the
// workgroup), NV vectors of 16 bytes a thread, every load of the row in flight
// before the sum, one pass over memory.  FULL: widths of whole vectors at aligned
// addresses; otherwise vectors load at element alignment (the hardware takes any
// address) and the row's last one element by element.
template <class T>
struct NormVec {
  static constexpr int N = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(N)));
  typedef T loose __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

template <class T, bool FULL>
__device__ __forceinline__ typename NormVec<T>::type norm_load(const T* row, int i, int width) {
  using V = NormVec<T>;
  typename V::type v{};
  const int c = i * V::N;
  if constexpr (FULL) {
    if (c < width) v = __builtin_nontemporal_load(reinterpret_cast<const typename V::type*>(row + c));
  } else {
    if (c + V::N <= width) {
      v = *reinterpret_cast<const typename V::loose*>(row + c);
    } else {
#pragma unroll
      for (int e = 0; e < V::N; ++e)
        if (c + e < width) v[e] = row[c + e];
    }
  }
  return v;
}

template <class T, bool FULL>
__device__ __forceinline__ void norm_store(T* row, int i, int width, typename NormVec<T>::type v) {
  using V = NormVec<T>;
  const int c = i * V::N;
  if constexpr (FULL) {
    if (c < width) __builtin_nontemporal_store(v, reinterpret_cast<typename V::type*>(row + c));
  } else {
    if (c + V::N <= width) {
      *reinterpret_cast<typename V::loose*>(row + c) = v;
    } else {
#pragma unroll
      for (int e = 0; e < V::N; ++e)
        if (c + e < width) row[c + e] = v[e];
    }
  }
}

// A weight's vector: read by every row, so no streaming load.
template <class T, bool FULL>
__device__ __forceinline__ typename NormVec<T>::type weight_load(const T* w, int i, int width) {
  if constexpr (FULL) {
    typename NormVec<T>::type v{};
    if (i * NormVec<T>::N < width) v = *reinterpret_cast<const typename NormVec<T>::type*>(w + i * NormVec<T>::N);
    return v;
  } else {
    return norm_load<T, false>(w, i, width);
  }
}

// The weights of vector i as floats (ones without any).
template <class T, bool FULL>
__device__ __forceinline__ void norm_weights(const void* w, bool wide, int i, int width, float (&out)[NormVec<T>::N]) {
  constexpr int N = NormVec<T>::N;
  if (w == nullptr) {
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = 1.f;
  } else if (!wide) {
    const typename NormVec<T>::type v = weight_load<T, FULL>(static_cast<const T*>(w), i, width);
#pragma unroll
    for (int e = 0; e < N; ++e) out[e] = to_float(static_cast<T>(v[e]));
  } else {
#pragma unroll
    for (int u = 0; u < N / 4; ++u) {
      const NormVec<float>::type v = weight_load<float, FULL>(static_cast<const float*>(w), i * (N / 4) + u, width);
#pragma unroll
      for (int e = 0; e < 4; ++e) out[4 * u + e] = v[e];
    }
  }
}

// Sum over the threads of a row (TPR == 64: the wave's).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* part) {
  v = group_sum<64>(v);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int u = 0; u < TPR / 64; ++u) v += part[u];
  }
  return v;
}

template <class T, bool Q, bool FULL, int TPR, int NV>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void add_norm_kernel(const AddNorm<T> a) {
  using V = NormVec<T>;
  constexpr int N = V::N;
  __shared__ float part[TPR / 64], top[TPR / 64];
  const int lane = TPR == 64 ? threadIdx.x & 63 : threadIdx.x;
  const int64_t row = TPR == 64 ? static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (TPR == 64 && row >= a.rows) return;  // whole waves; no barrier follows
  const int width = static_cast<int>(a.width);
  const int64_t at = row * width;
  typename V::type xv[NV], rv[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) xv[j] = norm_load<T, FULL>(a.x + at, lane + j * TPR, width);
  typename V::type wv[NV];  // asked for ahead of the sum
  if (a.w != nullptr && !a.wide_w) {
#pragma unroll
    for (int j = 0; j < NV; ++j) wv[j] = weight_load<T, FULL>(static_cast<const T*>(a.w), lane + j * TPR, width);
  }
  float ss = 0.f;
  if (a.r != nullptr) {
#pragma unroll
    for (int j = 0; j < NV; ++j) rv[j] = norm_load<T, FULL>(a.r + at, lane + j * TPR, width);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        xv[j][e] = from_compute<T>(to_float(static_cast<T>(xv[j][e])) + to_float(static_cast<T>(rv[j][e])));
      norm_store<T, FULL>(a.h + at, lane + j * TPR, width, xv[j]);
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float h = to_float(static_cast<T>(xv[j][e]));
      ss += h * h;
    }
  const float s = frsqrt(row_sum<TPR>(ss, part) / static_cast<float>(width) + a.eps);
  float y[NV][N];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = lane + j * TPR;
#pragma unroll
    for (int e = 0; e < N; ++e) y[j][e] = to_float(static_cast<T>(xv[j][e])) * s;
    if (a.w != nullptr && !a.wide_w) {
#pragma unroll
      for (int e = 0; e < N; ++e) y[j][e] *= to_float(static_cast<T>(wv[j][e]));
    } else if (a.w != nullptr) {
      float w[N];
      norm_weights<T, FULL>(a.w, true, i, width, w);
#pragma unroll
      for (int e = 0; e < N; ++e) y[j][e] *= w[e];
    }
  }
  if constexpr (!Q) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      typename V::type o;
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = from_compute<T>(y[j][e]);
      norm_store<T, FULL>(a.y + at, lane + j * TPR, width, o);
    }
  } else {
    // lanes of a group; a row's single group: all of them
    const bool whole = a.group == width;
    const int lanes = whole ? 64 : static_cast<int>(a.group) / N;
    float m[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      m[j] = 0.f;
#pragma unroll
      for (int e = 0; e < N; ++e) m[j] = nan_max(fabsf(y[j][e]), m[j]);
    }
    if (whole) {
#pragma unroll
      for (int j = 1; j < NV; ++j) m[0] = nan_max(m[j], m[0]);
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) m[0] = nan_max(__shfl_xor(m[0], off), m[0]);
      if constexpr (TPR > 64) {
        if ((lane & 63) == 0) top[lane >> 6] = m[0];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < TPR / 64; ++u) m[0] = nan_max(top[u], m[0]);
      }
#pragma unroll
      for (int j = 1; j < NV; ++j) m[j] = m[0];
    } else {
      for (int off = 1; off < lanes; off <<= 1)
#pragma unroll
        for (int j = 0; j < NV; ++j) m[j] = nan_max(__shfl_xor(m[j], off), m[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int i = lane + j * TPR, c = i * N;
      const float scale = group_scale(m[j]);
      if (c < width) {
        if (whole ? i == 0 : i % lanes == 0)
          a.scales[whole ? row : row * (width / a.group) + c / a.group] = scale;
        uint8_t* q = a.q + at + c;
        unsigned word[N / 4];
#pragma unroll
        for (int u = 0; u < N / 4; ++u) {
          const float* v = &y[j][4 * u];
          int p = __builtin_amdgcn_cvt_pk_fp8_f32(scaled(v[0], scale), scaled(v[1], scale), 0, false);
          word[u] = static_cast<unsigned>(__builtin_amdgcn_cvt_pk_fp8_f32(scaled(v[2], scale), scaled(v[3], scale), p, true));
        }
        if (FULL || c + N <= width) {
          struct __attribute__((packed, aligned(FULL ? N : 1))) Bytes {
            unsigned w[N / 4];
          };
          Bytes b;
#pragma unroll
          for (int u = 0; u < N / 4; ++u) b.w[u] = word[u];
          *reinterpret_cast<Bytes*>(q) = b;
        } else {
#pragma unroll
          for (int e = 0; e < N; ++e)
            if (c + e < width) q[e] = static_cast<uint8_t>(word[e / 4] >> (8 * (e % 4)));
        }
      }
    }
  }
}

template <class T>
struct AddNormBwd {
  const T *h, *dy, *dh;      // dh: may be null
  const void* w;             // null, or of T, or (wide_w) f32; the gradient dw alike
  bool wide_w;
  T* dx;
  void* dw;                  // may be null
  typename NormCompute<T>::type* s;     // [rows], for the weight gradient
  typename NormCompute<T>::type* part;  // [chunks, width] partial weight gradients
  int64_t rows, width, chunk;
  typename NormCompute<T>::type eps;
};

template <class T>
__global__ __launch_bounds__(256) void add_norm_bwd_row_kernel(const AddNormBwd<T> a) {
  using C = typename NormCompute<T>::type;
  __shared__ C part[4];
  const int64_t row = blockIdx.x, D = a.width, at = row * D;
  C ss = C(0), dot = C(0);
  auto wdy = [&](int64_t c) -> C {
    const C v = to_compute<C>(a.dy[at + c]);
    return a.w != nullptr ? v * norm_weight<T>(a.w, a.wide_w, c) : v;
  };
  for (int64_t c = threadIdx.x; c < D; c += 256) {
    const C h = to_compute<C>(a.h[at + c]);
    ss += h * h;
    dot += wdy(c) * h;
  }
  const C s = frsqrt(block_sum(ss, part) / C(D) + a.eps);
  const C back = s * s * (block_sum(dot, part) / C(D));
  for (int64_t c = threadIdx.x; c < D; c += 256) {
    C v = s * (wdy(c) - to_compute<C>(a.h[at + c]) * back);
    if (a.dh != nullptr) v += to_compute<C>(a.dh[at + c]);
    a.dx[at + c] = from_compute<T>(v);
  }
  if (threadIdx.x == 0 && a.s != nullptr) a.s[row] = s;
}

// The backward of rows in registers (as add_norm_kernel); the grid strides over the
// rows and each thread keeps the weight gradient of its columns, so the partial
// sums are one row a workgroup: no atomics, the same bits every time.  8192 x 7168
// bf16: 87 us for the rows (470 MB, 5.4 TB/s) and 5 us for the sums of 512
// workgroups; 256 workgroups take 108 us in all, 768 102 us, 1024 102 us.
template <class T, bool FULL, int TPR, int NV>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void add_norm_bwd_kernel(const AddNormBwd<T> a) {
  using V = NormVec<T>;
  constexpr int N = V::N;
  __shared__ float part[2][TPR / 64];
  const int tid = threadIdx.x, lane = TPR == 64 ? tid & 63 : tid;
  const int width = static_cast<int>(a.width);
  const int64_t group = TPR == 64 ? static_cast<int64_t>(blockIdx.x) * 4 + (tid >> 6) : blockIdx.x;
  const int64_t groups = static_cast<int64_t>(gridDim.x) * (TPR == 64 ? 4 : 1);
  float dw[NV][N] = {};
  float w[NV][N];
#pragma unroll
  for (int j = 0; j < NV; ++j) norm_weights<T, FULL>(a.w, a.wide_w, lane + j * TPR, width, w[j]);
  for (int64_t row = group; row < a.rows; row += groups) {
    const int64_t at = row * width;
    typename V::type hv[NV], yv[NV], uv[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      hv[j] = norm_load<T, FULL>(a.h + at, lane + j * TPR, width);
      yv[j] = norm_load<T, FULL>(a.dy + at, lane + j * TPR, width);
    }
    if (a.dh != nullptr) {
#pragma unroll
      for (int j = 0; j < NV; ++j) uv[j] = norm_load<T, FULL>(a.dh + at, lane + j * TPR, width);
    }
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float h = to_float(static_cast<T>(hv[j][e]));
        ss += h * h;
        dot += to_float(static_cast<T>(yv[j][e])) * w[j][e] * h;
      }
    ss = group_sum<64>(ss);
    dot = group_sum<64>(dot);
    if constexpr (TPR > 64) {
      __syncthreads();  // the last row's sums have been read
      if ((tid & 63) == 0) part[0][tid >> 6] = ss, part[1][tid >> 6] = dot;
      __syncthreads();
      ss = dot = 0.f;
#pragma unroll
      for (int u = 0; u < TPR / 64; ++u) ss += part[0][u], dot += part[1][u];
    }
    const float s = frsqrt(ss / static_cast<float>(width) + a.eps), back = s * s * (dot / static_cast<float>(width));
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      typename V::type o;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float h = to_float(static_cast<T>(hv[j][e])), dy = to_float(static_cast<T>(yv[j][e]));
        float v = s * (dy * w[j][e] - h * back);
        if (a.dh != nullptr) v += to_float(static_cast<T>(uv[j][e]));
        o[e] = from_compute<T>(v);
        dw[j][e] += dy * (h * s);
      }
      norm_store<T, FULL>(a.dx + at, lane + j * TPR, width, o);
    }
  }
  if (a.dw == nullptr) return;
  float* out = a.part + static_cast<int64_t>(blockIdx.x) * width;
  if constexpr (TPR == 64) {  // the four waves' columns meet
    __shared__ float meet[4][64 * NV * N];
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e) meet[tid >> 6][(lane + j * 64) * N + e] = dw[j][e];
    __syncthreads();
    for (int c = tid; c < width; c += 256) out[c] = (meet[0][c] + meet[1][c]) + (meet[2][c] + meet[3][c]);
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int c = (lane + j * TPR) * N + e;
        if (c < width) out[c] = dw[j][e];
      }
  }
}

// Weight gradient of a chunk of rows, 64 columns a workgroup; then the chunks' sum.
template <class T>
__global__ __launch_bounds__(256) void add_norm_dw_kernel(const AddNormBwd<T> a) {
  using C = typename NormCompute<T>::type;
  __shared__ C part[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane, r0 = static_cast<int64_t>(blockIdx.y) * a.chunk;
  const int64_t r1 = r0 + a.chunk < a.rows ? r0 + a.chunk : a.rows;
  C sum = C(0);
  if (c < a.width)
    for (int64_t r = r0 + wave; r < r1; r += 4)
      sum += to_compute<C>(a.dy[r * a.width + c]) * to_compute<C>(a.h[r * a.width + c]) * a.s[r];
  part[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < a.width)
    a.part[static_cast<int64_t>(blockIdx.y) * a.width + c] =
        (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
}

// The partial sums of 64 columns, sixteen waves each with every sixteenth part.
template <class T>
__global__ __launch_bounds__(1024) void add_norm_dw_sum_kernel(const AddNormBwd<T> a, int64_t parts) {
  using C = typename NormCompute<T>::type;
  __shared__ C part[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  C sum = C(0);
  if (c < a.width)
#pragma unroll 4
    for (int64_t k = wave; k < parts; k += 16) sum += a.part[k * a.width + c];
  part[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < a.width) {
    sum = part[0][lane];
#pragma unroll
    for (int u = 1; u < 16; ++u) sum += part[u][lane];
    if (a.wide_w)
      static_cast<float*>(a.dw)[c] = static_cast<float>(sum);
    else
      static_cast<T*>(a.dw)[c] = from_compute<T>(sum);
  }
}

}  // namespace kda

namespace kda_host {

using namespace kda;

static bool rows_fit(int64_t n) { return n <= 0x7fffffffLL; }

// A launch has fewer than 2^32 threads: more rows than that are served by several.
constexpr int64_t kLaunchThreads = int64_t(1) << 31;

// The weight gradient's sum has 1024 threads for 64 columns, in one launch.
constexpr int64_t kDwWidth = (int64_t(1) << 32) / 1024 * 64;

// The kernel for rows of `vectors` 16-byte vectors: a wave a row up to 256 of them,
// a workgroup of 256 or 1024 threads up to 4096, wider rows (0) value by value.
// With few rows the wave's four vectors go to four waves: latency.
struct RowShape {
  int threads, vectors;
};
static RowShape row_shape(int64_t width, int elem_bytes, int64_t rows) {
  const int64_t n = (width * elem_bytes + 15) / 16;
  if (elem_bytes == 8 || n > 4096) return {0, 0};
  if (n <= 64) return {64, 1};
  if (n <= 128) return {64, 2};
  if (n <= 256) return rows >= 1024 ? RowShape{64, 4} : RowShape{256, 1};
  if (n <= 512) return {256, 2};
  if (n <= 1024) return {256, 4};
  return n <= 2048 ? RowShape{1024, 2} : RowShape{1024, 4};
}

static bool whole_vectors(int64_t width, int elem_bytes, std::initializer_list<const void*> ptrs) {
  uintptr_t bits = static_cast<uintptr_t>(width * elem_bytes);
  for (const void* p : ptrs) bits |= reinterpret_cast<uintptr_t>(p);
  return bits % 16 == 0;
}

template <class T, bool Q, bool FULL>
static void launch_rows(const AddNorm<T>& a, RowShape r, hipStream_t s) {
  const unsigned rows = static_cast<unsigned>(a.rows), waves = static_cast<unsigned>((a.rows + 3) / 4);
  auto go = [&](auto kernel) {
    const dim3 grid(r.threads == 64 ? waves : rows), block(r.threads == 64 ? 256 : r.threads);
    hipLaunchKernelGGL(kernel, grid, block, 0, s, a);
  };
  if (r.threads == 64) {
    if (r.vectors == 1) go(add_norm_kernel<T, Q, FULL, 64, 1>);
    else if (r.vectors == 2) go(add_norm_kernel<T, Q, FULL, 64, 2>);
    else go(add_norm_kernel<T, Q, FULL, 64, 4>);
  } else if (r.threads == 256) {
    if (r.vectors == 1) go(add_norm_kernel<T, Q, FULL, 256, 1>);
    else if (r.vectors == 2) go(add_norm_kernel<T, Q, FULL, 256, 2>);
    else go(add_norm_kernel<T, Q, FULL, 256, 4>);
  } else {
    if (r.vectors == 2) go(add_norm_kernel<T, Q, FULL, 1024, 2>);
    else go(add_norm_kernel<T, Q, FULL, 1024, 4>);
  }
}

template <class T, bool Q>
static int run_add_norm_part(const AddNorm<T>& a, RowShape r, hipStream_t s) {
  if constexpr (sizeof(T) < 8) {
    if (r.threads != 0) {
      if (whole_vectors(a.width, sizeof(T), {a.x, a.r, a.w, a.h, a.y, a.q}))
        launch_rows<T, Q, true>(a, r, s);
      else
        launch_rows<T, Q, false>(a, r, s);
      return check_launch("add_norm");
    }
  }
  hipLaunchKernelGGL((add_norm_row_kernel<T, Q>), dim3(static_cast<unsigned>(a.rows)), dim3(256), 0, s, a);
  return check_launch("add_norm");
}

template <class T, bool Q>
static int run_add_norm(const AddNorm<T>& a, hipStream_t s) {
  const RowShape r = row_shape(a.width, sizeof(T), a.rows);
  const int64_t step = kLaunchThreads / (r.threads != 0 ? r.threads : 256);
  for (int64_t r0 = 0; r0 < a.rows; r0 += step) {
    AddNorm<T> b = a;
    const int64_t at = r0 * a.width;
    b.rows = a.rows - r0 < step ? a.rows - r0 : step;
    b.x += at;
    if (a.r != nullptr) b.r += at, b.h += at;
    if constexpr (Q)
      b.q += at, b.scales += r0 * (a.width / a.group);
    else
      b.y += at;
    const int rc = run_add_norm_part<T, Q>(b, r, s);
    if (rc != KDA_OK) return rc;
  }
  return KDA_OK;
}

template <class T>
static int add_norm_typed(const void* x, const void* r, const void* w, bool wide_w, void* h, void* y, void* q, float* scales,
                          int64_t group, int64_t rows, int64_t width, double eps, hipStream_t s) {
  AddNorm<T> a{};
  a.x = static_cast<const T*>(x), a.r = static_cast<const T*>(r), a.w = w;
  a.wide_w = wide_w && sizeof(T) == 2;
  a.h = static_cast<T*>(h), a.y = static_cast<T*>(y), a.q = static_cast<uint8_t*>(q), a.scales = scales;
  a.rows = rows, a.width = width, a.group = group, a.eps = static_cast<typename NormCompute<T>::type>(eps);
  if constexpr (!__is_same(T, double)) {
    if (q != nullptr) return run_add_norm<T, true>(a, s);
  }
  return run_add_norm<T, false>(a, s);
}

int launch_add_norm(const void* x, const void* r, const void* w, bool wide_w, void* h, void* y, void* q, float* scales,
                    int64_t group, int64_t rows, int64_t width, double eps, int dtype, hipStream_t s) {
  if (!rows_fit(rows)) {
    set_detail("add_rmsnorm: %lld rows", (long long)rows);
    return KDA_ERR_UNSUPPORTED;
  }
  switch (dtype) {
    case KDA_DTYPE_BF16: return add_norm_typed<bf16>(x, r, w, wide_w, h, y, q, scales, group, rows, width, eps, s);
    case KDA_DTYPE_F16: return add_norm_typed<f16>(x, r, w, wide_w, h, y, q, scales, group, rows, width, eps, s);
    case KDA_DTYPE_F32: return add_norm_typed<float>(x, r, w, wide_w, h, y, q, scales, group, rows, width, eps, s);
    default: return add_norm_typed<double>(x, r, w, wide_w, h, y, q, scales, group, rows, width, eps, s);
  }
}

// Partial weight gradients: one a workgroup of the strided backward, or of up to 64
// chunks of rows.
struct DwPlan {
  int64_t parts, chunk;
};
static DwPlan dw_plan(int64_t rows, int64_t width, int elem_bytes) {
  const RowShape r = row_shape(width, elem_bytes, rows);
  if (r.threads != 0) {
    const int64_t groups = r.threads == 64 ? (rows + 3) / 4 : rows, most = r.threads == 1024 ? 256 : 512;
    return {groups < most ? groups : most, 0};
  }
  const int64_t n = (rows + 63) / 64, chunk = n < 16 ? 16 : n;
  return {(rows + chunk - 1) / chunk, chunk};
}

static int elem_size(int dtype) { return dtype == KDA_DTYPE_F64 ? 8 : dtype == KDA_DTYPE_F32 ? 4 : 2; }

size_t add_norm_bwd_workspace_bytes(int64_t rows, int64_t width, int dtype) {
  const DwPlan p = dw_plan(rows, width, elem_size(dtype));
  const size_t c = dtype == KDA_DTYPE_F64 ? 8 : 4;
  return (static_cast<size_t>(p.parts) * width + (p.chunk != 0 ? rows : 0)) * c;
}

template <class T, bool FULL>
static void launch_bwd_rows(const AddNormBwd<T>& a, RowShape r, int64_t blocks, hipStream_t s) {
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(r.threads == 64 ? 256 : r.threads), 0, s, a);
  };
  if (r.threads == 64) {
    if (r.vectors == 1) go(add_norm_bwd_kernel<T, FULL, 64, 1>);
    else if (r.vectors == 2) go(add_norm_bwd_kernel<T, FULL, 64, 2>);
    else go(add_norm_bwd_kernel<T, FULL, 64, 4>);
  } else if (r.threads == 256) {
    if (r.vectors == 1) go(add_norm_bwd_kernel<T, FULL, 256, 1>);
    else if (r.vectors == 2) go(add_norm_bwd_kernel<T, FULL, 256, 2>);
    else go(add_norm_bwd_kernel<T, FULL, 256, 4>);
  } else {
    if (r.vectors == 2) go(add_norm_bwd_kernel<T, FULL, 1024, 2>);
    else go(add_norm_bwd_kernel<T, FULL, 1024, 4>);
  }
}

template <class T>
static int add_norm_bwd_typed(const void* h, const void* w, bool wide_w, const void* dy, const void* dh, void* dx, void* dw,
                              int64_t rows, int64_t width, double eps, void* ws, hipStream_t s) {
  using C = typename NormCompute<T>::type;
  AddNormBwd<T> a{};
  a.h = static_cast<const T*>(h), a.w = w, a.wide_w = wide_w && sizeof(T) == 2, a.dy = static_cast<const T*>(dy);
  a.dh = static_cast<const T*>(dh), a.dx = static_cast<T*>(dx), a.dw = dw;
  a.rows = rows, a.width = width, a.eps = static_cast<C>(eps);
  const RowShape r = row_shape(width, sizeof(T), rows);
  const DwPlan p = dw_plan(rows, width, sizeof(T));
  const unsigned columns = static_cast<unsigned>((width + 63) / 64);
  a.part = static_cast<C*>(ws), a.chunk = p.chunk;
  if (p.chunk != 0) {  // value by value
    if (dw != nullptr) a.s = a.part + p.parts * width;
    for (int64_t r0 = 0, step = kLaunchThreads / 256; r0 < rows; r0 += step) {
      AddNormBwd<T> b = a;
      const int64_t at = r0 * width;
      b.h += at, b.dy += at, b.dx += at;
      if (b.dh != nullptr) b.dh += at;
      if (b.s != nullptr) b.s += r0;
      const int64_t n = rows - r0 < step ? rows - r0 : step;
      hipLaunchKernelGGL((add_norm_bwd_row_kernel<T>), dim3(static_cast<unsigned>(n)), dim3(256), 0, s, b);
      const int rc = check_launch("add_norm_bwd");
      if (rc != KDA_OK) return rc;
    }
    if (dw != nullptr)
      hipLaunchKernelGGL((add_norm_dw_kernel<T>), dim3(columns, static_cast<unsigned>(p.parts)), dim3(256), 0, s, a);
  } else if constexpr (sizeof(T) < 8) {
    if (whole_vectors(width, sizeof(T), {h, w, dy, dh, dx}))
      launch_bwd_rows<T, true>(a, r, p.parts, s);
    else
      launch_bwd_rows<T, false>(a, r, p.parts, s);
  }
  if (dw != nullptr)
    hipLaunchKernelGGL((add_norm_dw_sum_kernel<T>), dim3(columns), dim3(1024), 0, s, a, p.parts);
  return check_launch("add_norm_bwd");
}

int launch_add_norm_bwd(const void* h, const void* w, bool wide_w, const void* dy, const void* dh, void* dx, void* dw, int64_t rows,
                        int64_t width, double eps, int dtype, void* ws, hipStream_t s) {
  if (!rows_fit(rows)) {
    set_detail("add_rmsnorm_bwd: %lld rows", (long long)rows);
    return KDA_ERR_UNSUPPORTED;
  }
  if (dw != nullptr && width >= kDwWidth) {
    set_detail("add_rmsnorm_bwd: the weight gradient of %lld columns", (long long)width);
    return KDA_ERR_UNSUPPORTED;
  }
  switch (dtype) {
    case KDA_DTYPE_BF16: return add_norm_bwd_typed<bf16>(h, w, wide_w, dy, dh, dx, dw, rows, width, eps, ws, s);
    case KDA_DTYPE_F16: return add_norm_bwd_typed<f16>(h, w, wide_w, dy, dh, dx, dw, rows, width, eps, ws, s);
    case KDA_DTYPE_F32: return add_norm_bwd_typed<float>(h, w, wide_w, dy, dh, dx, dw, rows, width, eps, ws, s);
    default: return add_norm_bwd_typed<double>(h, w, wide_w, dy, dh, dx, dw, rows, width, eps, ws, s);
  }
}

}  // namespace kda_host
