// RMSNorm with the residual's addition, its backward, and its 8-bit output.
//
//   h = round(x + r);  s = 1 / sqrt(mean(h^2) + eps);  y = h s w
// over rows of `width` elements; the norm reads the stored (rounded) sum, so
// the backward, which has h alone, differentiates the function that ran.  With
// 8-bit output, over each group of a row (or the row):
//   scale = max|y| / 448,  q = e4m3(y / scale)   (448: e4m3's largest value)
// and a group whose largest magnitude is under 2^-100 has scale 0 and zeros:
// its quotients would leave f32.
// Backward, with the gradients dy and dh of the two outputs:
//   dx = dr = dh + s (w dy - h s^2 mean(w dy h)),  dw = sum over rows of dy h s.
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
  const T *x, *r, *w;  // r, w: may be null
  T *h, *y;            // h: null without a residual (h is x)
  uint8_t* q;          // e4m3, in place of y
  float* scales;       // [rows, width / group]
  int64_t rows, width, group;
  typename NormCompute<T>::type eps;
};

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

// Any width, one workgroup a row, the sum kept in h (in x without a residual)
// between the passes: each thread reads back what it wrote itself.
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
    return a.w != nullptr ? v * to_compute<C>(a.w[c]) : v;
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
      const bool zero = m < kTinyGroup;
      const float inv = zero ? 0.f : kE4m3Max / m;
      for (int64_t c = first; c < a.group; c += step)
        a.q[at + g * a.group + c] = to_e4m3(static_cast<float>(value(g * a.group + c)) * inv);
      if (first == 0) a.scales[row * (D / a.group) + g] = zero ? 0.f : m / kE4m3Max;
    }
  }
}

template <class T>
struct AddNormBwd {
  const T *h, *w, *dy, *dh;  // w, dh: may be null
  T *dx, *dw;                // dw: may be null
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
    return a.w != nullptr ? v * to_compute<C>(a.w[c]) : v;
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

template <class T>
__global__ __launch_bounds__(256) void add_norm_dw_sum_kernel(const AddNormBwd<T> a, int64_t chunks) {
  using C = typename NormCompute<T>::type;
  __shared__ C part[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 64 + lane;
  C sum = C(0);
  if (c < a.width)
    for (int64_t k = wave; k < chunks; k += 4) sum += a.part[k * a.width + c];
  part[wave][lane] = sum;
  __syncthreads();
  if (wave == 0 && c < a.width)
    a.dw[c] = from_compute<T>((part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]));
}

}  // namespace kda

namespace kda_host {

using namespace kda;

static bool grid_fits(int64_t n) { return n <= 0x7fffffffLL; }

template <class T, bool Q>
static int run_add_norm(const AddNorm<T>& a, hipStream_t s) {
  hipLaunchKernelGGL((add_norm_row_kernel<T, Q>), dim3(static_cast<unsigned>(a.rows)), dim3(256), 0, s, a);
  return check_launch("add_norm");
}

template <class T>
static int add_norm_typed(const void* x, const void* r, const void* w, void* h, void* y, void* q, float* scales,
                          int64_t group, int64_t rows, int64_t width, double eps, hipStream_t s) {
  AddNorm<T> a{};
  a.x = static_cast<const T*>(x), a.r = static_cast<const T*>(r), a.w = static_cast<const T*>(w);
  a.h = static_cast<T*>(h), a.y = static_cast<T*>(y), a.q = static_cast<uint8_t*>(q), a.scales = scales;
  a.rows = rows, a.width = width, a.group = group, a.eps = static_cast<typename NormCompute<T>::type>(eps);
  if constexpr (!__is_same(T, double)) {
    if (q != nullptr) return run_add_norm<T, true>(a, s);
  }
  return run_add_norm<T, false>(a, s);
}

int launch_add_norm(const void* x, const void* r, const void* w, void* h, void* y, void* q, float* scales,
                    int64_t group, int64_t rows, int64_t width, double eps, int dtype, hipStream_t s) {
  if (!grid_fits(rows)) {
    set_detail("add_rmsnorm: %lld rows", (long long)rows);
    return KDA_ERR_UNSUPPORTED;
  }
  switch (dtype) {
    case KDA_DTYPE_BF16: return add_norm_typed<bf16>(x, r, w, h, y, q, scales, group, rows, width, eps, s);
    case KDA_DTYPE_F16: return add_norm_typed<f16>(x, r, w, h, y, q, scales, group, rows, width, eps, s);
    case KDA_DTYPE_F32: return add_norm_typed<float>(x, r, w, h, y, q, scales, group, rows, width, eps, s);
    default: return add_norm_typed<double>(x, r, w, h, y, q, scales, group, rows, width, eps, s);
  }
}

// Rows per chunk of the weight gradient's first pass: at most 64 chunks.
static int64_t dw_chunk(int64_t rows) {
  const int64_t n = (rows + 63) / 64;
  return n < 16 ? 16 : n;
}

size_t add_norm_bwd_workspace_bytes(int64_t rows, int64_t width, int dtype) {
  const int64_t chunk = dw_chunk(rows), chunks = (rows + chunk - 1) / chunk;
  return static_cast<size_t>(rows + chunks * width) * (dtype == KDA_DTYPE_F64 ? 8 : 4);
}

template <class T>
static int add_norm_bwd_typed(const void* h, const void* w, const void* dy, const void* dh, void* dx, void* dw,
                              int64_t rows, int64_t width, double eps, void* ws, hipStream_t s) {
  using C = typename NormCompute<T>::type;
  AddNormBwd<T> a{};
  a.h = static_cast<const T*>(h), a.w = static_cast<const T*>(w), a.dy = static_cast<const T*>(dy);
  a.dh = static_cast<const T*>(dh), a.dx = static_cast<T*>(dx), a.dw = static_cast<T*>(dw);
  a.rows = rows, a.width = width, a.eps = static_cast<typename NormCompute<T>::type>(eps), a.chunk = dw_chunk(rows);
  if (dw != nullptr) a.s = static_cast<C*>(ws), a.part = a.s + rows;
  hipLaunchKernelGGL((add_norm_bwd_row_kernel<T>), dim3(static_cast<unsigned>(rows)), dim3(256), 0, s, a);
  if (dw != nullptr) {
    const unsigned blocks = static_cast<unsigned>((width + 63) / 64);
    const int64_t chunks = (rows + a.chunk - 1) / a.chunk;
    hipLaunchKernelGGL((add_norm_dw_kernel<T>), dim3(blocks, static_cast<unsigned>(chunks)), dim3(256), 0, s, a);
    hipLaunchKernelGGL((add_norm_dw_sum_kernel<T>), dim3(blocks), dim3(256), 0, s, a, chunks);
  }
  return check_launch("add_norm_bwd");
}

int launch_add_norm_bwd(const void* h, const void* w, const void* dy, const void* dh, void* dx, void* dw, int64_t rows,
                        int64_t width, double eps, int dtype, void* ws, hipStream_t s) {
  if (!grid_fits(rows)) {
    set_detail("add_rmsnorm_bwd: %lld rows", (long long)rows);
    return KDA_ERR_UNSUPPORTED;
  }
  switch (dtype) {
    case KDA_DTYPE_BF16: return add_norm_bwd_typed<bf16>(h, w, dy, dh, dx, dw, rows, width, eps, ws, s);
    case KDA_DTYPE_F16: return add_norm_bwd_typed<f16>(h, w, dy, dh, dx, dw, rows, width, eps, ws, s);
    case KDA_DTYPE_F32: return add_norm_bwd_typed<float>(h, w, dy, dh, dx, dw, rows, width, eps, ws, s);
    default: return add_norm_bwd_typed<double>(h, w, dy, dh, dx, dw, rows, width, eps, ws, s);
  }
}

}  // namespace kda_host
