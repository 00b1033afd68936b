// Low-rank adapters of many requests beside a shared projection:
//   y_m = W x_m + bias + c_a B_a (A_a x_m),  a = the adapter of row m, or none.
// Row m's adapter is ids[m / span]: a negative id has none, an id past the stack
// gives a row of NaN (the host cannot see it without waiting for the GPU).
#include "kda_launch.h"

namespace kda {

template <class T>
struct Adapters {
  const T *x, *a, *b, *bias;  // x [rows, in], a [n, rank, in], b [n, out, rank], bias [out] or null
  const float* scaling;       // [n] or null (1)
  const void* ids;            // int32 or int64
  int ids64;
  int64_t span, rows;
  int in, out, rank, n;
  T* y;      // [rows, out]
  float* s;  // [rows, rank]
};

template <class T>
__device__ __forceinline__ int64_t adapter_of(const Adapters<T>& a, int64_t row) {
  const int64_t i = row / a.span;
  return a.ids64 != 0 ? static_cast<const int64_t*>(a.ids)[i] : static_cast<const int32_t*>(a.ids)[i];
}

// s_m = A x_m, a wave per (row, rank index)
template <class T>
__global__ __launch_bounds__(256) void adapter_down_kernel(const Adapters<T> a) {
  const int64_t row = blockIdx.x, id = adapter_of(a, row);
  if (id < 0 || id >= a.n) return;
  const int lane = threadIdx.x & 63;
  const T* x = a.x + row * a.in;
  for (int j = threadIdx.x >> 6; j < a.rank; j += 4) {
    const T* w = a.a + (id * a.rank + j) * a.in;
    float sum = 0.f;
    for (int k = lane; k < a.in; k += 64) sum += to_float(x[k]) * to_float(w[k]);
    sum = group_sum<64>(sum);
    if (lane == 0) a.s[row * a.rank + j] = sum;
  }
}

// y_m = bias + c B s_m, a thread per element
template <class T>
__global__ __launch_bounds__(256) void adapter_up_kernel(const Adapters<T> a) {
  const int64_t row = blockIdx.x, id = adapter_of(a, row);
  const int c = blockIdx.y * 256 + threadIdx.x;
  if (c >= a.out) return;
  float sum = 0.f;
  if (id >= a.n) {
    sum = __builtin_nanf("");
  } else if (id >= 0) {
    const T* w = a.b + (id * a.out + c) * a.rank;
    for (int j = 0; j < a.rank; ++j) sum += a.s[row * a.rank + j] * to_float(w[j]);
    if (a.scaling != nullptr) sum *= a.scaling[id];
  }
  if (a.bias != nullptr) sum += to_float(a.bias[c]);
  a.y[row * a.out + c] = from_compute<T>(sum);
}

}  // namespace kda

namespace kda_host {

using namespace kda;

size_t adapter_delta_workspace_bytes(const kda_adapter_args& d) { return static_cast<size_t>(d.rows) * d.rank * 4; }

template <class T>
static int run_adapter_delta(const kda_adapter_args& d, hipStream_t s) {
  Adapters<T> a{};
  a.x = static_cast<const T*>(d.x), a.a = static_cast<const T*>(d.a), a.b = static_cast<const T*>(d.b);
  a.bias = static_cast<const T*>(d.bias), a.scaling = d.scaling, a.ids = d.ids, a.ids64 = d.ids_are_int64;
  a.span = d.span, a.rows = d.rows, a.in = static_cast<int>(d.d_in), a.out = static_cast<int>(d.d_out);
  a.rank = static_cast<int>(d.rank), a.n = static_cast<int>(d.adapters);
  a.y = static_cast<T*>(d.y), a.s = static_cast<float*>(d.workspace);
  hipLaunchKernelGGL((adapter_down_kernel<T>), dim3(static_cast<unsigned>(d.rows)), dim3(256), 0, s, a);
  hipLaunchKernelGGL((adapter_up_kernel<T>),
                     dim3(static_cast<unsigned>(d.rows), static_cast<unsigned>((d.d_out + 255) / 256)), dim3(256), 0, s,
                     a);
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
