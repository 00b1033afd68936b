// The state cache in 8 bits: decode caches written into slots of a pool and
// read back, up to 64 tensors of any layers in one launch.
//
// A state row (entry, head, key channel) of V values has a scale of its own:
// the decay multiplies whole rows, so the rows of slow and fast channels differ
// by orders of magnitude while the values of one row do not.
//   scale = max|row| (1 / 127),  q = round_half_even(row / scale),  read back: q scale
// with 1 / 127 rounded to f32 (the scale is off by two roundings, the quotient by none).
// A row whose largest magnitude is under 2^-100 is held as zeros (its quotients
// would leave f32), one with a value that is not finite has scale NaN.  The
// other tensors of a cache (ShortConv histories, offsets) move as bytes.
//
// Bound: five bytes a value.  8 layers of 32 sequences and 32 heads, 128 x 128
// (713 MB): packed in one launch of 125 us (5.7 TB/s), read back in four of 37 us.
#include <algorithm>
#include <memory>
#include <new>

#include "kda_launch.h"

namespace kda {

constexpr int kMoveMax = 64;  // tensors per launch
constexpr int kMoveThreads = 256;
// Loads of a thread in flight.  8 layers x 32 sequences x 32 heads, 128 x 128: packing
// 125 us with 8, 130 with 4, 152 with 2; reading two of them back 38 us with 8, 37 with 4,
// 43 with 2.
constexpr int kPackSteps = 8;
constexpr int kMoveSteps = 4;
constexpr int64_t kMoveTiles = 0xffffffffLL / kMoveThreads;  // a launch has fewer than 2^32 threads
constexpr float kTinyRow = 0x1p-100f;

struct Move {
  const void* src;
  void* dst;
  float* scales;     // of the packed side
  int64_t rows;      // rows of an entry (bytes: 1)
  int64_t tile0;     // first tile of this tensor in the launch
  int32_t tiles;     // tiles of an entry
  int32_t width;     // values of a row (bytes: units of an entry)
  int16_t kind;      // KDA_MOVE_*
  int16_t lanes;     // lanes of a row, four values each (0: a wave a row, value by value; bytes: log2 of the unit)
  int32_t tile_rows;
};

struct MoveArgs {
  Move d[kMoveMax];
  const int64_t *src_index, *dst_index;  // entry of the source / destination, or null: i
  int64_t n, n_src, n_dst;
  int* status;
  int32_t count;
};
static_assert(sizeof(MoveArgs) <= 4096, "the descriptors travel in the kernel argument block");

// round_half_even(x / s) for |x| <= 127 s (1 + 2^-22), exactly: n is the whole
// number nearest to the rounded product x (1 / s), one off at most; the
// residual x - n s is exact in f32 (a multiple of half a step of s below its
// half), so comparing it with s / 2 decides.
__device__ __forceinline__ int quotient(float x, float s, float inv) {
  float n = rintf(x * inv);
  const float e = fmaf(-n, s, x), half = 0.5f * s;
  const bool odd = (static_cast<int>(n) & 1) != 0;
  if (e > half || (e == half && odd)) n += 1.f;
  if (e < -half || (e == -half && odd)) n -= 1.f;
  return static_cast<int>(n);
}

struct RowScale {
  float scale, inv;
};
// of a row's largest magnitude, as its bits
__device__ __forceinline__ RowScale row_scale(unsigned bits) {
  const float top = __builtin_bit_cast(float, bits);
  if (bits >= 0x7f800000u) return {__builtin_nanf(""), 0.f};
  if (top < kTinyRow) return {0.f, 0.f};
  const float s = top * (1.f / 127.f);
  return {s, frcp(s)};
}

// Four quotients as bytes, zeros for rows without a scale.  x inv + 1.5 2^23 holds the
// nearest whole number n in its low bits; x inv is off by 127 2^-23 at most, so n is
// the exact quotient's unless x inv lies within 2e-5 of a tie, where the residual
// decides.  (Deciding so for every value, 14 instructions each: 133 us against 125.)
__device__ __forceinline__ unsigned packed_four(const float (&x)[4], const RowScale& r) {
  constexpr float kWhole = 12582912.f;
  float n[4];
  bool near = false;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    n[e] = fmaf(x[e], r.inv, kWhole);
    near |= fabsf(fmaf(x[e], r.inv, -(n[e] - kWhole))) > 0.49998f;
  }
  unsigned b[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) b[e] = __builtin_bit_cast(unsigned, n[e]);
  if (__ballot(near) != 0) {  // about one wave in a hundred
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (r.inv != 0.f) b[e] = static_cast<unsigned>(quotient(x[e], r.scale, r.inv));
  }
  // the low bytes of the four
  const unsigned lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400u);
  return r.inv != 0.f ? lo | hi << 16 : 0u;
}

// The larger one of magnitudes' bits: as numbers, infinity over all, NaN over infinity.
__device__ __forceinline__ unsigned top_bits(float x, unsigned top) {
  const unsigned b = __builtin_bit_cast(unsigned, x) & 0x7fffffffu;
  return b > top ? b : top;
}
template <int ctrl>
__device__ __forceinline__ unsigned dpp_max(unsigned v) {
  const unsigned o = static_cast<unsigned>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), ctrl, 0xf, 0xf, false));
  return o > v ? o : v;
}
// over `lanes` neighbouring lanes (a power of two, the same in every lane)
__device__ __forceinline__ unsigned group_top(unsigned v, int lanes) {
  if (lanes >= 2) v = dpp_max<0xb1>(v);    // the moves of group_sum
  if (lanes >= 4) v = dpp_max<0x4e>(v);
  if (lanes >= 8) v = dpp_max<0x141>(v);
  if (lanes >= 16) v = dpp_max<0x140>(v);
  for (int off = 16; off < lanes; off <<= 1) {
    const unsigned o = __shfl_xor(v, off);
    v = o > v ? o : v;
  }
  return v;
}

typedef int8_t char4_t __attribute__((ext_vector_type(4)));

template <class T>
struct Four {
  typedef T type __attribute__((ext_vector_type(4)));
};

// `place()` finds the destination entry, -1 for none; every thread calls it, once,
// after the rows' loads have been asked for: its own loads and its barrier take as
// long again.
template <class T, class F>
__device__ __forceinline__ void pack_tile(const Move& d, int64_t from, int64_t row0, F place) {
  const T* src = static_cast<const T*>(d.src) + from * d.rows * d.width;
  const int tid = threadIdx.x;
  if (d.lanes != 0) {
    typedef typename Four<T>::type v4;
    const int c = 4 * (tid % d.lanes), step = kMoveThreads / d.lanes;
    const int64_t first = row0 + tid / d.lanes;
    v4 x[kPackSteps];
#pragma unroll
    for (int u = 0; u < kPackSteps; ++u) {
      const int64_t row = first + u * step;
      x[u] = v4{};
      if (row < d.rows && c < d.width)
        x[u] = __builtin_nontemporal_load(reinterpret_cast<const v4*>(src + row * d.width + c));
    }
    const int64_t to = place();
    if (to < 0) return;  // the whole workgroup
    int8_t* dst = static_cast<int8_t*>(d.dst) + to * d.rows * d.width;
    float* scales = d.scales + to * d.rows;
#pragma unroll
    for (int u = 0; u < kPackSteps; ++u) {
      float v[4];
      unsigned top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = to_float(static_cast<T>(x[u][e]));
        top = top_bits(v[e], top);
      }
      const RowScale r = row_scale(group_top(top, d.lanes));
      const unsigned q = packed_four(v, r);
      const int64_t row = first + u * step;
      if (row >= d.rows || c >= d.width) continue;
      __builtin_nontemporal_store(q, reinterpret_cast<unsigned*>(dst + row * d.width + c));
      if (c == 0) scales[row] = r.scale;
    }
    return;
  }
  const int64_t to = place();
  if (to < 0) return;
  int8_t* dst = static_cast<int8_t*>(d.dst) + to * d.rows * d.width;
  float* scales = d.scales + to * d.rows;
  const int lane = tid & 63;
  for (int64_t row = row0 + (tid >> 6); row < row0 + d.tile_rows && row < d.rows; row += kMoveThreads / 64) {
    const T* p = src + row * d.width;
    unsigned top = 0;
    for (int c = lane; c < d.width; c += 64) top = top_bits(to_float(p[c]), top);
    const RowScale r = row_scale(group_top(top, 64));
    for (int c = lane; c < d.width; c += 64)
      dst[row * d.width + c] = static_cast<int8_t>(r.inv != 0.f ? quotient(to_float(p[c]), r.scale, r.inv) : 0);
    if (lane == 0) scales[row] = r.scale;
  }
}

// `there`: whether the source slot exists; its rows are NaN otherwise
template <class T>
__device__ __forceinline__ void unpack_tile(const Move& d, int64_t from, int64_t to, int64_t row0, bool there) {
  const int8_t* src = static_cast<const int8_t*>(d.src) + (there ? from : 0) * d.rows * d.width;
  const float* scales = d.scales + (there ? from : 0) * d.rows;
  T* dst = static_cast<T*>(d.dst) + to * d.rows * d.width;
  const int tid = threadIdx.x;
  if (d.lanes != 0) {
    typedef typename Four<T>::type v4;
    const int c = 4 * (tid % d.lanes), step = kMoveThreads / d.lanes;
    const int64_t first = row0 + tid / d.lanes;
    char4_t q[kMoveSteps];
    float s[kMoveSteps];
#pragma unroll
    for (int u = 0; u < kMoveSteps; ++u) {
      const int64_t row = first + u * step;
      q[u] = char4_t{};
      s[u] = __builtin_nanf("");
      if (there && row < d.rows && c < d.width) {
        q[u] = __builtin_nontemporal_load(reinterpret_cast<const char4_t*>(src + row * d.width + c));
        s[u] = scales[row];
      }
    }
#pragma unroll
    for (int u = 0; u < kMoveSteps; ++u) {
      const int64_t row = first + u * step;
      if (row >= d.rows || c >= d.width) continue;
      v4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = from_compute<T>(static_cast<float>(q[u][e]) * s[u]);
      __builtin_nontemporal_store(v, reinterpret_cast<v4*>(dst + row * d.width + c));
    }
  } else {
    for (int64_t row = row0 + (tid >> 6); row < row0 + d.tile_rows && row < d.rows; row += kMoveThreads / 64) {
      const float s = there ? scales[row] : __builtin_nanf("");
      for (int c = tid & 63; c < d.width; c += 64)
        dst[row * d.width + c] = from_compute<T>((there ? static_cast<float>(src[row * d.width + c]) : 0.f) * s);
    }
  }
}

template <class U>
__device__ __forceinline__ void copy_tile(const Move& d, int64_t from, int64_t to, int64_t tile, bool there) {
  const U* src = static_cast<const U*>(d.src) + (there ? from : 0) * d.width;
  U* dst = static_cast<U*>(d.dst) + to * d.width;
  const int64_t c0 = tile * kMoveThreads * kMoveSteps + threadIdx.x;
#pragma unroll
  for (int u = 0; u < kMoveSteps; ++u) {
    const int64_t c = c0 + u * kMoveThreads;
    if (c < d.width) dst[c] = there ? src[c] : U{};
  }
}

// One workgroup a tile of one entry of one tensor.
template <class T>
__global__ __launch_bounds__(kMoveThreads) void state_move_kernel(const MoveArgs a) {
  const int64_t block = blockIdx.x;
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {  // tile0 ascends
    const int mid = (lo + hi + 1) >> 1;
    if (a.d[mid].tile0 <= block)
      lo = mid;
    else
      hi = mid - 1;
  }
  const Move& d = a.d[lo];
  const unsigned at = static_cast<unsigned>(block - d.tile0), tiles = static_cast<unsigned>(d.tiles);  // below 2^24
  const int64_t i = at / tiles, tile = at % tiles;
  const int64_t from = a.src_index != nullptr ? a.src_index[i] : i;
  const bool there = from >= 0 && from < a.n_src;
  if (!there && threadIdx.x == 0 && a.status != nullptr) *a.status = 1;
  auto place = [&]() -> int64_t {
    const int64_t to = a.dst_index != nullptr ? a.dst_index[i] : i;
    const bool fits = to >= 0 && to < a.n_dst;
    if (!fits && threadIdx.x == 0 && a.status != nullptr) *a.status = 1;
    if (a.dst_index != nullptr) {  // a slot that is named twice takes its last entry
      int later = 0;
      for (int64_t j = i + 1 + threadIdx.x; j < a.n; j += kMoveThreads) later |= a.dst_index[j] == to;
      if (__syncthreads_or(later)) return -1;
    }
    return fits ? to : -1;
  };
  if (d.kind == KDA_MOVE_PACK) {
    if (there) pack_tile<T>(d, from, tile * d.tile_rows, place);
    return;
  }
  const int64_t to = place();
  if (to < 0) return;
  switch (d.kind) {
    case KDA_MOVE_UNPACK:
      unpack_tile<T>(d, from, to, tile * d.tile_rows, there);
      break;
    default:
      switch (d.lanes) {
        case 4:
          typedef unsigned u4 __attribute__((ext_vector_type(4)));
          copy_tile<u4>(d, from, to, tile, there);
          break;
        case 3:
          copy_tile<uint64_t>(d, from, to, tile, there);
          break;
        case 2:
          copy_tile<uint32_t>(d, from, to, tile, there);
          break;
        case 1:
          copy_tile<uint16_t>(d, from, to, tile, there);
          break;
        default:
          copy_tile<uint8_t>(d, from, to, tile, there);
          break;
      }
  }
}

}  // namespace kda

namespace kda_host {

using namespace kda;

static_assert(sizeof(kda_state_tensor) == 48, "callers may pass records as six words");

static int float_bytes(int dtype) { return dtype == KDA_DTYPE_F32 ? 4 : 2; }

// Bytes of an entry on the two sides.
static int64_t side_bytes(const kda_state_tensor& t, int dtype, bool packed) {
  if (t.kind == KDA_MOVE_BYTES) return t.width;
  return t.rows * t.width * (packed ? 1 : float_bytes(dtype));
}

// What is written may not overlap what is read or written elsewhere: the spans in the
// order of their addresses, each against the furthest end before it (of any span for
// one that is written, of the written ones for one that is read).
static int check_overlap(const kda_state_tensor* t, int count, int dtype, int64_t n_src, int64_t n_dst) {
  struct Span {
    uintptr_t at, end;
    int tensor;
    bool written;
  };
  Span few[3 * kMoveMax];
  std::unique_ptr<Span[]> many(count > kMoveMax ? new (std::nothrow) Span[3 * static_cast<size_t>(count)] : nullptr);
  if (count > kMoveMax && !many) {
    set_detail("state_move: no host memory to check %d tensors", count);
    return KDA_ERR_UNSUPPORTED;
  }
  Span* spans = many ? many.get() : few;
  size_t n = 0;
  auto add = [&](const void* p, int64_t bytes, int tensor, bool written) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    spans[n++] = {at, at + static_cast<uintptr_t>(bytes), tensor, written};
  };
  for (int i = 0; i < count; ++i) {
    if (t[i].width == 0 || t[i].rows == 0) continue;
    const bool pack = t[i].kind == KDA_MOVE_PACK, unpack = t[i].kind == KDA_MOVE_UNPACK;
    add(t[i].src, side_bytes(t[i], dtype, unpack) * n_src, i, false);
    add(t[i].dst, side_bytes(t[i], dtype, pack) * n_dst, i, true);
    if (pack || unpack) add(t[i].scales, 4 * t[i].rows * (pack ? n_dst : n_src), i, pack);
  }
  std::sort(spans, spans + n, [](const Span& a, const Span& b) { return a.at < b.at; });
  const Span *any = nullptr, *written = nullptr;  // with the furthest end so far
  for (const Span* s = spans; s < spans + n; ++s) {
    const Span* before = s->written ? any : written;
    if (before != nullptr && s->at < before->end) {
      set_detail("state_move: tensors %d and %d overlap", before->tensor, s->tensor);
      return KDA_ERR_INVALID_ARGUMENT;
    }
    if (any == nullptr || s->end > any->end) any = s;
    if (s->written && (written == nullptr || s->end > written->end)) written = s;
  }
  return KDA_OK;
}

static int check_moves(const kda_state_tensor* t, int count, int dtype, int64_t n_src, int64_t n_dst) {
  for (int i = 0; i < count; ++i) {
    const bool bytes = t[i].kind == KDA_MOVE_BYTES;
    if (!bytes && t[i].kind != KDA_MOVE_PACK && t[i].kind != KDA_MOVE_UNPACK) {
      set_detail("state_move: tensor %d has kind %d", i, t[i].kind);
      return KDA_ERR_INVALID_ARGUMENT;
    }
    if (t[i].rows < 0 || t[i].width < 0 || t[i].width > 0x7fffffffLL ||
        (t[i].width > 0 && t[i].rows > INT64_MAX / 8 / t[i].width)) {
      set_detail("state_move: tensor %d has bad sizes", i);
      return KDA_ERR_INVALID_ARGUMENT;
    }
    const int64_t per = bytes ? t[i].width : t[i].rows * t[i].width;
    if (per == 0) continue;
    const int64_t most = n_src > n_dst ? n_src : n_dst;
    if (per > INT64_MAX / 8 / most) {
      set_detail("state_move: tensor %d is too large", i);
      return KDA_ERR_INVALID_ARGUMENT;
    }
    if (!t[i].src || !t[i].dst || (!bytes && !t[i].scales)) {
      set_detail("state_move: tensor %d has a null pointer", i);
      return KDA_ERR_INVALID_ARGUMENT;
    }
    const uintptr_t need = bytes ? 1 : float_bytes(dtype);
    const void* wide = t[i].kind == KDA_MOVE_PACK ? t[i].src : t[i].dst;
    if (!bytes && (reinterpret_cast<uintptr_t>(wide) % need != 0 || reinterpret_cast<uintptr_t>(t[i].scales) % 4 != 0)) {
      set_detail("state_move: tensor %d is not aligned to its elements", i);
      return KDA_ERR_INVALID_ARGUMENT;
    }
  }
  return check_overlap(t, count, dtype, n_src, n_dst);
}

static int launch_moves(const MoveArgs& a, int64_t tiles, int dtype, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(tiles)), block(kMoveThreads);
  if (dtype == KDA_DTYPE_F32)
    hipLaunchKernelGGL((state_move_kernel<float>), grid, block, 0, s, a);
  else if (dtype == KDA_DTYPE_BF16)
    hipLaunchKernelGGL((state_move_kernel<bf16>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((state_move_kernel<f16>), grid, block, 0, s, a);
  return check_launch("state_move");
}

int launch_state_move(const kda_state_tensor* t, int count, int dtype, const int64_t* src_index, int64_t n_src,
                      const int64_t* dst_index, int64_t n_dst, int64_t n, int* status, hipStream_t stream) {
  const int rc = check_moves(t, count, dtype, n_src, n_dst);
  if (rc != KDA_OK || n == 0) return rc;
  MoveArgs a{};
  a.src_index = src_index, a.dst_index = dst_index, a.n = n, a.n_src = n_src, a.n_dst = n_dst, a.status = status;
  int64_t tiles = 0;
  for (int i = 0; i < count; ++i) {
    if (t[i].width == 0 || t[i].rows == 0) continue;
    Move d{};
    d.src = t[i].src, d.dst = t[i].dst, d.scales = t[i].scales, d.kind = static_cast<int16_t>(t[i].kind);
    int64_t per;  // tiles of an entry
    if (t[i].kind == KDA_MOVE_BYTES) {
      const uintptr_t all = reinterpret_cast<uintptr_t>(t[i].src) | reinterpret_cast<uintptr_t>(t[i].dst) |
                            static_cast<uintptr_t>(t[i].width) | 16;
      int shift = 0;
      while (!(all >> shift & 1)) ++shift;
      d.rows = 1, d.lanes = static_cast<int16_t>(shift), d.width = static_cast<int32_t>(t[i].width >> shift);
      per = (int64_t{d.width} + kMoveThreads * kMoveSteps - 1) / (kMoveThreads * kMoveSteps);
    } else {
      d.rows = t[i].rows, d.width = static_cast<int32_t>(t[i].width);
      const bool pack = t[i].kind == KDA_MOVE_PACK;
      const uintptr_t wide = reinterpret_cast<uintptr_t>(pack ? t[i].src : t[i].dst);
      const uintptr_t narrow = reinterpret_cast<uintptr_t>(pack ? t[i].dst : t[i].src);
      int lanes = 0;
      if (d.width % 4 == 0 && d.width <= 256 && wide % (4 * float_bytes(dtype)) == 0 && narrow % 4 == 0)
        for (lanes = 1; lanes * 4 < d.width;) lanes *= 2;
      d.lanes = static_cast<int16_t>(lanes);
      d.tile_rows = kMoveThreads / (lanes != 0 ? lanes : 64) * (pack ? kPackSteps : kMoveSteps);
      per = (d.rows + d.tile_rows - 1) / d.tile_rows;
    }
    if (per > kMoveTiles / n) {
      set_detail("state_move: tensor %d is too large for one launch", i);
      return KDA_ERR_UNSUPPORTED;
    }
    d.tiles = static_cast<int32_t>(per);
    if (a.count == kMoveMax || tiles + per * n > kMoveTiles) {
      const int err = launch_moves(a, tiles, dtype, stream);
      if (err != KDA_OK) return err;
      a.count = 0, tiles = 0;
    }
    d.tile0 = tiles;
    tiles += per * n;
    a.d[a.count++] = d;
  }
  return a.count != 0 ? launch_moves(a, tiles, dtype, stream) : KDA_OK;
}

}  // namespace kda_host
