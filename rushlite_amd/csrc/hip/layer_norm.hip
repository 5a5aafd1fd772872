// Layer normalisation over rows, forward and backward.
//
//   y  = (x - mean) rstd w + b          mean, var over a row; rstd = 1 / sqrt(var + eps)
//   dx = rstd (u - avg(u) - z avg(u z)) z = (x - mean) rstd, u = g w
//   dw = sum over rows of g z,          db = sum over rows of g
//
// Both passes are bound by memory: forward reads x and writes y, backward reads
// g and x and writes dx.  A row stays in the registers of the L lanes that own
// it (16 lanes to 512), U units of 16 bytes each, so the variance is formed
// from the differences to the mean without a second read, and x is read once.
// Backward keeps the lane's columns of dw and db in registers over all rows of
// its workgroup: the weight's gradient costs one partial row per workgroup and a
// launch that folds the partials, in a fixed order.  Rows past the registers
// (16384 floats, 8192 doubles) are read again from the caches for each step.
//
// Measured (a copy of 1 GiB runs at 5.1 TB/s on the same card): forward of 8192 x
// 8192 floats 95 us = 5.6 TB/s (107 us with w and b read for every row and
// ordinary accesses); 12608 x 768, forward 13 us, backward 21 us = 5.5 TB/s and the
// fold 4.5, 41 us with the launches; 4095 x 3001 (no row aligned) 17, 30 and 5, 62 us;
// 4096 x 1024 doubles 13, 19 and 4, 41 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "common.hpp"
#include "lmp_hip_transformer.h"

namespace lmp_hip {
namespace {

#define LMP_WAVE_SWAP_SRC(...) __VA_ARGS__
#include "wave_swap.inc"
#undef LMP_WAVE_SWAP_SRC

// 16 bytes of T, read and written at any alignment of T.
template <typename T> struct Unit;
template <> struct Unit<float> {
  static constexpr int W = 4;
  typedef float V __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct Unit<double> {
  static constexpr int W = 2;
  typedef double V __attribute__((ext_vector_type(2), aligned(8)));
};

__device__ __forceinline__ float fma_of(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fma_of(double a, double b, double c) { return fma(a, b, c); }
__device__ __forceinline__ float root_of(float x) { return sqrtf(x); }
__device__ __forceinline__ double root_of(double x) { return sqrt(x); }

// Sum over the L lanes of a row, in every one of them.  L > 64: the waves' sums
// meet in `lds` (L / 64 values a slot; a barrier each call, so a caller takes
// its slots in turn, two at least).
template <int L, typename T>
__device__ __forceinline__ T row_sum(T v, T* lds) {
  v += lmp_swap<1>(v);
  v += lmp_swap<2>(v);
  v += lmp_swap<4>(v);
  v += lmp_swap<8>(v);
  if constexpr (L >= 64) {
    v += lmp_swap<16>(v);
    v += lmp_swap<32>(v);
  }
  if constexpr (L > 64) {
    constexpr int NW = L / 64;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) v += lds[i];
  }
  return v;
}

// The lane's U units of a row of n values; zeros past its end.  STREAM: with the
// nontemporal hint (kStreamBytes).
template <typename T, int L, int U, bool STREAM = false>
__device__ __forceinline__ void load_row(const T* p, int lane, int n,
                                         T (&v)[U * Unit<T>::W]) {
  constexpr int W = Unit<T>::W;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int c = (u * L + lane) * W;
    if (c + W <= n) {
      const auto* q = reinterpret_cast<const typename Unit<T>::V*>(p + c);
      const typename Unit<T>::V x = STREAM ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
      for (int j = 0; j < W; ++j) v[u * W + j] = x[j];
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) v[u * W + j] = c + j < n ? p[c + j] : T(0);
    }
  }
}
template <typename T, int L, int U, bool STREAM = false>
__device__ __forceinline__ void store_row(T* p, int lane, int n,
                                          const T (&v)[U * Unit<T>::W]) {
  constexpr int W = Unit<T>::W;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int c = (u * L + lane) * W;
    if (c + W <= n) {
      typename Unit<T>::V x;
#pragma unroll
      for (int j = 0; j < W; ++j) x[j] = v[u * W + j];
      auto* q = reinterpret_cast<typename Unit<T>::V*>(p + c);
      if constexpr (STREAM) __builtin_nontemporal_store(x, q);
      else *q = x;
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j)
        if (c + j < n) p[c + j] = v[u * W + j];
    }
  }
}

template <typename T>
struct NormArgs {
  int64_t rows;
  int n;
  const T* x;
  int64_t ldx;
  const T *w, *b;
  T eps;
  T* y;
  int64_t ldy;
  T *mean, *rstd;
  bool stream_in, stream_out;
};

template <typename T>
struct NormBackArgs {
  int64_t rows;
  int n;
  const T* g;
  int64_t ldg;
  const T* x;
  int64_t ldx;
  const T *w, *mean, *rstd;
  T* dx;
  int64_t lddx;
  T* part;      // [workgroup][dw, db][n], or null
  T *dw, *db;   // where one workgroup has all rows, and part is null
};

constexpr int threads_of(int lanes) { return lanes > 256 ? lanes : 256; }

template <typename T, int L, int U>
__global__ __launch_bounds__(threads_of(L)) void norm_rows(NormArgs<T> a) {
  constexpr int W = Unit<T>::W, R = threads_of(L) / L;
  __shared__ T meet[2][16];
  const int lane = threadIdx.x % L, sub = threadIdx.x / L;
  const T inv_n = T(1) / T(a.n);
  T w[U * W], b[U * W];
#pragma unroll
  for (int i = 0; i < U * W; ++i) {
    w[i] = T(1);
    b[i] = T(0);
  }
  if (a.w) load_row<T, L, U>(a.w, lane, a.n, w);
  if (a.b) load_row<T, L, U>(a.b, lane, a.n, b);
  for (int64_t first = int64_t(blockIdx.x) * R; first < a.rows; first += int64_t(gridDim.x) * R) {
    const bool live = first + sub < a.rows;
    const int64_t row = live ? first + sub : a.rows - 1;  // every lane takes part in the sums
    T v[U * W];
    if (a.stream_in) load_row<T, L, U, true>(a.x + row * a.ldx, lane, a.n, v);
    else load_row<T, L, U>(a.x + row * a.ldx, lane, a.n, v);
    T s = 0;
#pragma unroll
    for (int i = 0; i < U * W; ++i) s += v[i];
    const T mean = row_sum<L>(s, meet[0]) * inv_n;
    T q = 0;
#pragma unroll
    for (int i = 0; i < U * W; ++i) {
      v[i] -= mean;
      const int c = (i / W * L + lane) * W + i % W;
      q = c < a.n ? fma_of(v[i], v[i], q) : q;
    }
    const T rstd = T(1) / root_of(row_sum<L>(q, meet[1]) * inv_n + a.eps);
#pragma unroll
    for (int i = 0; i < U * W; ++i) v[i] = v[i] * rstd * w[i] + b[i];
    if (!live) continue;  // only rows of 64 lanes or fewer, which share no barrier
    if (a.stream_out) store_row<T, L, U, true>(a.y + row * a.ldy, lane, a.n, v);
    else store_row<T, L, U>(a.y + row * a.ldy, lane, a.n, v);
    if (lane == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
  }
}

// Rows longer than the registers hold: a workgroup per row, three passes.
template <typename T>
__global__ __launch_bounds__(1024) void norm_long_rows(NormArgs<T> a) {
  __shared__ T meet[2][16];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = a.x + row * a.ldx;
    T s = 0;
    for (int c = threadIdx.x; c < a.n; c += 1024) s += x[c];
    const T mean = row_sum<1024>(s, meet[0]) / T(a.n);
    T q = 0;
    for (int c = threadIdx.x; c < a.n; c += 1024) {
      const T d = x[c] - mean;
      q = fma_of(d, d, q);
    }
    const T rstd = T(1) / root_of(row_sum<1024>(q, meet[1]) / T(a.n) + a.eps);
    T* y = a.y + row * a.ldy;
    for (int c = threadIdx.x; c < a.n; c += 1024) {
      const T z = (x[c] - mean) * rstd * (a.w ? a.w[c] : T(1));
      y[c] = a.b ? z + a.b[c] : z;
    }
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = rstd;
    }
  }
}

template <typename T, int L, int U>
__global__ __launch_bounds__(threads_of(L)) void norm_back_rows(NormBackArgs<T> a) {
  constexpr int W = Unit<T>::W, R = threads_of(L) / L, N = U * W;
  __shared__ T meet[4][16];
  const int lane = threadIdx.x % L, sub = threadIdx.x / L;
  const T inv_n = T(1) / T(a.n);
  T w[N], dw[N], db[N];
  if (a.w) {
    load_row<T, L, U>(a.w, lane, a.n, w);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = T(1);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) dw[i] = db[i] = T(0);
  // The workgroup's rows are a contiguous run, so a lane's sums add neighbours.
  const int64_t groups = (a.rows + R - 1) / R;
  const int64_t begin = groups * blockIdx.x / gridDim.x, end = groups * (blockIdx.x + 1) / gridDim.x;
  int turn = 0;
  for (int64_t i_group = begin; i_group < end; ++i_group, turn ^= 2) {
    const bool live = i_group * R + sub < a.rows;
    const int64_t row = live ? i_group * R + sub : a.rows - 1;
    T x[N], g[N];
    load_row<T, L, U>(a.x + row * a.ldx, lane, a.n, x);
    load_row<T, L, U>(a.g + row * a.ldg, lane, a.n, g);
    const T mean = a.mean[row], rstd = a.rstd[row];
    T s1 = 0, s2 = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // Past the row's end g is zero, and z is kept finite where x is not there.
      x[i] = (x[i] - mean) * rstd;
      const int c = (i / W * L + lane) * W + i % W;
      if (live && c < a.n) {
        dw[i] = fma_of(g[i], x[i], dw[i]);
        db[i] += g[i];
      }
      g[i] *= w[i];
      s1 += g[i];
      s2 = c < a.n ? fma_of(g[i], x[i], s2) : s2;
    }
    if (!a.dx) continue;
    const T c1 = row_sum<L>(s1, meet[turn]) * inv_n, c2 = row_sum<L>(s2, meet[turn + 1]) * inv_n;
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = rstd * (g[i] - c1 - x[i] * c2);
    if (live) store_row<T, L, U>(a.dx + row * a.lddx, lane, a.n, g);
  }
  T* to_w = a.part ? a.part + int64_t(blockIdx.x) * 2 * a.n : a.dw;
  T* to_b = a.part ? to_w + a.n : a.db;
  if (!to_w && !to_b) return;
  if constexpr (R == 1) {
    if (to_w) store_row<T, L, U>(to_w, lane, a.n, dw);
    if (to_b) store_row<T, L, U>(to_b, lane, a.n, db);
  } else {
    __shared__ T sums[R][L * N];
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i)
        sums[sub][(i / W * L + lane) * W + i % W] = which ? db[i] : dw[i];
      __syncthreads();
      for (int c = threadIdx.x; c < a.n; c += threads_of(L)) {
        T s = sums[0][c];
#pragma unroll
        for (int r = 1; r < R; ++r) s += sums[r][c];
        if (T* to = which ? to_b : to_w) to[c] = s;
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void norm_back_long_rows(NormBackArgs<T> a) {
  __shared__ T meet[2][16];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = a.x + row * a.ldx;
    const T* g = a.g + row * a.ldg;
    const T mean = a.mean[row], rstd = a.rstd[row];
    T s1 = 0, s2 = 0;
    for (int c = threadIdx.x; c < a.n; c += 1024) {
      const T u = a.w ? g[c] * a.w[c] : g[c];
      s1 += u;
      s2 = fma_of(u, (x[c] - mean) * rstd, s2);
    }
    const T c1 = row_sum<1024>(s1, meet[0]) / T(a.n), c2 = row_sum<1024>(s2, meet[1]) / T(a.n);
    T* dx = a.dx + row * a.lddx;
    for (int c = threadIdx.x; c < a.n; c += 1024) {
      const T u = a.w ? g[c] * a.w[c] : g[c];
      dx[c] = rstd * (u - c1 - (x[c] - mean) * rstd * c2);
    }
  }
}

// dw and db of long rows: a lane per column, a run of rows per grid row.
template <typename T>
__global__ __launch_bounds__(256) void norm_back_columns(NormBackArgs<T> a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.n) return;
  const int64_t begin = a.rows * blockIdx.y / gridDim.y, end = a.rows * (blockIdx.y + 1) / gridDim.y;
  T dw = 0, db = 0;
  for (int64_t row = begin; row < end; ++row) {
    const T g = a.g[row * a.ldg + c];
    dw = fma_of(g, (a.x[row * a.ldx + c] - a.mean[row]) * a.rstd[row], dw);
    db += g;
  }
  T* out = a.part + int64_t(blockIdx.y) * 2 * a.n;
  out[c] = dw;
  out[a.n + c] = db;
}

// dw and db from the partials [parts][2][n]: 32 columns a workgroup, 32 lanes
// down the partials of each.
template <typename T>
__global__ __launch_bounds__(1024) void norm_back_fold(const T* part, int parts, int n, T* dw,
                                                       T* db) {
  __shared__ T sums[32][33];
  const int64_t width = 2 * int64_t(n);
  const int lane = threadIdx.x / 32;
  for (int64_t first = int64_t(blockIdx.x) * 32; first < width; first += int64_t(gridDim.x) * 32) {
    const int64_t c = first + threadIdx.x % 32;
    T s = 0;
    if (c < width) {
#pragma unroll 8
      for (int p = lane; p < parts; p += 32) s += part[p * width + c];
    }
    sums[lane][threadIdx.x % 32] = s;
    __syncthreads();
    for (int half = 16; half >= 1; half /= 2) {
      if (lane < half) sums[lane][threadIdx.x % 32] += sums[lane + half][threadIdx.x % 32];
      __syncthreads();
    }
    if (lane == 0 && c < width) {
      T* out = c < n ? dw : db;
      if (out) out[c < n ? c : c - n] = sums[0][threadIdx.x];
    }
    __syncthreads();
  }
}

template <typename T>
__global__ void norm_back_no_rows(int n, T* dw, T* db) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= n) return;
  if (dw) dw[c] = T(0);
  if (db) db[c] = T(0);
}

// Calls f with the lanes and units of the smallest variant that holds n values.
template <typename T, typename F>
bool with_variant(int64_t n, F&& f) {
  const int64_t units = (n + Unit<T>::W - 1) / Unit<T>::W;
  using std::integral_constant;
#define LMP_TRY(L, U) \
  if (units <= int64_t(L) * (U)) return f(integral_constant<int, L>{}, integral_constant<int, U>{}), true
  LMP_TRY(16, 1);
  LMP_TRY(16, 2);
  LMP_TRY(16, 4);
  LMP_TRY(64, 2);
  LMP_TRY(64, 3);
  LMP_TRY(64, 4);
  LMP_TRY(64, 8);
  LMP_TRY(256, 3);
  LMP_TRY(256, 4);
  LMP_TRY(256, 6);
  LMP_TRY(256, 8);
  LMP_TRY(512, 6);
  LMP_TRY(512, 8);
#undef LMP_TRY
  return false;
}

constexpr size_t kMaxCols = (size_t(1) << 31) - 65536;

// Grids stay below 2^32 threads; workgroups take further rows in turn.
int64_t capped(int64_t groups, int64_t most) { return std::max<int64_t>(1, std::min(groups, most)); }

template <typename T>
int layer_norm(Runtime* rt, const NormArgs<T>& a) {
  const int64_t cus = rt->cu_count;
  const bool held = with_variant<T>(a.n, [&](auto lanes, auto units) {
    constexpr int L = lanes, U = units, R = threads_of(L) / L;
    // Workgroups that run together, each over several rows with w and b in its
    // registers.
    const int64_t grid = capped((a.rows + R - 1) / R, cus * (L > 256 ? 2 : L > 64 ? 4 : 8));
    norm_rows<T, L, U><<<dim3(uint32_t(grid)), dim3(threads_of(L)), 0, rt->stream>>>(a);
  });
  if (!held)
    norm_long_rows<T><<<dim3(uint32_t(capped(a.rows, cus * 8))), dim3(1024), 0, rt->stream>>>(a);
  LMP_LAUNCH_CHECK("layer_norm");
  return LMP_OK;
}

template <typename T>
int layer_norm_backward(Runtime* rt, NormBackArgs<T> a, T* dw, T* db) {
  const int64_t cus = rt->cu_count;
  const bool columns = dw || db;
  // Workgroups over the rows: two waves' worth on every SIMD.  Up to four groups of
  // rows stay with one, which saves the launch that folds the partials.
  int64_t parts = 1;
  const bool held = with_variant<T>(a.n, [&](auto lanes, auto) {
    constexpr int L = lanes, R = threads_of(L) / L;
    const int64_t groups = (a.rows + R - 1) / R;
    parts = groups <= 4 ? 1 : std::min(groups, L > 256 ? cus : cus * 2);
  });
  if (!held) parts = capped(a.rows / 64, 64);
  const bool direct = held && parts == 1;
  if (direct) {
    a.dw = dw;
    a.db = db;
  } else if (columns) {
    a.part = static_cast<T*>(scratch_alloc(size_t(parts) * 2 * size_t(a.n) * sizeof(T)));
    if (!a.part) return LMP_ERR_OOM;
  }
  const auto run = [&]() -> int {
    if (held) {
      with_variant<T>(a.n, [&](auto lanes, auto units) {
        constexpr int L = lanes, U = units;
        norm_back_rows<T, L, U>
            <<<dim3(uint32_t(parts)), dim3(threads_of(L)), 0, rt->stream>>>(a);
      });
      LMP_LAUNCH_CHECK("layer_norm_backward");
    } else {
      if (columns) {  // first: dx may be g or x
        norm_back_columns<T><<<dim3(uint32_t((int64_t(a.n) + 255) / 256), uint32_t(parts)),
                               dim3(256), 0, rt->stream>>>(a);
        LMP_LAUNCH_CHECK("layer_norm_backward columns");
      }
      if (a.dx) {
        norm_back_long_rows<T>
            <<<dim3(uint32_t(capped(a.rows, cus * 8))), dim3(1024), 0, rt->stream>>>(a);
        LMP_LAUNCH_CHECK("layer_norm_backward");
      }
    }
    if (a.part) {
      norm_back_fold<T><<<dim3(uint32_t(capped((2 * int64_t(a.n) + 31) / 32, 1 << 20))), dim3(1024), 0,
                          rt->stream>>>(a.part, int(parts), a.n, dw, db);
      LMP_LAUNCH_CHECK("layer_norm_backward fold");
    }
    return LMP_OK;
  };
  const int status = run();
  if (a.part) scratch_free(a.part);
  return status;
}

int check_shape(const char* name, int dtype, size_t rows, size_t cols) {
  if (dtype != LMP_FLOAT32 && dtype != LMP_FLOAT64)
    return fail(LMP_ERR_INVALID, std::string(name) + ": dtype " + dtype_name(dtype) +
                                     " is neither Float32 nor Float64");
  if (cols == 0) return fail(LMP_ERR_INVALID, std::string(name) + ": rows of no values");
  if (cols > kMaxCols || rows > (size_t(1) << 40))
    return fail(LMP_ERR_UNSUPPORTED, std::string(name) + ": too many rows or columns");
  return LMP_OK;
}

}  // namespace
}  // namespace lmp_hip

using namespace lmp_hip;

extern "C" int lmp_k_layer_norm(int dtype, size_t rows, size_t cols, const void* x, size_t ldx,
                                const void* w, const void* b, double eps, void* y, size_t ldy,
                                void* mean, void* rstd) {
  if (int s = check_shape("lmp_k_layer_norm", dtype, rows, cols)) return s;
  if (!(eps >= 0) || std::isinf(eps))
    return fail(LMP_ERR_INVALID, "lmp_k_layer_norm: eps is negative or not finite");
  if (rows == 0) return LMP_OK;
  if (!x || !y) return fail(LMP_ERR_INVALID, "lmp_k_layer_norm: null buffer");
  if (ldx < cols || ldy < cols)
    return fail(LMP_ERR_INVALID, "lmp_k_layer_norm: leading dimension below cols");
  LMP_RUNTIME_OR_FAIL(rt);
  const auto go = [&](auto zero) {
    using T = decltype(zero);
    return layer_norm<T>(rt, {int64_t(rows), int(cols), static_cast<const T*>(x), int64_t(ldx),
                              static_cast<const T*>(w), static_cast<const T*>(b), T(eps),
                              static_cast<T*>(y), int64_t(ldy), static_cast<T*>(mean),
                              static_cast<T*>(rstd), rows * cols * sizeof(T) >= kStreamBytes,
                              rows * cols * sizeof(T) > kStreamStoreBytes});
  };
  return dtype == LMP_FLOAT64 ? go(double(0)) : go(float(0));
}

extern "C" int lmp_k_layer_norm_backward(int dtype, size_t rows, size_t cols, const void* g,
                                         size_t ldg, const void* x, size_t ldx, const void* w,
                                         const void* mean, const void* rstd, void* dx, size_t lddx,
                                         void* dw, void* db) {
  if (int s = check_shape("lmp_k_layer_norm_backward", dtype, rows, cols)) return s;
  if (!dx && !dw && !db) return LMP_OK;
  if (rows && (!g || !x || !mean || !rstd))
    return fail(LMP_ERR_INVALID, "lmp_k_layer_norm_backward: null buffer");
  if (rows && (ldg < cols || ldx < cols || (dx && lddx < cols)))
    return fail(LMP_ERR_INVALID, "lmp_k_layer_norm_backward: leading dimension below cols");
  LMP_RUNTIME_OR_FAIL(rt);
  const auto go = [&](auto zero) -> int {
    using T = decltype(zero);
    if (rows == 0) {
      if (!dw && !db) return LMP_OK;
      norm_back_no_rows<T><<<dim3(uint32_t((cols + 255) / 256)), dim3(256), 0, rt->stream>>>(
          int(cols), static_cast<T*>(dw), static_cast<T*>(db));
      LMP_LAUNCH_CHECK("layer_norm_backward of no rows");
      return LMP_OK;
    }
    NormBackArgs<T> a{int64_t(rows), int(cols), static_cast<const T*>(g), int64_t(ldg),
                      static_cast<const T*>(x), int64_t(ldx), static_cast<const T*>(w),
                      static_cast<const T*>(mean), static_cast<const T*>(rstd),
                      static_cast<T*>(dx), int64_t(lddx), nullptr, nullptr, nullptr};
    return layer_norm_backward<T>(rt, a, static_cast<T*>(dw), static_cast<T*>(db));
  };
  return dtype == LMP_FLOAT64 ? go(double(0)) : go(float(0));
}
