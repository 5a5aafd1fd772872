// Rotary positions: pairs of each head's values turned by position x frequency.
//
//   a = t f_j,  (u, v) -> s (u cos a - v sin a, v cos a + u sin a)
//
// with (u, v) values j and j + R / 2 of a head, or 2 j and 2 j + 1.  A gradient is turned
// back by the same kernel with sin negated.
//
// Bound by memory: every value read and written once.  A lane keeps one vector of
// pairs and goes over a row's heads with it, so that an angle's sine and cosine are
// formed once for all the heads of its lane; the loads of up to kHeads heads are on
// their way while they are.  8192 rows of 1536 take 21.8 us, 4.6 TB/s (16.5 from the memory-side
// cache); 16384 rows of 2048 float64 values 92 us, 5.8 TB/s.
//
// Angles.  t f_j / 2 pi in float64 is off by 2^-52 of itself, 2e-11 turns at a hundred
// thousand turns; what is left of it after the nearest quarter turn is exact and at most
// half a quarter, so rounding that to 32 bits moves the angle by at most pi / 2 x 2^-26
// = 2.3e-8.  Float64 rows take the angle t f_j, rounded to 64 bits, as it is.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "common.hpp"
#include "lmp_hip_transformer.h"

namespace lmp_hip {
namespace {

constexpr int kThreads = 256;
constexpr int kHeads = 4;  // heads of one lane whose loads are on their way together

// W values, which may start at any of them.
template <typename T, int W>
struct Values {
  typedef T type __attribute__((ext_vector_type(W), aligned(sizeof(T))));
};

template <typename T>
struct RotaryArgs {
  int64_t rows, ldx, ldy;
  const T* x;
  T* y;
  const int64_t* positions;
  const double* frequencies;
  double scale;
  int heads, dim, turned, plain;  // vectors per row, their size, how much of each turns, columns after them
  int pair_lanes, head_lanes;     // lanes over a head's pairs and over the heads: powers of two
  bool inverse, copy;             // copy: y is not x, so what does not turn is copied
};

// s cos a and s sin a of position t.
__device__ __forceinline__ void turn_of(double t, double f, double scale, float& c, float& s) {
  const double quarters = t * f * 0.63661977236758134308;  // 2 / pi
  const double whole = rint(quarters);
  const float rest = float(quarters - whole);
  float sn, cs;
  sincospif(0.5f * rest, &sn, &cs);
  const int q = int(whole - 4.0 * floor(whole * 0.25));
  const float a = q & 1 ? sn : cs, b = q & 1 ? cs : sn;
  // q: 0 (c, s), 1 (-s, c), 2 (-c, -s), 3 (s, -c)
  c = (q == 1 || q == 2 ? -a : a) * float(scale);
  s = (q >= 2 ? -b : b) * float(scale);
}
__device__ __forceinline__ void turn_of(double t, double f, double scale, double& c, double& s) {
  sincos(t * f, &s, &c);
  c *= scale;
  s *= scale;
}

// W values from or to memory; NT with the nontemporal hint.
template <typename T, int W, bool NT>
__device__ __forceinline__ void get(const T* p, T (&v)[W]) {
  using V = typename Values<T, W>::type;
  const V* q = reinterpret_cast<const V*>(p);
  const V r = NT ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
  for (int i = 0; i < W; ++i) v[i] = r[i];
}
template <typename T, int W, bool NT>
__device__ __forceinline__ void put(T* p, const T (&v)[W]) {
  using V = typename Values<T, W>::type;
  V r;
#pragma unroll
  for (int i = 0; i < W; ++i) r[i] = v[i];
  V* q = reinterpret_cast<V*>(p);
  if constexpr (NT) __builtin_nontemporal_store(r, q);
  else *q = r;
}
// n values by lanes `lane` of `lanes`.
template <typename T, int W, bool NT>
__device__ __forceinline__ void copy_run(T* y, const T* x, int n, int lane, int lanes) {
  for (int i = lane * W; i < n; i += lanes * W) {
    if (i + W <= n) {
      T v[W];
      get<T, W, NT>(x + i, v);
      put<T, W, NT>(y + i, v);
    } else {
      for (int j = i; j < n; ++j) y[j] = x[j];
    }
  }
}

// W: values of an access.  NEAR: pairs of neighbours, W / 2 of them in an access;
// otherwise W in two accesses.
template <typename T, int W, bool NEAR, bool NT>
__global__ __launch_bounds__(kThreads) void rotary_rows(RotaryArgs<T> a) {
  constexpr int P = NEAR ? W / 2 : W;  // pairs of a lane
  const int row_lanes = a.pair_lanes * a.head_lanes;
  const int in_row = threadIdx.x & (row_lanes - 1);
  const int pl = in_row & (a.pair_lanes - 1), hl = in_row / a.pair_lanes;
  const int per_group = kThreads / row_lanes;
  const int half = a.turned / 2, groups = half / P;
  for (int64_t row = int64_t(blockIdx.x) * per_group + threadIdx.x / row_lanes; row < a.rows;
       row += int64_t(gridDim.x) * per_group) {
    const T* x = a.x + row * a.ldx;
    T* y = a.y + row * a.ldy;
    const double t = double(a.positions[row]);
    for (int g = pl; g < groups; g += a.pair_lanes) {
      T c[P], s[P];
      bool fresh = true;
      for (int h0 = hl; h0 < a.heads; h0 += a.head_lanes * kHeads) {
        T u[kHeads][W], v[NEAR ? 1 : kHeads][W];
#pragma unroll
        for (int k = 0; k < kHeads; ++k) {
          const int h = h0 + k * a.head_lanes;
          if (h < a.heads) {
            const T* p = x + int64_t(h) * a.dim + g * W;
            get<T, W, NT>(p, u[k]);
            if constexpr (!NEAR) get<T, W, NT>(p + half, v[k]);
          }
        }
        if (fresh) {
#pragma unroll
          for (int i = 0; i < P; ++i) {
            turn_of(t, a.frequencies[g * P + i], a.scale, c[i], s[i]);
            if (a.inverse) s[i] = -s[i];
          }
          fresh = false;
        }
#pragma unroll
        for (int k = 0; k < kHeads; ++k) {
          const int h = h0 + k * a.head_lanes;
          if (h < a.heads) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
              T& p0 = NEAR ? u[k][2 * i] : u[k][i];
              T& p1 = NEAR ? u[k][2 * i + 1] : v[NEAR ? 0 : k][i];
              const T q0 = p0 * c[i] - p1 * s[i], q1 = p1 * c[i] + p0 * s[i];
              p0 = q0;
              p1 = q1;
            }
            T* p = y + int64_t(h) * a.dim + g * W;
            put<T, W, NT>(p, u[k]);
            if constexpr (!NEAR) put<T, W, NT>(p + half, v[k]);
          }
        }
      }
    }
    if (!a.copy) continue;
    if (a.dim > a.turned)
      for (int h = hl; h < a.heads; h += a.head_lanes) {
        const int64_t at = int64_t(h) * a.dim + a.turned;
        copy_run<T, W, NT>(y + at, x + at, a.dim - a.turned, pl, a.pair_lanes);
      }
    const int64_t at = int64_t(a.heads) * a.dim;
    copy_run<T, W, NT>(y + at, x + at, a.plain, in_row, row_lanes);
  }
}

int power_of_two(int64_t at_least, int most) {
  int p = 1;
  while (p < at_least && p < most) p *= 2;
  return p;
}

template <typename T, int W, bool NEAR>
int launch_rotary(Runtime* rt, RotaryArgs<T> a, bool stream) {
  constexpr int P = NEAR ? W / 2 : W;
  // A lane for every vector of pairs, as far as they go, and one for every kHeads heads.
  a.pair_lanes = power_of_two(std::max(1, a.turned / 2 / P), 64);
  a.head_lanes = power_of_two((a.heads + kHeads - 1) / kHeads, kThreads / a.pair_lanes);
  const int per_group = kThreads / (a.pair_lanes * a.head_lanes);
  const int64_t groups = (a.rows + per_group - 1) / per_group;
  const dim3 grid(uint32_t(std::min<int64_t>(groups, int64_t(rt->cu_count) * 64)));
  if (stream) rotary_rows<T, W, NEAR, true><<<grid, dim3(kThreads), 0, rt->stream>>>(a);
  else rotary_rows<T, W, NEAR, false><<<grid, dim3(kThreads), 0, rt->stream>>>(a);
  LMP_LAUNCH_CHECK("rotary");
  return LMP_OK;
}

// The widest access that the turned values are whole numbers of.
template <typename T, bool NEAR>
int rotary(Runtime* rt, const RotaryArgs<T>& a, bool stream) {
  const int unit = NEAR ? a.turned : a.turned / 2;
  if constexpr (sizeof(T) == 4)
    if (unit % 4 == 0) return launch_rotary<T, 4, NEAR>(rt, a, stream);
  if constexpr (!NEAR)
    if (unit % 2) return launch_rotary<T, 1, NEAR>(rt, a, stream);
  return launch_rotary<T, 2, NEAR>(rt, a, stream);
}

}  // namespace
}  // namespace lmp_hip

using namespace lmp_hip;

extern "C" int lmp_k_rotary(int dtype, size_t rows, size_t cols, size_t heads, size_t head_dim,
                            size_t rotary_dim, int interleaved, const void* x, size_t ldx,
                            const int64_t* positions, const double* frequencies, double scale,
                            int inverse, void* y, size_t ldy) {
  const std::string name = "lmp_k_rotary: ";
  if (dtype != LMP_FLOAT32 && dtype != LMP_FLOAT64)
    return fail(LMP_ERR_INVALID, name + "dtype " + dtype_name(dtype) + " is neither Float32 nor Float64");
  constexpr size_t kMost = (size_t(1) << 31) - 65536;
  if (heads > kMost || head_dim > kMost || cols > kMost || rows > (size_t(1) << 40))
    return fail(LMP_ERR_UNSUPPORTED, name + "too many rows or columns");
  if (rotary_dim % 2 || rotary_dim > head_dim)
    return fail(LMP_ERR_INVALID, name + "rotary_dim is odd or above head_dim");
  if (heads * head_dim > cols)
    return fail(LMP_ERR_INVALID, name + "rows have fewer than heads * head_dim columns");
  if (!std::isfinite(scale) || !std::isfinite(float(scale)))
    return fail(LMP_ERR_INVALID, name + "scale is not finite");
  if (rows == 0 || cols == 0) return LMP_OK;
  if (!x || !y || !positions || (rotary_dim && heads && !frequencies))
    return fail(LMP_ERR_INVALID, name + "null buffer");
  if (ldx < cols || ldy < cols) return fail(LMP_ERR_INVALID, name + "leading dimension below cols");
  const size_t size = dtype == LMP_FLOAT64 ? 8 : 4;
  if (x == y && ldx != ldy)
    return fail(LMP_ERR_INVALID, name + "in place, but the leading dimensions differ");
  if (x != y) {
    const auto bytes = [&](size_t ld) { return ((rows - 1) * ld + cols) * size; };
    const uintptr_t xa = reinterpret_cast<uintptr_t>(x), ya = reinterpret_cast<uintptr_t>(y);
    // Slices side by side in wider rows interleave without touching.
    const size_t apart = xa < ya ? (ya - xa) / size : (xa - ya) / size;
    const bool beside = ldx == ldy && apart < ldx && apart >= cols && ldx - apart >= cols;
    if (!beside && xa < ya + bytes(ldy) && ya < xa + bytes(ldx))
      return fail(LMP_ERR_INVALID, name + "x and y overlap without being the same rows");
  }
  if (x == y && (rotary_dim == 0 || heads == 0)) return LMP_OK;
  LMP_RUNTIME_OR_FAIL(rt);
  const auto go = [&](auto zero) {
    using T = decltype(zero);
    RotaryArgs<T> a{int64_t(rows), int64_t(ldx), int64_t(ldy), static_cast<const T*>(x), static_cast<T*>(y),
                    positions, frequencies, scale, int(heads), int(head_dim), int(rotary_dim),
                    int(cols - heads * head_dim), 1, 1, inverse != 0, x != y};
    const bool stream = rows * cols * sizeof(T) >= kStreamBytes;
    return interleaved ? rotary<T, true>(rt, a, stream) : rotary<T, false>(rt, a, stream);
  };
  return dtype == LMP_FLOAT64 ? go(double(0)) : go(float(0));
}
