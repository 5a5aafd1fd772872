// Dropout from a counter-based generator: y = residual + (kept ? x / (1 - rate) : 0).
//
// The generator is Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011): key (seed low, seed high), counter (place / 4
// low, high, call low, high).  Value i takes word i % 4 and is kept if that is at least
// rate 2^32, so what is kept is a function of (seed, call, place): nothing of it is
// stored, and the backward pass forms it again from the call's number.
//
// The count of calls lives on the device (as AdamW's count of steps does), so that a
// recorded call draws afresh at every replay; the last workgroup to finish advances it.
//
// Bound by memory: 8 bytes a value (12 with a residual).  Ten rounds cost 20 products of
// 32 by 32 bits per four values.  8192 x 8192 with a residual take 131 us, 6.1 TB/s, and
// backward 89 us, 6.0 TB/s.
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
constexpr int kUnits = 4;          // units of four values a lane, whose loads are on their way together
constexpr int kGroupsPerUnit = 16;  // workgroups per compute unit at most

template <typename T>
struct Four {
  typedef T type __attribute__((ext_vector_type(4), aligned(sizeof(T))));
};

template <typename T>
struct DropoutArgs {
  int64_t n;
  const T* x;
  const T* residual;
  T* y;
  T scale;
  uint32_t key0, key1;
  uint32_t last;  // words up to this are dropped, where `some`
  bool some;
  int64_t* state;       // forward: calls done, and the workgroups that finished
  int64_t* used;        // forward: takes the number of this call
  const int64_t* call;  // backward: the number of the forward call
};

__device__ __forceinline__ void philox(uint32_t (&c)[4], uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t p = uint64_t(c[0]) * 0xD2511F53u, q = uint64_t(c[2]) * 0xCD9E8D57u;
    c[0] = uint32_t(q >> 32) ^ c[1] ^ k0;
    c[2] = uint32_t(p >> 32) ^ c[3] ^ k1;
    c[1] = uint32_t(q);
    c[3] = uint32_t(p);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
}

// STREAM: accesses with the nontemporal hint.
template <typename T, bool FORWARD, bool STREAM>
__global__ __launch_bounds__(kThreads) void dropout_values(DropoutArgs<T> a) {
  using V = typename Four<T>::type;
  constexpr int64_t kPerGroup = int64_t(kThreads) * 4 * kUnits;
  const int64_t call = FORWARD ? a.state[0] : a.call[0];
  const auto load4 = [&](const T* from, int64_t at) -> V {
    V v = V(T(0));
    if (at + 4 <= a.n) {
      const V* q = reinterpret_cast<const V*>(from + at);
      return STREAM ? __builtin_nontemporal_load(q) : *q;
    }
    for (int j = 0; j < 4; ++j)
      if (at + j < a.n) v[j] = from[at + j];
    return v;
  };
  for (int64_t begin = blockIdx.x * kPerGroup; begin < a.n; begin += gridDim.x * kPerGroup) {
    const auto at_of = [&](int u) { return begin + (int64_t(u) * kThreads + threadIdx.x) * 4; };
    V x[kUnits], r[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      x[u] = load4(a.x, at_of(u));
      if (FORWARD && a.residual) r[u] = load4(a.residual, at_of(u));
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int64_t at = at_of(u);
      const uint64_t unit = uint64_t(at) / 4;
      uint32_t w[4] = {uint32_t(unit), uint32_t(unit >> 32), uint32_t(call), uint32_t(uint64_t(call) >> 32)};
      philox(w, a.key0, a.key1);
      V y;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // Selected, not multiplied by 0: an infinity or a NaN that is dropped leaves no trace.
        const T v = a.some && w[j] <= a.last ? T(0) : T(x[u][j] * a.scale);
        y[j] = FORWARD && a.residual ? r[u][j] + v : v;
      }
      if (at + 4 <= a.n) {
        V* q = reinterpret_cast<V*>(a.y + at);
        if constexpr (STREAM) __builtin_nontemporal_store(y, q);
        else *q = y;
      } else {
        for (int j = 0; j < 4; ++j)
          if (at + j < a.n) a.y[at + j] = y[j];
      }
    }
  }
  if constexpr (FORWARD) {
    // Every lane has read the count; the last workgroup to come here finds that all have,
    // and the next launch finds the counter at 0.
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned long long* done = reinterpret_cast<unsigned long long*>(a.state + 1);
      if (atomicAdd(done, 1ull) == gridDim.x - 1) {
        *done = 0;
        a.state[0] = call + 1;
        if (a.used) *a.used = call;
      }
    }
  }
}

template <typename T, bool FORWARD>
int launch_dropout(Runtime* rt, const DropoutArgs<T>& a, bool stream) {
  constexpr int64_t kPerGroup = int64_t(kThreads) * 4 * kUnits;
  // A call of nothing still counts.
  const int64_t groups = std::max<int64_t>(1, (a.n + kPerGroup - 1) / kPerGroup);
  const dim3 grid(uint32_t(std::min<int64_t>(groups, int64_t(rt->cu_count) * kGroupsPerUnit)));
  if (stream) dropout_values<T, FORWARD, true><<<grid, dim3(kThreads), 0, rt->stream>>>(a);
  else dropout_values<T, FORWARD, false><<<grid, dim3(kThreads), 0, rt->stream>>>(a);
  LMP_LAUNCH_CHECK("dropout");
  return LMP_OK;
}

int check_dropout(const std::string& name, int dtype, size_t n, double rate) {
  if (dtype != LMP_FLOAT32 && dtype != LMP_FLOAT64)
    return fail(LMP_ERR_INVALID, name + "dtype " + dtype_name(dtype) + " is neither Float32 nor Float64");
  if (!(rate >= 0 && rate <= 1)) return fail(LMP_ERR_INVALID, name + "rate lies in [0, 1]");
  if (n > (size_t(1) << 40)) return fail(LMP_ERR_UNSUPPORTED, name + "too many values");
  return LMP_OK;
}

// y is an operand or apart from it: workgroups have no order among them.
int check_apart(const std::string& name, int dtype, size_t n, const void* operand, const void* y) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(operand), b = reinterpret_cast<uintptr_t>(y);
  if (operand && a != b && (a < b ? b - a : a - b) < n * (dtype == LMP_FLOAT64 ? 8 : 4))
    return fail(LMP_ERR_INVALID, name + "the output overlaps an operand without being it");
  return LMP_OK;
}

template <typename T>
DropoutArgs<T> dropout_args(size_t n, const void* x, const void* residual, double rate, uint64_t seed,
                            void* y) {
  DropoutArgs<T> a{};
  a.n = int64_t(n);
  a.x = static_cast<const T*>(x);
  a.residual = static_cast<const T*>(residual);
  a.y = static_cast<T*>(y);
  const uint64_t dropped = uint64_t(std::llrint(rate * 4294967296.0));  // words below it
  a.some = dropped > 0;
  a.last = uint32_t(dropped - 1);
  a.scale = rate < 1 ? T(1 / (1 - rate)) : T(0);
  a.key0 = uint32_t(seed);
  a.key1 = uint32_t(seed >> 32);
  return a;
}

}  // namespace
}  // namespace lmp_hip

using namespace lmp_hip;

extern "C" int lmp_k_dropout(int dtype, size_t n, const void* x, const void* residual, double rate,
                             uint64_t seed, int64_t* state, int64_t* used, void* y) {
  if (int s = check_dropout("lmp_k_dropout: ", dtype, n, rate)) return s;
  if (!state || (n && (!x || !y))) return fail(LMP_ERR_INVALID, "lmp_k_dropout: null buffer");
  if (used && (used == state || used == state + 1))
    return fail(LMP_ERR_INVALID, "lmp_k_dropout: used is part of the state");
  for (const void* operand : {x, residual})
    if (int s = check_apart("lmp_k_dropout: ", dtype, n, operand, y)) return s;
  LMP_RUNTIME_OR_FAIL(rt);
  const auto go = [&](auto zero) {
    using T = decltype(zero);
    auto a = dropout_args<T>(n, x, residual, rate, seed, y);
    a.state = state;
    a.used = used;
    return launch_dropout<T, true>(rt, a, n * sizeof(T) >= kStreamBytes / 2);
  };
  return dtype == LMP_FLOAT64 ? go(double(0)) : go(float(0));
}

extern "C" int lmp_k_dropout_backward(int dtype, size_t n, const void* g, double rate, uint64_t seed,
                                      const int64_t* used, void* dx) {
  if (int s = check_dropout("lmp_k_dropout_backward: ", dtype, n, rate)) return s;
  if (n == 0) return LMP_OK;
  if (!g || !used || !dx) return fail(LMP_ERR_INVALID, "lmp_k_dropout_backward: null buffer");
  if (int s = check_apart("lmp_k_dropout_backward: ", dtype, n, g, dx)) return s;
  LMP_RUNTIME_OR_FAIL(rt);
  const auto go = [&](auto zero) {
    using T = decltype(zero);
    auto a = dropout_args<T>(n, g, nullptr, rate, seed, dx);
    a.call = used;
    return launch_dropout<T, false>(rt, a, n * sizeof(T) >= kStreamBytes / 2);
  };
  return dtype == LMP_FLOAT64 ? go(double(0)) : go(float(0));
}
