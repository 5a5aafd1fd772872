// One AdamW step over many tensors, its states in 32 or in 8 bits.
//
//   m = beta1 m + (1 - beta1) g,  v = beta2 v + (1 - beta2) g^2
//   p = p (1 - lr decay) - lr m^ / (sqrt(v^) + eps),  m^, v^ corrected by 1 - beta^t
//
// Bound by memory: 28 bytes a parameter with states of 32 bits (p, m, v read and
// written, g read), 16 with states of 8.  All tensors share a launch: their
// pointers ride in the kernel's arguments (kTensors of them), so nothing is
// copied to the device per step and a recorded step replays; a workgroup finds
// a chunk's tensor by bisection of the running chunk counts.  The step count
// lives on the device, and every workgroup forms the two bias corrections from it
// in float64 while its first loads are on their way.
//
// States of 8 bits: a wave owns a block of 256 values, four a lane, so the
// block's scale is a maximum over the wave and a state costs one 4-byte access
// per lane.  What bounds that form is the arithmetic, two hashes' worth of integer
// products and two roots a value, as much as the memory.
//
// Measured, 37.7 million parameters: 177 us = 6.0 TB/s with states of 32 bits; 143 us
// = 4.2 TB/s with states of 8 (178 us with the compiler's exact root and quotient),
// and 29 and 35 us to read them out.  17 thousand parameters in four tensors: 5.2 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <vector>

#include "common.hpp"
#include "lmp_hip_transformer.h"

namespace lmp_hip {
namespace {

constexpr int kTensors = 48;  // a launch's list: 48 x 64 bytes, inside the 4 KiB of arguments
constexpr int kThreads = 256;
// Chunks of UNITS units of four values a lane: four units, whose loads are all on
// their way at once, or one where four would leave compute units idle (17 thousand
// parameters: 8.5 us with four, 5.6 with one; 38 million: 250 us with two).
constexpr int chunk_of(int units) { return kThreads * 4 * units; }
// Workgroups per compute unit at most, each then over its share of the chunks: they
// count themselves done on one counter, 3.4 ns each (38 million parameters, 9216
// chunks: 185 us with 6 a unit, 180 with 18, 177 with 36).
constexpr int kGroupsPerUnit = 36;

typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u1_any __attribute__((aligned(1)));

struct AdamWList {
  float* p[kTensors];
  const float* g[kTensors];
  void* m[kTensors];
  void* v[kTensors];
  float* m_scale[kTensors];
  float* v_scale[kTensors];
  int64_t n[kTensors];
  float keep[kTensors];       // 1 - lr decay
  uint32_t first[kTensors];   // the tensor's first chunk
};

struct AdamWArgs {
  AdamWList list;
  int count;
  uint32_t chunks;
  uint32_t place;  // of the list's first tensor among all of the step's
  float beta1, rest1, beta2, rest2, eps;
  double lr, beta1_d, beta2_d;
  uint32_t seed;
  int64_t* step;
  int advance;  // the last workgroup to finish advances the step
};
static_assert(sizeof(AdamWArgs) <= 4096);

__device__ __forceinline__ double power(double base, int64_t t) {
  double r = 1;
  for (; t > 0; t >>= 1) {
    if (t & 1) r *= base;
    base *= base;
  }
  return r;
}

__device__ __forceinline__ uint32_t mixed(uint32_t x) {  // MurmurHash3's 32-bit finalizer
  x ^= x >> 16;
  x *= 0x85EBCA6Bu;
  x ^= x >> 13;
  x *= 0xC2B2AE35u;
  return x ^ (x >> 16);
}

// One value.  Each operation on the moments rounds once (no contraction), so that a
// state in 8 bits is a function of its inputs alone.  FAST: the parameter's root and
// quotient to a unit in their last places, where the arithmetic is what bounds the
// kernel; they take a v below float32's smallest normal for zero (fast_enough).
template <bool FAST>
__device__ __forceinline__ void step_one(const AdamWArgs& a, float keep, float size, float root,
                                         float g, float& p, float& m, float& v) {
  m = m * a.beta1 + g * a.rest1;
  v = v * a.beta2 + (g * g) * a.rest2;
  if constexpr (FAST)
    p = p * keep - size * (m * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v) * root + a.eps));
  else
    p = p * keep - size * (m / (sqrtf(v) * root + a.eps));
}

// Largest of the wave's values, which are not negative as integers: DPP within
// rows of 16 lanes, then the rows' broadcasts to the next, and lane 63 has it.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
#define LMP_STEP(ctrl, rows) \
  x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), ctrl, rows, 0xF, false)))
  LMP_STEP(0xB1, 0xF);
  LMP_STEP(0x4E, 0xF);
  LMP_STEP(0x141, 0xF);
  LMP_STEP(0x140, 0xF);
  LMP_STEP(0x142, 0xA);
  LMP_STEP(0x143, 0xC);
#undef LMP_STEP
  return uint32_t(__builtin_amdgcn_readlane(int(x), 63));
}

// Codes of a block's four values in this lane.  x scaled to [0, Q^2] has code c
// with c^2 <= t < (c + 1)^2, and moves up to c + 1 with probability
// (t - c^2) / (2 c + 1), the random 16 bits u being below it.  The root may be off
// by a unit in its last place: the two comparisons that follow settle c.
template <int Q>
__device__ __forceinline__ uint32_t encode(const float (&x)[4], const uint32_t (&r)[4],
                                           float* scale, bool first_lane) {
  // As integers, magnitudes order as they do as floats, and NaN is above all.
  uint32_t bits = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    bits = max(bits, __builtin_bit_cast(uint32_t, x[j]) & 0x7fffffffu);
  const float top = __builtin_bit_cast(float, wave_max(bits));
  const bool live = top >= 1e-30f && top < __builtin_inff();
  if (first_lane) *scale = live ? top : top < 1e-30f ? 0.0f : __builtin_nanf("");
  if (!live) return 0;
  const float inv = (1.0f / top) * float(Q * Q);
  uint32_t packed = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float t = fminf(fabsf(x[j]) * inv, float(Q * Q));
    float c = floorf(__builtin_amdgcn_sqrtf(t));
    c = c * c > t ? c - 1 : c;
    c = (c + 1) * (c + 1) <= t ? c + 1 : c;
    c = float(r[j]) * (1.0f / 65536) * (2 * c + 1) < t - c * c ? c + 1 : c;
    if (Q == 255) c = c == 0 && x[j] > 0 ? 1.0f : c;  // t may underflow
    c = fminf(c, float(Q));
    const int code = x[j] < 0 ? -int(c) : int(c);
    packed |= uint32_t(code & 255) << (8 * j);
  }
  return packed;
}

template <bool SIGNED>
__device__ __forceinline__ float decoded(uint32_t packed, int j, float unit) {
  const uint32_t byte = (packed >> (8 * j)) & 255;
  const float c = SIGNED ? float(int(int8_t(byte))) : float(byte);
  return (c * fabsf(c)) * unit;
}
constexpr float kUnitM = float(1.0 / (127 * 127)), kUnitV = float(1.0 / (255 * 255));

// STREAM: accesses with the nontemporal hint (38 million parameters: 197 us without,
// 177 with).
template <int BITS, int kUnits, bool STREAM, bool FAST>
__global__ __launch_bounds__(kThreads) void adamw_step(AdamWArgs a) {
  __shared__ float factors[2];
  const int64_t t = a.step[0] + 1;
  // The factors, one in each of two lanes, while the first loads are on their way.
  const auto corrections = [&] {
    if (threadIdx.x < 2) {
      const bool second = threadIdx.x == 1;
      const double rest = 1.0 - power(second ? a.beta2_d : a.beta1_d, t);
      factors[threadIdx.x] = float((second ? 1.0 : a.lr) / (second ? sqrt(rest) : rest));
    }
    __syncthreads();
  };
  for (uint32_t chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) {
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (chunk >= a.list.first[mid]) lo = mid;
      else hi = mid - 1;
    }
    const int i = lo;
    const int64_t n = a.list.n[i];
    float* p = a.list.p[i];
    const float* g = a.list.g[i];
    const float keep = a.list.keep[i];
    const int64_t begin = int64_t(chunk - a.list.first[i]) * chunk_of(kUnits);
    float pv[kUnits][4], gv[kUnits][4];
    const auto at_of = [&](int u) { return begin + (int64_t(u) * kThreads + threadIdx.x) * 4; };
    const auto load4 = [&](const float* from, int64_t at, float (&v)[4]) {
      if (at + 4 <= n) {
        const auto* q = reinterpret_cast<const f4*>(from + at);
        const f4 x = STREAM ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = x[j];
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = at + j < n ? from[at + j] : 0.0f;
      }
    };
    const auto store4 = [&](float* to, int64_t at, const float (&v)[4]) {
      if (at + 4 <= n) {
        auto* q = reinterpret_cast<f4*>(to + at);
        if constexpr (STREAM) __builtin_nontemporal_store(f4{v[0], v[1], v[2], v[3]}, q);
        else *q = f4{v[0], v[1], v[2], v[3]};
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (at + j < n) to[at + j] = v[j];
      }
    };
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      load4(p, at_of(u), pv[u]);
      load4(g, at_of(u), gv[u]);
    }
    if constexpr (BITS == 32) {
      float* m = static_cast<float*>(a.list.m[i]);
      float* v = static_cast<float*>(a.list.v[i]);
      float mv[kUnits][4], vv[kUnits][4];
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        load4(m, at_of(u), mv[u]);
        load4(v, at_of(u), vv[u]);
      }
      if (chunk == blockIdx.x) corrections();
      const float size = factors[0], root = factors[1];
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          step_one<FAST>(a, keep, size, root, gv[u][j], pv[u][j], mv[u][j], vv[u][j]);
        store4(p, at_of(u), pv[u]);
        store4(m, at_of(u), mv[u]);
        store4(v, at_of(u), vv[u]);
      }
    } else {
      uint8_t* m = static_cast<uint8_t*>(a.list.m[i]);
      uint8_t* v = static_cast<uint8_t*>(a.list.v[i]);
      uint32_t mc[kUnits], vc[kUnits];
      float ms[kUnits], vs[kUnits];
      const auto codes = [&](const uint8_t* from, int64_t at) -> uint32_t {
        if (at + 4 <= n) return *reinterpret_cast<const u1_any*>(from + at);
        uint32_t c = 0;
        for (int j = 0; j < 4; ++j)
          if (at + j < n) c |= uint32_t(from[at + j]) << (8 * j);
        return c;
      };
      const auto put = [&](uint8_t* to, int64_t at, uint32_t c) {
        if (at + 4 <= n) {
          *reinterpret_cast<u1_any*>(to + at) = c;
        } else {
          for (int j = 0; j < 4; ++j)
            if (at + j < n) to[at + j] = uint8_t(c >> (8 * j));
        }
      };
      // A wave's 64 lanes x 4 values of one unit are one block.
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int64_t block = at_of(u) / LMP_ADAMW_BLOCK;
        const bool there = block * LMP_ADAMW_BLOCK < n;
        mc[u] = codes(m, at_of(u));
        vc[u] = codes(v, at_of(u));
        ms[u] = there ? a.list.m_scale[i][block] : 0.0f;
        vs[u] = there ? a.list.v_scale[i][block] : 0.0f;
      }
      if (chunk == blockIdx.x) corrections();
      const float size = factors[0], root = factors[1];
      const uint32_t key = mixed(mixed(uint32_t(t) ^ a.seed) + 0x9E3779B9u * (a.place + uint32_t(i) + 1));
#pragma unroll
      for (int u = 0; u < kUnits; ++u) {
        const int64_t at = at_of(u), block = at / LMP_ADAMW_BLOCK;
        if (block * LMP_ADAMW_BLOCK >= n) continue;  // the whole wave
        const uint32_t key_here = key ^ (uint32_t(uint64_t(at) >> 32) * 0x85EBCA6Bu);
        float mv[4], vv[4];
        uint32_t lo16[4], hi16[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mv[j] = decoded<true>(mc[u], j, ms[u] * kUnitM);
          vv[j] = decoded<false>(vc[u], j, vs[u] * kUnitV);
          step_one<FAST>(a, keep, size, root, gv[u][j], pv[u][j], mv[j], vv[j]);
          if (at + j >= n) mv[j] = vv[j] = 0.0f;
          const uint32_t r = mixed(uint32_t(at + j) ^ key_here);
          lo16[j] = r & 0xFFFF;
          hi16[j] = r >> 16;
        }
        const bool first_lane = (threadIdx.x & 63) == 0;
        const uint32_t m2 = encode<127>(mv, lo16, a.list.m_scale[i] + block, first_lane);
        const uint32_t v2 = encode<255>(vv, hi16, a.list.v_scale[i] + block, first_lane);
        store4(p, at, pv[u]);
        put(m, at, m2);
        put(v, at, v2);
      }
    }
  }
  if (a.advance && threadIdx.x == 0) {
    // This workgroup read the step before its barrier; the last to come here
    // finds that all have, and the next launch finds the counter at 0.
    unsigned long long* done = reinterpret_cast<unsigned long long*>(a.step + 1);
    if (atomicAdd(done, 1ull) == gridDim.x - 1) {
      *done = 0;
      a.step[0] += 1;
    }
  }
}

__global__ void adamw_advance(int64_t* step) { step[0] += 1; }

template <bool SIGNED>
__global__ __launch_bounds__(kThreads) void adamw_values(const uint8_t* codes, const float* scales,
                                                         int64_t n, float* out, bool stream) {
  constexpr int kUnits = 4, kPerGroup = chunk_of(kUnits);
  constexpr float unit = SIGNED ? kUnitM : kUnitV;
  for (int64_t begin = int64_t(blockIdx.x) * kPerGroup; begin < n;
       begin += int64_t(gridDim.x) * kPerGroup) {
    uint32_t c[kUnits];
    float s[kUnits];
    const auto at_of = [&](int u) { return begin + (int64_t(u) * kThreads + threadIdx.x) * 4; };
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int64_t at = at_of(u);
      c[u] = 0;
      s[u] = at < n ? scales[at / LMP_ADAMW_BLOCK] * unit : 0.0f;
      if (at + 4 <= n) {
        c[u] = *reinterpret_cast<const u1_any*>(codes + at);
      } else {
        for (int j = 0; j < 4; ++j)
          if (at + j < n) c[u] |= uint32_t(codes[at + j]) << (8 * j);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int64_t at = at_of(u);
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = decoded<SIGNED>(c[u], j, s[u]);
      if (at + 4 <= n) {
        auto* q = reinterpret_cast<f4*>(out + at);
        if (stream) __builtin_nontemporal_store(f4{v[0], v[1], v[2], v[3]}, q);
        else *q = f4{v[0], v[1], v[2], v[3]};
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (at + j < n) out[at + j] = v[j];
      }
    }
  }
}

// Whether eps hides what the fast root and quotient take for zero: a v below 2^-126, whose
// corrected root is below 2^-63 / sqrt(1 - beta2), against 2^-24 of eps.
bool fast_enough(double eps, double beta2) { return eps >= 0x1p-39 / std::sqrt(1 - beta2); }

// Two of the buffers that a step writes, if any two overlap: workgroups take them
// without order, so an element that two entries hold would be stepped once or twice.
struct Written {
  uintptr_t begin, end;
  size_t tensor;
};
bool find_overlap(int bits, size_t count, const lmp_adamw_tensor* tensors, Written (&pair)[2]) {
  std::vector<Written> all;
  all.reserve(count * (bits == 8 ? 5 : 3));
  for (size_t i = 0; i < count; ++i) {
    const lmp_adamw_tensor& t = tensors[i];
    if (t.n == 0) continue;
    const auto add = [&](const void* p, uint64_t bytes) {
      const auto at = reinterpret_cast<uintptr_t>(p);
      all.push_back({at, at + bytes, i});
    };
    const uint64_t state = t.n * (bits == 8 ? 1 : 4);
    add(t.p, t.n * 4);
    add(t.m, state);
    add(t.v, state);
    if (bits == 8) {
      const uint64_t scales = (t.n + LMP_ADAMW_BLOCK - 1) / LMP_ADAMW_BLOCK * 4;
      add(t.m_scale, scales);
      add(t.v_scale, scales);
    }
  }
  std::sort(all.begin(), all.end(), [](const Written& x, const Written& y) { return x.begin < y.begin; });
  for (size_t i = 1; i < all.size(); ++i)
    if (all[i].begin < all[i - 1].end) {
      pair[0] = all[i - 1];
      pair[1] = all[i];
      return true;
    }
  return false;
}

}  // namespace
}  // namespace lmp_hip

using namespace lmp_hip;

extern "C" int lmp_k_adamw_f32(int bits, size_t count, const lmp_adamw_tensor* tensors, double lr,
                               double beta1, double beta2, double eps, uint64_t seed,
                               int64_t* step) {
  const char* name = "lmp_k_adamw_f32: ";
  if (bits != 32 && bits != 8)
    return fail(LMP_ERR_INVALID, std::string(name) + "states have 32 or 8 bits, not " +
                                     std::to_string(bits));
  if (!step) return fail(LMP_ERR_INVALID, std::string(name) + "null step");
  if (count && !tensors) return fail(LMP_ERR_INVALID, std::string(name) + "null list of tensors");
  if (!std::isfinite(lr)) return fail(LMP_ERR_INVALID, std::string(name) + "lr is not finite");
  if (!(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1))
    return fail(LMP_ERR_INVALID, std::string(name) + "beta1 and beta2 lie in [0, 1)");
  if (!(eps >= 0) || std::isinf(eps))
    return fail(LMP_ERR_INVALID, std::string(name) + "eps is negative or not finite");
  if (count > (size_t(1) << 31))
    return fail(LMP_ERR_UNSUPPORTED, std::string(name) + "more than 2^31 tensors");
  for (size_t i = 0; i < count; ++i) {
    const lmp_adamw_tensor& t = tensors[i];
    const std::string which = std::string(name) + "tensor " + std::to_string(i) + ": ";
    if (!std::isfinite(t.decay)) return fail(LMP_ERR_INVALID, which + "decay is not finite");
    if (t.n == 0) continue;
    if (!t.p || !t.g || !t.m || !t.v) return fail(LMP_ERR_INVALID, which + "null buffer");
    if (bits == 8 && (!t.m_scale || !t.v_scale))
      return fail(LMP_ERR_INVALID, which + "states of 8 bits need their scales");
    if (t.n > (uint64_t(1) << 35))
      return fail(LMP_ERR_UNSUPPORTED, which + "more than 2^35 values");
  }
  try {  // host memory can run out; no exception crosses the C boundary
    Written pair[2];
    if (find_overlap(bits, count, tensors, pair))
      return fail(LMP_ERR_INVALID, std::string(name) + "buffers that the step writes overlap: of tensors " +
                                       std::to_string(std::min(pair[0].tensor, pair[1].tensor)) + " and " +
                                       std::to_string(std::max(pair[0].tensor, pair[1].tensor)));
  } catch (const std::exception& e) {
    return fail(LMP_ERR_OOM, std::string(name) + e.what());
  }
  LMP_RUNTIME_OR_FAIL(rt);
  AdamWArgs a{};
  a.beta1 = float(beta1);
  a.rest1 = float(1 - beta1);
  a.beta2 = float(beta2);
  a.rest2 = float(1 - beta2);
  a.eps = float(eps);
  a.lr = lr;
  a.beta1_d = beta1;
  a.beta2_d = beta2;
  a.seed = uint32_t(seed);
  a.step = step;
  uint64_t values = 0;
  for (size_t i = 0; i < count; ++i) values += tensors[i].n;
  // Bytes of all tensors against the memory-side cache (kStreamBytes).
  const bool stream = values * (bits == 32 ? 16 : 10) >= kStreamBytes;
  const bool fast = fast_enough(eps, beta2);
  const bool few = values <= uint64_t(rt->cu_count) * chunk_of(4);
  const int chunk = chunk_of(few ? 1 : 4);
  uint64_t chunks = 0;
  bool advanced = false;
  const auto launch = [&]() -> int {
    a.chunks = uint32_t(chunks);
    const dim3 grid(uint32_t(std::min<uint64_t>(chunks, uint64_t(rt->cu_count) * kGroupsPerUnit)));
    const auto run = [&](auto kernel) { kernel<<<grid, dim3(kThreads), 0, rt->stream>>>(a); };
    if (bits == 32)
      run(few      ? adamw_step<32, 1, false, false>
          : stream ? adamw_step<32, 4, true, false>
                   : adamw_step<32, 4, false, false>);
    else if (!fast)
      run(few ? adamw_step<8, 1, false, false> : adamw_step<8, 4, false, false>);
    else
      run(few ? adamw_step<8, 1, false, true> : stream ? adamw_step<8, 4, true, true> : adamw_step<8, 4, false, true>);
    LMP_LAUNCH_CHECK("adamw_step");
    return LMP_OK;
  };
  // A launch takes tensors until its list is full or its chunks pass 32 bits (a
  // tensor alone does not).
  constexpr uint64_t kMostChunks = uint64_t(1) << 31;
  for (size_t i = 0; i < count; ++i) {
    const lmp_adamw_tensor& t = tensors[i];
    const uint64_t need = (t.n + chunk - 1) / chunk;
    if (need == 0 && a.count == 0) continue;
    if (a.count == kTensors || (a.count && chunks + need > kMostChunks)) {
      if (int s = launch()) return s;
      a.count = 0;
      chunks = 0;
      if (need == 0) continue;
    }
    if (a.count == 0) a.place = uint32_t(i);
    // A tensor without values keeps its place, and no chunk.
    const int k = a.count++;
    a.list.p[k] = t.p;
    a.list.g[k] = t.g;
    a.list.m[k] = t.m;
    a.list.v[k] = t.v;
    a.list.m_scale[k] = t.m_scale;
    a.list.v_scale[k] = t.v_scale;
    a.list.n[k] = int64_t(t.n);
    a.list.keep[k] = float(1 - lr * t.decay);
    a.list.first[k] = uint32_t(chunks);
    chunks += need;
  }
  if (chunks) {
    a.advance = 1;  // the last launch's last workgroup
    advanced = true;
    if (int s = launch()) return s;
  }
  if (!advanced) {
    adamw_advance<<<dim3(1), dim3(1), 0, rt->stream>>>(step);
    LMP_LAUNCH_CHECK("adamw_advance");
  }
  return LMP_OK;
}

extern "C" int lmp_k_adamw_decode(int signed_codes, const void* codes, const float* scales,
                                  size_t n, float* out) {
  if (n == 0) return LMP_OK;
  if (!codes || !scales || !out) return fail(LMP_ERR_INVALID, "lmp_k_adamw_decode: null buffer");
  if (n > (size_t(1) << 40)) return fail(LMP_ERR_UNSUPPORTED, "lmp_k_adamw_decode: too many values");
  LMP_RUNTIME_OR_FAIL(rt);
  const size_t groups = std::min<size_t>((n + chunk_of(4) - 1) / chunk_of(4), size_t(rt->cu_count) * 256);
  const bool stream = n * sizeof(float) > kStreamStoreBytes;
  const uint8_t* c = static_cast<const uint8_t*>(codes);
  if (signed_codes)
    adamw_values<true><<<dim3(uint32_t(groups)), dim3(kThreads), 0, rt->stream>>>(c, scales,
                                                                                   int64_t(n), out, stream);
  else
    adamw_values<false><<<dim3(uint32_t(groups)), dim3(kThreads), 0, rt->stream>>>(c, scales,
                                                                                    int64_t(n), out, stream);
  LMP_LAUNCH_CHECK("adamw_decode");
  return LMP_OK;
}
