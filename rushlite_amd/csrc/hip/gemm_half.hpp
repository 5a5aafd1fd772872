// fp32 products on the fp16 matrix cores, each operand in two fp16 parts.
//
// Why.  A value scaled by a power of two is x = h + m + r with h = fp16(x), m =
// fp16(x - h) and |r| <= 2^-22 |x|, so
//   a b = ah bh + ah bm + am bh + (am bm and what the r leave out: 3 x 2^-22 at most)
// is three fp16 MFMAs with fp32 accumulation, half of what three bf16 parts cost
// (gemm_bf3.hpp), with a product's error near that of rounding its operands: a sum's
// error is its own roundings'.
//
// Range.  Each row of A and each column of B has a power of two that takes its
// largest magnitude to [2^14, 2^15), found in a pass of its own (or by the kernel that
// makes the operand): values down to 2^-17 of the largest keep both parts whole,
// smaller ones lose at most 2^-40 of it.  The two powers leave the sum at the end, exactly.
// An infinity or a NaN leaves a sum that is not finite; a workgroup that finds one
// forms its tile again with fp32 MFMAs on the operands as they are.
//
// Structure.  A workgroup owns a BM x BN tile, its waves TM x TN blocks of 32 x 32; K
// advances 32 at a time through two LDS stages with one barrier a step.  Loads go
// through registers, one step ahead, are split there (five VALU operations a pair)
// and stored as two planes of 16-byte octets, [plane][k / 8][row], in which a fragment of
// one MFMA is one conflict-free 128-bit read a lane.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "gemm_plan.hpp"

namespace lmp_hip {
namespace {

typedef _Float16 hf2 __attribute__((ext_vector_type(2)));
typedef _Float16 hf8 __attribute__((ext_vector_type(8)));
typedef float hv2 __attribute__((ext_vector_type(2)));
typedef float hv4 __attribute__((ext_vector_type(4)));
typedef float hv4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef float hv16 __attribute__((ext_vector_type(16)));
typedef uint32_t hu4 __attribute__((ext_vector_type(4)));
typedef int hi4 __attribute__((ext_vector_type(4)));

// Kept out of the templates: a target builtin inside a kernel template keeps the host
// pass from emitting the kernel's launch stub.
__device__ __forceinline__ hv16 mfma_f16(hf8 a, hf8 b, hv16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ hv16 mfma_full(float a, float b, hv16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}
// Two values times s into the two parts, packed.
__device__ __forceinline__ void half_pair(float x, float y, float s, uint32_t& h, uint32_t& m) {
  const hf2 a = __builtin_convertvector(hv2{x * s, y * s}, hf2);
  hf2 b;
  b.x = _Float16(__builtin_fmaf(x, s, -float(a.x)));
  b.y = _Float16(__builtin_fmaf(y, s, -float(a.y)));
  h = __builtin_bit_cast(uint32_t, a);
  m = __builtin_bit_cast(uint32_t, b);
}

// The exponent of a row's power of two from the bits of its largest magnitude: [2^14,
// 2^15) where that is at least 2^-112 and finite.  Subnormal rows and rows of zeros take
// 2^126; infinities and NaN leave their mark whatever they are multiplied by.
__device__ __forceinline__ int half_exponent(uint32_t top) { return min(141 - int(top >> 23), 126); }
__device__ __forceinline__ float power_of(int e) {
  return __builtin_bit_cast(float, uint32_t(e + 127) << 23);
}

template <int WM_, int WN_, int TM_, int TN_, int MINB_>
struct HalfCfg {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, MINB = MINB_;
  static constexpr int NW = WM * WN, THREADS = 64 * NW;
  static constexpr int BM = WM * TM * 32, BN = WN * TN * 32;
  static constexpr int A_OCT = BM * 16 + 64, B_OCT = BN * 16 + 64;  // bytes
  static constexpr int A_PLANE = 4 * A_OCT, B_PLANE = 4 * B_OCT;
  static constexpr int STAGE = 2 * (A_PLANE + B_PLANE);
  static constexpr int SMEM = 2 * STAGE + 16;  // the stages and the fallback's flag
  static_assert(2 * STAGE >= NW * 32 * 36 * 4, "the epilogue's wave tiles fit");
  static_assert(2 * STAGE >= kHalfK * (BM + BN + 8) * 4, "the fallback's panels fit");
};

// One operand's panel of R rows (of m or n) x 32 k on its way from memory to LDS.  A
// thread holds ITEMS items of eight consecutive k of one row.  KMAJOR: k is contiguous.
template <int R, int THREADS, bool KMAJOR>
struct HalfPanel {
  static constexpr int ITEMS = R * 4 / THREADS;
  static constexpr int PAIRS = ITEMS * 4;
  static_assert(ITEMS * THREADS == R * 4, "items split evenly over the threads");
  // A load's address is a uniform base and the lane's own 32-bit offset, constant over K.
  const char* base;
  int ld, k[ITEMS], off[ITEMS];
  uint32_t at[ITEMS];
  float s[ITEMS];  // the row's power of two
  float v[ITEMS][8];

  static __device__ __forceinline__ int row_of(int i) {
    const int q = int(threadIdx.x) + i * THREADS;
    return KMAJOR ? q / 4 : q % R;
  }
  // `origin`: the value at k = 0 of the tile's first row; `local(r)`: how many rows after it
  // the tile's r-th is; `k0` the first k that load() reads; `tops`: the bits of the largest
  // magnitudes, from the tile's first row on.
  template <class Local>
  __device__ __forceinline__ void init(const float* origin, int ld_, Local&& local, int k0,
                                       int oct_bytes, const uint32_t* tops) {
    ld = ld_;
    base = reinterpret_cast<const char*>(origin + (KMAJOR ? int64_t(k0) : int64_t(k0) * ld));
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int q = int(threadIdx.x) + i * THREADS;
      const int row = row_of(i), oct = KMAJOR ? q % 4 : q / R;
      k[i] = 8 * oct;
      const int r = local(row);
      at[i] = 4u * (KMAJOR ? uint32_t(r) * uint32_t(ld) + uint32_t(k[i]) : uint32_t(k[i]) * uint32_t(ld) + uint32_t(r));
      off[i] = oct * oct_bytes + row * 16;
      s[i] = power_of(half_exponent(tops[r]));
    }
  }
  __device__ __forceinline__ const float* place(int64_t bytes, int i) const {
    return reinterpret_cast<const float*>(base + bytes + at[i]);
  }
  __device__ __forceinline__ void load(int i) {
    if constexpr (KMAJOR) {
#pragma unroll
      for (int j = 0; j < 8; j += 4) {
        const hv4_any x = *reinterpret_cast<const hv4_any*>(place(4 * j, i));
        v[i][j] = x.x; v[i][j + 1] = x.y; v[i][j + 2] = x.z; v[i][j + 3] = x.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = *place(int64_t(j) * ld * 4, i);
    }
  }
  __device__ __forceinline__ void move(int advance) { base += int64_t(advance) * (KMAJOR ? 4 : 4 * int64_t(ld)); }
  __device__ __forceinline__ void load_all(int advance) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) load(i);
    move(advance);
  }
  // A step of `left` values of k that starts `after` k past the base, zeros after them.
  __device__ __forceinline__ void load_tail(int after, int left) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] = 0.0f;
        if (k[i] + j < left) v[i][j] = *place(int64_t(after + j) * (KMAJOR ? 4 : 4 * int64_t(ld)), i);
      }
  }
  __device__ __forceinline__ void put(int i, char* lds, int plane, const uint32_t (&h)[4],
                                      const uint32_t (&m)[4]) const {
    *reinterpret_cast<hu4*>(lds + off[i]) = hu4{h[0], h[1], h[2], h[3]};
    *reinterpret_cast<hu4*>(lds + off[i] + plane) = hu4{m[0], m[1], m[2], m[3]};
  }
  __device__ __forceinline__ void store_all(char* lds, int plane) const {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      uint32_t h[4], m[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) half_pair(v[i][2 * j], v[i][2 * j + 1], s[i], h[j], m[j]);
      put(i, lds, plane, h, m);
    }
  }
  // The values themselves, [k][row] with R + 4 values per k (the fallback).
  __device__ __forceinline__ void store_values(float* lds) const {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int row = row_of(i);
#pragma unroll
      for (int j = 0; j < 8; ++j) lds[(k[i] + j) * (R + 4) + row] = v[i][j];
    }
  }
};

// A product op(A) [m, k] op(B) [k, n].  `a_top` and `b_top`: the bits of the largest
// magnitude of each row of op(A) and column of op(B), rounded up to 256 of them.
struct HalfArgs {
  const float *a, *b;
  int m, n, k, lda, ldb;  // lda, ldb below 2^22: a panel's offsets fit 32 bits
  const uint32_t *a_top, *b_top;
  int tiles_m, tiles_n;
  int splits, steps_per_split;  // K splits, and 32-wide k steps in each
};

// Where a work item lies: its tile's origin in tiles, and its split of K.
struct HalfItem {
  int tile_m, tile_n, split;
};

// Consecutive ids go round the eight XCDs: each takes a contiguous run of (split, tile),
// so that its L2 sees one range of k and neighbouring tiles, in groups of eight tile rows.
__device__ __forceinline__ HalfItem half_item(const HalfArgs& g, int id) {
  const int ntiles = g.tiles_m * g.tiles_n, total = ntiles * g.splits;
  {
    const int q = total / 8, r = total % 8, x = id % 8;
    id = x * q + min(x, r) + id / 8;
  }
  const int split = id / ntiles, tile = id - split * ntiles;
  constexpr int kGroup = 8;
  const int per_group = kGroup * g.tiles_n, group = tile / per_group;
  const int gsize = min(g.tiles_m - group * kGroup, kGroup);
  const int in_group = tile - group * per_group;
  return {group * kGroup + in_group % gsize, in_group / gsize, split};
}

// The tile's sums, scaled by the powers of two of rows and columns, into acc: block (i, j)
// of the wave, register r: row 8 (r / 4) + 4 (lane / 32) + r % 4, column lane % 32.
// The tile's first column of op(B) is b0, its c-th lies b_local(c) after it; rows and
// columns past the matrix repeat one of it.  Returns false where the sums come from the
// fallback: unscaled.
template <class C, bool TA, bool TB, class Local>
__device__ __forceinline__ bool half_tile(const HalfArgs& g, const HalfItem& at, int b0, Local&& b_local,
                                          char* smem, hv16 (&acc)[C::TM][C::TN]) {
  constexpr int TM = C::TM, TN = C::TN, MM = TM * TN;
  const int m0 = at.tile_m * C::BM;
  const int k_begin = at.split * g.steps_per_split * kHalfK;
  const int k_len = min(g.k - k_begin, g.steps_per_split * kHalfK);
  const int full = k_len / kHalfK, left = k_len % kHalfK, steps = full + (left ? 1 : 0);
  int* flag = reinterpret_cast<int*>(smem + 2 * C::STAGE);
  if (threadIdx.x == 0) *flag = 0;  // set after the K loop's barriers

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int li = lane & 31, lh = lane >> 5;

  const auto a_local = [&](int r) { return min(r, g.m - 1 - m0); };
  const float* a_origin = g.a + (TA ? int64_t(m0) : int64_t(m0) * g.lda);
  const float* b_origin = g.b + (TB ? int64_t(b0) * g.ldb : int64_t(b0));
  using PA = HalfPanel<C::BM, C::THREADS, !TA>;
  using PB = HalfPanel<C::BN, C::THREADS, TB>;
  PA pa;
  PB pb;
  // Loads past the last whole step repeat it (and are not used); a split without a whole
  // step reads the 32 k before the end of K for them (K >= 32).
  const int k_load = min(k_begin, g.k - kHalfK);
  pa.init(a_origin, g.lda, a_local, k_load, C::A_OCT, g.a_top + m0);
  pb.init(b_origin, g.ldb, b_local, k_load, C::B_OCT, g.b_top + b0);
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = hv16(0.0f);

  const int a_at = lh * C::A_OCT + (wm * TM * 32 + li) * 16;
  const int b_at = 2 * C::A_PLANE + lh * C::B_OCT + (wn * TN * 32 + li) * 16;
  // Fragments of 16 k: the leading parts of B in two sets, so that the next ones are read
  // while the leading product runs.
  hf8 ah[TM], am[TM], bh[2][TN], bm[TN];
  const auto read_a = [&](hf8 (&f)[TM], const char* s, int plane, int kh) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
      f[i] = *reinterpret_cast<const hf8*>(s + plane * C::A_PLANE + kh * 2 * C::A_OCT + a_at + i * 512);
  };
  const auto read_b = [&](hf8 (&f)[TN], const char* s, int plane, int kh) {
#pragma unroll
    for (int j = 0; j < TN; ++j)
      f[j] = *reinterpret_cast<const hf8*>(s + plane * C::B_PLANE + kh * 2 * C::B_OCT + b_at + j * 512);
  };
  const auto product = [&](const hf8 (&x)[TM], const hf8 (&y)[TN]) {
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = mfma_f16(x[i], y[j], acc[i][j]);
  };

  // The step with the end of K first (when 32 does not divide it), then the whole ones:
  // stage t % 2 holds step t, the registers the one after it.
  int ahead = full;  // whole steps not loaded yet
  const auto advance = [&]() { return ahead > 1 ? kHalfK : 0; };
  if (left) {
    pa.load_tail(k_begin - k_load + full * kHalfK, left);
    pb.load_tail(k_begin - k_load + full * kHalfK, left);
  } else {
    pa.load_all(advance());
    pb.load_all(advance());
    --ahead;
  }
  pa.store_all(smem, C::A_PLANE);
  pb.store_all(smem + 2 * C::A_PLANE, C::B_PLANE);
  {
    const int adv = advance();
    pa.load_all(adv);
    pb.load_all(adv);
    --ahead;
  }
  // The leading product of a step's second half is held past the barrier; zeros at first.
#pragma unroll
  for (int i = 0; i < TM; ++i) ah[i] = hf8(0);
#pragma unroll
  for (int j = 0; j < TN; ++j) bh[1][j] = hf8(0);
  constexpr int PAIRS = PA::PAIRS + PB::PAIRS;
  const auto step = [&](auto stage_c) {
    constexpr int stage = decltype(stage_c)::value;
    const char* s = smem + stage * C::STAGE;
    char* d = smem + (stage ^ 1) * C::STAGE;
    __syncthreads();
    const int adv = advance();
    --ahead;
    read_a(am, s, 1, 0);
    read_b(bh[0], s, 0, 0);
    __builtin_amdgcn_sched_barrier(0);
    product(ah, bh[1]);
    __builtin_amdgcn_sched_barrier(0);
    read_a(ah, s, 0, 0);
    read_b(bm, s, 1, 0);
    uint32_t h[4], m[4];
#pragma unroll
    for (int c = 0; c < PAIRS; ++c) {
      // The five products of the step in order, spread over the pairs; each one's fragments
      // are read when their registers fall free, a product ahead of it.
      const int q0 = c * 5 * MM / PAIRS, q1 = (c + 1) * 5 * MM / PAIRS;
      const bool of_a = c < PA::PAIRS;
      const int ca = of_a ? c : c - PA::PAIRS;
      const int it = ca / 4, pr = ca % 4;
      if (of_a) half_pair(pa.v[it][2 * pr], pa.v[it][2 * pr + 1], pa.s[it], h[pr], m[pr]);
      else half_pair(pb.v[it][2 * pr], pb.v[it][2 * pr + 1], pb.s[it], h[pr], m[pr]);
#pragma unroll
      for (int q = q0; q < q1; ++q) {
        if (q == MM) read_a(am, s, 1, 1);
        if (q == 2 * MM) read_b(bh[1], s, 0, 1);
        if (q == 2 * MM) read_b(bm, s, 1, 1);
        if (q == 3 * MM) read_a(ah, s, 0, 1);
        const int pp = q / MM, i = (q % MM) / TN, j = q % TN;
        const hf8 x = pp == 0 || pp == 3 ? am[i] : ah[i];
        const hf8 y = pp == 0 || pp == 2 ? bh[0][j] : pp == 3 ? bh[1][j] : bm[j];
        acc[i][j] = mfma_f16(x, y, acc[i][j]);
      }
      if (of_a && pr == 3) {
        pa.put(it, d, C::A_PLANE, h, m);
        pa.load(it);
      }
      if (!of_a && pr == 3) {
        pb.put(it, d + 2 * C::A_PLANE, C::B_PLANE, h, m);
        pb.load(it);
      }
      // Masks: 0x8 MFMA, 0x100 LDS read, 0x2 VALU.
#pragma unroll
      for (int q = q0; q < q1; ++q) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);
      }
      if (c < PAIRS - 1) __builtin_amdgcn_sched_barrier(0);
    }
    pa.move(adv);
    pb.move(adv);
  };
  int t = 0;
  while (t + 1 < steps) {
    step(std::integral_constant<int, 0>{});
    ++t;
    step(std::integral_constant<int, 1>{});
    ++t;
  }
  if (t < steps) step(std::integral_constant<int, 0>{});
  product(ah, bh[1]);
  __syncthreads();

  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        top = max(top, __builtin_bit_cast(uint32_t, float(acc[i][j][r])) & 0x7fffffffu);
  if (top >= 0x7f800000u) *flag = 1;
  __syncthreads();
  if (!*flag) return true;

  // fp32 MFMAs on the values as they are.
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = hv16(0.0f);
  pa.init(a_origin, g.lda, a_local, k_load, C::A_OCT, g.a_top + m0);
  pb.init(b_origin, g.ldb, b_local, k_load, C::B_OCT, g.b_top + b0);
  constexpr int PITCH_A = C::BM + 4, PITCH_B = C::BN + 4;
  float* sa = reinterpret_cast<float*>(smem);
  float* sb = sa + kHalfK * PITCH_A;
#pragma unroll 1
  for (int u = 0; u < steps; ++u) {
    if (u == 0 && left) {
      pa.load_tail(k_begin - k_load + full * kHalfK, left);
      pb.load_tail(k_begin - k_load + full * kHalfK, left);
    } else {
      const int adv = u + 1 < steps ? kHalfK : 0;
      pa.load_all(adv);
      pb.load_all(adv);
    }
    __syncthreads();  // the step before is read
    pa.store_values(sa);
    pb.store_values(sb);
    __syncthreads();
#pragma unroll 4
    for (int k = 0; k < kHalfK; k += 2) {
      float xa[TM], xb[TN];
#pragma unroll
      for (int i = 0; i < TM; ++i) xa[i] = sa[(k + lh) * PITCH_A + (wm * TM + i) * 32 + li];
#pragma unroll
      for (int j = 0; j < TN; ++j) xb[j] = sb[(k + lh) * PITCH_B + (wn * TN + j) * 32 + li];
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma_full(xa[i], xb[j], acc[i][j]);
    }
  }
  __syncthreads();  // the epilogue writes over the panels
  return false;
}

// Calls f(row, column, values) for every four consecutive columns of the wave's rows: values
// [j] are block column j's at columns column + 32 j of the tile (so a lane has the same place
// of every block), unscaled.  Through a wave-private LDS tile of 16 rows (LDS requests
// of one wave complete in order).
template <class C, class F>
__device__ __forceinline__ void half_epilogue(const HalfArgs& g, const HalfItem& at, bool scaled,
                                              char* smem, const uint32_t* const (&b_tops)[C::TN],
                                              hv16 (&acc)[C::TM][C::TN], F&& f) {
  constexpr int TM = C::TM, TN = C::TN, PITCH = 32 * TN + 4;
  static_assert(2 * C::STAGE >= C::NW * 16 * PITCH * 4, "the wave tiles fit");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / C::WN, wn = wave % C::WN;
  const int li = lane & 31, lh = lane >> 5;
  float* w = reinterpret_cast<float*>(smem) + wave * (16 * PITCH);
  const int c4 = 4 * (lane & 7);
  hi4 eb[TN];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) eb[j][e] = scaled ? half_exponent(b_tops[j][c4 + e]) : 0;
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 8; ++r)
          w[((r / 4) * 8 + lh * 4 + r % 4) * PITCH + j * 32 + li] = acc[i][j][8 * half + r];
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int rr = q * 8 + (lane >> 3);
        const int row = at.tile_m * C::BM + (wm * TM + i) * 32 + half * 16 + rr;
        const int ea = scaled ? half_exponent(g.a_top[row]) : 0;
        hv4 v[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          v[j] = *reinterpret_cast<const hv4*>(w + rr * PITCH + j * 32 + c4);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][e] = ldexpf(v[j][e], -(ea + eb[j][e]));
        }
        f(row, c4, v);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
}

// Four values of a row from `col` on, as far as the row's n go.
__device__ __forceinline__ void store_four(float* row, int col, int n, hv4 v) {
  if (col + 4 <= n) {
    *reinterpret_cast<hv4_any*>(row + col) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < n) row[col + e] = v[e];
  }
}

using HalfBig = HalfCfg<2, 4, 4, 2, 1>;   // 256 x 256, 8 waves of 128 x 64
using HalfWide = HalfCfg<4, 2, 2, 2, 2>;  // 256 x 128, 8 waves of 64 x 64
using HalfMid = HalfCfg<4, 2, 1, 2, 4>;   // 128 x 128, 8 waves of 32 x 64, two a CU
using HalfFlat = HalfCfg<2, 2, 1, 2, 2>;  // 64 x 128, 4 waves of 32 x 64, three a CU

// kHalfTiles is what these types are.
template <class C>
constexpr bool half_is(int cfg) {
  return kHalfTiles[cfg].bm == C::BM && kHalfTiles[cfg].bn == C::BN && kHalfTiles[cfg].threads == C::THREADS;
}
static_assert(half_is<HalfBig>(0) && half_is<HalfWide>(1) && half_is<HalfMid>(2) && half_is<HalfFlat>(3));
static_assert(HalfBig::TN == 2 && HalfWide::TN == 2 && HalfMid::TN == 2 && HalfFlat::TN == 2);

// Calls f with the configuration's type.
template <class F>
int with_half_cfg(int cfg, F&& f) {
  switch (cfg) {
    case 0: return f(HalfBig{});
    case 1: return f(HalfWide{});
    case 2: return f(HalfMid{});
    default: return f(HalfFlat{});
  }
}

// The launch arguments of a product under `plan`.
inline HalfArgs half_args(const float* a, int lda, const float* b, int ldb, int m, int n, int k,
                          const uint32_t* a_top, const uint32_t* b_top, const HalfPlan& plan) {
  const HalfTile& t = kHalfTiles[plan.cfg];
  const int steps = (k + kHalfK - 1) / kHalfK, each = (steps + plan.splits - 1) / plan.splits;
  return {a, b, m, n, k, lda, ldb, a_top, b_top, (m + t.bm - 1) / t.bm, (n + t.bn - 1) / t.bn,
          (steps + each - 1) / each, each};
}
inline uint32_t half_items(const HalfArgs& g) { return uint32_t(int64_t(g.tiles_m) * g.tiles_n * g.splits); }

}  // namespace
}  // namespace lmp_hip
