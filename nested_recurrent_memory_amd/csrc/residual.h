// What the residual norm's two passes (residual.hip, residual_bwd.hip) share: a
// row's layout over lanes, loads and stores of any width and alignment, and
// sums over a row.
//
// A row of D values is held by G lanes of a wave (G < 64: D <= 8 G) or by
// blockDim.x / 64 / slots whole waves, 8 V values a lane: chunk v of lane l is
// columns (v L + l) 8 ... + 7 of a row's L lanes. Where D is no multiple of
// eight the last lane's chunk starts at D - 8, and its first values, which the
// lane before has, count in no sum and are not stored; lanes behind the row
// read the same eight, with none that counts. So every load is one or two of 16
// bytes, at the alignment of a value (which the hardware takes), no load lies
// under a branch, and none leaves the row. Rows of fewer than eight values
// (TINY) are read value by value.
#pragma once

#include "ngdn_kernels.h"
#include "philox.h"

namespace ngdn {

enum GateKind { GATE_NONE, GATE_CHANNEL, GATE_SEQUENCE, GATE_TOKEN, GATE_FULL };

template <typename E> struct Raw8;
template <> struct Raw8<float> { f4 a, b; };
template <> struct Raw8<bf16> { bf16x8 a; };

struct Chunk {
  int base, first;      // its first column, and the first of its eight values that counts
  int n;                // TINY: values in the row (lane 0's), else unused
};

template <bool TINY>
__device__ __forceinline__ Chunk chunk_of(int lane, int D) {
  Chunk c;
  const int c0 = lane * 8;
  if (TINY) {
    c.base = 0; c.first = 0; c.n = lane == 0 ? D : 0;
  } else {
    c.base = c0 < D - 8 ? c0 : D - 8;
    c.first = c0 - c.base;
    c.n = 8;
  }
  return c;
}
template <bool TINY>
__device__ __forceinline__ bool counts(const Chunk& c, int e) { return TINY ? e < c.n : e >= c.first; }

template <bool TINY, typename E>
__device__ __forceinline__ Raw8<E> raw8(const E* row, const Chunk& c) {
  Raw8<E> r;
  if (TINY) {
    E t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = e < c.n ? row[e] : (E)0.f;
    __builtin_memcpy(&r, t, sizeof r);
  } else {
    __builtin_memcpy(&r, row + c.base, sizeof r);
  }
  return r;
}
__device__ __forceinline__ void widen(const Raw8<float>& r, float* o) {
#pragma unroll
  for (int e = 0; e < 4; ++e) { o[e] = r.a[e]; o[4 + e] = r.b[e]; }
}
__device__ __forceinline__ void widen(const Raw8<bf16>& r, float* o) {
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = (float)r.a[e];
}
// a parameter's or gate's eight values, in either type
template <bool TINY>
__device__ __forceinline__ void load_param(const void* p, int dtype, long long at, const Chunk& c, float* o) {
  if (dtype == NGDN_BF16) widen(raw8<TINY>(static_cast<const bf16*>(p) + at, c), o);
  else widen(raw8<TINY>(static_cast<const float*>(p) + at, c), o);
}
__device__ __forceinline__ float load_one(const void* p, int dtype, long long at) {
  return dtype == NGDN_BF16 ? (float)static_cast<const bf16*>(p)[at] : static_cast<const float*>(p)[at];
}
template <bool TINY, typename E>
__device__ __forceinline__ void put8(E* row, const Chunk& c, const float* x) {
  if (!TINY && c.first == 0) {
    Raw8<E> r;
    if constexpr (std::is_same<E, float>::value) {
#pragma unroll
      for (int e = 0; e < 4; ++e) { r.a[e] = x[e]; r.b[e] = x[4 + e]; }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) r.a[e] = (bf16)x[e];
    }
    __builtin_memcpy(row + c.base, &r, sizeof r);
  } else if (TINY || c.first < 8) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (counts<TINY>(c, e)) row[c.base + e] = (E)x[e];
  }
}

// sums over a row of N values a lane, the same in each of its lanes. A row over
// several waves goes through s [2][32], its halves in turn: a half is written again
// only behind the next sum's barrier, so one barrier a sum is enough
template <int G, int N>
__device__ __forceinline__ void row_sum(float* v, int waves, float* s, int& side) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1)
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] += __shfl_xor(v[j], o, WAVE);
  if (G == WAVE && waves > 1) {
    float* t = s + side * 32;
    side ^= 1;
    const int w = wave_id(), w0 = w - w % waves;
    if (lane_id() == 0) {
#pragma unroll
      for (int j = 0; j < N; ++j) t[w * N + j] = v[j];
    }
    lds_barrier();
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = 0.f;
    for (int i = 0; i < waves; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] += t[(w0 + i) * N + j];
  }
}

// which of the values i ... i + 7 of the stream are kept: word >= threshold (1 to 2^32)
__device__ __forceinline__ void drop8(const ResidualArgs& a, const PhiloxKey& key, uint64_t i, bool* kept) {
  uint32_t w[8];
  philox8(key, i, (a.D & 3) == 0, w);
#pragma unroll
  for (int e = 0; e < 8; ++e) kept[e] = w[e] > (uint32_t)(a.threshold - 1);
}

__device__ __forceinline__ PhiloxKey residual_key(const ResidualArgs& a) {
  return PhiloxKey((uint64_t)(a.seed_ptr ? *a.seed_ptr : a.seed), (uint64_t)a.offset);
}

}  // namespace ngdn
