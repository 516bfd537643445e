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
// scale times post_weight and times a gate of channels (with sequence, one of a sequence too,
// whose row begins at gate_at), where there are such
template <bool TINY>
__device__ __forceinline__ void branch_factor(const ResidualArgs& a, bool sequence, long long gate_at, const Chunk& c,
                                              float scale, float* o) {
  float t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = scale;
  if (a.post_weight) {
    load_param<TINY>(a.post_weight, a.pw_dtype, 0, c, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= t[e];
  }
  if (a.gate_kind == GATE_CHANNEL || (sequence && a.gate_kind == GATE_SEQUENCE)) {
    load_param<TINY>(a.gate, a.gate_dtype, gate_at, c, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= t[e];
  }
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

// v of another lane of the row, by the vector unit's own lane moves (no trip through LDS)
template <int CTRL, int ROWS>
__device__ __forceinline__ float moved(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, false));
}
// the sum over a wave, in a scalar register
__device__ __forceinline__ float wave_sum_uniform(float v) {
  v += moved<0x111, 0xf>(v);      // row_shr 1, 2, 4, 8: the sum of 16 lanes in their last
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);      // row_bcast 15 into rows 1 and 3, row_bcast 31 into 2 and 3
  v += moved<0x143, 0xc>(v);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), WAVE - 1));
}

// sums over a row of N values a lane, the same in each of its lanes. A row over
// several waves goes through s [2][32], its halves in turn: a half is written again
// only behind the next sum's barrier, so one barrier a sum is enough
template <int G, int N>
__device__ __forceinline__ void row_sum(float* v, int waves, float* s, int& side) {
  if constexpr (G < WAVE) {
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1)
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] += __shfl_xor(v[j], o, WAVE);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = wave_sum_uniform(v[j]);
    if (waves > 1) {
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
}

// a sum over a lane's values p(e) that count. Where D is a multiple of eight (uniform)
// a lane's count all or none
template <bool TINY, typename F>
__device__ __forceinline__ float lane_sum(const Chunk& c, bool eights, F p) {
  float s = 0.f;
  if (!TINY && eights) {
#pragma unroll
    for (int e = 0; e < 8; ++e) s += p(e);
    return c.first == 0 ? s : 0.f;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) s += counts<TINY>(c, e) ? p(e) : 0.f;
  return s;
}
// 1 / sqrt(mean + eps): the hardware's, which is up to a unit off, and a Newton step on it, with
// what the product loses, after which only the rounding is left (4 x 8192 rows of 2048, bf16, with
// dropout, both passes: 271 us, as without; 275 by a root and a quotient). Zeros and infinities
// as they are
__device__ __forceinline__ float inverse_root(float sum, float inv, float eps) {
  const float v = sum * inv + eps, r = rsqrtf(v), t = v * r;
  const float e = fmaf(-t, r, 1.f) - fmaf(v, r, -t) * r;       // 1 - v r^2
  return v > 0.f && v < INFINITY ? fmaf(0.5f * r, e, r) : r;
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
