// Dropout, and the forward of the residual norm: a block's output added to its
// residual stream, with the norms on both sides of the sum.
//
//   z = branch rstd(branch) post_weight          (post_weight NULL: z = branch)
//   h = residual_scale x + branch_scale drop(gate z)
//   y = h rstd(h) weight                         (weight NULL: no y)
//   rstd(v) = 1 / sqrt(mean(v^2) + eps) over a row
//
// One pass: a row is read once into registers, both statistics are sums over
// its lanes, and h and y are written from there. y is formed from h before h is
// rounded to its type, so it carries one rounding; the backward forms h again from
// x and branch (the same up to fp32 roundings: its factors come in another order), which
// costs no more bytes than reading h would where a norm or a gate on the branch needs
// the branch anyway.
// All arithmetic is in fp32.
#include "residual.h"

namespace ngdn {

// ---------------------------------------------------------------- dropout

// y[i] = kept(i) ? x[i] keep : 0, kept(i): word i of the generator >= threshold.
// Eight values a lane and step. The mask is formed again in the backward, which
// is the same kernel on the gradient. HBM-bound at 5.6 to 6.6 TB/s (46 M bf16 values,
// 184 MB, in 33 us), with the generator just behind: the vector units are busy 64% of the
// cycles, counting its products (14 for four values, at a quarter of the rate) as one each.
template <typename E>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs a) {
  const PhiloxKey key((uint64_t)(a.seed_ptr ? *a.seed_ptr : a.seed), (uint64_t)a.offset);
  const uint32_t last = (uint32_t)(a.threshold - 1);      // the largest word that is dropped
  const E* x = static_cast<const E*>(a.x);
  E* y = static_cast<E*>(a.y);
  const long long step = (long long)gridDim.x * 256 * 8;
  for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 8; i < a.n; i += step) {
    uint32_t w[8];
    float v[8];
    if (i + 8 <= a.n) {
      Raw8<E> r;
      __builtin_memcpy(&r, x + i, sizeof r);
      philox8(key, (uint64_t)i, true, w);
      widen(r, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = w[e] > last ? v[e] * a.keep : 0.f;
      put8<false>(y + i, Chunk{0, 0, 8}, v);
    } else {
      philox8(key, (uint64_t)i, true, w);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (i + e < a.n) y[i + e] = (E)(w[e] > last ? (float)x[i + e] * a.keep : 0.f);
    }
  }
}

hipError_t dropout(const DropoutArgs& a, int dtype, hipStream_t st) {
  if (a.n == 0) return hipSuccess;
  const long long blocks = (a.n + 2047) / 2048, most = 1 << 20;     // work-items below 2^32
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
  if (dtype == NGDN_BF16) hipLaunchKernelGGL(dropout_kernel<bf16>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(dropout_kernel<float>, grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------- the residual norm

// A row of G < 64 lanes, of one wave (four rows a workgroup, each wave on its own)
// or of a workgroup. A workgroup stays and takes rows in steps of the grid, its
// parameters in registers; the next row's values are in flight while a row is worked
// on, in two sets of registers in turn (a copy from one into the other would wait
// for them).
//
// HBM-bound: 4 x 4096 rows of 2048, fp32 stream and bf16 branch, 403 MB in 77-78 us
// (5.2 TB/s, a copy's rate); 4 x 8192 rows of 2048, bf16, with dropout, 537 MB in 109
// to 113 us (4.75 to 4.9 TB/s). A workgroup a row with its parameters loaded each time took 111 and
// 226 us, and 12 us for 128 rows, the latencies of four loads in a row, where this takes
// 4.5. Of the second case's 226 us the generator and the sums' arithmetic were as much as
// the loads: xor of three in one instruction, wave sums by lane moves instead of through
// LDS and one factor for post_weight, gate and scales took it from 157 to 113.
template <typename X, typename R, typename Y, int G, int V, bool PRE, bool TINY>
__global__ __launch_bounds__(1024) void residual_fwd_kernel(ResidualArgs a, int waves) {
  __shared__ float s_sum[2 * 32];
  int side = 0;
  const int lanes = G < WAVE ? G : waves * WAVE, slots = blockDim.x / lanes;
  const int slot = G < WAVE ? threadIdx.x / G : wave_id() / waves, li = threadIdx.x - slot * lanes;
  const PhiloxKey key = residual_key(a);
  const float inv = 1.f / (float)a.D;
  const bool eights = (a.D & 7) == 0;
  const bool rows_gate = a.gate_kind == GATE_SEQUENCE || a.gate_kind == GATE_FULL;
  Chunk c[V];
#pragma unroll
  for (int v = 0; v < V; ++v) c[v] = chunk_of<TINY>(v * lanes + li, a.D);

  struct Row {
    Raw8<X> x[V];
    Raw8<R> b[V];
  };
  auto fetch = [&](long long row, Row& r) __attribute__((always_inline)) {
    const long long at = row * a.D;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      r.b[v] = raw8<TINY>(static_cast<const R*>(a.branch) + at, c[v]);
      r.x[v] = raw8<TINY>(static_cast<const X*>(a.x) + at, c[v]);
    }
  };
  const long long step = (long long)gridDim.x * slots;
  long long row = (long long)blockIdx.x * slots + slot;
  // the rows of a wave under 64 lanes end together
  const long long last = a.rows - 1;
  Row r0, r1;
  if (G < WAVE || row <= last) fetch(row < last ? row : last, r0);
  // pg: what a normalised value of the branch is multiplied by
  float w[V][8], pg[V][8];
  const float scale = a.branch_scale * (a.threshold ? a.keep : 1.f);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (PRE) load_param<TINY>(a.weight, a.w_dtype, 0, c[v], w[v]);
    branch_factor<TINY>(a, false, 0, c[v], scale, pg[v]);
  }

  auto work = [&](Row& r, Row& next) __attribute__((always_inline)) {
    const bool live = row <= last;
    const long long at = (live ? row : last) * a.D;
    if (G < WAVE || row + step <= last) fetch(row + step < last ? row + step : last, next);
    float z[V][8], t[8], rstd_b = 1.f;
#pragma unroll
    for (int v = 0; v < V; ++v) widen(r.b[v], z[v]);
    if (a.post_weight) {
      float ss = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) ss += lane_sum<TINY>(c[v], eights, [&](int e) { return z[v][e] * z[v][e]; });
      row_sum<G, 1>(&ss, waves, s_sum, side);
      rstd_b = inverse_root(ss, inv, a.eps);
    }
    if (rows_gate) {
      const long long ga = a.gate_kind == GATE_FULL ? at : (long long)((uint32_t)(live ? row : last) / (uint32_t)a.seq) * a.D;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        load_param<TINY>(a.gate, a.gate_dtype, ga, c[v], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[v][e] *= rstd_b * (pg[v][e] * t[e]);
      }
    } else {
      const float one = a.gate_kind == GATE_TOKEN ? rstd_b * load_one(a.gate, a.gate_dtype, live ? row : last) : rstd_b;
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) z[v][e] *= one * pg[v][e];
    }
    if (a.threshold) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        bool kept[8];
        drop8(a, key, (uint64_t)at + c[v].base, kept);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[v][e] = kept[e] ? z[v][e] : 0.f;
      }
    }
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      widen(r.x[v], t);
#pragma unroll
      for (int e = 0; e < 8; ++e) z[v][e] += a.residual_scale * t[e];      // h
      if (PRE) ss += lane_sum<TINY>(c[v], eights, [&](int e) { return z[v][e] * z[v][e]; });
      if (G == WAVE || live) put8<TINY>(static_cast<X*>(a.h) + at, c[v], z[v]);
    }
    if (PRE) {
      row_sum<G, 1>(&ss, waves, s_sum, side);
      const float rstd = inverse_root(ss, inv, a.eps);
#pragma unroll
      for (int v = 0; v < V; ++v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) z[v][e] *= rstd * w[v][e];
        if (G == WAVE || live) put8<TINY>(static_cast<Y*>(a.y) + at, c[v], z[v]);
      }
      if (a.rstd_h && live && li == 0) a.rstd_h[row] = rstd;
    }
    if (a.rstd_b && a.post_weight && live && li == 0) a.rstd_b[row] = rstd_b;
    row += step;
  };
  // lanes of a wave and waves of a row end together: rows in one step differ by less than slots
  if constexpr (G < WAVE) {
    for (long long first = (long long)blockIdx.x * slots; first <= last; first += 2 * step) {
      work(r0, r1);
      work(r1, r0);
    }
  } else {
    while (row <= last) {
      work(r0, r1);
      if (row > last) break;
      work(r1, r0);
    }
  }
}

// types of (x and h, branch, y)
bool residual_types(int xd, int rd, int yd) {
  return xd == NGDN_F32 ? (rd == NGDN_F32 || rd == NGDN_BF16) && (yd == NGDN_F32 || yd == NGDN_BF16)
                        : xd == NGDN_BF16 && rd == NGDN_BF16 && yd == NGDN_BF16;
}

namespace {

template <typename X, typename R, typename Y, bool PRE>
hipError_t launch_fwd(const ResidualArgs& a, hipStream_t st) {
  const int D = a.D;
  // As many whole workgroups as 16 waves a CU hold (four a SIMD, at the registers that a
  // row takes): 12 and 20 waves take 77 and 86 us where 16 take 77 (fp32 stream), 139 and
  // 143 where 16 take 126 (dropout); part of a round more, 47 where 37 (2816 columns).
  // Rows of up to 8192 by eight values a lane: sixteen take 62 us where eight take 47 (8192
  // columns), and 24.5 where 20 (768 columns, one wave where two). Rows of up to 256 share
  // a wave: one a wave takes 22.8 us where eight take 8.3 (65536 rows of 64), 25.9 where 22.5
  // (of 256)
  auto go = [&](auto kernel, int threads, int slots, int waves) {
    const long long want = (a.rows + slots - 1) / slots, most = 256LL * (threads < 1024 ? 1024 / threads : 1);
    hipLaunchKernelGGL(kernel, dim3((unsigned)(want < most ? want : most)), dim3(threads), 0, st, a, waves);
    return hipGetLastError();
  };
  if (D < 8) return go(residual_fwd_kernel<X, R, Y, 8, 1, PRE, true>, 256, 32, 1);
  if (D <= 64) return go(residual_fwd_kernel<X, R, Y, 8, 1, PRE, false>, 256, 32, 1);
  if (D <= 128) return go(residual_fwd_kernel<X, R, Y, 16, 1, PRE, false>, 256, 16, 1);
  if (D <= 256) return go(residual_fwd_kernel<X, R, Y, 32, 1, PRE, false>, 256, 8, 1);
  const int waves = (D + 511) / 512;
  if (waves == 1) return go(residual_fwd_kernel<X, R, Y, 64, 1, PRE, false>, 256, 4, 1);
  if (waves <= 16) return go(residual_fwd_kernel<X, R, Y, 64, 1, PRE, false>, waves * 64, 1, waves);
  return go(residual_fwd_kernel<X, R, Y, 64, 2, PRE, false>, (waves + 1) / 2 * 64, 1, (waves + 1) / 2);
}

template <typename X, typename R, typename Y>
hipError_t launch_fwd(const ResidualArgs& a, hipStream_t st) {
  return a.weight ? launch_fwd<X, R, Y, true>(a, st) : launch_fwd<X, R, X, false>(a, st);
}

}  // namespace

hipError_t residual_fwd(const ResidualArgs& a, hipStream_t st) {
  if (!residual_types(a.x_dtype, a.branch_dtype, a.y_dtype) || a.D < 1 || a.D > RESIDUAL_MOST)
    return hipErrorInvalidValue;
  if (a.rows == 0) return hipSuccess;
  if (a.x_dtype == NGDN_BF16) return launch_fwd<bf16, bf16, bf16>(a, st);
  if (a.branch_dtype == NGDN_BF16)
    return a.y_dtype == NGDN_BF16 ? launch_fwd<float, bf16, bf16>(a, st) : launch_fwd<float, bf16, float>(a, st);
  return a.y_dtype == NGDN_BF16 ? launch_fwd<float, float, bf16>(a, st) : launch_fwd<float, float, float>(a, st);
}

}  // namespace ngdn
