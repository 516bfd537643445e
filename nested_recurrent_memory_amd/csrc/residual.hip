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
// rounded to its type, so it carries one rounding; the backward forms the same h
// from x and branch again, which costs no more bytes than reading h would.
// All arithmetic is in fp32.
#include "residual.h"

namespace ngdn {

// ---------------------------------------------------------------- dropout

// y[i] = kept(i) ? x[i] keep : 0, kept(i): word i of the generator >= threshold.
// Eight values a lane and step. The mask is formed again in the backward, which
// is the same kernel on the gradient.
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

template <typename X, typename R, typename Y, int G, int V, bool TINY>
__global__ __launch_bounds__(1024) void residual_fwd_kernel(ResidualArgs a, int waves) {
  __shared__ float s_sum[2 * 32];
  int side = 0;
  const int lanes = G < WAVE ? G : waves * WAVE, slots = blockDim.x / lanes;
  const int slot = G < WAVE ? threadIdx.x / G : wave_id() / waves, li = threadIdx.x - slot * lanes;
  const PhiloxKey key = residual_key(a);
  Chunk c[V];
#pragma unroll
  for (int v = 0; v < V; ++v) c[v] = chunk_of<TINY>(v * lanes + li, a.D);
  const float inv = 1.f / (float)a.D;
  for (long long r0 = (long long)blockIdx.x * slots; r0 < a.rows; r0 += (long long)gridDim.x * slots) {
    const bool live = r0 + slot < a.rows;
    const long long row = live ? r0 + slot : a.rows - 1, at = row * a.D;
    Raw8<X> rx[V];
    Raw8<R> rb[V];
    float z[V][8], t[8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      rx[v] = raw8<TINY>(static_cast<const X*>(a.x) + at, c[v]);
      rb[v] = raw8<TINY>(static_cast<const R*>(a.branch) + at, c[v]);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) widen(rb[v], z[v]);
    if (a.post_weight) {
      float ss = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += counts<TINY>(c[v], e) ? z[v][e] * z[v][e] : 0.f;
      row_sum<G, 1>(&ss, waves, s_sum, side);
      const float rstd = 1.f / sqrtf(ss * inv + a.eps);
      if (a.rstd_b && live && li == 0) a.rstd_b[row] = rstd;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        load_param<TINY>(a.post_weight, a.pw_dtype, 0, c[v], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[v][e] *= rstd * t[e];
      }
    }
    if (a.gate_kind == GATE_TOKEN) {
      const float g = load_one(a.gate, a.gate_dtype, row);
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) z[v][e] *= g;
    } else if (a.gate_kind != GATE_NONE) {
      const long long ga = a.gate_kind == GATE_FULL ? at : a.gate_kind == GATE_SEQUENCE ? row / a.seq * a.D : 0;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        load_param<TINY>(a.gate, a.gate_dtype, ga, c[v], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[v][e] *= t[e];
      }
    }
    float scale = a.branch_scale;
    if (a.threshold) {
      scale *= a.keep;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        bool kept[8];
        drop8(a, key, (uint64_t)at + c[v].base, kept);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[v][e] = kept[e] ? z[v][e] * scale : 0.f;
      }
      scale = 1.f;
    }
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      widen(rx[v], t);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        z[v][e] = a.residual_scale * t[e] + scale * z[v][e];      // h
        ss += counts<TINY>(c[v], e) ? z[v][e] * z[v][e] : 0.f;
      }
      if (live) put8<TINY>(static_cast<X*>(a.h) + at, c[v], z[v]);
    }
    if (a.weight) {
      row_sum<G, 1>(&ss, waves, s_sum, side);
      const float rstd = 1.f / sqrtf(ss * inv + a.eps);
      if (a.rstd_h && live && li == 0) a.rstd_h[row] = rstd;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        load_param<TINY>(a.weight, a.w_dtype, 0, c[v], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[v][e] *= rstd * t[e];
        if (live) put8<TINY>(static_cast<Y*>(a.y) + at, c[v], z[v]);
      }
    }
  }
}

// types of (x and h, branch, y)
bool residual_types(int xd, int rd, int yd) {
  return xd == NGDN_F32 ? (rd == NGDN_F32 || rd == NGDN_BF16) && (yd == NGDN_F32 || yd == NGDN_BF16)
                        : xd == NGDN_BF16 && rd == NGDN_BF16 && yd == NGDN_BF16;
}

namespace {

template <typename X, typename R, typename Y>
hipError_t launch_fwd(const ResidualArgs& a, hipStream_t st) {
  const int D = a.D;
  // work-items below 2^32; a workgroup takes further rows in steps of the grid
  auto go = [&](auto kernel, int threads, int slots, int waves) {
    const long long want = (a.rows + slots - 1) / slots, most = 1 << 21;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(want < most ? want : most)), dim3(threads), 0, st, a, waves);
    return hipGetLastError();
  };
  if (D < 8) return go(residual_fwd_kernel<X, R, Y, 8, 1, true>, 256, 32, 1);
  if (D <= 64) return go(residual_fwd_kernel<X, R, Y, 8, 1, false>, 256, 32, 1);
  if (D <= 128) return go(residual_fwd_kernel<X, R, Y, 16, 1, false>, 256, 16, 1);
  if (D <= 256) return go(residual_fwd_kernel<X, R, Y, 32, 1, false>, 256, 8, 1);
  const int waves = (D + 511) / 512;
  if (waves <= 2) return go(residual_fwd_kernel<X, R, Y, 64, 1, false>, 256, 4 / waves, waves);
  if (waves <= 16) return go(residual_fwd_kernel<X, R, Y, 64, 1, false>, waves * 64, 1, waves);
  return go(residual_fwd_kernel<X, R, Y, 64, 2, false>, (waves + 1) / 2 * 64, 1, (waves + 1) / 2);
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
