// The backward of the residual norm (residual.hip has its formulas):
//
//   dH = dh + rstd_h (dy w - hn mean(dy w hn)),  hn = h rstd_h,  dweight = sum dy hn
//   dx = residual_scale dH
//   du = branch_scale drop(dH)
//   dgate = du z summed over what the gate was broadcast over,  dz = du gate
//   dpost_weight = sum dz bn,  bn = branch rstd_b
//   dbranch = rstd_b (dz post_weight - bn mean(dz post_weight bn))
//
// z and h are formed again from branch and x with the forward's statistics, the
// mask from its counter. With q the kept part of dH (times the gate where it is a
// token's or a value's) the sums over rows of post_weight and of a gate of channels
// are one: sum q bn, times branch_scale and the other parameter. Sums over rows are kept in registers by a workgroup for
// the rows that it takes, written once as its partial row, and added in a second
// launch in the order of the workgroups: the same inputs give the same bits.
#include "residual.h"

namespace ngdn {

namespace {

// Workgroups of a pass: each leaves one partial row of every sum over rows; each group
// (the rows that share a gate of a sequence; one group else) has its own.
struct Plan {
  int lanes, threads, slots, waves, V;
  long long groups, per, blocks;     // rows of a group, workgroups a group
};

// Two rows a slot at least, which halves the partial rows of a small batch.
constexpr int BWD_ROWS = 2;

Plan plan_bwd(const ResidualArgs& a) {
  Plan p;
  const int D = a.D;
  p.V = 1;
  if (D <= 256) {
    p.lanes = D <= 64 ? 8 : D <= 128 ? 16 : 32;
    p.threads = 256; p.waves = 1;
  } else {
    p.waves = (D + 511) / 512;
    if (p.waves > 16) { p.V = 2; p.waves = (p.waves + 1) / 2; }
    p.lanes = p.waves * 64;
    p.threads = p.waves == 1 ? 256 : p.lanes;
  }
  p.slots = p.threads / p.lanes;
  p.groups = a.gate_kind != GATE_SEQUENCE ? 1 : a.rows > 0 ? a.rows / a.seq : 0;
  p.per = a.gate_kind == GATE_SEQUENCE ? a.seq : a.rows;
  // a CU's share: 12 waves in small workgroups (16 are no faster and leave more partial
  // rows), else as many workgroups as 16 waves hold
  const long long want = (p.per + p.slots * BWD_ROWS - 1) / (p.slots * BWD_ROWS);
  const long long all = 256LL * (p.threads <= 256 ? 768 / p.threads : 1024 / p.threads);
  const long long most = p.groups > 0 && all / p.groups > 1 ? all / p.groups : 1;
  p.blocks = want < most ? want : most;
  return p;
}

}  // namespace

// ws: three arrays [groups x blocks][D], of dweight, dpost_weight and dgate
int64_t residual_ws(const ResidualArgs& a) {
  const Plan p = plan_bwd(a);
  return 3 * p.groups * p.blocks * a.D;
}

// A row's layout is the forward's. A workgroup stays, its parameters and its sums over
// rows in registers.
//
// HBM-bound: 4 x 8192 rows of 2048, bf16, a gate a channel and dropout move 805 MB (x
// and branch read again, dh, dy, dx, dbranch) in 167-171 us, 4.8 TB/s of the 4.9-5.2
// that a copy reaches; the sum over partial rows takes 5. Of the arithmetic, 42 full-rate
// operations a value (17 of them the generator's), one sum for post_weight and gate
// instead of two took the pass from 181 to 170 us. The next row's values in flight in a
// second set of registers, as in the forward, changed nothing (167), nor did a variant
// without a branch over any load or store.
template <typename X, typename R, typename Y, int G, int V, int TH, bool TINY>
__global__ __launch_bounds__(TH) void residual_bwd_kernel(ResidualArgs a, int waves, long long per, long long blocks) {
  extern __shared__ float s_row[];          // [slots][D]
  __shared__ float s_sum[2 * 32];
  int side = 0;
  const int lanes = G < WAVE ? G : waves * WAVE, slots = blockDim.x / lanes;
  const int slot = G < WAVE ? threadIdx.x / G : wave_id() / waves, li = threadIdx.x - slot * lanes;
  const PhiloxKey key = residual_key(a);
  const float inv = 1.f / (float)a.D;
  const bool eights = (a.D & 7) == 0;
  const bool cols = a.gate_kind == GATE_CHANNEL || a.gate_kind == GATE_SEQUENCE;
  const bool norm = a.weight && a.dy, has_dh = a.dh;
  const float scale = a.branch_scale * (a.threshold ? a.keep : 1.f);
  // the group's rows, from its block-th run of slots in steps of its workgroups
  const long long group = blockIdx.x / blocks, block = blockIdx.x - group * blocks;
  const long long g0 = group * per, last = (g0 + per < a.rows ? g0 + per : a.rows) - 1;
  const long long step = blocks * slots;
  Chunk c[V];
  float sw[V][8], sb[V][8], w[V][8], pg[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    c[v] = chunk_of<TINY>(v * lanes + li, a.D);
#pragma unroll
    for (int e = 0; e < 8; ++e) sw[v][e] = sb[v][e] = 0.f;
  }

  auto work = [&](long long row, bool live) __attribute__((always_inline)) {
    const long long at = row * a.D;
    Raw8<X> rx[V], rh[V];
    Raw8<R> rb[V];
    Raw8<Y> ry[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      rb[v] = raw8<TINY>(static_cast<const R*>(a.branch) + at, c[v]);
      if (norm) {
        rx[v] = raw8<TINY>(static_cast<const X*>(a.x) + at, c[v]);
        ry[v] = raw8<TINY>(static_cast<const Y*>(a.dy) + at, c[v]);
      }
      if (has_dh) rh[v] = raw8<TINY>(static_cast<const X*>(a.dh) + at, c[v]);
    }
    const float rstd_h = norm ? a.rstd_h[row] : 0.f, rstd_b = a.post_weight ? a.rstd_b[row] : 1.f;
    const bool full = a.gate_kind == GATE_FULL, token = a.gate_kind == GATE_TOKEN;
    const float one = token ? load_one(a.gate, a.gate_dtype, row) : 1.f;
    // bn; hn, then what dz is of the kept dH; dH, then dz post_weight
    float b[V][8], u[V][8], d[V][8], t[8];
    bool kept[V][8];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      widen(rb[v], b[v]);
#pragma unroll
      for (int e = 0; e < 8; ++e) { b[v][e] *= rstd_b; kept[v][e] = true; }
      if (a.threshold) drop8(a, key, (uint64_t)at + c[v].base, kept[v]);
    }
    if (norm) {
      float dot = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float x[8];
        if (full) {
          load_param<TINY>(a.gate, a.gate_dtype, at, c[v], t);
#pragma unroll
          for (int e = 0; e < 8; ++e) u[v][e] = b[v][e] * (pg[v][e] * t[e]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) u[v][e] = b[v][e] * (one * pg[v][e]);
        }
        widen(rx[v], x);
        widen(ry[v], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          u[v][e] = (a.residual_scale * x[e] + (kept[v][e] ? u[v][e] : 0.f)) * rstd_h;
          if (G == WAVE || live) sw[v][e] += t[e] * u[v][e];
          d[v][e] = t[e] * w[v][e];
        }
        dot += lane_sum<TINY>(c[v], eights, [&](int e) { return d[v][e] * u[v][e]; });
      }
      row_sum<G, 1>(&dot, waves, s_sum, side);
      dot *= inv;
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) d[v][e] = rstd_h * (d[v][e] - u[v][e] * dot);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) d[v][e] = 0.f;
    }
    float sums[2] = {0.f, 0.f};       // dz post_weight bn, and the token gate's
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (has_dh) {
        widen(rh[v], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[v][e] += t[e];
      }
      if (a.dx && (G == WAVE || live)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = a.residual_scale * d[v][e];
        put8<TINY>(static_cast<X*>(a.dx) + at, c[v], t);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) d[v][e] = kept[v][e] ? d[v][e] : 0.f;
      if (full) {
        float g[8];
        load_param<TINY>(a.gate, a.gate_dtype, at, c[v], g);
        if (a.dgate && (G == WAVE || live)) {
#pragma unroll
          for (int e = 0; e < 8; ++e) t[e] = d[v][e] * (b[v][e] * pg[v][e]);
          if (a.gate_dtype == NGDN_BF16) put8<TINY>(static_cast<bf16*>(a.dgate) + at, c[v], t);
          else put8<TINY>(static_cast<float*>(a.dgate) + at, c[v], t);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) d[v][e] *= g[e];
      } else if (token) {
        sums[1] += lane_sum<TINY>(c[v], eights, [&](int e) { return d[v][e] * (b[v][e] * pg[v][e]); });
#pragma unroll
        for (int e = 0; e < 8; ++e) d[v][e] *= one;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (G == WAVE || live) sb[v][e] += d[v][e] * b[v][e];
        d[v][e] *= pg[v][e];
      }
      if (a.post_weight) sums[0] += lane_sum<TINY>(c[v], eights, [&](int e) { return d[v][e] * b[v][e]; });
    }
    if (a.post_weight || (token && a.dgate)) row_sum<G, 2>(sums, waves, s_sum, side);
    if (a.dbranch) {
      const float mean = sums[0] * inv;      // 0 without a norm on the branch
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (a.post_weight) {
#pragma unroll
          for (int e = 0; e < 8; ++e) d[v][e] = rstd_b * (d[v][e] - b[v][e] * mean);
        }
        if (G == WAVE || live) put8<TINY>(static_cast<R*>(a.dbranch) + at, c[v], d[v]);
      }
    }
    if (token && a.dgate && live && li == 0) {
      if (a.gate_dtype == NGDN_BF16) static_cast<bf16*>(a.dgate)[row] = (bf16)sums[1];
      else static_cast<float*>(a.dgate)[row] = sums[1];
    }
  };

#pragma unroll
  for (int v = 0; v < V; ++v) {
    if (norm) load_param<TINY>(a.weight, a.w_dtype, 0, c[v], w[v]);
    branch_factor<TINY>(a, true, group * a.D, c[v], scale, pg[v]);
  }
  if constexpr (G < WAVE) {
    // the rows of a wave: those behind the last are the last again, and leave nothing
    for (long long first = g0 + block * slots; first <= last; first += step) {
      const bool live = first + slot <= last;
      work(live ? first + slot : last, live);
    }
  } else {
    for (long long row = g0 + block * slots + slot; row <= last; row += step) work(row, true);
  }

  // the workgroup's sums over rows: its slots in their order
  auto leave = [&](int k, float (&s)[V][8]) __attribute__((always_inline)) {
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (counts<TINY>(c[v], e)) s_row[slot * a.D + c[v].base + e] = s[v][e];
    __syncthreads();
    float* out = a.ws + ((long long)k * gridDim.x + blockIdx.x) * a.D;
    for (int j = threadIdx.x; j < a.D; j += blockDim.x) {
      float t = 0.f;
      for (int i = 0; i < slots; ++i) t += s_row[i * a.D + j];
      out[j] = t;
    }
  };
  if (a.dweight && norm) leave(0, sw);
  float t[8];
  if (a.dpost_weight) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[v][e] = sb[v][e] * scale;
      if (cols) {
        load_param<TINY>(a.gate, a.gate_dtype, group * a.D, c[v], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[v][e] *= t[e];
      }
    }
    leave(1, w);
  }
  if (cols && a.dgate) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[v][e] = sb[v][e] * scale;
      if (a.post_weight) {
        load_param<TINY>(a.post_weight, a.pw_dtype, 0, c[v], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[v][e] *= t[e];
      }
    }
    leave(2, w);
  }
}

// out[j] = sum over parts of ws[p][j], rounded to its type: a workgroup has 32
// columns, its 32 slices every 32nd part, joined in order
constexpr int SUM_COLS = 32, SUM_SLICES = 32;

struct RowSumArgs {
  const float* ws[3];
  void* out[3];
  int dtype[3];
  long long parts[3], groups[3];
  int D;
};

__global__ __launch_bounds__(1024) void residual_sum_kernel(RowSumArgs a) {
  __shared__ float s[SUM_SLICES][SUM_COLS + 1];
  const int k = blockIdx.z;
  if (!a.out[k]) return;
  const int col = threadIdx.x % SUM_COLS, slice = threadIdx.x / SUM_COLS;
  const int j = blockIdx.x * SUM_COLS + col;
  for (long long g = blockIdx.y; g < a.groups[k]; g += gridDim.y) {
    const float* ws = a.ws[k] + g * a.parts[k] * a.D;
    float v = 0.f;
    if (j < a.D)
#pragma unroll 8
      for (long long p = slice; p < a.parts[k]; p += SUM_SLICES) v += ws[p * a.D + j];
    __syncthreads();
    s[slice][col] = v;
    __syncthreads();
    if (slice == 0 && j < a.D) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < SUM_SLICES; ++i) sum += s[i][col];
      if (a.dtype[k] == NGDN_BF16) static_cast<bf16*>(a.out[k])[g * a.D + j] = (bf16)sum;
      else static_cast<float*>(a.out[k])[g * a.D + j] = sum;
    }
  }
}

namespace {

template <typename X, typename R, typename Y>
hipError_t launch_bwd(const ResidualArgs& a, const Plan& p, hipStream_t st) {
  const dim3 grid((unsigned)(p.groups * p.blocks));
  const size_t lds = (size_t)p.slots * a.D * 4;
#define NGDN_GO(G, V, TH, TINY)                                                                             \
  hipLaunchKernelGGL((residual_bwd_kernel<X, R, Y, G, V, TH, TINY>), grid, dim3(p.threads), lds, st, a, p.waves, \
                     p.per, p.blocks)
  if (a.D < 8) NGDN_GO(8, 1, 256, true);
  else if (p.lanes == 8) NGDN_GO(8, 1, 256, false);
  else if (p.lanes == 16) NGDN_GO(16, 1, 256, false);
  else if (p.lanes == 32) NGDN_GO(32, 1, 256, false);
  else if (p.V == 1) NGDN_GO(64, 1, 1024, false);
  else NGDN_GO(64, 2, 1024, false);
#undef NGDN_GO
  return hipGetLastError();
}

}  // namespace

hipError_t residual_bwd(const ResidualArgs& a, hipStream_t st) {
  if (!residual_types(a.x_dtype, a.branch_dtype, a.y_dtype) || a.D < 1 || a.D > RESIDUAL_MOST)
    return hipErrorInvalidValue;
  const Plan p = plan_bwd(a);
  hipError_t e = hipSuccess;
  if (a.rows > 0) {
    if (a.x_dtype == NGDN_BF16) e = launch_bwd<bf16, bf16, bf16>(a, p, st);
    else if (a.branch_dtype == NGDN_BF16)
      e = a.y_dtype == NGDN_BF16 ? launch_bwd<float, bf16, bf16>(a, p, st) : launch_bwd<float, bf16, float>(a, p, st);
    else
      e = a.y_dtype == NGDN_BF16 ? launch_bwd<float, float, bf16>(a, p, st) : launch_bwd<float, float, float>(a, p, st);
    if (e) return e;
  }
  // without rows the sums are over nothing: zeros
  RowSumArgs s{};
  const long long parts = a.rows > 0 ? p.groups * p.blocks : 0;
  s.D = a.D;
  s.out[0] = a.dweight; s.dtype[0] = a.w_dtype; s.parts[0] = a.dy ? parts : 0; s.groups[0] = 1;
  s.out[1] = a.dpost_weight; s.dtype[1] = a.pw_dtype; s.parts[1] = parts; s.groups[1] = 1;
  if (a.gate_kind == GATE_CHANNEL || a.gate_kind == GATE_SEQUENCE) {
    s.out[2] = a.dgate; s.dtype[2] = a.gate_dtype; s.parts[2] = a.rows > 0 ? p.blocks : 0; s.groups[2] = p.groups;
  }
  for (int k = 0; k < 3; ++k) s.ws[k] = a.ws + k * parts * a.D;
  if (!s.out[0] && !s.out[1] && !s.out[2]) return hipSuccess;
  const long long groups = s.out[2] ? (p.groups < 4096 ? p.groups : 4096) : 1;
  hipLaunchKernelGGL(residual_sum_kernel, dim3((a.D + SUM_COLS - 1) / SUM_COLS, (unsigned)(groups > 0 ? groups : 1), 3),
                     dim3(SUM_COLS * SUM_SLICES), 0, st, s);
  return hipGetLastError();
}

}  // namespace ngdn
