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
// mask from its counter. Sums over rows are kept in registers by a workgroup for
// the rows that it takes, written once as its partial row, and added in a second
// launch in the order of the workgroups: the same inputs give the same bits.
#include "residual.h"

namespace ngdn {

namespace {

// Workgroups of a pass: for sums over rows, few partial rows; each group (the
// rows that share a gate of a sequence; one group else) has its own.
struct Plan {
  int lanes, threads, slots, waves, V;
  long long groups, per, blocks;     // rows of a group, workgroups a group
};

constexpr long long BWD_BLOCKS = 1024;

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
    p.threads = p.waves <= 2 ? 256 : p.lanes;
  }
  p.slots = p.threads / p.lanes;
  p.groups = a.gate_kind != GATE_SEQUENCE ? 1 : a.rows > 0 ? a.rows / a.seq : 0;
  p.per = a.gate_kind == GATE_SEQUENCE ? a.seq : a.rows;
  const long long want = (p.per + p.slots - 1) / p.slots;
  const long long most = p.groups > 0 && BWD_BLOCKS / p.groups > 1 ? BWD_BLOCKS / p.groups : 1;
  p.blocks = want < most ? want : most;
  return p;
}

}  // namespace

// ws: three arrays [groups x blocks][D], of dweight, dpost_weight and dgate
int64_t residual_ws(const ResidualArgs& a) {
  const Plan p = plan_bwd(a);
  return 3 * p.groups * p.blocks * a.D;
}

template <typename X, typename R, typename Y, int G, int V, bool TINY>
__global__ __launch_bounds__(1024) void residual_bwd_kernel(ResidualArgs a, int waves, long long per,
                                                            long long blocks) {
  extern __shared__ float s_row[];          // [slots][D]
  __shared__ float s_sum[2 * 32];
  int side = 0;
  const int lanes = G < WAVE ? G : waves * WAVE, slots = blockDim.x / lanes;
  const int slot = G < WAVE ? threadIdx.x / G : wave_id() / waves, li = threadIdx.x - slot * lanes;
  const PhiloxKey key = residual_key(a);
  const float inv = 1.f / (float)a.D;
  const bool cols = a.gate_kind == GATE_CHANNEL || a.gate_kind == GATE_SEQUENCE;
  // the group's rows, from its block-th run of slots in steps of its workgroups
  const long long group = blockIdx.x / blocks, block = blockIdx.x - group * blocks;
  const long long g0 = group * per, g1 = g0 + per < a.rows ? g0 + per : a.rows;
  Chunk c[V];
  float sw[V][8], sp[V][8], sg[V][8];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    c[v] = chunk_of<TINY>(v * lanes + li, a.D);
#pragma unroll
    for (int e = 0; e < 8; ++e) sw[v][e] = sp[v][e] = sg[v][e] = 0.f;
  }
  for (long long r0 = g0 + block * slots; r0 < g1; r0 += blocks * slots) {
    const bool live = r0 + slot < g1;
    const long long row = live ? r0 + slot : g1 - 1, at = row * a.D;
    Raw8<X> rx[V], rh[V];
    Raw8<R> rb[V];
    Raw8<Y> ry[V];
    float z[V][8], u[V][8], d[V][8], t[8];
    const bool norm = a.weight != nullptr && a.dy != nullptr;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      rb[v] = raw8<TINY>(static_cast<const R*>(a.branch) + at, c[v]);
      if (norm) {
        rx[v] = raw8<TINY>(static_cast<const X*>(a.x) + at, c[v]);
        ry[v] = raw8<TINY>(static_cast<const Y*>(a.dy) + at, c[v]);
      }
      if (a.dh) rh[v] = raw8<TINY>(static_cast<const X*>(a.dh) + at, c[v]);
    }
    const float rstd_b = a.post_weight ? a.rstd_b[row] : 1.f;
    const float one = a.gate_kind == GATE_TOKEN ? load_one(a.gate, a.gate_dtype, row) : 1.f;
    const long long ga = a.gate_kind == GATE_FULL ? at : a.gate_kind == GATE_SEQUENCE ? group * a.D : 0;
    const bool wide = a.gate_kind != GATE_NONE && a.gate_kind != GATE_TOKEN;
    unsigned kept[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      kept[v] = 0xff;
      if (a.threshold) {
        bool k[8];
        drop8(a, key, (uint64_t)at + c[v].base, k);
        kept[v] = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) kept[v] |= (unsigned)k[e] << e;
      }
    }
    const float scale = a.branch_scale * (a.threshold ? a.keep : 1.f);
    // z, and the sum over the row for the norm of h
#pragma unroll
    for (int v = 0; v < V; ++v) {
      widen(rb[v], z[v]);
      if (a.post_weight) {
        load_param<TINY>(a.post_weight, a.pw_dtype, 0, c[v], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) z[v][e] *= rstd_b * t[e];
      }
    }
    if (norm) {
      const float rstd = a.rstd_h[row];
      float dot = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float g[8], x[8], dy[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) g[e] = one;
        if (wide) load_param<TINY>(a.gate, a.gate_dtype, ga, c[v], g);
        widen(rx[v], x);
        widen(ry[v], dy);
        load_param<TINY>(a.weight, a.w_dtype, 0, c[v], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float b = kept[v] >> e & 1 ? z[v][e] * g[e] * scale : 0.f;
          u[v][e] = (a.residual_scale * x[e] + b) * rstd;          // hn
          if (live) sw[v][e] += dy[e] * u[v][e];
          d[v][e] = dy[e] * t[e];
          dot += counts<TINY>(c[v], e) ? d[v][e] * u[v][e] : 0.f;
        }
      }
      row_sum<G, 1>(&dot, waves, s_sum, side);
      dot *= inv;
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) d[v][e] = rstd * (d[v][e] - u[v][e] * dot);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int e = 0; e < 8; ++e) d[v][e] = 0.f;
    }
    float sums[2] = {0.f, 0.f};       // dz post_weight bn, and the token gate's
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float g[8];
      if (a.dh) {
        widen(rh[v], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[v][e] += t[e];               // dH
      }
      if (a.dx && live) {
#pragma unroll
        for (int e = 0; e < 8; ++e) t[e] = a.residual_scale * d[v][e];
        put8<TINY>(static_cast<X*>(a.dx) + at, c[v], t);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = one;
      if (wide) load_param<TINY>(a.gate, a.gate_dtype, ga, c[v], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        d[v][e] = kept[v] >> e & 1 ? d[v][e] * scale : 0.f;        // du
        z[v][e] *= d[v][e];                                        // du z
        d[v][e] *= g[e];                                           // dz
        if (counts<TINY>(c[v], e)) sums[1] += z[v][e];
      }
      if (a.gate_kind == GATE_FULL && a.dgate && live) {
        if (a.gate_dtype == NGDN_BF16) put8<TINY>(static_cast<bf16*>(a.dgate) + at, c[v], z[v]);
        else put8<TINY>(static_cast<float*>(a.dgate) + at, c[v], z[v]);
      }
      if (cols && live) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sg[v][e] += z[v][e];
      }
      if (a.post_weight) {
        widen(rb[v], u[v]);
        load_param<TINY>(a.post_weight, a.pw_dtype, 0, c[v], t);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          u[v][e] *= rstd_b;                                       // bn
          if (live) sp[v][e] += d[v][e] * u[v][e];
          d[v][e] *= t[e];
          if (counts<TINY>(c[v], e)) sums[0] += d[v][e] * u[v][e];
        }
      }
    }
    const bool token = a.gate_kind == GATE_TOKEN && a.dgate;
    if (a.post_weight || token) {
      row_sum<G, 2>(sums, waves, s_sum, side);
      if (token && live && li == 0) {
        if (a.gate_dtype == NGDN_BF16) static_cast<bf16*>(a.dgate)[row] = (bf16)sums[1];
        else static_cast<float*>(a.dgate)[row] = sums[1];
      }
    }
    if (a.dbranch && live) {
      const float mean = sums[0] * inv;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (a.post_weight) {
#pragma unroll
          for (int e = 0; e < 8; ++e) d[v][e] = rstd_b * (d[v][e] - u[v][e] * mean);
        }
        put8<TINY>(static_cast<R*>(a.dbranch) + at, c[v], d[v]);
      }
    }
  }
  // the workgroup's sums over rows: its slots in their order
  for (int k = 0; k < 3; ++k) {
    const bool wanted = k == 0 ? a.dweight && a.dy : k == 1 ? a.dpost_weight != nullptr : cols && a.dgate;
    if (!wanted) continue;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (counts<TINY>(c[v], e)) s_row[slot * a.D + c[v].base + e] = k == 0 ? sw[v][e] : k == 1 ? sp[v][e] : sg[v][e];
    __syncthreads();
    for (int j = threadIdx.x; j < a.D; j += blockDim.x) {
      float s = 0.f;
      for (int i = 0; i < slots; ++i) s += s_row[i * a.D + j];
      a.ws[((long long)k * gridDim.x + blockIdx.x) * a.D + j] = s;
    }
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
#define NGDN_GO(G, V, TINY)                                                                              \
  hipLaunchKernelGGL((residual_bwd_kernel<X, R, Y, G, V, TINY>), grid, dim3(p.threads), lds, st, a, p.waves, \
                     p.per, p.blocks)
  if (a.D < 8) NGDN_GO(8, 1, true);
  else if (p.lanes == 8) NGDN_GO(8, 1, false);
  else if (p.lanes == 16) NGDN_GO(16, 1, false);
  else if (p.lanes == 32) NGDN_GO(32, 1, false);
  else if (p.V == 1) NGDN_GO(64, 1, false);
  else NGDN_GO(64, 2, false);
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
