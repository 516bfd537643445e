// A gated linear recurrence with one state value a channel, forward, backward
// and as a decoding step. Per channel d of head h(d):
//   z = f + dt_bias,  g = -exp(A_log[h]) softplus(z),  a = e^g,
//   h_t = a_t h_(t-1) + beta_t s_t x_t,  beta = sqrt(1 - a^2), s = sigmoid(wz), y_t = h_t
// so h keeps the variance of the gated inputs at any decay. Backward, with
// lam_t = dy_t + a_(t+1) lam_(t+1) (the last token of a sequence: dy_t + dfinal):
//   dx = lam beta s, dwz = lam beta s (1 - s) x, dh0 = a_0 lam_0,
//   dg = lam (a h_(t-1) - (a^2 / beta) s x), df = -exp(A_log) sigmoid(z) dg,
//   d dt_bias = sum df, d A_log = sum dg g.
// Everything between loads and stores is fp32. The recurrence is linear, so a
// run of tokens acts on the state before it as h -> A h + H with A = prod a;
// runs of SEG tokens are reduced to (A, H), joined in order, and then formed
// from the state that enters them.
#include <initializer_list>

#include "ngdn_kernels.h"

namespace ngdn {

namespace {

constexpr int SEG = REC_SEG;

constexpr float LOG2E = 1.44269504088896340736f;

// e^(ln2 p) - 1 = ln2 p (1 + ...): the coefficients of -(2^p - 1) / p
constexpr float EM1 = 0.69314718055994531f, EM2 = 0.24022650695910071f, EM3 = 0.05550410866482158f,
                EM4 = 0.00961812910762848f;

// What a token's decay needs: a = e^g, q = 1 - a^2, g2 = g log2(e), and the
// sigmoid's parts (e = e^-|z|, up = z >= 0).
struct Decay {
  float a, q, g2, e;
  bool up;
};

// z2 = z log2(e) = f log2(e) + bias2, nrate = -exp(A_log).
// softplus(z) log2(e) = max(z2, 0) + log2(1 + e): the logarithm as e P(e), P
// the degree-7 polynomial of least relative error on [0, 1] (3e-7 in fp32),
// which keeps its relative precision for the small e where decays usually sit;
// log2(1 + e) itself loses e's low bits there.
// 1 - a from the series of e^g - 1 for -g < 1/16 (relative error 1e-7), where
// the subtraction would cancel, and q = (1 - a)(1 + a).
__device__ __forceinline__ Decay decay(float f, float bias2, float nrate) {
  Decay d;
  const float z2 = fmaf(f, LOG2E, bias2);
  d.up = z2 >= 0.f;
  d.e = __builtin_amdgcn_exp2f(-fabsf(z2));
  const float e = d.e;
  float p = -0.012319466099143028f;
  p = fmaf(p, e, 0.06360787153244019f);
  p = fmaf(p, e, -0.15535186231136322f);
  p = fmaf(p, e, 0.2560097277164459f);
  p = fmaf(p, e, -0.35339483618736267f);
  p = fmaf(p, e, 0.48006370663642883f);
  p = fmaf(p, e, -0.7213100790977478f);
  p = fmaf(p, e, 1.4426947832107544f);
  d.g2 = nrate * fmaf(p, e, fmaxf(z2, 0.f));
  d.a = __builtin_amdgcn_exp2f(d.g2);
  const float g2 = d.g2;
  const float s = -g2 * fmaf(g2, fmaf(g2, fmaf(g2, EM4, EM3), EM2), EM1);
  const float t = g2 > -LOG2E / 16.f ? s : 1.f - d.a;
  d.q = t * (2.f - t);
  return d;
}

__device__ __forceinline__ float sigmoid2(float w) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-LOG2E * w));
}

// beta and 1 / beta. A q of 0 (a decay that rounds to 1) is lifted so that
// 1 / beta stays finite: it is multiplied by e, which is 0 there.
__device__ __forceinline__ void root(float q, float& beta, float& inv) {
  inv = __builtin_amdgcn_rsqf(fmaxf(q, 1e-37f));
  beta = q * inv;
}

template <typename E, int VEC>
__device__ __forceinline__ void loadv(const E* p, float* o) {
  if constexpr (VEC == 1) {
    o[0] = to_f(*p);
  } else {
    struct alignas(VEC * sizeof(E)) Pack { E v[VEC]; };
    const Pack k = *reinterpret_cast<const Pack*>(p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) o[i] = to_f(k.v[i]);
  }
}
template <typename E, int VEC>
__device__ __forceinline__ void storev(E* p, const float* x) {
  if constexpr (VEC == 1) {
    *p = from_f<E>(x[0]);
  } else {
    struct alignas(VEC * sizeof(E)) Pack { E v[VEC]; };
    Pack k;
#pragma unroll
    for (int i = 0; i < VEC; ++i) k.v[i] = from_f<E>(x[i]);
    *reinterpret_cast<Pack*>(p) = k;
  }
}

// Where the tokens [t0, t0 + n) of a packed row stand: bit j of start / end /
// used says whether token t0 + j is the first / the last of its sequence / in
// one at all; cur is the sequence of token t0 (or the one before it), last that
// of the run's last token. Nothing is read or assumed of cu beyond its S + 1
// values, so a cu that is not sorted gives wrong rows but no access outside.
struct Run {
  unsigned start, end, used;
  int cur, last;
};
__device__ __forceinline__ Run run_of(const int* cu, int S, int t0, int n, int T) {
  Run r{0u, 0u, 0u, 0, 0};
  int lo = 0, hi = S + 1;                  // first boundary at or behind t0
  while (lo < hi) {
    const int m = (lo + hi) / 2;
    if (cu[m] < t0) lo = m + 1; else hi = m;
  }
  int s = lo;
  r.cur = s - 1;
  for (int j = 0; j < n; ++j) {
    while (s <= S && cu[s] <= t0 + j) {
      if (cu[s] == t0 + j) r.start |= 1u << j;
      ++s;
    }
    if (s >= 1 && s <= S) {
      r.used |= 1u << j;
      if (cu[s] == t0 + j + 1 || t0 + j + 1 == T) r.end |= 1u << j;
    }
  }
  r.last = s - 1;
  return r;
}
// the sequence that token t starts: the last one with that boundary, from
// sequence cur on
__device__ __forceinline__ int seq_from(const int* cu, int S, int cur, int t) {
  if (cur < 0) cur = 0;
  while (cur + 1 <= S && cu[cur + 1] <= t) ++cur;
  return cur < S ? cur : S - 1;
}
// the sequence of token t, from sequence cur (behind it) down
__device__ __forceinline__ int seq_before(const int* cu, int S, int cur, int t) {
  while (cur > 0 && cu[cur] > t) --cur;
  return cur < S ? cur : S - 1;
}

// One thread's VEC channels of one run.
struct Place {
  int b, seg, t0, n;
  long long d;
  bool live;
};
template <int VEC>
__device__ __forceinline__ Place place(const RecArgs& a) {
  const int nseg = (a.T + SEG - 1) / SEG, strips = (a.D + 64 * VEC - 1) / (64 * VEC);
  const long long quads = (nseg + 3) / 4;
  long long k = blockIdx.x;
  Place p;
  const int strip = (int)(k % strips);
  k /= strips;
  p.seg = (int)(k % quads) * 4 + wave_id();
  p.b = (int)(k / quads);
  p.t0 = p.seg * SEG;
  p.n = a.T - p.t0 < SEG ? a.T - p.t0 : SEG;
  p.d = (long long)strip * 64 * VEC + lane_id() * VEC;
  p.live = p.seg < nseg && p.d < a.D;
  return p;
}

template <int VEC>
__device__ __forceinline__ void params(const RecArgs& a, long long d, float* bias2, float* nrate) {
  const int per = a.D / a.H;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    bias2[i] = a.dt_bias[d + i] * LOG2E;
    nrate[i] = -__builtin_amdgcn_exp2f(a.A_log[(d + i) / per] * LOG2E);
  }
}

}  // namespace

// ---------------------------------------------------------------- forward

// (A, H) of every run.
template <typename E, int VEC>
__global__ __launch_bounds__(256) void rec_reduce_fwd(RecArgs a) {
  const Place p = place<VEC>(a);
  if (!p.live) return;
  float bias2[VEC], nrate[VEC], A[VEC], H[VEC];
  params<VEC>(a, p.d, bias2, nrate);
  Run r{0u, 0u, ~0u, 0, 0};
  if (a.cu) r = run_of(a.cu, a.S, p.t0, p.n, a.T);
  int cur = r.cur;
#pragma unroll
  for (int i = 0; i < VEC; ++i) { A[i] = 1.f; H[i] = 0.f; }
  for (int j = 0; j < p.n; ++j) {
    const long long t = p.t0 + j;
    float x[VEC], f[VEC], w[VEC];
    loadv<E, VEC>(static_cast<const E*>(a.x) + p.b * a.x_b + t * a.x_t + p.d, x);
    loadv<E, VEC>(static_cast<const E*>(a.f) + p.b * a.f_b + t * a.f_t + p.d, f);
    loadv<E, VEC>(static_cast<const E*>(a.wz) + p.b * a.w_b + t * a.w_t + p.d, w);
    const bool st = r.start >> j & 1, us = r.used >> j & 1;
    if (st) cur = seq_from(a.cu, a.S, cur, (int)t);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const Decay k = decay(f[i], bias2[i], nrate[i]);
      float beta, inv;
      root(k.q, beta, inv);
      float u = beta * sigmoid2(w[i]) * x[i], keep = k.a;
      if (st) {
        if (a.h0 && us) u += k.a * a.h0[(long long)cur * a.D + p.d + i];
        keep = 0.f;
      }
      if (!us) { u = 0.f; keep = 0.f; H[i] = 0.f; }
      H[i] = st ? u : keep * H[i] + u;
      A[i] *= keep;
    }
  }
  const long long nseg = (a.T + SEG - 1) / SEG;
  const long long o = ((long long)p.b * nseg + p.seg) * a.D + p.d;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    a.ws[o + i] = A[i];
    a.hs[o + i] = H[i];
  }
}

// The state entering every run (hs: H in, the state out), and for rows that
// are not packed the final state.
__global__ __launch_bounds__(64) void rec_carry_fwd(RecArgs a) {
  const long long c = (long long)blockIdx.x * 64 + threadIdx.x;
  if (c >= (long long)a.B * a.D) return;
  const long long b = c / a.D, d = c % a.D, nseg = (a.T + SEG - 1) / SEG;
  float h = (a.h0 && !a.cu) ? a.h0[c] : 0.f;
  for (long long s = 0; s < nseg; ++s) {
    const long long o = (b * nseg + s) * a.D + d;
    const float H = a.hs[o];
    a.hs[o] = h;
    const float A = a.ws[o];
    h = A == 0.f ? H : A * h + H;
  }
  if (a.final_state && !a.cu) a.final_state[c] = h;
}

// Every token from the state entering its run.
template <typename E, int VEC>
__global__ __launch_bounds__(256) void rec_apply_fwd(RecArgs a) {
  const Place p = place<VEC>(a);
  if (!p.live) return;
  float bias2[VEC], nrate[VEC], h[VEC];
  params<VEC>(a, p.d, bias2, nrate);
  const long long nseg = (a.T + SEG - 1) / SEG;
#pragma unroll
  for (int i = 0; i < VEC; ++i) h[i] = a.hs[(p.b * nseg + p.seg) * a.D + p.d + i];
  Run r{0u, 0u, ~0u, 0, 0};
  if (a.cu) r = run_of(a.cu, a.S, p.t0, p.n, a.T);
  int cur = r.cur;
  for (int j = 0; j < p.n; ++j) {
    const long long t = p.t0 + j;
    float x[VEC], f[VEC], w[VEC], y[VEC];
    loadv<E, VEC>(static_cast<const E*>(a.x) + p.b * a.x_b + t * a.x_t + p.d, x);
    loadv<E, VEC>(static_cast<const E*>(a.f) + p.b * a.f_b + t * a.f_t + p.d, f);
    loadv<E, VEC>(static_cast<const E*>(a.wz) + p.b * a.w_b + t * a.w_t + p.d, w);
    const bool st = r.start >> j & 1, us = r.used >> j & 1, en = r.end >> j & 1;
    if (st) cur = seq_from(a.cu, a.S, cur, (int)t);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const Decay k = decay(f[i], bias2[i], nrate[i]);
      float beta, inv;
      root(k.q, beta, inv);
      const float u = beta * sigmoid2(w[i]) * x[i];
      if (st) h[i] = (a.h0 && us) ? a.h0[(long long)cur * a.D + p.d + i] : 0.f;
      h[i] = us ? k.a * h[i] + u : 0.f;
      if (en && a.final_state) a.final_state[(long long)cur * a.D + p.d + i] = h[i];
      y[i] = h[i];
    }
    storev<E, VEC>(static_cast<E*>(a.y) + ((long long)p.b * a.T + t) * a.D + p.d, y);
  }
}

// Sequences without tokens: out = in (or 0). Their final state is their
// initial one, their initial state's gradient the final one's.
__global__ __launch_bounds__(256) void rec_empty(RecArgs a, const float* in, float* out) {
  const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
  if (c >= (long long)a.S * a.D) return;
  const long long s = c / a.D;
  const int lo = a.cu[s] < a.T ? a.cu[s] : a.T, hi = a.cu[s + 1] < a.T ? a.cu[s + 1] : a.T;
  if (lo >= hi) out[c] = in ? in[c] : 0.f;
}

// ---------------------------------------------------------------- backward

// (A, C) of every run in reverse: what flows to the token before it,
// c = A c_in + C, c_t = a_t lam_t.
template <typename E, int VEC>
__global__ __launch_bounds__(256) void rec_reduce_bwd(RecArgs a) {
  const Place p = place<VEC>(a);
  if (!p.live) return;
  float bias2[VEC], nrate[VEC], A[VEC], C[VEC];
  params<VEC>(a, p.d, bias2, nrate);
  Run r{0u, 0u, ~0u, 0, 0};
  if (a.cu) r = run_of(a.cu, a.S, p.t0, p.n, a.T);
  int cur = r.last;
#pragma unroll
  for (int i = 0; i < VEC; ++i) { A[i] = 1.f; C[i] = 0.f; }
  for (int j = p.n - 1; j >= 0; --j) {
    const long long t = p.t0 + j;
    float f[VEC], g[VEC];
    loadv<E, VEC>(static_cast<const E*>(a.f) + p.b * a.f_b + t * a.f_t + p.d, f);
    loadv<E, VEC>(static_cast<const E*>(a.dy) + p.b * a.dy_b + t * a.dy_t + p.d, g);
    const bool us = r.used >> j & 1, en = r.end >> j & 1;
    if (en) cur = seq_before(a.cu, a.S, cur, (int)t);
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const Decay k = decay(f[i], bias2[i], nrate[i]);
      if (en) {
        A[i] = 0.f;
        C[i] = a.dfinal ? a.dfinal[(long long)cur * a.D + p.d + i] : 0.f;
      }
      C[i] = us ? k.a * (g[i] + C[i]) : 0.f;
      A[i] = us ? k.a * A[i] : 0.f;
    }
  }
  const long long nseg = (a.T + SEG - 1) / SEG, n = (long long)a.B * nseg * a.D;
  const long long o = ((long long)p.b * nseg + p.seg) * a.D + p.d;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    a.ws[o + i] = A[i];
    a.ws[n + o + i] = C[i];
  }
}

__global__ __launch_bounds__(64) void rec_carry_bwd(RecArgs a) {
  const long long c = (long long)blockIdx.x * 64 + threadIdx.x;
  if (c >= (long long)a.B * a.D) return;
  const long long b = c / a.D, d = c % a.D, nseg = (a.T + SEG - 1) / SEG;
  const long long n = (long long)a.B * nseg * a.D;
  float h = (a.dfinal && !a.cu) ? a.dfinal[c] : 0.f;
  for (long long s = nseg - 1; s >= 0; --s) {
    const long long o = (b * nseg + s) * a.D + d;
    const float C = a.ws[n + o], A = a.ws[o];
    a.ws[n + o] = h;
    h = A == 0.f ? C : A * h + C;
  }
  if (a.dh0 && !a.cu) a.dh0[c] = h;
}

// Every token's gradients from the state entering its run and the gradient
// entering it from behind; the two sums over tokens a run at a time into ws
// behind the carries.
template <typename E, int VEC>
__global__ __launch_bounds__(256) void rec_apply_bwd(RecArgs a) {
  const Place p = place<VEC>(a);
  if (!p.live) return;
  float bias2[VEC], nrate[VEC], h[VEC], c[VEC], sb[VEC], sa[VEC];
  params<VEC>(a, p.d, bias2, nrate);
  const long long nseg = (a.T + SEG - 1) / SEG, n = (long long)a.B * nseg * a.D;
  const long long o = ((long long)p.b * nseg + p.seg) * a.D + p.d;
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    h[i] = a.hs[o + i];
    c[i] = a.ws[n + o + i];
    sb[i] = sa[i] = 0.f;
  }
  Run r{0u, 0u, ~0u, 0, 0};
  if (a.cu) r = run_of(a.cu, a.S, p.t0, p.n, a.T);
  float prev[SEG][VEC];
  int cur = r.cur;
#pragma unroll
  for (int j = 0; j < SEG; ++j) {
    if (j < p.n) {
      const long long t = p.t0 + j;
      float x[VEC], f[VEC], w[VEC];
      loadv<E, VEC>(static_cast<const E*>(a.x) + p.b * a.x_b + t * a.x_t + p.d, x);
      loadv<E, VEC>(static_cast<const E*>(a.f) + p.b * a.f_b + t * a.f_t + p.d, f);
      loadv<E, VEC>(static_cast<const E*>(a.wz) + p.b * a.w_b + t * a.w_t + p.d, w);
      const bool st = r.start >> j & 1, us = r.used >> j & 1;
      if (st) cur = seq_from(a.cu, a.S, cur, (int)t);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const Decay k = decay(f[i], bias2[i], nrate[i]);
        float beta, inv;
        root(k.q, beta, inv);
        if (st) h[i] = (a.h0 && us) ? a.h0[(long long)cur * a.D + p.d + i] : 0.f;
        prev[j][i] = h[i];
        h[i] = us ? k.a * h[i] + beta * sigmoid2(w[i]) * x[i] : 0.f;
      }
    }
  }
  cur = r.last;
#pragma unroll
  for (int j = SEG - 1; j >= 0; --j) {
    if (j < p.n) {
      const long long t = p.t0 + j;
      float x[VEC], f[VEC], w[VEC], g[VEC], dx[VEC], df[VEC], dw[VEC];
      loadv<E, VEC>(static_cast<const E*>(a.x) + p.b * a.x_b + t * a.x_t + p.d, x);
      loadv<E, VEC>(static_cast<const E*>(a.f) + p.b * a.f_b + t * a.f_t + p.d, f);
      loadv<E, VEC>(static_cast<const E*>(a.wz) + p.b * a.w_b + t * a.w_t + p.d, w);
      loadv<E, VEC>(static_cast<const E*>(a.dy) + p.b * a.dy_b + t * a.dy_t + p.d, g);
      const bool st = r.start >> j & 1, us = r.used >> j & 1, en = r.end >> j & 1;
      if (en) cur = seq_before(a.cu, a.S, cur, (int)t);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        if (en) c[i] = a.dfinal ? a.dfinal[(long long)cur * a.D + p.d + i] : 0.f;
        if (!us) {
          dx[i] = df[i] = dw[i] = c[i] = 0.f;
          continue;
        }
        const Decay k = decay(f[i], bias2[i], nrate[i]);
        float beta, inv;
        root(k.q, beta, inv);
        const float s = sigmoid2(w[i]), lam = g[i] + c[i];
        const float one = __builtin_amdgcn_rcpf(1.f + k.e), sz = k.up ? one : k.e * one;
        const float dg = lam * (k.a * prev[j][i] - k.a * k.a * inv * s * x[i]);
        dx[i] = lam * beta * s;
        dw[i] = dx[i] * x[i] * (1.f - s);
        df[i] = nrate[i] * sz * dg;
        sb[i] += df[i];
        sa[i] += dg * k.g2;
        c[i] = k.a * lam;
        if (st && a.dh0) a.dh0[(long long)cur * a.D + p.d + i] = c[i];
      }
      const long long q = ((long long)p.b * a.T + t) * a.D + p.d;
      storev<E, VEC>(static_cast<E*>(a.dx) + q, dx);
      storev<E, VEC>(static_cast<E*>(a.df) + q, df);
      storev<E, VEC>(static_cast<E*>(a.dwz) + q, dw);
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    a.ws[2 * n + o + i] = sb[i];
    a.ws[3 * n + o + i] = sa[i];
  }
}

// Sums over runs, a slice of them a workgroup row: part[slice][2][D].
__global__ __launch_bounds__(256) void rec_sum_runs(RecArgs a, const float* parts, long long rows,
                                                    float* out) {
  __shared__ float s[2][4][64];
  const int d = blockIdx.x * 64 + lane_id(), w = wave_id();
  const long long per = (rows + REC_SLICES - 1) / REC_SLICES, r0 = blockIdx.y * per;
  const long long r1 = r0 + per < rows ? r0 + per : rows;
  float b = 0.f, g = 0.f;
  if (d < a.D) {
    for (long long r = r0 + w; r < r1; r += 4) {
      b += parts[r * a.D + d];
      g += parts[(rows + r) * a.D + d];
    }
  }
  s[0][w][lane_id()] = b;
  s[1][w][lane_id()] = g;
  __syncthreads();
  if (w < 2 && d < a.D) {
    const int l = lane_id();
    out[((long long)blockIdx.y * 2 + w) * a.D + d] = s[w][0][l] + s[w][1][l] + s[w][2][l] + s[w][3][l];
  }
}

// The last sum, a wave a head: dt_bias' gradient a channel, A_log's a head.
__global__ __launch_bounds__(64) void rec_sum_heads(RecArgs a, const float* part) {
  const int h = blockIdx.x, per = a.D / a.H;
  float s = 0.f;
  for (int i = threadIdx.x; i < per; i += 64) {
    const int d = h * per + i;
    float b = 0.f, g = 0.f;
    for (int k = 0; k < REC_SLICES; ++k) {
      b += part[(k * 2LL) * a.D + d];
      g += part[(k * 2LL + 1) * a.D + d];
    }
    a.ddt_bias[d] = b;
    s += g;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, WAVE);
  if (threadIdx.x == 0) a.dA_log[h] = s * 0.69314718055994531f;     // g2 -> g
}

// ---------------------------------------------------------------- one token

// y = h' = a h + beta s x for B rows of D channels, VEC channels a thread.
template <typename E, int VEC>
__global__ __launch_bounds__(256) void rec_step_kernel(RecArgs a) {
  const int per = a.D / VEC;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)a.B * per) return;
  const long long b = i / per, d = (i - b * per) * VEC;
  float x[VEC], f[VEC], w[VEC], h[VEC], bias2[VEC], nrate[VEC];
  loadv<E, VEC>(static_cast<const E*>(a.x) + b * a.x_b + d, x);
  loadv<E, VEC>(static_cast<const E*>(a.f) + b * a.f_b + d, f);
  loadv<E, VEC>(static_cast<const E*>(a.wz) + b * a.w_b + d, w);
  loadv<float, VEC>(a.h0 + b * a.D + d, h);
  params<VEC>(a, d, bias2, nrate);
#pragma unroll
  for (int v = 0; v < VEC; ++v) {
    const Decay k = decay(f[v], bias2[v], nrate[v]);
    float beta, inv;
    root(k.q, beta, inv);
    h[v] = k.a * h[v] + beta * sigmoid2(w[v]) * x[v];
  }
  storev<float, VEC>(a.final_state + b * a.D + d, h);
  storev<E, VEC>(static_cast<E*>(a.y) + b * a.D + d, h);
}

// ---------------------------------------------------------------- launches

namespace {

// channels a thread can take at once: every row of every tensor it reads or
// writes starts on a multiple of that many elements
int vec_of(const RecArgs& a, size_t esz, std::initializer_list<const void*> ts,
           std::initializer_list<int64_t> strides) {
  if (a.D % 2) return 1;
  for (int64_t s : strides)
    if (s % 2) return 1;
  for (const void* t : ts)
    if (reinterpret_cast<uintptr_t>(t) % (2 * esz)) return 1;
  return 2;
}

template <int VEC>
dim3 run_grid(const RecArgs& a) {
  const long long nseg = (a.T + SEG - 1) / SEG;
  return dim3((unsigned)((a.D + 64 * VEC - 1) / (64 * VEC) * ((nseg + 3) / 4) * a.B));
}

template <typename E, int VEC>
hipError_t fwd(const RecArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((rec_reduce_fwd<E, VEC>), run_grid<VEC>(a), dim3(256), 0, st, a);
  hipLaunchKernelGGL(rec_carry_fwd, dim3((unsigned)(((long long)a.B * a.D + 63) / 64)), dim3(64), 0, st, a);
  hipLaunchKernelGGL((rec_apply_fwd<E, VEC>), run_grid<VEC>(a), dim3(256), 0, st, a);
  if (a.cu && a.final_state && a.S > 0)
    hipLaunchKernelGGL(rec_empty, dim3((unsigned)(((long long)a.S * a.D + 255) / 256)), dim3(256), 0,
                       st, a, a.h0, a.final_state);
  return hipGetLastError();
}

template <typename E, int VEC>
hipError_t bwd(const RecArgs& a, hipStream_t st) {
  const long long nseg = (a.T + SEG - 1) / SEG, rows = a.B * nseg;
  hipLaunchKernelGGL((rec_reduce_bwd<E, VEC>), run_grid<VEC>(a), dim3(256), 0, st, a);
  hipLaunchKernelGGL(rec_carry_bwd, dim3((unsigned)(((long long)a.B * a.D + 63) / 64)), dim3(64), 0, st, a);
  hipLaunchKernelGGL((rec_apply_bwd<E, VEC>), run_grid<VEC>(a), dim3(256), 0, st, a);
  if (a.cu && a.dh0 && a.S > 0)
    hipLaunchKernelGGL(rec_empty, dim3((unsigned)(((long long)a.S * a.D + 255) / 256)), dim3(256), 0,
                       st, a, a.dfinal, a.dh0);
  float* parts = a.ws + 2 * rows * a.D;
  float* sums = a.ws + 4 * rows * a.D;
  hipLaunchKernelGGL(rec_sum_runs, dim3((a.D + 63) / 64, REC_SLICES), dim3(256), 0, st, a,
                     (const float*)parts, rows, sums);
  hipLaunchKernelGGL(rec_sum_heads, dim3(a.H), dim3(64), 0, st, a, (const float*)sums);
  return hipGetLastError();
}

}  // namespace

int64_t rec_ws(int64_t B, int64_t T, int64_t D, bool backward) {
  const int64_t nseg = (T + SEG - 1) / SEG;
  if (!backward) return B * nseg * D;
  return 4 * B * nseg * D + 2 * REC_SLICES * D;
}

hipError_t rec_fwd(const RecArgs& a, int dtype, hipStream_t st) {
  const size_t esz = dtype == NGDN_BF16 ? 2 : 4;
  const int v = vec_of(a, esz, {a.x, a.f, a.wz, a.y}, {a.x_b, a.x_t, a.f_b, a.f_t, a.w_b, a.w_t});
  if (dtype == NGDN_BF16) return v == 2 ? fwd<bf16, 2>(a, st) : fwd<bf16, 1>(a, st);
  return v == 2 ? fwd<float, 2>(a, st) : fwd<float, 1>(a, st);
}

hipError_t rec_bwd(const RecArgs& a, int dtype, hipStream_t st) {
  const size_t esz = dtype == NGDN_BF16 ? 2 : 4;
  const int v = vec_of(a, esz, {a.x, a.f, a.wz, a.dy, a.dx, a.df, a.dwz},
                       {a.x_b, a.x_t, a.f_b, a.f_t, a.w_b, a.w_t, a.dy_b, a.dy_t});
  if (dtype == NGDN_BF16) return v == 2 ? bwd<bf16, 2>(a, st) : bwd<bf16, 1>(a, st);
  return v == 2 ? bwd<float, 2>(a, st) : bwd<float, 1>(a, st);
}

hipError_t rec_step(const RecArgs& a, int dtype, hipStream_t st) {
  const size_t esz = dtype == NGDN_BF16 ? 2 : 4;
  int v = vec_of(a, esz, {a.x, a.f, a.wz, a.y}, {a.x_b, a.f_b, a.w_b});
  if (v == 2) v = vec_of(a, 4, {a.h0, a.final_state}, {});
  const dim3 grid((unsigned)(((long long)a.B * (a.D / v) + 255) / 256));
  if (dtype == NGDN_BF16) {
    if (v == 2) hipLaunchKernelGGL((rec_step_kernel<bf16, 2>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((rec_step_kernel<bf16, 1>), grid, dim3(256), 0, st, a);
  } else {
    if (v == 2) hipLaunchKernelGGL((rec_step_kernel<float, 2>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((rec_step_kernel<float, 1>), grid, dim3(256), 0, st, a);
  }
  return hipGetLastError();
}

}  // namespace ngdn
