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
// runs are formed from zero in registers, joined in order, and completed from
// the state that enters them.
#include <algorithm>

#include "ngdn_kernels.h"

namespace ngdn {

namespace {

constexpr int N = REC_RUN;          // tokens a run, which a wave has in registers

constexpr float LOG2E = 1.44269504088896340736f;

// (1 - 4^p) / -p by its series: with p = g log2(e) 1 - e^2g
constexpr float Q1 = 1.3862943611198906f, Q2 = 0.96090602783640278f, Q3 = 0.44403286931857261f,
                Q4 = 0.15389006572205563f, Q5 = 0.042667386068571012f;

// What a token's decay needs: a = e^g, q = 1 - a^2, g2 = g log2(e), and ls = log2
// of sigmoid(z).
struct Decay {
  float a, q, g2, ls;
};

// The first coefficients of both polynomials. An instruction takes one constant:
// held in registers, where there are any left, they save two moves a token.
struct First {
  float p, q;
};
constexpr First FIRST{-0.012319466099143028f, Q5};
__device__ __forceinline__ First held() {
  First k = FIRST;
  asm volatile("" : "+v"(k.p), "+v"(k.q));
  return k;
}

// z2 = z log2(e) = f log2(e) + bias2, nrate = -exp(A_log).
// softplus(z) log2(e) = max(z2, 0) + log2(1 + e), e = e^-|z|: the logarithm as
// e P(e), P the degree-7 polynomial of least relative error on [0, 1] (3e-7 in
// fp32), which keeps its relative precision for the small e where decays usually
// sit; log2(1 + e) itself loses e's low bits there. And log2 sigmoid(z) =
// min(z2, 0) - e P(e), in one instruction where a reciprocal took six.
// q from the series for -g < 1/16 (its error 4e-8), where 1 - a^2 would cancel.
__device__ __forceinline__ Decay decay(float f, float bias2, float nrate, const First& k) {
  Decay d;
  const float z2 = fmaf(f, LOG2E, bias2);
  const float e = __builtin_amdgcn_exp2f(-fabsf(z2));
  float p = fmaf(k.p, e, 0.06360787153244019f);
  p = fmaf(p, e, -0.15535186231136322f);
  p = fmaf(p, e, 0.2560097277164459f);
  p = fmaf(p, e, -0.35339483618736267f);
  p = fmaf(p, e, 0.48006370663642883f);
  p = fmaf(p, e, -0.7213100790977478f);
  p = fmaf(p, e, 1.4426947832107544f);
  d.g2 = nrate * fmaf(p, e, fmaxf(z2, 0.f));
  d.ls = fmaf(-p, e, fminf(z2, 0.f));
  d.a = __builtin_amdgcn_exp2f(d.g2);
  const float g2 = d.g2;
  const float s = -g2 * fmaf(g2, fmaf(g2, fmaf(g2, fmaf(g2, k.q, Q4), Q3), Q2), Q1);
  d.q = g2 > -LOG2E / 16.f ? s : fmaf(-d.a, d.a, 1.f);
  return d;
}

__device__ __forceinline__ float sigmoid2(float w) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-LOG2E * w));
}
// s = sigmoid(w) and 1 - s = e^-w s, which a subtraction loses where the gate is open
// (all of it from w = 17). e^-w is held below 2^126 there: where it is more, s may be
// 0, and so is what 1 - s multiplies.
__device__ __forceinline__ float sigmoid2(float w, float& rest) {
  const float e = __builtin_amdgcn_exp2f(-LOG2E * w), s = __builtin_amdgcn_rcpf(1.f + e);
  rest = fminf(e, 0x1p126f) * s;
  return s;
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
__device__ Run run_of(const int* cu, int S, int t0, int n, int T) {
  Run r{0u, 0u, 0u, 0, 0};
  int lo = 0, hi = S + 1;                  // first boundary at or behind t0
  while (lo < hi) {
    const int m = (lo + hi) / 2;
    if (cu[m] < t0) lo = m + 1; else hi = m;
  }
  int s = lo;
  r.cur = s - 1;
  // from boundary to boundary (a boundary that lies lower than one before it counts
  // as there)
  for (int at = t0;;) {
    const int next = s <= S ? (cu[s] > at ? cu[s] : at) : 0x7fffffff, to = next < t0 + n ? next : t0 + n;
    if (s >= 1 && s <= S && to > at) {
      r.used |= (1u << (to - t0)) - (1u << (at - t0));
      if (next == to || to == T) r.end |= 1u << (to - 1 - t0);
    }
    if (next >= t0 + n) break;
    r.start |= 1u << (next - t0);
    at = next;
    ++s;
  }
  r.last = s - 1;
  return r;
}
__device__ __forceinline__ int4 pack(const Run& r) {
  return make_int4((int)(r.start | r.end << 16), (int)r.used, r.cur, r.last);
}
// A wave's run, by a scalar load: it does not queue behind the tokens' loads.
__device__ __forceinline__ Run unpack(const int4* at) {
  typedef int I4 __attribute__((ext_vector_type(4)));
  const I4 v = *(const __attribute__((address_space(4))) I4*)at;
  const unsigned m = v.x;
  return Run{m & 0xffffu, m >> 16, (unsigned)v.y, v.z, v.w};
}
// the sequence that token t starts: the last one with that boundary, from
// sequence cur on
using Scalar = const __attribute__((address_space(4))) int;
__device__ __forceinline__ int seq_from(const int* boundaries, int S, int cur, int t) {
  Scalar* cu = (Scalar*)boundaries;
  if (cur < 0) cur = 0;
  while (cur + 1 <= S && cu[cur + 1] <= t) ++cur;
  return cur < S ? cur : S - 1;
}
// the sequence of token t, from sequence cur (behind it) down
__device__ __forceinline__ int seq_before(const int* boundaries, int S, int cur, int t) {
  Scalar* cu = (Scalar*)boundaries;
  while (cur > 0 && cu[cur] > t) --cur;
  return cur < S ? cur : S - 1;
}

// bias2 and nrate of a channel
__device__ __forceinline__ void params(const RecArgs& a, unsigned d, float& bias2, float& nrate) {
  bias2 = a.dt_bias[d] * LOG2E;
  nrate = -__builtin_amdgcn_exp2f(a.A_log[d / (unsigned)(a.D / a.H)] * LOG2E);
}

// ---------------------------------------------------------------- joining runs
//
// A workgroup has W waves, each a run of N tokens of 64 channels (a strip): a
// tile of W runs. The state that enters a tile comes from the tiles before it (in
// the backward: behind it) while those are still running, through device memory:
// every tile publishes its (A, H) as soon as it has them; the last of a group of
// W EACH also the state behind it. A tile takes the state at its group's start and
// the (A, H) of the tiles between, so the chain over a long row has a link a
// group, and the order of the arithmetic does not depend on timing. EACH 1, 2, 4,
// both passes: 65536 x 64 100, 70, 59 us; 4 x 8192 x 2048 323, 327, 332.
// One 64-bit (32-bit) value is its own flag: all bits set before it is
// published, which no published value has (a NaN of that pattern is changed).
// A strip's tiles are handed out by a counter, so all a tile waits for was
// started before it and waits only for tiles before itself: every wait ends.
// A counter for each strip: 512 workgroups that start together on one counter
// take 6 us to get their numbers.
// Against reducing, joining and applying in three launches: inputs are read
// and their gates computed once instead of twice (65536 x 2048 bf16 forward
// 1900 us, then 250).
// One channel a lane leaves room for three or four workgroups a CU (two in the
// backward), whose loading, computing and waiting overlap; with two channels
// (4-byte loads of bf16) half of that fits. When it was decided: 16384 x 1024
// packed, both passes, 146 us against 135, 333 x 1024 forward 13.7 against 11.1,
// 65536 x 2048 forward 234 against 243.

constexpr int W = REC_WAVES;
constexpr int LINE = 32;            // ints in a cache line
constexpr int EACH = 2;             // tiles that a wave looks at, W EACH of them a group

struct Sync {
  int* ticket;                      // [nstrip] counters, LINE apart (NULL: one tile a row, nothing to join)
  unsigned long long* agg;          // [nchunk][nstrip][64] (A, H)
  unsigned* base;                   // [groups][nstrip][64]
  const int4* runs;                 // packed rows: every run's Run
  int nchunk, nstrip, strips;       // nstrip = B strips
};

__device__ __forceinline__ unsigned bits(float x) { return __float_as_uint(x); }
constexpr unsigned RESET = 0x80000000u;      // A = -0: nothing before passes (a >= +0 is never it)

// (A2, H2) after (A1, H1); a reset keeps what is not finite before it out
template <bool PACKED>
__device__ __forceinline__ void join(float& A1, float& H1, float2 v) {
  if (PACKED && bits(v.x) == RESET) {
    A1 = v.x;
    H1 = v.y;
  } else {
    H1 = fmaf(v.x, H1, v.y);
    A1 = PACKED && bits(A1) == RESET ? A1 : A1 * v.x;
  }
}
template <bool PACKED>
__device__ __forceinline__ float pass(float h, float2 v) {
  return PACKED && bits(v.x) == RESET ? v.y : fmaf(v.x, h, v.y);
}

__device__ __forceinline__ void publish(unsigned long long* p, float A, float H) {
  const unsigned a = bits(A) == ~0u ? 0x7fc00000u : bits(A);
  __hip_atomic_store(p, (unsigned long long)a << 32 | bits(H), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void publish(unsigned* p, float h) {
  __hip_atomic_store(p, bits(h) == ~0u ? 0x7fc00000u : bits(h), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename U>
__device__ __forceinline__ U peek(const U* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename U>
__device__ __forceinline__ U await(const U* p, U v) {
  while (v == (U)~(U)0) {
    __builtin_amdgcn_s_sleep(1);
    v = peek(p);
  }
  return v;
}
__device__ __forceinline__ float2 pair(unsigned long long v) {
  return make_float2(__uint_as_float((unsigned)(v >> 32)), __uint_as_float((unsigned)v));
}

struct Joint {
  float2 wave[W][64];               // (A, H) of the tile's waves, in the order of the scan
  float2 before[W][64];             // of the group's tiles before it
  float base[64];
  int step;
};

// A lane's element of a row: the row's address is the wave's and the lane's part
// 32 bits, so that the next token costs scalar additions and no vector instruction
// (a vector 64-bit address for each load: 4 x 8192 x 2048, both passes, 358 us
// against 330, 65536 x 2048 forward 243 against 228).
template <typename E>
using Device = __attribute__((address_space(1))) E;
template <typename E>
__device__ __forceinline__ E load_at(const E* row, unsigned bytes) {
  return *(const Device<E>*)((const Device<char>*)row + bytes);
}
template <typename E>
__device__ __forceinline__ void store_at(E* row, unsigned bytes, float x) {
  *(Device<E>*)((Device<char>*)row + bytes) = from_f<E>(x);
}
// Two tokens' rows, one conversion.
template <typename E>
__device__ __forceinline__ void store_two(E* r0, E* r1, unsigned bytes, float x0, float x1) {
  typedef E Pair __attribute__((ext_vector_type(2)));
  typedef float Two __attribute__((ext_vector_type(2)));
  const Pair p = __builtin_convertvector((Two{x0, x1}), Pair);
  *(Device<E>*)((Device<char>*)r0 + bytes) = p.x;
  *(Device<E>*)((Device<char>*)r1 + bytes) = p.y;
}
// The compiler takes that form only where it sees the 32 bits widened in the same block.
__device__ __forceinline__ unsigned here(unsigned bytes) {
  asm volatile("" : "+v"(bytes));
  return bytes;
}
// The run's n tokens of K tensors, token by token; p: their first tokens' rows, row:
// elements from one to the next. Behind the n the last again. (The barrier keeps
// the sum in scalar registers, where it would be rearranged into vector ones.)
template <int K, typename E>
__device__ __forceinline__ void load_run(E (&v)[K][N], const E* (&p)[K], const long long (&row)[K], int n,
                                         unsigned bytes) {
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k][j] = load_at(p[k], bytes);
      if (j + 1 < N) {
        p[k] += j + 1 < n ? row[k] : 0;
        asm volatile("" : "+s"(p[k]));
      }
    }
}

// From wave (A, H) to the state entering the wave. step: the tile's place in the
// scan's order (0 first), wv the wave's. first: the state entering tile 0.
template <bool PACKED>
__device__ __forceinline__ float join_tiles(Joint& s, const Sync& y, int step, int strip, int wv, float A, float H,
                                            float first) {
  const int l = lane_id();
  s.wave[wv][l] = make_float2(A, H);
  lds_barrier();
  float h = first;
  if (y.ticket) {
    constexpr int per = W * EACH;
    const int group = step / per, n = step - group * per;      // n tiles from the group's start
    const bool go = step + 1 < y.nchunk, link = n == per - 1 && go;
    auto agg = [&](int k) { return y.agg + ((long long)k * y.nstrip + strip) * 64 + l; };
    auto base = [&](int k) { return y.base + ((long long)k * y.nstrip + strip) * 64 + l; };
    float tA = 1.f, tH = 0.f;                                 // the whole tile
    if (wv == W - 1 && go) {
#pragma unroll
      for (int k = 0; k < W; ++k) join<PACKED>(tA, tH, s.wave[k][l]);
      publish(agg(step), tA, tH);
    }
    if (step > 0) {
      // each wave EACH of the n tiles in order; the last wave also the state at the
      // group's start. All are looked at before the first is waited for
      const int k0 = wv * EACH, k1 = k0 + EACH < n ? k0 + EACH : n;
      const bool far = wv == W - 1 && group > 0;
      const unsigned hb = far ? peek(base(group)) : bits(first);
      unsigned long long v[EACH];
#pragma unroll
      for (int i = 0; i < EACH; ++i) v[i] = k0 + i < k1 ? peek(agg(group * per + k0 + i)) : 0;
      float bA = 1.f, bH = 0.f;
#pragma unroll
      for (int i = 0; i < EACH; ++i)
        if (k0 + i < k1) join<PACKED>(bA, bH, pair(await(agg(group * per + k0 + i), v[i])));
      s.before[wv][l] = make_float2(bA, bH);
      // the group's last tile is a link of the chain: everything up to its own end is
      // joined before the state at its start is there, which then goes on in one operation
      if (link) lds_barrier();
      if (wv == W - 1) {
        float gA = 1.f, gH = 0.f;
        if (link) {
          for (int k = 0; k * EACH < n; ++k) join<PACKED>(gA, gH, s.before[k][l]);
          join<PACKED>(gA, gH, make_float2(tA, tH));
        }
        h = __uint_as_float(far ? await(base(group), hb) : hb);
        if (link) publish(base(group + 1), pass<PACKED>(h, make_float2(gA, gH)));
        s.base[l] = h;
      }
      lds_barrier();
      h = s.base[l];
      for (int k = 0; k * EACH < n; ++k) h = pass<PACKED>(h, s.before[k][l]);
    }
  }
  for (int k = 0; k < wv; ++k) h = pass<PACKED>(h, s.wave[k][l]);
  return h;
}

// A workgroup's strip: every nstrip workgroups one of each, turned on by one
// each time, so that the workgroups of one XCD (every 8th) go over all strips. A
// strip's rows lie a whole row apart and fall on few of the XCD's L2 channels:
// with a strip always on the same XCD, 65536 x 2048 took 278 us, turned 243.
__device__ __forceinline__ int strip_of(const Sync& y) {
  const unsigned q = blockIdx.x / y.nstrip, r = blockIdx.x - q * y.nstrip;
  return (r + q) % y.nstrip;
}
// The tile's place in its strip's scan.
__device__ __forceinline__ int take(const Sync& y, int strip, Joint& s) {
  if (!y.ticket) return 0;
  if (threadIdx.x == 0)
    s.step = __hip_atomic_fetch_add(y.ticket + strip * LINE, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(s.step);
}

// Before either pass: the flags' patterns, the counters, where the boundaries of
// packed sequences fall in each run, and sequences without tokens (out = in or
// 0: their final state is their initial one, their initial state's gradient the
// final one's). 2 to 6 us, a launch and 0.8 % of the pass's bytes.
__global__ __launch_bounds__(256) void rec_init(RecArgs a, uint4* fill, long long n16, int* ticket, int tickets,
                                                int4* runs, const float* in, float* out) {
  const unsigned i0 = blockIdx.x * 256 + threadIdx.x, step = gridDim.x * 256;
  if (a.cu) {
    // the search and the walk are chains of reads: from LDS where the boundaries fit
    constexpr int FIT = 4096;
    __shared__ int s_cu[FIT];
    const int* cu = a.cu;
    if (a.S < FIT) {
      for (int i = threadIdx.x; i <= a.S; i += 256) s_cu[i] = a.cu[i];
      __syncthreads();
      cu = s_cu;
    }
    const unsigned nrun = (a.T + N - 1u) / N, n = out ? (unsigned)a.S * a.D : 0u;     // S D < 2^31
    for (unsigned i = i0; i < nrun; i += step) {
      const int t0 = (int)i * N;
      runs[i] = pack(run_of(cu, a.S, t0, a.T - t0 < N ? a.T - t0 : N, a.T));
    }
    for (unsigned c = i0; c < n; c += step) {
      const unsigned s = c / (unsigned)a.D;
      const int lo = cu[s] < a.T ? cu[s] : a.T, hi = cu[s + 1] < a.T ? cu[s + 1] : a.T;
      if (lo >= hi) out[c] = in ? in[c] : 0.f;
    }
  }
  for (unsigned i = i0; i < (unsigned)tickets; i += step) ticket[(long long)i * LINE] = 0;
  for (long long i = i0; i < n16; i += step) fill[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
}

}  // namespace

// ---------------------------------------------------------------- forward

// A wave has the gates of its run in registers, then within the run
// h_t = H_t + P_t h_in from one pass, then y.
// Three values of a token and channel are read and one written, in bf16 8 bytes:
// 65536 x 2048 in 225 us, 4.8 TB/s where a large copy reaches 5.2. Behind that
// bound lies the next: vector instructions are issued 4/5 of the time (42 a token, 5
// of them transcendental). More waves a CU (64 registers, a few spilled) took 251 us.
// 333 x 1024: 7.5 us, three tiles' loads and joins.
template <typename E, bool PACKED>
__global__ __launch_bounds__(64 * W, 4) void rec_fwd_kernel(RecArgs a, Sync sy) {
  __shared__ Joint s_join;
  const int strip = strip_of(sy), chunk = take(sy, strip, s_join), wv = wave_id(), b = strip / sy.strips;
  const int d = strip % sy.strips * 64 + lane_id();
  const bool live = d < a.D;
  // lanes behind D work on channel 0 and store nothing
  const unsigned dl = live ? d : 0, lane = dl * (unsigned)sizeof(E);
  const int t0 = (chunk * W + wv) * N, n = a.T - t0 < N ? a.T - t0 : N;     // n <= 0: no token
  const long long ts = n > 0 ? t0 : a.T - 1;
  E v[3][N];                                          // f, wz, x
  const long long row[3] = {a.f_t, a.w_t, a.x_t};
  const E* p[3] = {static_cast<const E*>(a.f) + b * a.f_b + ts * a.f_t,
                   static_cast<const E*>(a.wz) + b * a.w_b + ts * a.w_t,
                   static_cast<const E*>(a.x) + b * a.x_b + ts * a.x_t};
  load_run(v, p, row, n, lane);
  float bias2, nrate;
  params(a, dl, bias2, nrate);
  const float first = a.h0 && !PACKED ? a.h0[(long long)b * a.D + dl] : 0.f;
  Run r{0u, 0u, 0u, 0, 0};
  if (PACKED && n > 0) r = unpack(sy.runs + t0 / N);
  const First c0 = FIRST;
  float P[N], H[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const Decay k = decay(to_f(v[0][j]), bias2, nrate, c0);
    P[j] = k.a;
    H[j] = __builtin_amdgcn_sqrtf(k.q) * sigmoid2(to_f(v[1][j])) * to_f(v[2][j]);
  }
  if (n < N) {                                        // behind the row: the state passes
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j >= n) {
        P[j] = 1.f;
        H[j] = 0.f;
      }
  }
  // the first token that the state before the run does not reach
  int cut = N;
  if (PACKED) {
    const unsigned stop = r.start | (~r.used & ((1u << N) - 1));
    if (stop) cut = __builtin_ctz(stop);
    int cur = r.cur;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const bool st = r.start >> j & 1, us = r.used >> j & 1;
      if (st || !us) {
        if (st) cur = seq_from(a.cu, a.S, cur, t0 + j);
        const float h = a.h0 && st && us ? a.h0[(long long)cur * a.D + dl] : 0.f;
        H[j] = us ? fmaf(P[j], h, H[j]) : 0.f;
        P[j] = 0.f;
      } else if (j > 0) {
        H[j] = fmaf(P[j], H[j - 1], H[j]);
        P[j] *= P[j - 1];
      }
    }
  } else {
#pragma unroll
    for (int j = 1; j < N; ++j) {
      H[j] = fmaf(P[j], H[j - 1], H[j]);
      P[j] *= P[j - 1];
    }
  }
  const float A = PACKED && cut < N ? __uint_as_float(RESET) : P[N - 1];
  const float h = join_tiles<PACKED>(s_join, sy, chunk, strip, wv, A, H[N - 1], first);
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (!PACKED || j < cut) H[j] = fmaf(P[j], h, H[j]);
  if (n <= 0 || !live) return;
  if (a.hs) a.hs[(b * ((a.T + N - 1LL) / N) + t0 / N) * a.D + d] = h;
  E* yp = static_cast<E*>(a.y) + ((long long)b * a.T + t0) * a.D;
  if (n >= N) {
    const unsigned o = here(lane);
#pragma unroll
    for (int j = 0; j < N; j += 2, yp += 2LL * a.D) store_two(yp, yp + a.D, o, H[j], H[j + 1]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j, yp += a.D)
      if (j < n) store_at(yp, lane, H[j]);
  }
  if (!a.final_state) return;
  if (PACKED) {
    if (!r.end) return;
    int cur = r.cur;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (r.start >> j & 1) cur = seq_from(a.cu, a.S, cur, t0 + j);
      if (r.end >> j & 1) {
        if (cur < 0) cur = 0;
        a.final_state[(long long)cur * a.D + d] = H[j];
      }
    }
  } else if (t0 + N >= a.T) {
    // tokens behind the row pass the state on, so the last register has it
    a.final_state[(long long)b * a.D + d] = H[N - 1];
  }
}

// ---------------------------------------------------------------- backward

// One pass over the run's tokens in order forms the gates again, the states from
// hs, what lam_t multiplies in each gradient, and (A, C) with c = A c_in + C for
// what flows out of the run backwards (c_t = a_t lam_t). The parameter gradients'
// sums over tokens: dt_bias' of df as it is formed; A_log's, sum lam_t k_t with k_t =
// ki_t g_t, needs no second array: with G_t = a_t G_(t-1) + k_t it is
// sum dy_t G_t + c_in G_last.
// Four values of a token and channel are read, three written: 4 x 8192 x 2048 in
// bf16 195 us, 4.8 TB/s. Its 71 vector instructions a token are issued 3/4 of the
// time; a tenth fewer (sigmoid(z) from its logarithm, df summed as it is formed)
// took 1 % off. A branch a token where a row or sequence may end: straight code for
// rows of whole runs was no faster, and two copies of the loop spill.
template <typename E, bool PACKED>
__global__ __launch_bounds__(64 * W, 4) void rec_bwd_kernel(RecArgs a, Sync sy, float* parts) {
  __shared__ Joint s_join;
  const int strip = strip_of(sy), step = take(sy, strip, s_join), wv = wave_id();
  const int chunk = sy.nchunk - 1 - step, b = strip / sy.strips, d = strip % sy.strips * 64 + lane_id();
  const bool live = d < a.D;
  const unsigned dl = live ? d : 0, lane = dl * (unsigned)sizeof(E);
  const int t0 = (chunk * W + wv) * N, n = a.T - t0 < N ? a.T - t0 : N;
  const long long ts = n > 0 ? t0 : a.T - 1;
  E v[4][N];                                          // f, wz, x, dy
  const long long row[4] = {a.f_t, a.w_t, a.x_t, a.dy_t};
  const E* p[4] = {static_cast<const E*>(a.f) + b * a.f_b + ts * a.f_t,
                   static_cast<const E*>(a.wz) + b * a.w_b + ts * a.w_t,
                   static_cast<const E*>(a.x) + b * a.x_b + ts * a.x_t,
                   static_cast<const E*>(a.dy) + b * a.dy_b + ts * a.dy_t};
  load_run(v, p, row, n, lane);
  float bias2, nrate;
  params(a, dl, bias2, nrate);
  const float last = a.dfinal && !PACKED ? a.dfinal[(long long)b * a.D + dl] : 0.f;
  float h = n > 0 ? a.hs[(b * ((a.T + N - 1LL) / N) + t0 / N) * a.D + dl] : 0.f;
  Run r{0u, 0u, 0u, 0, 0};
  if (PACKED && n > 0) r = unpack(sy.runs + t0 / N);
  float aa[N], bs[N], kw[N], kf[N], dy[N];
  const First c0 = held();
  float A = 1.f, C = 0.f, Ga = 0.f, sb = 0.f, sa = 0.f;
  int cur = r.cur;
  bool open = true;                        // no sequence has ended in the run yet
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const bool st = PACKED && (r.start >> j & 1), us = PACKED ? (r.used >> j & 1) : j < n;
    const bool en = PACKED && (r.end >> j & 1);
    if (!us) {
      aa[j] = PACKED ? 0.f : 1.f;          // behind the row the gradient passes
      bs[j] = kw[j] = kf[j] = dy[j] = 0.f;
      if (PACKED) Ga = 0.f;
      continue;
    }
    if (PACKED && (st || en)) {
      if (st) cur = seq_from(a.cu, a.S, cur, t0 + j);
      if (cur < 0) cur = 0;
    }
    const Decay k = decay(to_f(v[0][j]), bias2, nrate, c0);
    // 1 / beta; a q of 0 (a decay that rounds to 1) is lifted so that it stays finite
    const float inv = __builtin_amdgcn_rsqf(fmaxf(k.q, 1e-37f));
    float rest;
    const float xv = to_f(v[2][j]), s = sigmoid2(to_f(v[1][j]), rest), si = s * inv;
    if (st) h = a.h0 ? a.h0[(long long)cur * a.D + dl] : 0.f;
    aa[j] = k.a;
    bs[j] = k.q * si;
    const float u = bs[j] * xv;
    const float ki = fmaf(k.a, h, -(k.a * k.a) * (si * xv));        // dg = lam ki
    kw[j] = u * rest;
    kf[j] = nrate * __builtin_amdgcn_exp2f(k.ls) * ki;
    dy[j] = to_f(v[3][j]);
    if (en && a.dfinal) dy[j] += a.dfinal[(long long)cur * a.D + dl];
    h = fmaf(k.a, h, u);
    Ga = st ? ki * k.g2 : fmaf(k.a, Ga, ki * k.g2);
    sa = fmaf(dy[j], Ga, sa);
    if (open) {
      A *= k.a;
      C = fmaf(A, dy[j], C);
    }
    if (en) open = false;
  }
  constexpr unsigned ALL = (1u << N) - 1;
  if (PACKED && (!open || r.used != ALL)) A = __uint_as_float(RESET);
  float c = join_tiles<PACKED>(s_join, sy, step, strip, W - 1 - wv, A, C, last);
  // what comes from behind a run whose last token is the last of its sequence
  // (or in none) is not for it
  if (PACKED && (n < N || (r.end >> (N - 1) & 1) || !(r.used >> (N - 1) & 1))) c = 0.f;
  sa = fmaf(c, Ga, sa);
  if (live) {
    const long long o = ((long long)b * a.T + t0) * a.D;
    if (PACKED ? !(r.start | r.end) && r.used == ALL : n >= N) {
      E *dx = static_cast<E*>(a.dx) + o + (N - 1LL) * a.D, *df = static_cast<E*>(a.df) + o + (N - 1LL) * a.D;
      E* dw = static_cast<E*>(a.dwz) + o + (N - 1LL) * a.D;
      const unsigned l = here(lane);
#pragma unroll
      for (int j = N - 1; j > 0; j -= 2, dx -= 2LL * a.D, df -= 2LL * a.D, dw -= 2LL * a.D) {
        const float l1 = dy[j] + c, l0 = fmaf(aa[j], l1, dy[j - 1]), f1 = l1 * kf[j], f0 = l0 * kf[j - 1];
        c = aa[j - 1] * l0;
        sb += f1;
        sb += f0;
        store_two(dx, dx - a.D, l, l1 * bs[j], l0 * bs[j - 1]);
        store_two(df, df - a.D, l, f1, f0);
        store_two(dw, dw - a.D, l, l1 * kw[j], l0 * kw[j - 1]);
      }
    } else {
      cur = r.last;
#pragma unroll
      for (int j = N - 1; j >= 0; --j) {
        const bool st = PACKED && (r.start >> j & 1), us = !PACKED || (r.used >> j & 1);
        if (PACKED && (!us || (r.end >> j & 1))) c = 0.f;
        const float lam = dy[j] + c;
        c = aa[j] * lam;
        if (j < n) {
          const long long q = o + (long long)j * a.D + d;
          static_cast<E*>(a.dx)[q] = from_f<E>(lam * bs[j]);
          const float fj = lam * kf[j];
          sb += fj;
          static_cast<E*>(a.df)[q] = from_f<E>(fj);
          static_cast<E*>(a.dwz)[q] = from_f<E>(lam * kw[j]);
          if (PACKED && st && us && a.dh0) {
            cur = seq_before(a.cu, a.S, cur, t0 + j);
            a.dh0[(long long)cur * a.D + d] = c;
          }
        }
      }
    }
    if (!PACKED && t0 == 0 && a.dh0) a.dh0[(long long)b * a.D + d] = c;
  }
  // the tile's sums, its waves' in order
  lds_barrier();
  s_join.wave[wv][lane_id()] = make_float2(sb, sa);
  lds_barrier();
  if (wv == 0 && live) {
    const long long rows = (long long)a.B * sy.nchunk, row = (long long)b * sy.nchunk + chunk;
    sb = sa = 0.f;
    for (int k = 0; k < W; ++k) {
      sb += s_join.wave[k][lane_id()].x;
      sa += s_join.wave[k][lane_id()].y;
    }
    parts[row * a.D + d] = sb;
    parts[(rows + row) * a.D + d] = sa;
  }
}

// Sums over tiles ([2][rows][D]), a slice of them a workgroup row: [2][slices][D].
// 5 us for 256 tiles of 2048 channels, the latency of its reads.
__global__ __launch_bounds__(256) void rec_sum_runs(const float* parts, long long rows, int D, int slices, float* out) {
  __shared__ float s[2][4][64];
  const int d = blockIdx.x * 64 + lane_id(), w = wave_id();
  const long long per = (rows + slices - 1) / slices, r0 = blockIdx.y * per;
  const long long r1 = r0 + per < rows ? r0 + per : rows;
  float b = 0.f, g = 0.f;
  if (d < D) {
#pragma unroll 8
    for (long long r = r0 + w; r < r1; r += 4) {
      b += parts[r * D + d];
      g += parts[(rows + r) * D + d];
    }
  }
  s[0][w][lane_id()] = b;
  s[1][w][lane_id()] = g;
  __syncthreads();
  if (w < 2 && d < D) {
    const int l = lane_id();
    out[((long long)w * slices + blockIdx.y) * D + d] = s[w][0][l] + s[w][1][l] + s[w][2][l] + s[w][3][l];
  }
}

// The last sum over n rows ([2][n][D]), a workgroup a head (several where there are
// more than a grid can have): dt_bias' gradient a channel, A_log's the sum over the
// head's. Four waves have a quarter of the rows of 64 channels each; a wide head has
// up to 16 waves, 256 channels at once (one head of 2048 channels: 4000 tokens, both
// passes, 82 us with 4 waves, 71 with 16).
__global__ __launch_bounds__(1024) void rec_sum_heads(RecArgs a, const float* part, int n) {
  __shared__ float s[2][16][64], s_sum[4];
  const int per = a.D / a.H, l = lane_id(), w = wave_id(), q = w % 4, sets = blockDim.x / (4 * WAVE);
  for (unsigned h = blockIdx.x; h < (unsigned)a.H; h += gridDim.x) {
    float sum = 0.f;
    for (int i0 = 0; i0 < per; i0 += 64 * sets) {
      const int i = i0 + w / 4 * 64 + l;
      const bool live = i < per;
      const int d = (int)h * per + (live ? i : 0);
      float b = 0.f, g = 0.f;
#pragma unroll 8
      for (int k = q; k < n; k += 4) {
        b += part[(long long)k * a.D + d];
        g += part[(long long)(n + k) * a.D + d];
      }
      __syncthreads();
      s[0][w][l] = b;
      s[1][w][l] = g;
      __syncthreads();
      if (q == 0 && live) {
        a.ddt_bias[d] = s[0][w][l] + s[0][w + 1][l] + s[0][w + 2][l] + s[0][w + 3][l];
        sum += s[1][w][l] + s[1][w + 1][l] + s[1][w + 2][l] + s[1][w + 3][l];
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, WAVE);
    if (q == 0 && l == 0) s_sum[w / 4] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int k = 1; k < sets; ++k) sum += s_sum[k];
      a.dA_log[h] = sum * 0.69314718055994531f;     // g2 -> g
    }
  }
}

// ---------------------------------------------------------------- one token

// y = h' = a h + beta s x for B rows of D channels, a channel a thread: 1024
// channels 2.4 us, 256 x 2048 in bf16 4.8 us (8.4 MB, from the cache), both a
// launch's and a read's latency.
template <typename E>
__global__ __launch_bounds__(256) void rec_step_kernel(RecArgs a) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long long)a.B * a.D) return;
  const unsigned b = (unsigned)i / (unsigned)a.D, d = (unsigned)i - b * a.D;      // B D < 2^31
  const float x = to_f(static_cast<const E*>(a.x)[b * a.x_b + d]), f = to_f(static_cast<const E*>(a.f)[b * a.f_b + d]);
  const float w = to_f(static_cast<const E*>(a.wz)[b * a.w_b + d]);
  float bias2, nrate;
  params(a, d, bias2, nrate);
  const Decay k = decay(f, bias2, nrate, FIRST);
  const float h = fmaf(k.a, a.h0[i], __builtin_amdgcn_sqrtf(k.q) * sigmoid2(w) * x);
  a.final_state[i] = h;
  static_cast<E*>(a.y)[i] = from_f<E>(h);
}

// ---------------------------------------------------------------- launches

namespace {

long long up(long long n, long long m) { return (n + m - 1) / m * m; }

// The parts of ws (fp32 units): counters, (A, H) pairs, states at groups, runs of
// packed rows, then the backward's sums over tokens a tile and over slices of them.
struct Space {
  long long agg, base, runs, parts, sums, all, nchunk;
};
Space space(long long B, long long T, long long D, bool backward) {
  const long long wide = B * up(D, 64);
  Space s;
  s.nchunk = (T + W * N - 1) / (W * N);
  const bool many = s.nchunk > 1;
  s.agg = many ? wide / 64 * LINE : 16;
  s.base = s.agg + (many ? 2 * s.nchunk * wide : 0);
  s.runs = s.base + (many ? (s.nchunk / (W * EACH) + 1) * wide : 0);
  s.parts = s.runs + (B == 1 ? 4 * ((T + N - 1) / N) : 0);
  s.sums = s.parts + (backward ? 2 * B * s.nchunk * D : 0);
  s.all = s.sums + (backward ? 2 * REC_SLICES * D : 0);
  return s;
}

Sync prepare(const RecArgs& a, const Space& s, const float* in, float* out, hipStream_t st) {
  Sync y{};
  y.nchunk = (int)s.nchunk;
  y.strips = (a.D + 63) / 64;
  y.nstrip = y.strips * a.B;
  long long n16 = 0;
  if (s.nchunk > 1) {
    y.ticket = reinterpret_cast<int*>(a.ws);
    y.agg = reinterpret_cast<unsigned long long*>(a.ws + s.agg);
    y.base = reinterpret_cast<unsigned*>(a.ws + s.base);
    n16 = (s.runs - s.agg) / 4;
  }
  int4* runs = a.cu ? reinterpret_cast<int4*>(a.ws + s.runs) : nullptr;
  y.runs = runs;
  if (n16 || a.cu) {
    long long n = std::max<long long>(n16, y.nstrip);
    if (a.cu) n = std::max(n, std::max((long long)(a.T + N - 1) / N, out ? (long long)a.S * a.D : 0));
    const unsigned grid = (unsigned)std::min<long long>((n + 255) / 256, 1024);
    hipLaunchKernelGGL(rec_init, dim3(grid), dim3(256), 0, st, a, reinterpret_cast<uint4*>(a.ws + s.agg),
                       n16, y.ticket, y.ticket ? y.nstrip : 0, runs, in, out);
  }
  return y;
}

template <typename E>
hipError_t fwd(const RecArgs& a, hipStream_t st) {
  const Space s = space(a.B, a.T, a.D, false);
  const Sync y = prepare(a, s, a.h0, a.final_state, st);
  const dim3 grid((unsigned)(s.nchunk * y.nstrip));
  if (a.cu) hipLaunchKernelGGL((rec_fwd_kernel<E, true>), grid, dim3(64 * W), 0, st, a, y);
  else hipLaunchKernelGGL((rec_fwd_kernel<E, false>), grid, dim3(64 * W), 0, st, a, y);
  return hipGetLastError();
}

template <typename E>
hipError_t bwd(const RecArgs& a, hipStream_t st) {
  const Space s = space(a.B, a.T, a.D, true);
  const Sync y = prepare(a, s, a.dfinal, a.dh0, st);
  const dim3 grid((unsigned)(s.nchunk * y.nstrip));
  float* parts = a.ws + s.parts;
  if (a.cu) hipLaunchKernelGGL((rec_bwd_kernel<E, true>), grid, dim3(64 * W), 0, st, a, y, parts);
  else hipLaunchKernelGGL((rec_bwd_kernel<E, false>), grid, dim3(64 * W), 0, st, a, y, parts);
  // many tiles: first slices of them, over the whole card
  const long long rows = s.nchunk * a.B;
  const unsigned wide = 4 * WAVE * (unsigned)std::min(4, (a.D / a.H + 63) / 64);
  // a grid has under 2^32 work-items, and a decay for every channel may be 2^24 heads
  const dim3 heads((unsigned)std::min<long long>(a.H, (1LL << 30) / wide));
  if (rows > REC_SLICES) {
    float* sums = a.ws + s.sums;
    hipLaunchKernelGGL(rec_sum_runs, dim3((a.D + 63) / 64, REC_SLICES), dim3(256), 0, st, (const float*)parts,
                       rows, a.D, REC_SLICES, sums);
    hipLaunchKernelGGL(rec_sum_heads, heads, dim3(wide), 0, st, a, (const float*)sums, REC_SLICES);
  } else {
    hipLaunchKernelGGL(rec_sum_heads, heads, dim3(wide), 0, st, a, (const float*)parts, (int)rows);
  }
  return hipGetLastError();
}

}  // namespace

int64_t rec_ws(int64_t B, int64_t T, int64_t D, bool backward) { return space(B, T, D, backward).all; }

hipError_t rec_fwd(const RecArgs& a, int dtype, hipStream_t st) {
  return dtype == NGDN_F32 ? fwd<float>(a, st) : fwd<bf16>(a, st);
}

hipError_t rec_bwd(const RecArgs& a, int dtype, hipStream_t st) {
  return dtype == NGDN_F32 ? bwd<float>(a, st) : bwd<bf16>(a, st);
}

hipError_t rec_step(const RecArgs& a, int dtype, hipStream_t st) {
  const dim3 grid((unsigned)(((long long)a.B * a.D + 255) / 256));
  if (dtype == NGDN_F32) hipLaunchKernelGGL((rec_step_kernel<float>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((rec_step_kernel<bf16>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace ngdn
