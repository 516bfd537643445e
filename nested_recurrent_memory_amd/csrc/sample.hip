// A token a row of logits, from a given random number u in [0, 1): with
// w_i = exp((l_i - max l) / t), the top_k largest; of those, largest first, the
// ones before which less than top_p of their sum lies; of those the ones with
// w_i >= min_p; and of those, in index order, the first with the weights up to
// and with it above u times their sum. Equal logits rank by index. t = 0: the
// first of the largest logits.
//
// Nothing is sorted. What is kept is a run of the order by (logit, index), so it
// is given by its last member: a logit and an index. That one is found by
// histograms, first of max l - l in equal bins over the range in which w is not
// 0, then of the bits of the logits that share the bin in which the count (or
// the weight) is reached, a part of the remaining range at a time. Weights are
// formed in fp64 and summed as integers, in units of 2^-s with s as large as V
// of them allow (2^-46 at 131072): sums have no rounding, so they do not depend
// on the order in which lanes and atomics come, and the same inputs give the
// same token.
//
// A workgroup of 1024 threads has a row.
#include "ngdn_kernels.h"

namespace ngdn {

namespace {

typedef unsigned long long u64;

constexpr int TH = 1024, WV = TH / WAVE, NB = 2048, STEP = TH * 8;

// order of the logits as integers; NaN above all
__device__ __forceinline__ uint32_t key_of(float l) {
  if (l != l) return 0xffffffffu;
  const uint32_t b = __float_as_uint(l + 0.f);      // -0 as 0
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t k) {
  return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}
constexpr uint32_t KEY_INF = 0xff800000u, KEY_NINF = 0x007fffffu;      // of +inf and -inf

template <typename E>
__device__ __forceinline__ void load_logits(const E* row, int i0, int V, float* l) {
  if (i0 + 8 <= V) {
    E t[8];
    __builtin_memcpy(t, row + i0, sizeof t);
#pragma unroll
    for (int e = 0; e < 8; ++e) l[e] = (float)t[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) l[e] = i0 + e < V ? (float)row[i0 + e] : -INFINITY;
  }
}

struct Weigh {
  float max;
  double rate, unit;        // 1 / t, 2^s
  __device__ __forceinline__ u64 operator()(float l) const {
    return (u64)__double2ull_rn(exp(((double)l - (double)max) * rate) * unit);
  }
};

struct Shared {
  u64 weight[NB];
  uint32_t count[NB];
  u64 wave_w[WV];
  uint32_t wave_c[WV];
  // what a search found: the bin, and what lies before it
  int bin;
  u64 before_w, in_w;
  uint32_t before_c, in_c;
  uint32_t lo, hi;
  u64 best;
};

template <typename T>
__device__ __forceinline__ T scan_wave(T v) {        // inclusive
#pragma unroll
  for (int o = 1; o < WAVE; o <<= 1) {
    const T t = __shfl_up(v, o, WAVE);
    if (lane_id() >= o) v += t;
  }
  return v;
}

// this thread's exclusive sum over the workgroup, and the whole sum
__device__ __forceinline__ void scan_block(Shared& s, uint32_t c, u64 w, uint32_t& c0, u64& w0, uint32_t& ct, u64& wt) {
  const uint32_t ci = scan_wave(c);
  const u64 wi = scan_wave(w);
  __syncthreads();
  if (lane_id() == WAVE - 1) { s.wave_c[wave_id()] = ci; s.wave_w[wave_id()] = wi; }
  __syncthreads();
  c0 = ci - c; w0 = wi - w; ct = 0; wt = 0;
#pragma unroll
  for (int i = 0; i < WV; ++i) {
    const uint32_t a = s.wave_c[i];
    const u64 b = s.wave_w[i];
    if (i < wave_id()) { c0 += a; w0 += b; }
    ct += a; wt += b;
  }
}

__device__ __forceinline__ void clear_bins(Shared& s) {
  __syncthreads();
  for (int i = threadIdx.x; i < NB; i += TH) { s.weight[i] = 0; s.count[i] = 0; }
  __syncthreads();
}

// the first bin with which the count (by_weight: the weight) reaches target >= 1,
// which lies within the bins' whole; base_c and base_w lie before bin 0
__device__ __forceinline__ void find_bin(Shared& s, bool by_weight, u64 target, uint32_t base_c, u64 base_w) {
  __syncthreads();
  const int i = threadIdx.x * 2;
  const uint32_t ca = s.count[i], cb = s.count[i + 1];
  const u64 wa = s.weight[i], wb = s.weight[i + 1];
  uint32_t c, ct;
  u64 w, wt;
  scan_block(s, ca + cb, wa + wb, c, w, ct, wt);
  c += base_c; w += base_w;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t cj = j ? cb : ca;
    const u64 wj = j ? wb : wa;
    const u64 from = by_weight ? w : c, to = by_weight ? w + wj : (u64)(c + cj);
    if (from < target && to >= target) {
      s.bin = i + j; s.before_c = c; s.before_w = w; s.in_c = cj; s.in_w = wj;
    }
    c += cj; w += wj;
  }
  __syncthreads();
}

struct Cut {
  uint32_t key;              // the last logit that is kept
  uint32_t ties, kept;       // how many have it, and how many of them are kept
  u64 sum;                   // the weight of all that is kept
};

// the first f(i) > target in index order: f summed over segments (a step's
// elements of one wave), the segment's elements by its wave
template <typename E, typename F>
__device__ __forceinline__ int select_index(Shared& s, const E* row, int V, F f, u64 (*target_of)(u64, double), double arg) {
  const int steps = (V + STEP - 1) / STEP;
  __syncthreads();
  for (int i = threadIdx.x; i < NB; i += TH) s.weight[i] = 0;
  __syncthreads();
  for (int k = 0; k < steps; ++k) {
    const int i0 = k * STEP + threadIdx.x * 8;
    float l[8];
    load_logits(row, i0, V, l);
    u64 sum = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += f(i0 + e, l[e]);
#pragma unroll
    for (int o = WAVE / 2; o > 0; o >>= 1) sum += __shfl_xor(sum, o, WAVE);
    if (lane_id() == 0) s.weight[k * WV + wave_id()] = sum;
  }
  __syncthreads();
  const int j = threadIdx.x * 2;
  const u64 a = s.weight[j], b = s.weight[j + 1];
  uint32_t c, ct;
  u64 w, wt;
  scan_block(s, 0, a + b, c, w, ct, wt);
  const u64 target = target_of(wt, arg);
  if (w <= target && w + a > target) { s.bin = j; s.before_w = w; }
  else if (w + a <= target && w + a + b > target) { s.bin = j + 1; s.before_w = w + a; }
  __syncthreads();
  const int seg = s.bin;
  if (wave_id() == seg % WV) {
    const int i0 = seg / WV * STEP + threadIdx.x * 8;
    float l[8];
    u64 v[8], sum = 0;
    load_logits(row, i0, V, l);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += v[e] = f(i0 + e, l[e]);
    u64 at = s.before_w + scan_wave(sum) - sum;
    if (at <= target && at + sum > target) {
      int found = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (at <= target && at + v[e] > target) found = i0 + e;
        at += v[e];
      }
      s.lo = (uint32_t)found;
    }
  }
  __syncthreads();
  return (int)s.lo;
}

__device__ u64 as_given(u64, double target) { return (u64)target; }
__device__ u64 share_of(u64 whole, double u) {
  const double t = u * (double)whole;
  return t < (double)whole ? (u64)t < whole ? (u64)t : whole - 1 : whole - 1;
}

}  // namespace

template <typename E>
__global__ __launch_bounds__(TH) void sample_kernel(SampleArgs a, double unit, float range) {
  __shared__ Shared s;
  const long long r = blockIdx.x;
  const int V = a.V, steps = (V + STEP - 1) / STEP;
  const E* row = static_cast<const E*>(a.logits) + r * a.stride;
  const float t = a.temperature_ptr ? a.temperature_ptr[r] : a.temperature;
  const float top_p = a.top_p_ptr ? a.top_p_ptr[r] : a.top_p;
  const float min_p = a.min_p_ptr ? a.min_p_ptr[r] : a.min_p;
  const long long k = a.top_k_ptr ? (a.top_k_wide ? static_cast<const long long*>(a.top_k_ptr)[r]
                                                  : static_cast<const int*>(a.top_k_ptr)[r])
                                  : a.top_k;
  const double u = a.u_wide ? static_cast<const double*>(a.u)[r] : (double)static_cast<const float*>(a.u)[r];

  // the largest logit and its first place
  if (threadIdx.x == 0) s.best = 0;
  __syncthreads();
  u64 best = 0;
  for (int j = 0; j < steps; ++j) {
    const int i0 = j * STEP + threadIdx.x * 8;
    float l[8];
    load_logits(row, i0, V, l);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const u64 v = (u64)key_of(l[e]) << 32 | (uint32_t)~(i0 + e);
      best = v > best ? v : best;
    }
  }
#pragma unroll
  for (int o = WAVE / 2; o > 0; o >>= 1) {
    const u64 v = __shfl_xor(best, o, WAVE);
    best = v > best ? v : best;
  }
  if (lane_id() == 0) atomicMax(&s.best, best);
  __syncthreads();
  best = s.best;
  const uint32_t top = (uint32_t)(best >> 32);
  const bool fits = top > KEY_NINF && top < KEY_INF && t >= 0.f && t < INFINITY && top_p >= 0.f && min_p >= 0.f &&
                    min_p <= 1.f && u >= 0. && u <= 1.;
  if (!fits || t == 0.f) {
    if (threadIdx.x == 0) a.token[r] = fits ? (long long)(uint32_t)~best : -1;
    return;
  }
  const Weigh weigh{logit_of(top), 1. / (double)t, unit};

  // what top_k and top_p keep
  Cut cut{0, 0, 0, 0};
  if (k >= 1 && k < V || top_p < 1.f) {
    const float scale = fminf(fmaxf((float)NB / (range * t), 1e-30f), 1e30f);
    auto bin_of = [&](float l) { return (int)fminf((weigh.max - l) * scale, (float)(NB - 1)); };
    clear_bins(s);
    for (int j = 0; j < steps; ++j) {
      float l[8];
      load_logits(row, j * STEP + threadIdx.x * 8, V, l);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const u64 w = weigh(l[e]);
        if (w) {
          const int b = bin_of(l[e]);
          atomicAdd(&s.count[b], 1u);
          atomicAdd(&s.weight[b], w);
        }
      }
    }
    __syncthreads();
    uint32_t c, live;
    u64 w, whole;
    {
      const int i = threadIdx.x * 2;
      scan_block(s, s.count[i] + s.count[i + 1], s.weight[i] + s.weight[i + 1], c, w, live, whole);
    }
    // the last that is kept when target of the count (or the weight) is to be reached
    auto search = [&](bool by_weight, u64 target) {
      find_bin(s, by_weight, target, 0, 0);
      const int bin = s.bin;
      uint32_t before_c = s.before_c;
      u64 before_w = s.before_w;
      // the range of the logits in this bin
      if (threadIdx.x == 0) { s.lo = 0xffffffffu; s.hi = 0; }
      __syncthreads();
      uint32_t lo = 0xffffffffu, hi = 0;
      for (int j = 0; j < steps; ++j) {
        float l[8];
        load_logits(row, j * STEP + threadIdx.x * 8, V, l);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (bin_of(l[e]) == bin && weigh(l[e])) {
            const uint32_t key = key_of(l[e]);
            lo = key < lo ? key : lo;
            hi = key > hi ? key : hi;
          }
        }
      }
      atomicMin(&s.lo, lo);
      atomicMax(&s.hi, hi);
      __syncthreads();
      lo = s.lo; hi = s.hi;
      for (;;) {
        const uint32_t width = hi - lo;
        const int bits = width ? 32 - __clz(width) : 0, shift = bits > 11 ? bits - 11 : 0;
        clear_bins(s);
        for (int j = 0; j < steps; ++j) {
          float l[8];
          load_logits(row, j * STEP + threadIdx.x * 8, V, l);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t key = key_of(l[e]);
            if (key >= lo && key <= hi) {
              atomicAdd(&s.count[(hi - key) >> shift], 1u);
              atomicAdd(&s.weight[(hi - key) >> shift], weigh(l[e]));
            }
          }
        }
        find_bin(s, by_weight, target, before_c, before_w);
        const uint32_t b = (uint32_t)s.bin;
        const uint32_t in_c = s.in_c;
        const u64 in_w = s.in_w;
        before_c = s.before_c; before_w = s.before_w;
        hi -= b << shift;
        if (shift == 0) {
          Cut x;
          const u64 each = in_w / in_c;            // equal logits have equal weights
          x.key = hi; x.ties = in_c;
          x.kept = by_weight ? (uint32_t)((target - before_w + each - 1) / each) : (uint32_t)(target - before_c);
          x.sum = before_w + x.kept * each;
          return x;
        }
        const uint32_t span = (1u << shift) - 1;
        lo = hi - lo > span ? hi - span : lo;
      }
    };
    if (k >= 1 && (u64)k < live) {
      cut = search(false, (u64)k);
      whole = cut.sum;
    }
    if (top_p < 1.f) {
      // the first is kept whatever its share
      const double want = ceil((double)top_p * (double)whole);
      if (cut.key) {                               // the bins of the whole row again
        clear_bins(s);
        for (int j = 0; j < steps; ++j) {
          float l[8];
          load_logits(row, j * STEP + threadIdx.x * 8, V, l);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const u64 w = weigh(l[e]);
            if (w) {
              const int b = bin_of(l[e]);
              atomicAdd(&s.count[b], 1u);
              atomicAdd(&s.weight[b], w);
            }
          }
        }
      }
      const u64 target = want < 1. ? 1 : want < (double)whole ? (u64)want : whole;
      cut = search(true, target);
    }
  }
  int last = V;                                     // equal ones up to here are kept
  if (cut.kept < cut.ties) {
    const uint32_t key = cut.key;
    last = select_index(s, row, V, [&](int, float l) -> u64 { return key_of(l) == key; }, as_given, (double)(cut.kept - 1));
  }
  const double floor = (double)min_p * unit;
  const int token = select_index(s, row, V, [&](int i, float l) -> u64 {
    const uint32_t key = key_of(l);
    if (key < cut.key || (key == cut.key && i > last)) return 0;
    const u64 w = weigh(l);
    return (double)w >= floor ? w : 0;
  }, share_of, u);
  if (threadIdx.x == 0) a.token[r] = token;
}

hipError_t sample(const SampleArgs& a, int dtype, hipStream_t st) {
  if (a.rows == 0) return hipSuccess;
  int bits = 0;
  while ((1LL << bits) < a.V) ++bits;
  const int s = 62 - bits;                          // V weights of at most 2^s stay below 2^63
  const double unit = (double)(1ULL << s);
  // w is 0 from exp(-x) 2^s < 1/2: x > (s + 1) ln 2; the bins reach a little further
  const float range = (float)((s + 2) * 0.6931471805599453);
  if (dtype == NGDN_BF16) hipLaunchKernelGGL(sample_kernel<bf16>, dim3((unsigned)a.rows), dim3(TH), 0, st, a, unit, range);
  else hipLaunchKernelGGL(sample_kernel<float>, dim3((unsigned)a.rows), dim3(TH), 0, st, a, unit, range);
  return hipGetLastError();
}

}  // namespace ngdn
