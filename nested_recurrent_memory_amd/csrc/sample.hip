// A token a row of logits, from a given random number u in [0, 1): with
// w_i = exp((l_i - max l) / t), the top_k largest; of those, largest first, the
// ones before which less than top_p of their sum lies; of those the ones with
// w_i >= min_p; and of those, in index order, the first with the weights up to
// and with it above u times their sum. Equal logits rank by index. t = 0: the
// first of the largest logits.
//
// Nothing is sorted. What is kept is a run of the order by (logit, index), so it is
// given by its last member. Weights are formed in fp64 and summed as integers, in
// units of 2^-s with s as large as V of them allow (2^-45 at 131072): the sums have no
// rounding, so they do not depend on the order in which lanes and atomics come, and
// the same inputs give the same token. Forming a weight rounds it, by half a unit at
// most: sums are off by V 2^-(s+1) at most, and what weighs less than half a unit of
// the largest is never drawn.
//
// A workgroup of 1024 threads has a row, each wave a run of it. What bounds it is the one
// CU that a row has: 256 rows of 131072 fp32, top_k 50 and top_p 0.95, 38 us, of which 26 to
// 29 read the 134 MB (4.6 to 5.2 TB/s) and the rest are latencies; a row of 32000 bf16 with
// top_p 0.9 19 us: 2.6 to read, 8 the weights by bins (5.7 of them fp64 arithmetic), 3 to
// find the bin, 4 for the candidates.
//
// The row is read once for its maximum, and the largest value of each lane's groups of
// columns is kept: a later pass looks only into groups that can hold what it looks for.
//  * top_k: below the k-th largest of the lanes' maxima none of the top_k lies. What
//    reaches it (or its bin, see below), a few more than k, is listed.
//  * top_p without it: the weights of the row in 2048 equal bins of max l - l. What is
//    in the bin in which top_p is reached, or above, is listed. min_p: what reaches it.
//  * In a list of at most LIST each member counts what is above it and sums its weights,
//    and then what is kept before it in index order.
// Where more than that is kept, the last member is found in the bin alone, by its list
// or, if that is too long too (many equal or close logits), by bins of the logits' bits,
// a part of the remaining range at a time, and the token by the sums of kept weights
// over segments of the row.
#include "ngdn_kernels.h"

namespace ngdn {

namespace {

typedef unsigned long long u64;

constexpr int TH = 1024, WV = TH / WAVE, NB = 2048, RUN = WAVE * 8, GROUPS = 8;
// Members of a list, and runs of eight columns that are looked into for it. A row of 32000
// with 500 kept takes 32 us with lists of 256, 38 of 512 and 58 of 1024 (the count is of
// their square), one of 131072 with top_p 0.95 no less; of 1000 with hundreds kept 16 and 28
constexpr int LIST = 256, PARTS = 1024;

// order of the logits as integers
__device__ __forceinline__ uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l + 0.f);      // -0 as 0
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t k) {
  return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}
// order by logit, then the lower index first
__device__ __forceinline__ u64 place_of(float l, int i) { return (u64)key_of(l) << 32 | (uint32_t)~i; }

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

// exp((l - max) / t) in units of 2^-s, to the nearest: 2^(y / 64) with y = 64 (l - max)
// log2(e) / t as 2^n times a 64th power from a table (which holds 2^(j / 64 + s)) times a
// polynomial of the rest, |r| <= 1/2 (the exponential series to r^5: relative error below
// 2^-54). 13 fp64 operations; the library's exp takes three times as many.
struct Weigh {
  double max, rate, least;        // 64 log2(e) / t; least: below it the weight is 0
  const double* table;
  __device__ __forceinline__ u64 operator()(float l) const {
    const double y = fmax(((double)l - max) * rate, least);
    const double m = y + 0x1.8p52;                                  // to the nearest integer
    const uint32_t k = (uint32_t)__double_as_longlong(m);
    const double r = y - (m - 0x1.8p52);
    constexpr double C = 0.69314718055994530942 / 64;
    double p = fma(r, C * C * C * C * C / 120, C * C * C * C / 24);
    p = fma(r, p, C * C * C / 6);
    p = fma(r, p, C * C / 2);
    p = fma(r, p, C);
    p = fma(r, p, 1.);
    const double power = table[k & 63];                             // times 2^(k >> 6)
    const double scaled = __hiloint2double(__double2hiint(power) + (int)((k & ~63u) << 14), __double2loint(power));
    const double w = fma(p, scaled, 0x1p52);                        // below 2^52: its integer
    return (u64)__double_as_longlong(w) & 0xfffffffffffffull;
  }
};

struct Shared {
  u64 weight[NB];
  uint32_t count[NB];
  float most[GROUPS][TH];         // a lane's largest logit of a group of its columns
  // a list: places, weights, and what a count over it found for each
  u64 place[LIST], amount[LIST], before[LIST];
  uint32_t rank[LIST];
  uint32_t part[PARTS];           // runs of eight columns to look into
  double table[64];
  u64 wave_w[WV];
  uint32_t wave_c[WV];
  // what a search found: the bin, and what lies before it
  int bin;
  u64 before_w, in_w;
  uint32_t before_c, in_c;
  uint32_t lo, hi, listed, parts;
  u64 sum, best;
  int bad, token;
};

// what a row's passes go by
template <typename E>
struct Row {
  const E* p;
  int V, iters, each;             // runs of 512 columns a wave, and in a group of them
  __device__ __forceinline__ int at(int it) const { return (wave_id() * iters + it) * RUN + lane_id() * 8; }
};

// f of this lane's columns in the groups whose largest logit want() takes, the next run's
// loads ahead of this one's use
template <typename E, typename W, typename F>
__device__ __forceinline__ void visit(const Shared& s, const Row<E>& row, W want, F f) {
  float next[8];
  load_logits(row.p, row.at(0), row.V, next);
  for (int it = 0; it < row.iters; ++it) {
    float l[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) l[e] = next[e];
    if (it + 1 < row.iters) load_logits(row.p, row.at(it + 1), row.V, next);
    if (!want(s.most[it / row.each][threadIdx.x])) continue;
    const int i0 = row.at(it);
#pragma unroll
    for (int e = 0; e < 8; ++e) f(l[e], i0 + e);
  }
}

// n = the counter's value for the first of the lanes that are here, and one more for each
__device__ __forceinline__ uint32_t take(uint32_t* counter) {
  const u64 here = __ballot(1);
  const int first = __ffsll((long long)here) - 1;
  uint32_t n = 0;
  if (lane_id() == first) n = atomicAdd(counter, (uint32_t)__popcll(here));
  return __shfl(n, first, WAVE) + (uint32_t)__popcll(here & ((1ull << lane_id()) - 1));
}

// Lists the places of the logits that pred() takes, which it does of none in a group whose
// largest want() does not take; false if there are more than LIST. First the runs of eight
// to look into, then their logits, one a thread: one load's latency in all. With too
// many runs every column, if sweep is set. Ends behind a barrier
template <typename E, typename W, typename P>
__device__ __forceinline__ bool gather(Shared& s, const Row<E>& row, bool sweep, W want, P pred) {
  __syncthreads();
  if (threadIdx.x == 0) { s.listed = 0; s.parts = 0; }
  __syncthreads();
  for (int g = 0; g * row.each < row.iters; ++g) {
    if (!want(s.most[g][threadIdx.x])) continue;
    const int end = (g + 1) * row.each < row.iters ? (g + 1) * row.each : row.iters;
    for (int it = g * row.each; it < end; ++it) {
      const uint32_t n = take(&s.parts);
      if (n < PARTS) s.part[n] = (uint32_t)row.at(it);
    }
  }
  __syncthreads();
  const int parts = (int)s.parts;
  auto add = [&](float l, int i) {
    if (pred(l)) {
      const uint32_t n = take(&s.listed);
      if (n < LIST) s.place[n] = place_of(l, i);
    }
  };
  if (parts <= PARTS) {
    for (int j = threadIdx.x; j < parts * 8; j += TH) {
      const int i = (int)s.part[j / 8] + j % 8;
      if (i < row.V) add((float)row.p[i], i);
    }
  } else {
    if (!sweep) return false;
    visit(s, row, [&](float m) { return want(m) && *(volatile uint32_t*)&s.listed <= LIST; }, add);
  }
  __syncthreads();
  return s.listed <= LIST;
}

template <typename T>
__device__ __forceinline__ T scan_wave(T v) {        // inclusive
#pragma unroll
  for (int o = 1; o < WAVE; o <<= 1) {
    const T t = __shfl_up(v, o, WAVE);
    if (lane_id() >= o) v += t;
  }
  return v;
}
__device__ __forceinline__ u64 wave_total(u64 v) {
#pragma unroll
  for (int o = WAVE / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, WAVE);
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

// the first bin with which the count (by_weight: the weight) reaches target_of(the bins'
// whole), 1 at least; none where the whole does not reach it. base_c and base_w lie before
// bin 0. Gives the whole
struct Whole { uint32_t count; u64 weight; };
template <typename T>
__device__ __forceinline__ Whole find_bin(Shared& s, bool by_weight, T target_of, uint32_t base_c, u64 base_w) {
  __syncthreads();
  const int i = threadIdx.x * 2;
  const uint32_t ca = s.count[i], cb = s.count[i + 1];
  const u64 wa = s.weight[i], wb = s.weight[i + 1];
  uint32_t c;
  u64 w;
  Whole all;
  scan_block(s, ca + cb, wa + wb, c, w, all.count, all.weight);
  c += base_c; w += base_w;
  const u64 target = target_of(all);
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
  return all;
}

// the first index with f(l, i) summed up to and with it above target(whole sum): sums over
// segments (a wave's group of columns), then along the one that holds it
template <typename E, typename W, typename F, typename T>
__device__ __forceinline__ int select_index(Shared& s, const Row<E>& row, W want, F f, T target_of) {
  __syncthreads();
  if (threadIdx.x < 2 * WAVE) s.weight[threadIdx.x] = 0;
  __syncthreads();
  {
    float next[8];
    u64 sum = 0;
    load_logits(row.p, row.at(0), row.V, next);
    for (int it = 0; it < row.iters; ++it) {
      float l[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) l[e] = next[e];
      if (it + 1 < row.iters) load_logits(row.p, row.at(it + 1), row.V, next);
      const int g = it / row.each, i0 = row.at(it);
      if (want(s.most[g][threadIdx.x])) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sum += f(l[e], i0 + e);
      }
      if ((it + 1) % row.each == 0 || it + 1 == row.iters) {
        sum = wave_total(sum);
        if (lane_id() == 0) s.weight[wave_id() * GROUPS + g] = sum;
        sum = 0;
      }
    }
  }
  __syncthreads();
  // 128 segments: two a lane of every wave, which so all know the sum
  const u64 a = s.weight[lane_id() * 2], b = s.weight[lane_id() * 2 + 1];
  u64 before = scan_wave(a + b);
  const u64 target = target_of(__shfl(before, WAVE - 1, WAVE));
  before -= a + b;
  const bool in_a = before <= target && before + a > target;
  const bool in_b = before + a <= target && before + a + b > target;
  const u64 hit = __ballot(in_a || in_b);
  const int lane = __ffsll((long long)hit) - 1;
  const int seg = __shfl(lane_id() * 2 + (in_b ? 1 : 0), lane, WAVE);
  u64 from = __shfl(in_b ? before + a : before, lane, WAVE);
  if (wave_id() == seg / GROUPS) {
    const int g = seg % GROUPS, end = (g + 1) * row.each < row.iters ? (g + 1) * row.each : row.iters;
    for (int it = g * row.each; it < end; ++it) {
      float l[8];
      u64 v[8], sum = 0;
      const int i0 = row.at(it);
      load_logits(row.p, i0, row.V, l);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += v[e] = f(l[e], i0 + e);
      const u64 upto = from + scan_wave(sum);
      u64 at = upto - sum;
      if (at <= target && upto > target) {
        int found = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (at <= target && at + v[e] > target) found = i0 + e;
          at += v[e];
        }
        s.token = found;
      }
      from = __shfl(upto, WAVE - 1, WAVE);
      if (from > target) break;
    }
  }
  __syncthreads();
  return s.token;
}

__device__ __forceinline__ u64 share_of(u64 whole, double u) {
  const double t = u * (double)whole;
  return t < (double)whole ? (u64)t < whole ? (u64)t : whole - 1 : whole - 1;
}
// the smallest integer weight with which top_p of whole is reached, the first's at least
__device__ __forceinline__ u64 part_of(u64 whole, float top_p) {
  const double want = ceil((double)top_p * (double)whole);
  return want < 1. ? 1 : want < (double)whole ? (u64)want : whole;
}

// the sum over the workgroup, by one atomic a wave
__device__ __forceinline__ u64 block_total(Shared& s, u64 v) {
  __syncthreads();
  if (threadIdx.x == 0) s.sum = 0;
  __syncthreads();
  v = wave_total(v);
  if (lane_id() == 0 && v) atomicAdd(&s.sum, v);
  __syncthreads();
  return s.sum;
}

// for each member of the list its rank, and in before the amounts of those that come first:
// above it, or (BY_INDEX, without the rank) at a lower index. A wave has a part of the list
// to count, a lane every 64th member to count for. Ends behind a barrier
template <bool BY_INDEX>
__device__ __forceinline__ void count_before(Shared& s, int n) {
  if ((int)threadIdx.x < n) { s.before[threadIdx.x] = 0; s.rank[threadIdx.x] = 0; }
  __syncthreads();
  constexpr int EACH = LIST / WAVE;
  const int len = (n + WV - 1) / WV, j0 = wave_id() * len, j1 = j0 + len < n ? j0 + len : n;
  u64 me[EACH], sum[EACH];
  uint32_t rank[EACH];
#pragma unroll
  for (int q = 0; q < EACH; ++q) {
    const int i = q * WAVE + lane_id();
    me[q] = s.place[i < n ? i : 0]; sum[q] = 0; rank[q] = 0;
  }
#pragma unroll 4
  for (int j = j0; j < j1; ++j) {
    const u64 p = s.place[j], w = s.amount[j];
#pragma unroll
    for (int q = 0; q < EACH; ++q) {
      const bool first = BY_INDEX ? (uint32_t)p > (uint32_t)me[q] : p > me[q];
      sum[q] += first ? w : 0;
      rank[q] += first ? 1 : 0;
    }
  }
#pragma unroll
  for (int q = 0; q < EACH; ++q) {
    const int i = q * WAVE + lane_id();
    if (i < n && rank[q]) {
      atomicAdd(&s.before[i], sum[q]);
      if (!BY_INDEX) atomicAdd(&s.rank[i], rank[q]);
    }
  }
  __syncthreads();
}

}  // namespace

template <typename E>
__global__ __launch_bounds__(TH) void sample_kernel(SampleArgs a, int s_bits, float range) {
  __shared__ Shared s;
  const long long r = blockIdx.x;
  Row<E> row;
  row.p = static_cast<const E*>(a.logits) + r * a.stride;
  row.V = a.V;
  row.iters = (a.V + WV * RUN - 1) / (WV * RUN);
  row.each = (row.iters + GROUPS - 1) / GROUPS;
  const float t = a.temperature_ptr ? a.temperature_ptr[r] : a.temperature;
  const float top_p = a.top_p_ptr ? a.top_p_ptr[r] : a.top_p;
  const float min_p = a.min_p_ptr ? a.min_p_ptr[r] : a.min_p;
  const long long k = a.top_k_ptr ? (a.top_k_wide ? static_cast<const long long*>(a.top_k_ptr)[r]
                                                  : static_cast<const int*>(a.top_k_ptr)[r])
                                  : a.top_k;
  const double u = a.u_wide ? static_cast<const double*>(a.u)[r] : (double)static_cast<const float*>(a.u)[r];
  if (threadIdx.x == 0) { s.best = 0; s.bad = 0; }
  if (threadIdx.x < 64) s.table[threadIdx.x] = exp2(threadIdx.x * 0x1p-6 + (double)s_bits);
  __syncthreads();

  // the largest logit, of each lane's groups too
  float mine = -INFINITY;
  bool bad = false;
  for (int g = 0; g * row.each < row.iters; ++g) {
    const int end = (g + 1) * row.each < row.iters ? (g + 1) * row.each : row.iters;
    float most = -INFINITY;
#pragma unroll 4
    for (int it = g * row.each; it < end; ++it) {
      float l[8];
      load_logits(row.p, row.at(it), row.V, l);
#pragma unroll
      for (int e = 0; e < 8; ++e) { most = fmaxf(most, l[e]); bad |= l[e] != l[e]; }
    }
    s.most[g][threadIdx.x] = most;
    mine = fmaxf(mine, most);
  }
  float top = mine;
#pragma unroll
  for (int o = WAVE / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, WAVE));
  if (lane_id() == 0) atomicMax(&s.best, (u64)key_of(top));
  if (__any(bad) && lane_id() == 0) s.bad = 1;
  __syncthreads();
  top = logit_of((uint32_t)s.best);
  const bool fits = !s.bad && top > -INFINITY && top < INFINITY && t >= 0.f && t < INFINITY && top_p >= 0.f &&
                    top_p <= 1.f && min_p >= 0.f && min_p <= 1.f && u >= 0. && u <= 1.;
  if (!fits) {
    if (threadIdx.x == 0) a.token[r] = -1;
    return;
  }
  if (t == 0.f) {                                   // the first of the largest
    if (threadIdx.x == 0) s.lo = 0xffffffffu;
    auto is_top = [&](float l) { return l == top; };
    if (gather(s, row, false, is_top, is_top)) {
      if (threadIdx.x < s.listed) atomicMin(&s.lo, ~(uint32_t)s.place[threadIdx.x]);
    } else {
      __syncthreads();
      uint32_t first = 0xffffffffu;
      visit(s, row, is_top, [&](float l, int i) {
        if (l == top && (uint32_t)i < first) first = (uint32_t)i;
      });
      atomicMin(&s.lo, first);
    }
    __syncthreads();
    if (threadIdx.x == 0) a.token[r] = s.lo;
    return;
  }
  const Weigh weigh{(double)top, 64 * 1.4426950408889634074 / (double)t, -64. * (s_bits + 3), s.table};
  const u64 floor = (u64)ceil((double)min_p * (double)(1ull << s_bits));
  const float scale = fminf(fmaxf((float)NB / (range * t), 1e-30f), 1e30f);
  auto bin_of = [&](float l) { return (int)fminf((top - l) * scale, (float)(NB - 1)); };
  auto every = [](float) { return true; };

  // the token from a list with all that is kept: below limit by rank, below top_p of the
  // whole (0: of what limit leaves) by weight
  auto weigh_list = [&](int n) {
    if ((int)threadIdx.x < n) s.amount[threadIdx.x] = weigh(logit_of((uint32_t)(s.place[threadIdx.x] >> 32)));
    __syncthreads();
  };
  auto from_list = [&](long long limit, u64 whole) {
    const int n = (int)s.listed;
    const bool in = (int)threadIdx.x < n;
    weigh_list(n);
    count_before<false>(s, n);
    u64 w = in ? s.amount[threadIdx.x] : 0;
    const u64 before = in ? s.before[threadIdx.x] : 0;
    const bool ranked = in && s.rank[threadIdx.x] < limit;
    if (top_p < 1.f && whole == 0) whole = block_total(s, ranked ? w : 0);
    if (!ranked || w < floor || (top_p < 1.f && before >= part_of(whole, top_p))) w = 0;
    const u64 target = share_of(block_total(s, w), u);
    if (in) s.amount[threadIdx.x] = w;
    __syncthreads();
    count_before<true>(s, n);
    if (w && s.before[threadIdx.x] <= target && s.before[threadIdx.x] + w > target)
      a.token[r] = (long long)(uint32_t)~(uint32_t)s.place[threadIdx.x];
  };

  const bool some = k >= 1 && k < a.V;
  if (some && k <= LIST) {
    // the bin that the k-th largest of the lanes' maxima is in: at least k logits are in it
    // or above
    clear_bins(s);
    if (mine > -INFINITY) atomicAdd(&s.count[bin_of(mine)], 1u);
    if (threadIdx.x == 0) s.bin = NB - 1;           // fewer than k lanes have one
    find_bin(s, false, [&](Whole) { return (u64)k; }, 0, 0);
    const int bin = s.bin;
    auto there = [&](float l) { return l > -INFINITY && bin_of(l) <= bin; };
    if (gather(s, row, false, there, there)) {
      from_list(k, 0);
      return;
    }
  }

  // the weights of the row by bins
  auto histogram = [&]() {
    clear_bins(s);
    visit(s, row, every, [&](float l, int) {
      const u64 w = weigh(l);
      if (w) {
        const int b = bin_of(l);
        if (some) atomicAdd(&s.count[b], 1u);
        atomicAdd(&s.weight[b], w);
      }
    });
    __syncthreads();
  };
  u64 cut = 0;                                      // the place of the last that is kept
  if (some || top_p < 1.f) {
    histogram();
    // the bin in which top_k ends, or without it top_p
    const Whole all = find_bin(s, !some, [&](Whole v) { return some ? (u64)k : part_of(v.weight, top_p); }, 0, 0);
    u64 whole = all.weight;
    bool spoilt = false;
    // the last that is kept when target of the count (or the weight) is to be reached, and
    // in sum the weight up to it; found: its bin is known
    auto search = [&](bool by_weight, u64 target, bool found, u64& sum) -> u64 {
      if (!found) find_bin(s, by_weight, [&](Whole) { return target; }, 0, 0);
      const int bin = s.bin;
      uint32_t before_c = s.before_c;
      u64 before_w = s.before_w;
      if (gather(s, row, true, [&](float m) { return m > -INFINITY && bin_of(m) <= bin; },
                 [&](float l) { return l > -INFINITY && bin_of(l) == bin; })) {
        const int n = (int)s.listed;
        weigh_list(n);
        count_before<false>(s, n);
        if ((int)threadIdx.x < n) {
          const u64 w = s.amount[threadIdx.x], upto = before_w + s.before[threadIdx.x];
          const u64 from = by_weight ? upto : before_c + s.rank[threadIdx.x];
          if (from < target && from + (by_weight ? w : 1) >= target) {
            s.best = s.place[threadIdx.x];
            s.sum = upto + w;
          }
        }
        __syncthreads();
        sum = s.sum;
        return s.best;
      }
      spoilt = true;
      // the range of the logits in this bin; near the last bins some of them weigh nothing
      const bool live_bin = bin < NB - 2 * NB / (s_bits + 2);
      if (threadIdx.x == 0) { s.lo = 0xffffffffu; s.hi = 0; }
      __syncthreads();
      uint32_t lo = 0xffffffffu, hi = 0;
      visit(s, row, [&](float m) { return bin_of(m) <= bin; }, [&](float l, int) {
        if (bin_of(l) == bin && (live_bin || weigh(l))) {
          const uint32_t key = key_of(l);
          lo = key < lo ? key : lo;
          hi = key > hi ? key : hi;
        }
      });
      atomicMin(&s.lo, lo);
      atomicMax(&s.hi, hi);
      __syncthreads();
      lo = s.lo; hi = s.hi;
      // a bf16's key is its upper half: the lower is 0, or all ones below zero
      constexpr int LOW = sizeof(E) == 2 ? 16 : 0;
      auto value_of = [](uint32_t k) { return logit_of(LOW ? k << LOW | (k >> 15 ? 0u : 0xffffu) : k); };
      lo >>= LOW;
      hi >>= LOW;
      for (;;) {
        const uint32_t width = hi - lo;
        const int bits = width ? 32 - __clz(width) : 0, shift = bits > 11 ? bits - 11 : 0;
        const bool single = shift == 0;                // a bin for each value: counts are enough
        const float least = value_of(lo);
        clear_bins(s);
        visit(s, row, [&](float m) { return m >= least; }, [&](float l, int) {
          const uint32_t key = key_of(l) >> LOW;
          if (key >= lo && key <= hi) {
            atomicAdd(&s.count[(hi - key) >> shift], 1u);
            if (!single) atomicAdd(&s.weight[(hi - key) >> shift], weigh(l));
          }
        });
        __syncthreads();
        if (single)
          for (uint32_t i = threadIdx.x; i <= width; i += TH) s.weight[i] = s.count[i] * weigh(value_of(hi - i));
        find_bin(s, by_weight, [&](Whole) { return target; }, before_c, before_w);
        const uint32_t b = (uint32_t)s.bin, in_c = s.in_c;
        const u64 in_w = s.in_w;
        before_c = s.before_c; before_w = s.before_w;
        hi -= b << shift;
        if (single) {
          const u64 each = in_w / in_c;                // equal logits have equal weights
          const u64 kept = by_weight ? (target - before_w + each - 1) / each : target - before_c;
          const float value = value_of(hi);
          sum = before_w + kept * each;
          int last = row.V;                            // every index
          if (kept < in_c)
            last = select_index(s, row, [&](float m) { return m >= value; },
                                [&](float l, int) -> u64 { return l == value; }, [&](u64) { return kept - 1; });
          return (u64)key_of(value) << 32 | (uint32_t)~last;
        }
        const uint32_t span = (1u << shift) - 1;
        lo = hi - lo > span ? hi - span : lo;
      }
    };
    if (some && (u64)k < all.count) {
      cut = search(false, (u64)k, true, whole);
      if (top_p < 1.f && spoilt) histogram();
    }
    if (top_p < 1.f) {
      const u64 target = part_of(whole, top_p);
      const bool first = !cut;
      if (first) {
        if (some) find_bin(s, true, [&](Whole) { return target; }, 0, 0);
        const int bin = s.bin;
        auto there = [&](float l) { return l > -INFINITY && bin_of(l) <= bin; };
        if (gather(s, row, false, there, there)) {
          from_list(LIST + 1, whole);
          return;
        }
      }
      u64 sum;
      cut = search(true, target, first, sum);
    }
  } else if (min_p > 0.f) {
    auto there = [&](float l) { return weigh(l) >= floor; };
    if (gather(s, row, false, there, there)) {
      from_list(LIST + 1, 0);
      return;
    }
  }
  auto target_of = [&](u64 whole) { return share_of(whole, u); };
  int token;
  if (!cut && floor == 0) {
    token = select_index(s, row, every, [&](float l, int) { return weigh(l); }, target_of);
  } else {
    const float least = cut ? logit_of((uint32_t)(cut >> 32)) : -INFINITY;
    const int last = cut ? (int)~(uint32_t)cut : a.V;
    auto there = [&](float m) { return m >= least; };
    auto kept = [&](float l, int i) { return l > least || (l == least && i <= last); };
    if (floor == 0)
      token = select_index(s, row, there, [&](float l, int i) { return kept(l, i) ? weigh(l) : 0; }, target_of);
    else
      token = select_index(s, row, there, [&](float l, int i) -> u64 {
        const u64 w = weigh(l);
        return w >= floor && kept(l, i) ? w : 0;
      }, target_of);
  }
  if (threadIdx.x == 0) a.token[r] = token;
}

hipError_t sample(const SampleArgs& a, int dtype, hipStream_t st) {
  if (a.rows == 0) return hipSuccess;
  int bits = 0;
  while ((1LL << bits) < a.V) ++bits;
  // V weights of at most 2^s stay below 2^63, and a weight is an integer of fp64's 52 bits
  const int s = bits > 11 ? 62 - bits : 51;
  // w is 0 from exp(-x) 2^s < 1/2: x > (s + 1) ln 2; the bins reach a little further
  const float range = (float)((s + 2) * 0.6931471805599453);
  if (dtype == NGDN_BF16) hipLaunchKernelGGL(sample_kernel<bf16>, dim3((unsigned)a.rows), dim3(TH), 0, st, a, s, range);
  else hipLaunchKernelGGL(sample_kernel<float>, dim3((unsigned)a.rows), dim3(TH), 0, st, a, s, range);
  return hipGetLastError();
}

}  // namespace ngdn
