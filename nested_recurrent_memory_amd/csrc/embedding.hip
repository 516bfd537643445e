// Rows of a [V,D] table by id, times a scale, and the table's gradient.
//   forward   y[n,:] = scale w[ids[n],:]
//   backward  dw[v,:] = scale sum_{n: ids[n] = v} dy[n,:]
// Sums are fp32 and rounded once; their order is that of the positions n, so
// the same ids give the same bits.
#include <algorithm>
#include <utility>

#include "ngdn_kernels.h"

namespace ngdn {

namespace {

// VEC values at p, aligned to their size
template <typename E, int VEC>
__device__ __forceinline__ void get(const E* p, float* o) {
  typedef E Vec __attribute__((ext_vector_type(4)));
  if constexpr (VEC == 8) {
    load8f(p, o);
  } else if constexpr (VEC == 4) {
    const Vec v = *reinterpret_cast<const Vec*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (float)v[e];
  } else {
    o[0] = to_f(*p);
  }
}
template <typename E, int VEC>
__device__ __forceinline__ void put(E* p, const float* x) {
  typedef E Vec __attribute__((ext_vector_type(4)));
  if constexpr (VEC == 8) {
    store8f(p, x);
  } else if constexpr (VEC == 4) {
    Vec v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (E)x[e];
    *reinterpret_cast<Vec*>(p) = v;
  } else {
    *p = from_f<E>(x[0]);
  }
}

}  // namespace

// 2^lg lanes a row (the least that hold it in one pass, at most a wave), each
// taking VEC values at a time. Bound by HBM: 32768 x 1024 from fp32 to bf16 20 us
// (102 MB with the distinct rows of the table), 131072 x 2048 182 us (870 MB; 196 in a
// training pass, behind the gradient of the one before).
template <typename W, typename Y, int VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(EmbedArgs a, int lg) {
  // loads before the first store: 131072 x 2048 from fp32 to bf16 184 us one at a
  // time, 181 two, 175 four; bf16 189 us four, 186 two
  constexpr int AHEAD = sizeof(W) * VEC > 16 ? 4 : 2;
  const long long n = ((long long)blockIdx.x * 256 + threadIdx.x) >> lg;
  if (n >= a.N) return;
  const long long v = a.ids[n];
  const bool ok = v >= 0 && v < a.V;
  const W* w = static_cast<const W*>(a.w) + (ok ? v : 0) * a.D;
  Y* y = static_cast<Y*>(a.y) + n * a.D;
  const int step = VEC << lg;
  for (int c = (threadIdx.x & ((1 << lg) - 1)) * VEC; c < a.D; c += AHEAD * step) {
    float t[AHEAD][VEC];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      if (c + u * step < a.D) get<W, VEC>(w + c + u * step, t[u]);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (c + u * step < a.D) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) t[u][i] = ok ? a.scale * t[u][i] : __builtin_nanf("");
        put<Y, VEC>(y + c + u * step, t[u]);
      }
    }
  }
}

// ---------------------------------------------------------------- sorting the ids
//
// The gradient's sums need the positions of each id together and in order: a
// stable radix sort of (id, position), from the low digit up. Ids that get no
// gradient sort behind the others, as V. Up to ONE ids one workgroup sorts in
// LDS; above, every pass is a count and a scatter over blocks of BLOCK ids.
// Every launch of the sort also clears a share of dw's last rows with workgroups
// of its own: the sort waits on latency, the clearing on HBM, and the rows with a
// sum are written after both. What does not fit beside the sort is cleared beside
// the sums, there only the rows without one (embed_sum).

namespace {

constexpr int ST = 1024, SW = ST / WAVE;       // threads and waves of a sorting workgroup
constexpr int ROUNDS = 4, BLOCK = ST * ROUNDS;
constexpr int ONE_ROUNDS = 8, ONE = ST * ONE_ROUNDS;
constexpr int DIGIT = 9, BUCKETS = 1 << DIGIT;
// behind the last id: every digit is the largest, and equal digits keep their
// order, so it stays behind them in every pass
constexpr int FILLER = 0x7fffffff;

struct SortArgs {
  const long long* ids;
  int* key[2];            // sorted ids and their positions; a pass reads one and writes the other
  int* pos[2];
  int* table;             // [nblock][BUCKETS] counts of a pass (embed_offsets: their sums, and a row of totals)
  int* owners;            // count of runs that cross segments, then their segments
  uint4* dw;              // cleared: [w0, w1), by the workgroups that do not sort
  long long w0, w1;
  unsigned short* tail;   // and, in the last launch, what is left of dw behind w1
  int tails;
  int N, V, pad, shift, bits, passes, nblock;
};

__device__ __forceinline__ int key_of(const SortArgs& s, long long id) {
  return id >= 0 && id < s.V && id != s.pad ? (int)id : s.V;
}

__device__ __forceinline__ void clear(const SortArgs& s, int block, int blocks) {
  for (long long i = s.w0 + (long long)block * ST + threadIdx.x; i < s.w1; i += (long long)blocks * ST)
    s.dw[i] = make_uint4(0, 0, 0, 0);
  if (block == 0 && (int)threadIdx.x < s.tails) s.tail[threadIdx.x] = 0;
}

// lanes of the wave with this lane's digit
__device__ __forceinline__ unsigned long long peers(int digit, int bits) {
  unsigned long long m = ~0ull;
  for (int b = 0; b < bits; ++b) {
    const bool one = digit >> b & 1;
    const unsigned long long v = __ballot(one);
    m &= one ? v : ~v;
  }
  return m;
}

// Ranks of the workgroup's keys among the equal digits before them: a wave's
// keys are R rounds of 64 in order; count[wave][digit] ends as the number of
// that digit in the waves before, total as that of the workgroup.
template <int R>
__device__ __forceinline__ void rank_keys(const int* key, int* rank, int shift, int bits,
                                          int (*count)[BUCKETS], int* total) {
  const int w = wave_id(), l = lane_id();
  for (int i = threadIdx.x; i < SW * BUCKETS; i += ST) (&count[0][0])[i] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int dg = key[r] >> shift & ((1 << bits) - 1);
    const unsigned long long m = peers(dg, bits);
    const int before = __popcll(m & ((1ull << l) - 1));
    const int c = count[w][dg];
    rank[r] = c + before;
    __builtin_amdgcn_wave_barrier();
    if (before == 0) count[w][dg] = c + __popcll(m);
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
  if (threadIdx.x < BUCKETS) {
    int sum = 0;
    for (int k = 0; k < SW; ++k) {
      const int c = count[k][threadIdx.x];
      count[k][threadIdx.x] = sum;
      sum += c;
    }
    total[threadIdx.x] = sum;
  }
  __syncthreads();
}

// exclusive sums of v over the threads below BUCKETS (all threads call)
__device__ __forceinline__ int scan_digits(int v, int* s_part) {
  const int w = wave_id(), l = lane_id();
  int x = v;
#pragma unroll
  for (int o = 1; o < WAVE; o <<= 1) {
    const int y = __shfl_up(x, o, WAVE);
    if (l >= o) x += y;
  }
  if (l == WAVE - 1) s_part[w] = x;
  __syncthreads();
  int before = 0;
  for (int k = 0; k < w; ++k) before += s_part[k];
  return before + x - v;
}

}  // namespace

// The whole sort of at most ONE ids (block 0); the other blocks clear dw. 8192 ids
// of a table of 32000 rows: 21.5 us, two passes' latency in one workgroup, beside
// which 128 MiB are cleared.
__global__ __launch_bounds__(ST) void embed_sort_one(SortArgs s) {
  __shared__ int s_key[ONE], s_pos[ONE], s_count[SW][BUCKETS], s_total[BUCKETS], s_part[SW];
  if (blockIdx.x > 0) {
    clear(s, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  if (threadIdx.x == 0) *s.owners = 0;
  const int first = wave_id() * (ONE_ROUNDS * WAVE) + lane_id();
  int key[ONE_ROUNDS], pos[ONE_ROUNDS], rank[ONE_ROUNDS];
#pragma unroll
  for (int r = 0; r < ONE_ROUNDS; ++r) {
    pos[r] = first + r * WAVE;
    key[r] = pos[r] < s.N ? key_of(s, s.ids[pos[r]]) : FILLER;
  }
  for (int p = 0; p < s.passes; ++p) {
    rank_keys<ONE_ROUNDS>(key, rank, p * s.bits, s.bits, s_count, s_total);
    const int base = scan_digits(threadIdx.x < BUCKETS ? s_total[threadIdx.x] : 0, s_part);
    if (threadIdx.x < BUCKETS) s_total[threadIdx.x] = base;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ONE_ROUNDS; ++r) {
      const int dg = key[r] >> (p * s.bits) & ((1 << s.bits) - 1);
      const int at = s_total[dg] + s_count[wave_id()][dg] + rank[r];
      s_key[at] = key[r];
      s_pos[at] = pos[r];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ONE_ROUNDS; ++r) {
      key[r] = s_key[first + r * WAVE];
      pos[r] = s_pos[first + r * WAVE];
    }
  }
#pragma unroll
  for (int r = 0; r < ONE_ROUNDS; ++r) {
    const int i = first + r * WAVE;
    if (i < s.N) {
      s.key[0][i] = key[r];
      s.pos[0][i] = pos[r];
    }
  }
}

__device__ __forceinline__ int pass_key(const SortArgs& s, int i) {
  return i >= s.N ? FILLER : s.shift == 0 ? key_of(s, s.ids[i]) : s.key[0][i];
}

// One pass over blocks: their counts of every digit. 131072 ids 9 us, the scatter 15.
__global__ __launch_bounds__(ST) void embed_count(SortArgs s) {
  __shared__ int s_count[BUCKETS];
  if ((int)blockIdx.x >= s.nblock) {
    clear(s, blockIdx.x - s.nblock, gridDim.x - s.nblock);
    return;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *s.owners = 0;
  if (threadIdx.x < BUCKETS) s_count[threadIdx.x] = 0;
  __syncthreads();
  const int first = blockIdx.x * BLOCK + wave_id() * (ROUNDS * WAVE) + lane_id();
  int key[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) key[r] = pass_key(s, first + r * WAVE);
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int dg = key[r] >> s.shift & ((1 << s.bits) - 1);
    const unsigned long long m = peers(dg, s.bits);
    if ((m & ((1ull << lane_id()) - 1)) == 0) atomicAdd(&s_count[dg], __popcll(m));
  }
  __syncthreads();
  if (threadIdx.x < BUCKETS) s.table[blockIdx.x * BUCKETS + threadIdx.x] = s_count[threadIdx.x];
}

// Above MANY blocks the counts are summed once, not by every block again, which grows
// with their square: 64 columns of the table a workgroup, each of its waves a stretch of
// the blocks. The gradient of 2^18 ids into 32000 x 16: 116 us, 119 with this launch;
// 2^19 179 and 177, 2^20 305 and 286, 2^24 5127 and 1867.
constexpr int MANY = 128;
__global__ __launch_bounds__(ST) void embed_offsets(SortArgs s) {
  __shared__ int s_sum[SW][WAVE];
  const int w = wave_id(), l = lane_id(), per = (s.nblock + SW - 1) / SW, b0 = w * per;
  const int b1 = b0 + per < s.nblock ? b0 + per : s.nblock;
  int* t = s.table + blockIdx.x * WAVE + l;
  int sum = 0;
#pragma unroll 16
  for (int b = b0; b < b1; ++b) sum += t[b * BUCKETS];
  s_sum[w][l] = sum;
  __syncthreads();
  int at = 0;
  for (int k = 0; k < w; ++k) at += s_sum[k][l];
  for (int b = b0; b < b1; b += 16) {
    int c[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) c[u] = b + u < b1 ? t[(b + u) * BUCKETS] : 0;
#pragma unroll
    for (int u = 0; u < 16; ++u) {
      if (b + u < b1) t[(b + u) * BUCKETS] = at;
      at += c[u];
    }
  }
  if (w == SW - 1) t[s.nblock * BUCKETS] = at;
}

// One pass over blocks: every id to its place.
__global__ __launch_bounds__(ST) void embed_scatter(SortArgs s) {
  __shared__ int s_count[SW][BUCKETS], s_total[BUCKETS], s_part[SW];
  if ((int)blockIdx.x >= s.nblock) {
    clear(s, blockIdx.x - s.nblock, gridDim.x - s.nblock);
    return;
  }
  const int first = blockIdx.x * BLOCK + wave_id() * (ROUNDS * WAVE) + lane_id();
  int key[ROUNDS], pos[ROUNDS], rank[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int i = first + r * WAVE;
    key[r] = pass_key(s, i);
    pos[r] = s.shift == 0 || i >= s.N ? i : s.pos[0][i];
  }
  int all = 0, before = 0;
  if (s.nblock > MANY) {
    if (threadIdx.x < BUCKETS) {
      all = s.table[s.nblock * BUCKETS + threadIdx.x];
      before = s.table[blockIdx.x * BUCKETS + threadIdx.x];
    }
  } else if (threadIdx.x < BUCKETS) {
    // 16 loads ahead of their additions: one at a time, beside the clearing, a
    // table of 32 blocks took 50 us to add
    for (int b = 0; b < s.nblock; b += 16) {
      int c[16];
#pragma unroll
      for (int u = 0; u < 16; ++u) c[u] = b + u < s.nblock ? s.table[(b + u) * BUCKETS + threadIdx.x] : 0;
#pragma unroll
      for (int u = 0; u < 16; ++u) {
        all += c[u];
        before += b + u < (int)blockIdx.x ? c[u] : 0;
      }
    }
  }
  rank_keys<ROUNDS>(key, rank, s.shift, s.bits, s_count, s_total);
  const int base = scan_digits(all, s_part) + before;
  if (threadIdx.x < BUCKETS) s_total[threadIdx.x] = base;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int dg = key[r] >> s.shift & ((1 << s.bits) - 1);
    const int at = s_total[dg] + s_count[wave_id()][dg] + rank[r];
    if (at < s.N) {                           // the filler's places are behind N
      s.key[1][at] = key[r];
      s.pos[1][at] = pos[r];
    }
  }
}

// ---------------------------------------------------------------- summing
//
// The sorted positions are cut into segments of `seg` (at most a wave): a wave
// takes a segment and 64 VEC columns, whichever ids are in it, so a frequent
// id's rows are spread over many waves. An id whose positions lie in one
// segment is summed there; of one that crosses segments each leaves its part
// (parts[2 k] what came into segment k from before, [2 k + 1] what starts in it
// and goes on), added in order by embed_join.
// 131072 x 2048 in bf16 into 131072 rows of fp32: 315 us, 0.54 GB read and 0.94 GB
// written (rows without a sum are cleared here), at 4.7 TB/s; clearing first or
// mixed among the sums 342 and 334, with non-temporal stores 470.

struct EmbedSum {
  const int* key; const int* pos;
  const void* dy; void* dw;
  float* parts;
  int* owners;
  int N, V, D, seg, nseg, tiles;
  int sums;               // workgroups that sum; those behind clear rows [0, rows) that no id has
  int rows;
  float scale;
};

// Rows of dw that no sorted key is: a wave looks for ROWS of them at once.
constexpr int ROWS = 16;
template <typename T, int VEC>
__device__ __forceinline__ void clear_rows(const EmbedSum& a, int wave) {
  const int l = lane_id(), v0 = wave * ROWS;
  bool gone = false;
  if (l < ROWS && v0 + l < a.rows) {
    int lo = 0, hi = a.N;
    while (lo < hi) {
      const int m = (lo + hi) / 2;
      if (a.key[m] < v0 + l) lo = m + 1; else hi = m;
    }
    gone = lo == a.N || a.key[lo] != v0 + l;
  }
  unsigned long long m = __ballot(gone);
  float zero[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) zero[e] = 0.f;
  while (m) {
    T* row = static_cast<T*>(a.dw) + (long long)(v0 + __builtin_ctzll(m)) * a.D;
    m &= m - 1;
    for (int c = l * VEC; c < a.D; c += WAVE * VEC) put<T, VEC>(row + c, zero);
  }
}

template <typename G, typename T, int VEC>
__global__ __launch_bounds__(256) void embed_sum(EmbedSum a) {
  constexpr int AHEAD = 8;                    // rows loaded before the first is added
  if ((int)blockIdx.x >= a.sums) {
    clear_rows<T, VEC>(a, (blockIdx.x - a.sums) * 4 + wave_id());
    return;
  }
  const long long item = (long long)blockIdx.x * 4 + wave_id();
  const int k = (int)(item / a.tiles), l = lane_id();
  if (k >= a.nseg) return;
  const int tile = (int)(item % a.tiles), c = (tile * WAVE + l) * VEC;
  const bool live = c < a.D;
  const int i0 = k * a.seg, m = a.N - i0 < a.seg ? a.N - i0 : a.seg;
  const int key = l < m ? a.key[i0 + l] : a.V, pos = l < m ? a.pos[i0 + l] : 0;
  const int n = __popcll(__ballot(key < a.V));          // those with a gradient come first
  if (n == 0) return;
  const int before = i0 > 0 ? a.key[i0 - 1] : -1, after = i0 + m < a.N ? a.key[i0 + m] : -1;
  const int down = __shfl_down(key, 1, WAVE), next = l + 1 < m ? down : after;
  const unsigned long long ends = __ballot(l + 1 == n || key != next);
  const bool open = __builtin_amdgcn_readlane(key, n - 1) == after;
  bool in = __builtin_amdgcn_readlane(key, 0) == before;
  const G* dy = static_cast<const G*>(a.dy) + (live ? c : 0);
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  for (int i = 0; i < n; i += AHEAD) {
    float v[AHEAD][VEC];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int j = i + u < n ? i + u : n - 1;
      get<G, VEC>(dy + (long long)__builtin_amdgcn_readlane(pos, j) * a.D, v[u]);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (i + u < n) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += v[u][e];
        if (ends >> (i + u) & 1) {
          const bool out = open && i + u == n - 1;
          if (live) {
            if (in || out) {
              put<float, VEC>(a.parts + (2LL * k + (in ? 0 : 1)) * a.D + c, acc);
            } else {
              const int id = __builtin_amdgcn_readlane(key, i + u);
#pragma unroll
              for (int e = 0; e < VEC; ++e) acc[e] *= a.scale;
              put<T, VEC>(static_cast<T*>(a.dw) + (long long)id * a.D + c, acc);
            }
          }
          if (out && !in && tile == 0 && l == 0) a.owners[1 + atomicAdd(a.owners, 1)] = k;
          in = false;
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
        }
      }
    }
  }
}

// The ids that cross segments: the part of the segment they start in and of
// those behind it, each of the workgroup's waves a stretch of them in order.
// The list of segments is in any order, what is added for one is not. 20 us at
// the same size: the most frequent ids' parts, one after another.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void embed_join(EmbedSum a) {
  __shared__ float s_acc[4][WAVE * VEC];
  const int w = wave_id(), l = lane_id(), c = (blockIdx.x * WAVE + l) * VEC;
  const bool live = c < a.D;
  const int count = *a.owners;
  for (int o = blockIdx.y; o < count; o += gridDim.y) {
    const int k = a.owners[1 + o];
    const int id = a.key[(k + 1) * a.seg];
    int more = 0;                              // segments behind k with rows of this id
    for (int s = k + 1;; s += WAVE) {
      const int q = s + l;
      const unsigned long long hit = __ballot(q < a.nseg && a.key[q < a.nseg ? q * a.seg : 0] == id);
      more += __popcll(hit);
      if (hit != ~0ull) break;
    }
    const int per = (more + 1 + 3) / 4, r0 = w * per, r1 = r0 + per < more + 1 ? r0 + per : more + 1;
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    if (live) {
#pragma unroll 8
      for (int r = r0; r < r1; ++r) {
        float v[VEC];
        get<float, VEC>(a.parts + (2LL * (k + r) + (r == 0 ? 1 : 0)) * a.D + c, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += v[e];
      }
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VEC; ++e) s_acc[w][l * VEC + e] = acc[e];
    __syncthreads();
    if (w == 0 && live) {
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        acc[e] = a.scale * (s_acc[0][l * VEC + e] + s_acc[1][l * VEC + e] + s_acc[2][l * VEC + e] +
                            s_acc[3][l * VEC + e]);
      put<T, VEC>(static_cast<T*>(a.dw) + (long long)id * a.D + c, acc);
    }
  }
}

// The whole gradient of at most FEW ids in one launch: a workgroup has HAND rows
// of dw, looks all ids over for them, and its waves take the rows' tiles of 64
// VEC columns in turn, to clear them or to add what points at them. 256 ids into
// 32000 x 1024: 25 us (131 MB cleared), 33 sorted; every workgroup reads all ids, so
// not beyond the ids that a workgroup has threads for.
constexpr int FEW = 256, HAND = 16;
template <typename G, typename T, int VEC>
__global__ __launch_bounds__(FEW) void embed_few(EmbedArgs a) {
  constexpr int AHEAD = 8;
  __shared__ int s_row[FEW], s_at[FEW], s_pos[FEW], s_count[FEW / WAVE], s_first[HAND + 1];
  const int l = lane_id(), w = wave_id(), n = threadIdx.x;
  const long long v0 = (long long)blockIdx.x * HAND;
  const long long id = n < a.N ? a.ids[n] : -1;
  const bool mine = id >= v0 && id < v0 + HAND && id < a.V && id != a.padding_idx;
  const unsigned long long m = __ballot(mine);
  if (l == 0) s_count[w] = __popcll(m);
  __syncthreads();
  int at = __popcll(m & ((1ull << l) - 1)), count = 0;
#pragma unroll
  for (int k = 0; k < FEW / WAVE; ++k) {
    at += k < w ? s_count[k] : 0;
    count += s_count[k];
  }
  if (mine) {
    s_row[at] = (int)(id - v0);
    s_at[at] = n;
  }
  __syncthreads();
  // by row, in the order of their positions within one
  if (n < count) {
    int rank = 0;
    for (int k = 0; k < count; ++k) rank += s_row[k] < s_row[n] || (s_row[k] == s_row[n] && k < n);
    s_pos[rank] = s_at[n];
  }
  if (n <= HAND) {
    int first = 0;
    for (int k = 0; k < count; ++k) first += s_row[k] < n;
    s_first[n] = first;
  }
  __syncthreads();
  const int tiles = (a.D + WAVE * VEC - 1) / (WAVE * VEC);
  const int rows = a.V - v0 < HAND ? (int)(a.V - v0) : HAND;
  for (int item = w; item < rows * tiles; item += FEW / WAVE) {
    const int r = item / tiles, c = (item % tiles * WAVE + l) * VEC;
    if (c >= a.D) continue;
    const G* dy = static_cast<const G*>(a.dy) + c;
    const int k1 = s_first[r + 1];
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    for (int k = s_first[r]; k < k1; k += AHEAD) {
      float v[AHEAD][VEC];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) get<G, VEC>(dy + (long long)s_pos[k + u < k1 ? k + u : k1 - 1] * a.D, v[u]);
#pragma unroll
      for (int u = 0; u < AHEAD; ++u)
        if (k + u < k1)
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] += v[u][e];
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] *= a.scale;
    put<T, VEC>(static_cast<T*>(a.dw) + (v0 + r) * a.D + c, acc);
  }
}

namespace {

long long up4(long long n) { return (n + 3) / 4 * 4; }

// The parts of ws (int32 units).
struct Space {
  long long pos0, key1, pos1, table, owners, parts, all;
  int seg, nseg, nblock;
};
Space space(long long N, long long V, long long D) {
  Space s;
  s.nblock = (int)((N + BLOCK - 1) / BLOCK);
  // Long segments leave fewer parts, short ones more waves: the longest that gives
  // 16 waves a CU at 512 columns a wave. 131072 x 2048: sums and joining 226 us with
  // segments of 64, 247 with 32, 272 with 16
  s.seg = 16;
  while (s.seg < WAVE && (N / (2 * s.seg)) * ((D + 511) / 512) >= 4096) s.seg *= 2;
  s.nseg = (int)((N + s.seg - 1) / s.seg);
  s.pos0 = up4(N);
  s.key1 = s.pos0 + up4(N);
  s.pos1 = s.key1 + (N > ONE ? up4(N) : 0);
  s.table = s.pos1 + (N > ONE ? up4(N) : 0);
  s.owners = s.table + (N > ONE ? (s.nblock + 1LL) * BUCKETS : 0);
  s.parts = s.owners + up4(s.nseg + 1);
  s.all = s.parts + (s.nseg > 1 ? 2LL * s.nseg * D : 0);
  return s;
}

template <typename W, typename Y>
hipError_t fwd(const EmbedArgs& a, hipStream_t st) {
  if (a.N == 0) return hipSuccess;
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(a.y);
  // 16 bytes a lane each way; 8 values of fp32 are two loads, which pays where they
  // are one store (32768 x 2048 fp32 90 us with 8 values, 81.5 with 4; to bf16 59.8
  // and 59.7, 32768 x 256 9.0 and 9.6)
  constexpr int WIDE = sizeof(W) == 4 && sizeof(Y) == 4 ? 4 : 8;
  const int vec = a.D % 8 == 0 && at % 16 == 0 ? WIDE : 1;
  int lg = 0;
  while (lg < 6 && (vec << lg) < a.D) ++lg;
  const dim3 grid((unsigned)(((a.N << lg) + 255) / 256));
  if (vec > 1) hipLaunchKernelGGL((embed_fwd_kernel<W, Y, WIDE>), grid, dim3(256), 0, st, a, lg);
  else hipLaunchKernelGGL((embed_fwd_kernel<W, Y, 1>), grid, dim3(256), 0, st, a, lg);
  return hipGetLastError();
}

template <typename G, typename W, int VEC>
hipError_t sum(const EmbedArgs& a, const Space& s, const int* key, const int* pos, int rows, hipStream_t st) {
  EmbedSum m{};
  m.key = key;
  m.pos = pos;
  m.dy = a.dy; m.dw = a.dw;
  m.parts = reinterpret_cast<float*>(a.ws + s.parts);
  m.owners = a.ws + s.owners;
  m.N = (int)a.N; m.V = (int)a.V; m.D = a.D; m.seg = s.seg; m.nseg = s.nseg; m.scale = a.scale;
  m.tiles = (a.D + WAVE * VEC - 1) / (WAVE * VEC);
  m.sums = (int)(((long long)m.nseg * m.tiles + 3) / 4);
  m.rows = rows;
  hipLaunchKernelGGL((embed_sum<G, W, VEC>), dim3(m.sums + (rows + 4 * ROWS - 1) / (4 * ROWS)), dim3(256), 0, st, m);
  if (m.nseg > 1) {
    const unsigned rows = (unsigned)std::min(m.nseg - 1, std::max(1, 1024 / m.tiles));
    hipLaunchKernelGGL((embed_join<W, VEC>), dim3(m.tiles, rows), dim3(256), 0, st, m);
  }
  return hipGetLastError();
}

template <typename G, typename W>
hipError_t bwd(const EmbedArgs& a, hipStream_t st) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.dy) | reinterpret_cast<uintptr_t>(a.dw) |
                       reinterpret_cast<uintptr_t>(a.ws);
  const bool vec = a.D % 8 == 0 && at % 16 == 0;
  if (a.N <= FEW) {
    const dim3 grid((unsigned)((a.V + HAND - 1) / HAND));
    if (vec) hipLaunchKernelGGL((embed_few<G, W, 8>), grid, dim3(FEW), 0, st, a);
    else hipLaunchKernelGGL((embed_few<G, W, 1>), grid, dim3(FEW), 0, st, a);
    return hipGetLastError();
  }
  const Space s = space(a.N, a.V, a.D);
  // what is cleared beside the sort: 128 MiB take about as long as it does
  constexpr long long BESIDE = 128LL << 20;
  const long long row = a.D * (long long)sizeof(W), bytes = a.V * row, all = bytes / 16;
  const int rows = bytes <= BESIDE ? 0 : (int)(a.V - BESIDE / row);
  const long long from = rows * row / 16, words = all - from;
  int bits = 1;
  while ((1LL << bits) <= a.V) ++bits;               // ids 0..V
  SortArgs r{};
  r.ids = a.ids;
  r.key[0] = a.ws; r.pos[0] = a.ws + s.pos0;
  r.key[1] = a.ws + s.key1; r.pos[1] = a.ws + s.pos1;
  r.table = a.ws + s.table;
  r.owners = a.ws + s.owners;
  r.dw = static_cast<uint4*>(a.dw);
  r.tail = reinterpret_cast<unsigned short*>(static_cast<char*>(a.dw) + all * 16);
  r.N = (int)a.N; r.V = (int)a.V;
  r.pad = a.padding_idx >= 0 && a.padding_idx < a.V ? (int)a.padding_idx : -1;
  r.passes = (bits + DIGIT - 1) / DIGIT;
  r.bits = (bits + r.passes - 1) / r.passes;
  const int clears = (int)std::min<long long>(512, (words + ST - 1) / ST + 1);
  const int *key = r.key[0], *pos = r.pos[0];
  r.w0 = from;
  r.w1 = all;
  r.tails = (int)(bytes - all * 16) / 2;
  if (a.N <= ONE) {
    hipLaunchKernelGGL(embed_sort_one, dim3(1 + clears), dim3(ST), 0, st, r);
  } else {
    r.nblock = s.nblock;
    const int launches = 2 * r.passes;
    for (int p = 0; p < launches; ++p) {
      r.w0 = from + words * p / launches;
      r.w1 = from + words * (p + 1) / launches;
      r.shift = p / 2 * r.bits;
      if (p % 2 == 0) {
        hipLaunchKernelGGL(embed_count, dim3(s.nblock + clears), dim3(ST), 0, st, r);
        if (s.nblock > MANY) hipLaunchKernelGGL(embed_offsets, dim3(BUCKETS / WAVE), dim3(ST), 0, st, r);
      } else {
        hipLaunchKernelGGL(embed_scatter, dim3(s.nblock + clears), dim3(ST), 0, st, r);
        std::swap(r.key[0], r.key[1]);
        std::swap(r.pos[0], r.pos[1]);
      }
    }
    key = r.key[0];
    pos = r.pos[0];
  }
  if (vec) return sum<G, W, 8>(a, s, key, pos, rows, st);
  return sum<G, W, 1>(a, s, key, pos, rows, st);
}

}  // namespace

int64_t embed_ws(int64_t N, int64_t V, int64_t D) { return space(N, V, D).all; }

hipError_t embed_fwd(const EmbedArgs& a, int wd, int yd, hipStream_t st) {
  if (wd == NGDN_BF16) return yd == NGDN_BF16 ? fwd<bf16, bf16>(a, st) : fwd<bf16, float>(a, st);
  return yd == NGDN_BF16 ? fwd<float, bf16>(a, st) : fwd<float, float>(a, st);
}

hipError_t embed_bwd(const EmbedArgs& a, int gd, int wd, hipStream_t st) {
  if (gd == NGDN_BF16) return wd == NGDN_BF16 ? bwd<bf16, bf16>(a, st) : bwd<bf16, float>(a, st);
  return wd == NGDN_BF16 ? bwd<float, bf16>(a, st) : bwd<float, float>(a, st);
}

}  // namespace ngdn
