// Rows of a [V,D] table by id, times a scale, and the table's gradient.
//   forward   y[n,:] = scale w[ids[n],:]
//   backward  dw[v,:] = scale sum_{n: ids[n] = v} dy[n,:]
// Sums are fp32 and rounded once; their order is that of the positions n, so
// the same ids give the same bits.
#include "ngdn_kernels.h"

namespace ngdn {

namespace {

template <typename E, int VEC>
__device__ __forceinline__ void get(const E* p, float* o) {
  if constexpr (VEC == 8) load8f(p, o);
  else o[0] = to_f(*p);
}
template <typename E, int VEC>
__device__ __forceinline__ void put(E* p, const float* x) {
  if constexpr (VEC == 8) store8f(p, x);
  else *p = from_f<E>(x[0]);
}

}  // namespace

// 2^lg lanes a row (the least that hold it in one pass, at most a wave), each
// taking VEC values at a time.
template <typename W, typename Y, int VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(EmbedArgs a, int lg) {
  const long long n = ((long long)blockIdx.x * 256 + threadIdx.x) >> lg;
  if (n >= a.N) return;
  const long long v = a.ids[n];
  const bool ok = v >= 0 && v < a.V;
  const W* w = static_cast<const W*>(a.w) + (ok ? v : 0) * a.D;
  Y* y = static_cast<Y*>(a.y) + n * a.D;
  for (int c = (threadIdx.x & ((1 << lg) - 1)) * VEC; c < a.D; c += VEC << lg) {
    float t[VEC];
    get<W, VEC>(w + c, t);
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = ok ? a.scale * t[i] : __builtin_nanf("");
    put<Y, VEC>(y + c, t);
  }
}

// A workgroup a row of the table: it looks through the ids 256 at a time and
// adds the rows of dy that point at it.
template <typename G, typename W>
__global__ __launch_bounds__(256) void embed_bwd_kernel(EmbedArgs a) {
  __shared__ unsigned long long s_hit[4];
  const long long v = blockIdx.x;
  W* dw = static_cast<W*>(a.dw) + v * a.D;
  for (int c0 = 0; c0 < a.D; c0 += 1024) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (long long n0 = 0; n0 < a.N && v != a.padding_idx; n0 += 256) {
      const long long n = n0 + threadIdx.x;
      const unsigned long long hit = __ballot(n < a.N && a.ids[n < a.N ? n : 0] == v);
      if (lane_id() == 0) s_hit[wave_id()] = hit;
      __syncthreads();
      for (int w = 0; w < 4; ++w) {
        unsigned long long m = s_hit[w];
        while (m) {
          const long long r = n0 + w * 64 + __builtin_ctzll(m);
          m &= m - 1;
          const G* dy = static_cast<const G*>(a.dy) + r * a.D;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int c = c0 + i * 256 + threadIdx.x;
            if (c < a.D) acc[i] += to_f(dy[c]);
          }
        }
      }
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = c0 + i * 256 + threadIdx.x;
      if (c < a.D) dw[c] = from_f<W>(a.scale * acc[i]);
    }
  }
}

int64_t embed_ws(int64_t N, int64_t V, int64_t D) { return 1; }

namespace {

template <typename W, typename Y>
hipError_t fwd(const EmbedArgs& a, hipStream_t st) {
  if (a.N == 0) return hipSuccess;
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.w) | reinterpret_cast<uintptr_t>(a.y);
  const int vec = a.D % 8 == 0 && at % 16 == 0 ? 8 : 1;
  int lg = 0;
  while (lg < 6 && (vec << lg) < a.D) ++lg;
  const dim3 grid((unsigned)(((a.N << lg) + 255) / 256));
  if (vec == 8) hipLaunchKernelGGL((embed_fwd_kernel<W, Y, 8>), grid, dim3(256), 0, st, a, lg);
  else hipLaunchKernelGGL((embed_fwd_kernel<W, Y, 1>), grid, dim3(256), 0, st, a, lg);
  return hipGetLastError();
}

template <typename G, typename W>
hipError_t bwd(const EmbedArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((embed_bwd_kernel<G, W>), dim3((unsigned)a.V), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace

hipError_t embed_fwd(const EmbedArgs& a, int wd, int yd, hipStream_t st) {
  if (wd == NGDN_BF16) return yd == NGDN_BF16 ? fwd<bf16, bf16>(a, st) : fwd<bf16, float>(a, st);
  return yd == NGDN_BF16 ? fwd<float, bf16>(a, st) : fwd<float, float>(a, st);
}

hipError_t embed_bwd(const EmbedArgs& a, int gd, int wd, hipStream_t st) {
  if (gd == NGDN_BF16) return wd == NGDN_BF16 ? bwd<bf16, bf16>(a, st) : bwd<bf16, float>(a, st);
  return wd == NGDN_BF16 ? bwd<float, bf16>(a, st) : bwd<float, float>(a, st);
}

}  // namespace ngdn
