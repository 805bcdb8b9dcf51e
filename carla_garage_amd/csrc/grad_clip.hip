// Norm of the gradients of a model and their clipping (train.py:900-906: unscale, clip_grad_norm_), over any number of tensors:
//   norm = || s g ||_p  over all elements of all tensors (p = 2, 1 or the largest magnitude)     coef = min(1, max_norm / (norm + 1e-6))
//   out  = s coef g     (s: the inverse of the loss scale)
// A table in device memory holds one 32-byte entry per chunk of at most GC_CHUNK elements, whatever tensor it belongs to, so 1332 tensors
// cost the same two launches as one.  Bounded by HBM: the gradient is read for the norm, read again and written for the clipping.
//   1. grad_norm_kernel: workgroup w takes the chunks w, w + G, ... and leaves ONE partial.  Sums are double: fp32 squares of gradients
//      around 1e-23 (or 1e20) underflow (overflow), and the f64 rate is far above what 4 B / element asks for.
//   2. grad_clip_kernel: EVERY workgroup adds the partials in index order (<= 16 KB out of L2, bit-identical in all of them and from run
//      to run; no ticket, no atomics, no state between calls), then writes its chunks -- walked from the LAST chunk to the first, since
//      the end of the gradient is what launch 1 left in the 256 MB memory-side cache.  In place with s coef == 1 nothing is touched.
// Measured: 1332 tensors, 480 MB of fp32: 104 us (4.6 TB/s) and 184 us (960 MB, 5.2 TB/s; a large copy reaches 5.1); 80 MB of bf16 in 300 tensors:
// 34 us and 41 us (3.9 TB/s): two or three chunks a workgroup, so starting and draining them shows.
#include <type_traits>

#include "common.h"
#include "../../include/tfpp.h"

namespace {
constexpr int GC_THREADS = 256;
constexpr int GC_GRID = 2048;    // 8 workgroups per CU
constexpr int GC_CHUNK = 16384;  // most elements of a chunk; the table's maker takes 16 or 64 KB of the source, so that 2048 workgroups end together
enum { GC_SRC_BF16 = 1, GC_DST_BF16 = 2, GC_VEC = 4 };

__device__ __forceinline__ float max_nan(float m, float v) { return (v > m || v != v) ? v : m; }  // NaN wins and stays

template <int P> __device__ __forceinline__ void accumulate(double& s, float& m, float v) {
  if constexpr (P == 2) s = fma((double)v, (double)v, s);
  else if constexpr (P == 1) s += (double)fabsf(v);
  else m = max_nan(m, fabsf(v));
}

template <int P, typename T> __device__ __forceinline__ void chunk_norm(const T* __restrict__ p, int n, bool vec, double& s, float& m) {
  constexpr int V = ElemTraits<T>::VEC, U = 4;  // (four 16-byte loads in flight)
  int done = 0;
  if (vec) {
    const int nv = n / V;
    int i = threadIdx.x;
#pragma unroll 2
    for (; i + (U - 1) * GC_THREADS < nv; i += U * GC_THREADS) {
      uint4 r[U];
#pragma unroll
      for (int u = 0; u < U; ++u) r[u] = reinterpret_cast<const uint4*>(p)[i + u * GC_THREADS];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[V];
        unpack16<T>(r[u], f);
#pragma unroll
        for (int e = 0; e < V; ++e) accumulate<P>(s, m, f[e]);
      }
    }
    for (; i < nv; i += GC_THREADS) {
      float f[V];
      load_vec<T>(p + (size_t)i * V, f);
#pragma unroll
      for (int e = 0; e < V; ++e) accumulate<P>(s, m, f[e]);
    }
    done = nv * V;
  }
  for (int i = done + threadIdx.x; i < n; i += GC_THREADS) accumulate<P>(s, m, ElemTraits<T>::to_f(p[i]));
}

template <int P> __global__ __launch_bounds__(GC_THREADS) void grad_norm_kernel(const tfpp_grad_chunk* __restrict__ table, int chunks, double* __restrict__ partial) {
  __shared__ double sm[GC_THREADS / 64];
  double s = 0.0;
  float m = 0.f;
  tfpp_grad_chunk next = table[blockIdx.x];
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const tfpp_grad_chunk t = next;
    if (c + (int)gridDim.x < chunks) next = table[c + gridDim.x];  // (one table entry ahead of its data)
    if (t.flags & GC_SRC_BF16) chunk_norm<P, bf16_t>((const bf16_t*)t.src, t.n, t.flags & GC_VEC, s, m);
    else chunk_norm<P, float>((const float*)t.src, t.n, t.flags & GC_VEC, s, m);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    if constexpr (P == 0) m = max_nan(m, __shfl_xor(m, o, 64));
    else s += __shfl_xor(s, o, 64);
  }
  if constexpr (P == 0) s = (double)m;
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double t = sm[0];
    for (int w = 1; w < GC_THREADS / 64; ++w) t = P == 0 ? (double)max_nan((float)t, (float)sm[w]) : t + sm[w];
    partial[blockIdx.x] = t;
  }
}

// every thread returns the same (norm, coef); partials added in an order that depends on their number only
template <int P> __device__ __forceinline__ float2 norm_and_coef(const double* __restrict__ partial, int n, float max_norm, float scale) {
  __shared__ double sm[GC_THREADS / 64];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += GC_THREADS) {
    const double v = partial[i];
    if constexpr (P == 0) s = (double)max_nan((float)s, (float)v);
    else s += v;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const double v = __shfl_xor(s, o, 64);
    if constexpr (P == 0) s = (double)max_nan((float)s, (float)v);
    else s += v;
  }
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = s;
  __syncthreads();
  s = sm[0];
#pragma unroll
  for (int w = 1; w < GC_THREADS / 64; ++w) s = P == 0 ? (double)max_nan((float)s, (float)sm[w]) : s + sm[w];
  if constexpr (P == 2) s = sqrt(s);
  const float norm = (float)(s * fabs((double)scale));
  const float c = max_norm / (norm + 1e-6f);
  return make_float2(norm, c > 1.f ? 1.f : c);  // (a NaN norm gives a NaN coefficient, an infinite one 0: torch's clamp keeps both too)
}

template <typename S, typename D> __device__ __forceinline__ void chunk_scale(const S* src, D* dst, int n, bool vec, float f) {
  constexpr int V = 8;  // two float4 or one 16-byte vector of bf16
  int done = 0;
  if (vec) {
    const int nv = n / V;
    int i = threadIdx.x;
    auto step = [&](auto count) {
      constexpr int U = decltype(count)::value;
      uint4 r[U][V / ElemTraits<S>::VEC];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < V; e += ElemTraits<S>::VEC) r[u][e / ElemTraits<S>::VEC] = *reinterpret_cast<const uint4*>(src + (size_t)(i + u * GC_THREADS) * V + e);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[V];
#pragma unroll
        for (int e = 0; e < V; e += ElemTraits<S>::VEC) unpack16<S>(r[u][e / ElemTraits<S>::VEC], x + e);
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] *= f;
#pragma unroll
        for (int e = 0; e < V; e += ElemTraits<D>::VEC) store_vec<D>(dst + (size_t)(i + u * GC_THREADS) * V + e, x + e);
      }
      i += U * GC_THREADS;
    };
    while (i + 3 * GC_THREADS < nv) step(std::integral_constant<int, 4>());
    while (i < nv) step(std::integral_constant<int, 1>());
    done = nv * V;
  }
  for (int i = done + threadIdx.x; i < n; i += GC_THREADS) dst[i] = ElemTraits<D>::from_f(ElemTraits<S>::to_f(src[i]) * f);
}

template <int P> __global__ __launch_bounds__(GC_THREADS) void grad_clip_kernel(const tfpp_grad_chunk* __restrict__ table, int chunks, const double* __restrict__ partial,
                                                                                int npart, float max_norm, float scale, float* __restrict__ norm_coef, int apply) {
  const float2 nc = norm_and_coef<P>(partial, npart, max_norm, scale);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    norm_coef[0] = nc.x;
    norm_coef[1] = nc.y;
  }
  if (!apply) return;
  const float f = (float)((double)scale * (double)nc.y);
  if ((int)blockIdx.x >= chunks) return;
  tfpp_grad_chunk next = table[chunks - 1 - (int)blockIdx.x];
  for (int c = chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const tfpp_grad_chunk t = next;
    if (c >= (int)gridDim.x) next = table[c - (int)gridDim.x];
    if (t.src == t.dst && f == 1.f) continue;
    const bool vec = t.flags & GC_VEC;
    switch (t.flags & (GC_SRC_BF16 | GC_DST_BF16)) {
      case 0: chunk_scale<float, float>((const float*)t.src, (float*)t.dst, t.n, vec, f); break;
      case GC_SRC_BF16: chunk_scale<bf16_t, float>((const bf16_t*)t.src, (float*)t.dst, t.n, vec, f); break;
      case GC_DST_BF16: chunk_scale<float, bf16_t>((const float*)t.src, (bf16_t*)t.dst, t.n, vec, f); break;
      default: chunk_scale<bf16_t, bf16_t>((const bf16_t*)t.src, (bf16_t*)t.dst, t.n, vec, f); break;
    }
  }
}

template <int P> int launch(const tfpp_grad_chunk* table, int chunks, double* ws, float max_norm, float scale, float* norm_coef, int apply, hipStream_t st) {
  const int grid = chunks < GC_GRID ? chunks : GC_GRID;
  if (grid > 0) hipLaunchKernelGGL((grad_norm_kernel<P>), dim3(grid), dim3(GC_THREADS), 0, st, table, chunks, ws);
  TFPP_CHECK_LAUNCH();
  hipLaunchKernelGGL((grad_clip_kernel<P>), dim3(apply && grid > 0 ? grid : 1), dim3(GC_THREADS), 0, st, table, chunks, ws, grid, max_norm, scale, norm_coef, apply);
  TFPP_CHECK_LAUNCH();
  return 0;
}
}  // namespace

extern "C" int tfpp_grad_clip_chunk(void) { return GC_CHUNK; }
extern "C" int tfpp_grad_clip_partials(int chunks) { return chunks < GC_GRID ? (chunks > 0 ? chunks : 1) : GC_GRID; }

extern "C" int tfpp_grad_clip(const tfpp_grad_chunk* table, int chunks, double* ws, float max_norm, int norm_type, float grad_scale, float* norm_coef, int apply,
                              void* stream) {
  if (chunks < 0 || (chunks > 0 && !table) || !ws || !norm_coef || !(max_norm >= 0.f)) return TFPP_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  switch (norm_type) {
    case 0: return launch<0>(table, chunks, ws, max_norm, grad_scale, norm_coef, apply, st);
    case 1: return launch<1>(table, chunks, ws, max_norm, grad_scale, norm_coef, apply, st);
    case 2: return launch<2>(table, chunks, ws, max_norm, grad_scale, norm_coef, apply, st);
    default: return TFPP_EINVAL;
  }
}
