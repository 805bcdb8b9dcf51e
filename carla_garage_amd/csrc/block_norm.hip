// What stands between two blocks of a residual network, in one pass over the row (channels-last, fp32 or bf16 storage, fp32 arithmetic):
//   n = post(a)                 norm behind the block that produced a        (optional)
//   y = alpha x + s * act(g) * n   residual scale alpha, layer scale s [C], gate g (per sample [B, C] or per token, act: none / sigmoid / tanh)
//   h = pre(y)                  norm in front of the next block              (optional)
// LayerNorm: (v - mean) rstd w + b;  RMS: v rstd w + b, rstd = 1 / sqrt(mean(v^2) + eps).
// Both directions are bounded by HBM.  Unfused, y and n make a round trip each; here forward reads x, a (, g) and writes y, h.  Backward recomputes n and
// y from x, a, g and the four saved row statistics -- y is NOT read back, so its rounding to bf16 does not reach any gradient -- and reads
// dy, dh, x, a (, g), writes dx, da (, dg):
//   dY = dy + pre'(dh)     dx = alpha dY     dn = dY s act(g)     dg = dY s n act'(g)     ds = sum dY act(g) n     da = post'(dn)
//   LayerNorm': rstd (dz w - mean(dz w) - xh mean(dz w xh));  RMS': without the middle term;  dw = sum dz xh, db = sum dz.
// Layout: a row belongs to TPR threads (64 .. 512, at most 8 elements each: 16 would not fit the registers beside their column sums, hence C <= 4096), a workgroup holds max(TPR, 256) threads;
// row sums are wave shuffles plus one LDS exchange when TPR > 64.  Column sums (the parameter gradients) stay in registers over all rows of the
// workgroup, one row of partials per workgroup, added in a fixed order by block_norm_colsum_kernel: bit-reproducible.
#include "common.h"
#include "../../include/tfpp.h"

namespace {
enum { GATE_NONE = 0, GATE_SAMPLE = 1, GATE_TOKEN = 2 };
constexpr int K_SUMS = 6;  // partial rows of one workgroup: dw_pre, db_pre, dw_post, db_post, dscale, dgate of the sample

// element e of thread t in a row: 16-byte chunks (ALIGNED) or single elements TPR apart (any C, any alignment)
template <typename T, int TPR, int EPT, bool ALIGNED> struct Row {
  static constexpr int V = ElemTraits<T>::VEC;
  __device__ static __forceinline__ int col(int t, int e) { return ALIGNED ? ((e / V) * TPR + t) * V + e % V : e * TPR + t; }
  __device__ static __forceinline__ void load(const T* __restrict__ p, int t, int C, float (&f)[EPT]) {
    if constexpr (ALIGNED) {
#pragma unroll
      for (int e = 0; e < EPT; e += V) {
        if (col(t, e) < C) load_vec<T>(p + col(t, e), f + e);
        else
#pragma unroll
          for (int i = 0; i < V; ++i) f[e + i] = 0.f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < EPT; ++e) f[e] = col(t, e) < C ? ElemTraits<T>::to_f(p[col(t, e)]) : 0.f;
    }
  }
  __device__ static __forceinline__ void store(T* __restrict__ p, int t, int C, const float (&f)[EPT]) {
    if constexpr (ALIGNED) {
#pragma unroll
      for (int e = 0; e < EPT; e += V)
        if (col(t, e) < C) store_vec<T>(p + col(t, e), f + e);
    } else {
#pragma unroll
      for (int e = 0; e < EPT; ++e)
        if (col(t, e) < C) p[col(t, e)] = ElemTraits<T>::from_f(f[e]);
    }
  }
};
// per-channel fp32 parameter (null: the given constant)
template <typename R, int EPT> __device__ __forceinline__ void load_param(const float* __restrict__ p, float none, int t, int C, float (&f)[EPT]) {
#pragma unroll
  for (int e = 0; e < EPT; ++e) f[e] = (p && R::col(t, e) < C) ? p[R::col(t, e)] : none;
}

// Sums of N values over the TPR threads of a row, the same in all of them.  `sm` alternates between two halves so that one barrier per call is
// enough: a wave may write the other half while slower waves still read this one.
template <int TPR, int NT, int N> __device__ __forceinline__ void row_sums(float (&v)[N], float* sm, int& phase) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if constexpr (TPR > 64) {
    constexpr int W = NT / 64, WR = TPR / 64;
    float* s = sm + phase * (2 * W);
    phase ^= 1;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) s[i * W + wave] = v[i];
    __syncthreads();
    const int first = wave / WR * WR;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.f;
#pragma unroll
      for (int w = 0; w < WR; ++w) v[i] += s[i * W + first + w];
    }
  }
}

__device__ __forceinline__ float gate_act(float v, int act) {
  if (act == ACT_SIGMOID) return 1.f / (1.f + __expf(-v));
  if (act == ACT_TANH) return tanhf(v);
  return v;
}
__device__ __forceinline__ float gate_slope(float g, int act) {  // from the activated value
  if (act == ACT_SIGMOID) return g * (1.f - g);
  if (act == ACT_TANH) return 1.f - g * g;
  return 1.f;
}

// mean (LayerNorm only) and rstd of a row held in registers: the mean first, then the centred squares (no cancellation)
template <typename R, int TPR, int NT, int EPT> __device__ __forceinline__ void stats(const float (&f)[EPT], int t, int C, int layer, float eps, float* sm, int& phase, float& mean,
                                                                                    float& rstd) {
  mean = 0.f;
  const float inv = 1.f / (float)C;
  if (layer) {
    float s[1] = {0.f};
#pragma unroll
    for (int e = 0; e < EPT; ++e) s[0] += f[e];
    row_sums<TPR, NT, 1>(s, sm, phase);
    mean = s[0] * inv;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int e = 0; e < EPT; ++e) {
    const float d = R::col(t, e) < C ? f[e] - mean : 0.f;
    q[0] += d * d;
  }
  row_sums<TPR, NT, 1>(q, sm, phase);
  rstd = 1.f / sqrtf(q[0] * inv + eps);
}

template <typename T, int TPR, int EPT, bool ALIGNED> __global__ __launch_bounds__(TPR > 256 ? TPR : 256) void block_norm_fwd_kernel(tfpp_block_norm_params p) {
  constexpr int NT = TPR > 256 ? TPR : 256, RPB = NT / TPR;
  typedef Row<T, TPR, EPT, ALIGNED> R;
  __shared__ float sm[4 * (NT / 64)];
  int phase = 0;
  const int t = threadIdx.x % TPR, C = p.C;
  const long row = (long)blockIdx.x * RPB + threadIdx.x / TPR, rows = (long)p.B * p.T;
  const bool live = row < rows;  // (rows past the end compute on row 0 and store nothing: every wave reaches the barriers)
  const long r = live ? row : 0;
  float x[EPT], a[EPT], w[EPT], b[EPT];
  R::load((const T*)p.x + r * p.ld_x, t, C, x);
  R::load((const T*)p.a + r * p.ld_a, t, C, a);
  float g[EPT];
  if (p.gate_mode) {
    R::load((const T*)p.gate + (p.gate_mode == GATE_TOKEN ? r : r / p.T) * p.ld_g, t, C, g);
#pragma unroll
    for (int e = 0; e < EPT; ++e) g[e] = gate_act(g[e], p.gate_act);
  } else {
#pragma unroll
    for (int e = 0; e < EPT; ++e) g[e] = 1.f;
  }
  float mean, rstd;
  if (p.post) {
    load_param<R>(p.post_w, 1.f, t, C, w);
    load_param<R>(p.post_b, 0.f, t, C, b);
    stats<R, TPR, NT>(a, t, C, p.layer, p.eps, sm, phase, mean, rstd);
    if (live && t == 0 && p.stat) {
      p.stat[r * 4] = mean;
      p.stat[r * 4 + 1] = rstd;
    }
#pragma unroll
    for (int e = 0; e < EPT; ++e) a[e] = (a[e] - mean) * rstd * w[e] + b[e];
  }
  load_param<R>(p.scale, 1.f, t, C, w);
#pragma unroll
  for (int e = 0; e < EPT; ++e) x[e] = R::col(t, e) < C ? p.alpha * x[e] + w[e] * g[e] * a[e] : 0.f;
  if (live) R::store((T*)p.y + r * (long)C, t, C, x);
  if (p.pre) {
    load_param<R>(p.pre_w, 1.f, t, C, w);
    load_param<R>(p.pre_b, 0.f, t, C, b);
    stats<R, TPR, NT>(x, t, C, p.layer, p.eps, sm, phase, mean, rstd);
    if (live && t == 0 && p.stat) {
      p.stat[r * 4 + 2] = mean;
      p.stat[r * 4 + 3] = rstd;
    }
#pragma unroll
    for (int e = 0; e < EPT; ++e) x[e] = (x[e] - mean) * rstd * w[e] + b[e];
    if (live) R::store((T*)p.h + r * (long)C, t, C, x);
  }
}

// grid (blocks per sample, B): a workgroup's rows belong to one sample, so its partial of the sample's gate gradient is one row
template <typename T, int TPR, int EPT, bool ALIGNED> __global__ __launch_bounds__(TPR > 256 ? TPR : 256) void block_norm_bwd_kernel(tfpp_block_norm_params p) {
  constexpr int NT = TPR > 256 ? TPR : 256, RPB = NT / TPR;
  typedef Row<T, TPR, EPT, ALIGNED> R;
  extern __shared__ float red[];  // RPB > 1: column sums of the row groups
  __shared__ float sm[4 * (NT / 64)];
  int phase = 0;
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, C = p.C;
  const float inv = 1.f / (float)C;
  float pw[EPT], pb[EPT], qw[EPT], sc[EPT];
  load_param<R>(p.post_w, 1.f, t, C, pw);
  load_param<R>(p.post_b, 0.f, t, C, pb);
  load_param<R>(p.pre_w, 1.f, t, C, qw);
  load_param<R>(p.scale, 1.f, t, C, sc);
  float gs[EPT];
#pragma unroll
  for (int e = 0; e < EPT; ++e) gs[e] = 1.f;
  if (p.gate_mode == GATE_SAMPLE) {
    R::load((const T*)p.gate + (long)blockIdx.y * p.ld_g, t, C, gs);
#pragma unroll
    for (int e = 0; e < EPT; ++e) gs[e] = gate_act(gs[e], p.gate_act);
  }
  float acc[K_SUMS][EPT];
#pragma unroll
  for (int k = 0; k < K_SUMS; ++k)
#pragma unroll
    for (int e = 0; e < EPT; ++e) acc[k][e] = 0.f;
  const int per = (p.T + (int)gridDim.x - 1) / (int)gridDim.x;
  const int t0 = (int)blockIdx.x * per, t1 = t0 + per < p.T ? t0 + per : p.T;
  for (int tt = t0; tt < t1; tt += RPB) {
    const bool live = tt + sub < t1;
    const long r = (long)blockIdx.y * p.T + (live ? tt + sub : t0);
    float dy[EPT], dh[EPT], x[EPT], n[EPT], g[EPT];
    R::load((const T*)p.x + r * p.ld_x, t, C, x);
    R::load((const T*)p.a + r * p.ld_a, t, C, n);
    if (p.dy) R::load((const T*)p.dy + r * p.ld_dy, t, C, dy);
    if (p.dh) R::load((const T*)p.dh + r * p.ld_dh, t, C, dh);
    if (p.gate_mode == GATE_TOKEN) {
      R::load((const T*)p.gate + r * p.ld_g, t, C, g);
#pragma unroll
      for (int e = 0; e < EPT; ++e) g[e] = gate_act(g[e], p.gate_act);
    } else {
#pragma unroll
      for (int e = 0; e < EPT; ++e) g[e] = gs[e];
    }
    if (!p.dy)
#pragma unroll
      for (int e = 0; e < EPT; ++e) dy[e] = 0.f;
    const float4 st = *reinterpret_cast<const float4*>(p.stat + r * 4);
    if (p.post)
#pragma unroll
      for (int e = 0; e < EPT; ++e) n[e] = (n[e] - st.x) * st.y;  // normalised a
    if (p.dh) {  // y recomputed, normalised; dY = dy + pre'(dh)
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int e = 0; e < EPT; ++e) {
        const float nn = p.post ? n[e] * pw[e] + pb[e] : n[e];
        const float xh = (p.alpha * x[e] + sc[e] * g[e] * nn - st.z) * st.w;
        if (live) {
          acc[0][e] += dh[e] * xh;
          acc[1][e] += dh[e];
        }
        const bool in = R::col(t, e) < C;
        dh[e] *= qw[e];
        s[0] += in ? dh[e] : 0.f;
        s[1] += in ? dh[e] * xh : 0.f;
        x[e] = xh;
      }
      row_sums<TPR, NT, 2>(s, sm, phase);
      const float c0 = p.layer ? s[0] * inv : 0.f, c1 = s[1] * inv;
#pragma unroll
      for (int e = 0; e < EPT; ++e) dy[e] += st.w * (dh[e] - c0 - x[e] * c1);
    }
#pragma unroll
    for (int e = 0; e < EPT; ++e) x[e] = p.alpha * dy[e];
    if (live) R::store((T*)p.dx + r * (long)C, t, C, x);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < EPT; ++e) {
      const float nn = p.post ? n[e] * pw[e] + pb[e] : n[e];
      const float d = dy[e];
      const float dg = d * sc[e] * nn * gate_slope(g[e], p.gate_act), dn = d * sc[e] * g[e];
      if (live) {
        acc[4][e] += d * g[e] * nn;
        acc[5][e] += dg;
        acc[2][e] += dn * n[e];
        acc[3][e] += dn;
      }
      x[e] = dg;
      const bool in = R::col(t, e) < C;
      dy[e] = dn * pw[e];
      s[0] += in ? dy[e] : 0.f;
      s[1] += in ? dy[e] * n[e] : 0.f;
    }
    if (live && p.gate_mode == GATE_TOKEN && p.dgate) R::store((T*)p.dgate + r * (long)C, t, C, x);
    if (p.post) {
      row_sums<TPR, NT, 2>(s, sm, phase);
      const float c0 = p.layer ? s[0] * inv : 0.f, c1 = s[1] * inv;
#pragma unroll
      for (int e = 0; e < EPT; ++e) dy[e] = st.y * (dy[e] - c0 - n[e] * c1);
    }
    if (live) R::store((T*)p.da + r * (long)C, t, C, dy);
  }
  float* out = p.partial + ((long)blockIdx.y * gridDim.x + blockIdx.x) * K_SUMS * C;
#pragma unroll
  for (int k = 0; k < K_SUMS; ++k) {
    if (k == K_SUMS - 1 && p.gate_mode != GATE_SAMPLE) break;
    if constexpr (RPB > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < EPT; ++e) red[e * NT + threadIdx.x] = acc[k][e];
      __syncthreads();
      if (sub == 0)
#pragma unroll
        for (int e = 0; e < EPT; ++e)
          for (int s = 1; s < RPB; ++s) acc[k][e] += red[e * NT + s * TPR + t];
    }
    if (sub == 0)
#pragma unroll
      for (int e = 0; e < EPT; ++e)
        if (R::col(t, e) < C) out[(long)k * C + R::col(t, e)] = acc[k][e];
  }
}

// out[k][c] (+)= sum over the workgroups' partials, 64 columns x 4 slices of them per workgroup; z = 0 .. 4: the parameter gradients over all workgroups,
// z = 5 + b: the gate gradient of sample b over that sample's workgroups, in the gate's type
template <typename T> __global__ __launch_bounds__(256) void block_norm_colsum_kernel(tfpp_block_norm_params p, int bps) {
  __shared__ float sm[256];
  const int k = blockIdx.y < 5 ? (int)blockIdx.y : 5, c = (int)blockIdx.x * 64 + ((int)threadIdx.x & 63), slice = threadIdx.x >> 6, C = p.C;
  float* const outs[5] = {p.dpre_w, p.dpre_b, p.dpost_w, p.dpost_b, p.dscale};
  float* out = nullptr;
#pragma unroll
  for (int i = 0; i < 5; ++i)
    if (k == i) out = outs[i];
  const int b = (int)blockIdx.y - 5;
  if (k < 5 && !out) return;
  const long lo = k < 5 ? 0 : (long)b * bps, hi = k < 5 ? (long)p.B * bps : lo + bps;
  float s = 0.f;
  if (c < C)
    for (long i = lo + slice; i < hi; i += 4) s += p.partial[(i * K_SUMS + k) * C + c];
  sm[threadIdx.x] = s;
  __syncthreads();
  if (slice == 0 && c < C) {
    s = (sm[threadIdx.x] + sm[threadIdx.x + 64]) + (sm[threadIdx.x + 128] + sm[threadIdx.x + 192]);
    if (k < 5) out[c] = (p.accumulate >> k) & 1 ? out[c] + s : s;
    else reinterpret_cast<T*>(p.dgate)[(long)b * C + c] = ElemTraits<T>::from_f(s);
  }
}

int blocks_per_sample(const tfpp_block_norm_params& p) {
  // 512 workgroups of 256 threads fill the chip at this register count; each has at least 4 rows, since its 6 rows of partials are traffic too
  const int tpr = p.C <= 512 ? 64 : (p.C <= 1024 ? 128 : (p.C <= 2048 ? 256 : 512)), rpb = tpr < 256 ? 256 / tpr : 1;
  long n = (512 + p.B - 1) / p.B;
  const long most = (p.T + 4L * rpb - 1) / (4L * rpb);
  if (n > most) n = most;
  return n < 1 ? 1 : (int)n;
}

bool aligned16(const tfpp_block_norm_params& p, int vec) {
  const void* ptrs[] = {p.x, p.a, p.gate, p.y, p.h, p.dy, p.dh, p.dx, p.da, p.gate_mode == GATE_TOKEN ? p.dgate : nullptr};
  for (const void* q : ptrs)
    if ((uintptr_t)q & 15) return false;
  const int64_t lds[] = {p.ld_x, p.ld_a, p.gate_mode ? p.ld_g : 0, p.dy ? p.ld_dy : 0, p.dh ? p.ld_dh : 0, p.C};
  for (int64_t l : lds)
    if (l % vec) return false;
  return true;
}

bool valid(const tfpp_block_norm_params& p, int dtype) {
  return (dtype == TFPP_F32 || dtype == TFPP_BF16) && p.C >= 1 && p.C <= 4096 && p.B >= 1 && p.T >= 1 && p.x && p.a && p.gate_mode >= 0 && p.gate_mode <= 2 &&
         (!p.gate_mode || p.gate) && (p.gate_act == ACT_NONE || p.gate_act == ACT_SIGMOID || p.gate_act == ACT_TANH);
}

template <typename T, int TPR, int EPT, bool AL> void launch(const tfpp_block_norm_params& p, bool bwd, int bps, hipStream_t st) {
  constexpr int NT = TPR > 256 ? TPR : 256, RPB = NT / TPR;
  if (bwd) {
    const size_t lds = RPB > 1 ? (size_t)EPT * NT * 4 : 0;
    hipLaunchKernelGGL((block_norm_bwd_kernel<T, TPR, EPT, AL>), dim3(bps, p.B), dim3(NT), lds, st, p);
  } else {
    const long rows = (long)p.B * p.T;
    hipLaunchKernelGGL((block_norm_fwd_kernel<T, TPR, EPT, AL>), dim3((unsigned)((rows + RPB - 1) / RPB)), dim3(NT), 0, st, p);
  }
}
template <typename T> void dispatch(const tfpp_block_norm_params& p, bool bwd, int bps, hipStream_t st) {
  const bool al = aligned16(p, ElemTraits<T>::VEC);
#define BN_GO(TPR, EPT) (al ? launch<T, TPR, EPT, true>(p, bwd, bps, st) : launch<T, TPR, EPT, false>(p, bwd, bps, st))
  if (p.C <= 512) BN_GO(64, 8);
  else if (p.C <= 1024) BN_GO(128, 8);
  else if (p.C <= 2048) BN_GO(256, 8);
  else BN_GO(512, 8);
#undef BN_GO
}
}  // namespace

extern "C" int tfpp_block_norm_fwd(const tfpp_block_norm_params* p, int dtype, void* stream) {
  if (!p || !valid(*p, dtype) || !p->y || (p->pre && !p->h)) return TFPP_EINVAL;
  if ((long)p->B * p->T > 0x7fffffffL) return TFPP_EINVAL;  // one workgroup holds at least one row: the grid's x limit
  if (dtype == TFPP_F32) dispatch<float>(*p, false, 0, (hipStream_t)stream);
  else dispatch<bf16_t>(*p, false, 0, (hipStream_t)stream);
  TFPP_CHECK_LAUNCH();
  return 0;
}

extern "C" int tfpp_block_norm_bwd_partial_floats(const tfpp_block_norm_params* p, int64_t* out) {
  if (!p || !out || p->B < 1 || p->T < 1 || p->C < 1) return TFPP_EINVAL;
  *out = (int64_t)blocks_per_sample(*p) * p->B * K_SUMS * p->C;
  return 0;
}

extern "C" int tfpp_block_norm_bwd(const tfpp_block_norm_params* p, int dtype, void* stream) {
  if (!p || !valid(*p, dtype) || !p->dx || !p->da || !p->stat || ((uintptr_t)p->stat & 15) || !p->partial || (!p->dy && !p->dh) || (p->dh && !p->pre)) return TFPP_EINVAL;
  if (p->gate_mode == GATE_SAMPLE && !p->dgate) return TFPP_EINVAL;
  if (p->B > 65530) return TFPP_EINVAL;  // samples lie in the grid's y dimension
  hipStream_t st = (hipStream_t)stream;
  const int bps = blocks_per_sample(*p);
  if (dtype == TFPP_F32) dispatch<float>(*p, true, bps, st);
  else dispatch<bf16_t>(*p, true, bps, st);
  TFPP_CHECK_LAUNCH();
  const dim3 grid((p->C + 63) / 64, 5 + (p->gate_mode == GATE_SAMPLE ? p->B : 0));
  if (dtype == TFPP_F32) hipLaunchKernelGGL(block_norm_colsum_kernel<float>, grid, dim3(256), 0, st, *p, bps);
  else hipLaunchKernelGGL(block_norm_colsum_kernel<bf16_t>, grid, dim3(256), 0, st, *p, bps);
  TFPP_CHECK_LAUNCH();
  return 0;
}
