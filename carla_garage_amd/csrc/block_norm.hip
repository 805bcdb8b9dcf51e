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
// Layout: a row belongs to TPR threads (64 .. 512, at most 8 elements each: 16 would not fit the registers beside their column sums, hence C <= 4096);
// row sums are DPP moves plus one LDS exchange when TPR > 64.  Column sums (the parameter gradients) stay in registers over all rows of the
// workgroup, one row of partials per workgroup, added in a fixed order by block_norm_colsum_kernel: bit-reproducible.
// Measured, 16384 rows of 2048 in bf16 with a gate for each token: forward 67 us (336 MB, 5.0 TB/s; a large copy reaches 5.1), backward 134 us (537 MB,
// 4.0 TB/s: 12 waves a CU is what the column sums leave) and 6 us for their sum; 3840 rows of 576, a gate for each sample: 12 + 25 + 6 us, latency.
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
  // a row as it lies in memory, fetched one iteration ahead of its use (aligned rows: 16 bytes of it are 4 registers)
  struct Raw { uint4 u[ALIGNED ? EPT / V : 1]; };
  __device__ static __forceinline__ void fetch(const T* __restrict__ p, int t, int C, Raw& r) {
    if constexpr (ALIGNED)
#pragma unroll
      for (int e = 0; e < EPT; e += V) r.u[e / V] = col(t, e) < C ? *reinterpret_cast<const uint4*>(p + col(t, e)) : make_uint4(0, 0, 0, 0);
  }
  __device__ static __forceinline__ void take(const Raw& r, const T* __restrict__ p, int t, int C, float (&f)[EPT]) {
    if constexpr (ALIGNED)
#pragma unroll
      for (int e = 0; e < EPT; e += V) unpack16<T>(r.u[e / V], f + e);
    else load(p, t, C, f);
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
template <typename T, int TPR, int EPT, bool ALIGNED> __device__ __forceinline__ void load_param(const float* __restrict__ p, float none, int t, int C, float (&f)[EPT]) {
  typedef Row<T, TPR, EPT, ALIGNED> R;
#pragma unroll
  for (int e = 0; e < EPT; ++e) f[e] = none;
  if (!p) return;
  if constexpr (ALIGNED) {
#pragma unroll
    for (int e = 0; e < EPT; e += 4)
      if (R::col(t, e) < C) load_vec<float>(p + R::col(t, e), f + e);
  } else {
#pragma unroll
    for (int e = 0; e < EPT; ++e)
      if (R::col(t, e) < C) f[e] = p[R::col(t, e)];
  }
}

// Sum over a wave by DPP moves (register to register; __shfl_xor goes through LDS, ~100 cycles a step, and a row needs up to four sums one after the other)
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) { return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true)); }
__device__ __forceinline__ float row_wave_sum(float v) {
  v = dpp_add<0xB1>(v);   // lane ^ 1
  v = dpp_add<0x4E>(v);   // lane ^ 2
  v = dpp_add<0x141>(v);  // mirror within 8
  v = dpp_add<0x140>(v);  // mirror within 16
  const int i = __float_as_int(v);
  return (__int_as_float(__builtin_amdgcn_readlane(i, 0)) + __int_as_float(__builtin_amdgcn_readlane(i, 16))) +
         (__int_as_float(__builtin_amdgcn_readlane(i, 32)) + __int_as_float(__builtin_amdgcn_readlane(i, 48)));
}

constexpr int threads_of(int tpr) { return tpr > 64 ? tpr : 256; }  // one row a workgroup, four where a row is one wave (no barrier at all)

// Sums of N values over the TPR threads of a row, the same in all of them.  `sm` alternates between two halves so that one barrier per call is
// enough: a wave may write the other half while slower waves still read this one.
template <int TPR, int N> __device__ __forceinline__ void row_sums(float (&v)[N], float* sm, int& phase) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = row_wave_sum(v[i]);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    float* s = sm + phase * (2 * W);
    phase ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) s[i * W + (threadIdx.x >> 6)] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) v[i] += s[i * W + w];
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
template <typename R, int TPR, int EPT> __device__ __forceinline__ void stats(const float (&f)[EPT], int t, int C, int layer, float eps, float* sm, int& phase, float& mean, float& rstd) {
  mean = 0.f;
  const float inv = 1.f / (float)C;
  if (layer) {
    float s[1] = {0.f};
#pragma unroll
    for (int e = 0; e < EPT; ++e) s[0] += f[e];
    row_sums<TPR, 1>(s, sm, phase);
    mean = s[0] * inv;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int e = 0; e < EPT; ++e) {
    const float d = R::col(t, e) < C ? f[e] - mean : 0.f;
    q[0] += d * d;
  }
  row_sums<TPR, 1>(q, sm, phase);
  rstd = 1.f / sqrtf(q[0] * inv + eps);
}

// A workgroup keeps the parameters in registers and takes the rows w, w + G, ..; the next row is on its way while this one is worked on.
template <typename T, int TPR, int EPT, bool ALIGNED> __global__ __launch_bounds__(threads_of(TPR)) void block_norm_fwd_kernel(tfpp_block_norm_params p) {
  constexpr int NT = threads_of(TPR), RPB = NT / TPR;
  typedef Row<T, TPR, EPT, ALIGNED> R;
  __shared__ float sm[4 * (NT / 64)];
  int phase = 0;
  const int t = threadIdx.x % TPR, C = p.C;
  const long rows = (long)p.B * p.T, stride = (long)gridDim.x * RPB;
  float pw[EPT], pb[EPT], qw[EPT], qb[EPT], sc[EPT];
  load_param<T, TPR, EPT, ALIGNED>(p.post_w, 1.f, t, C, pw);
  load_param<T, TPR, EPT, ALIGNED>(p.post_b, 0.f, t, C, pb);
  load_param<T, TPR, EPT, ALIGNED>(p.pre_w, 1.f, t, C, qw);
  load_param<T, TPR, EPT, ALIGNED>(p.pre_b, 0.f, t, C, qb);
  load_param<T, TPR, EPT, ALIGNED>(p.scale, 1.f, t, C, sc);
  auto gate_row = [&](long r) { return (const T*)p.gate + (p.gate_mode == GATE_TOKEN ? r : r / p.T) * p.ld_g; };
  typename R::Raw rx, ra, rg;
  long first = (long)blockIdx.x * RPB;
  auto fetch = [&](long base) {  // (rows past the end fetch and compute the last row and store nothing: every wave reaches the barriers)
    long r = base + threadIdx.x / TPR;
    if (r >= rows) r = rows - 1;
    R::fetch((const T*)p.x + r * p.ld_x, t, C, rx);
    R::fetch((const T*)p.a + r * p.ld_a, t, C, ra);
    if (p.gate_mode) R::fetch(gate_row(r), t, C, rg);
  };
  fetch(first);
  for (long base = first; base < rows; base += stride) {
    long r = base + threadIdx.x / TPR;
    const bool live = r < rows;
    if (!live) r = rows - 1;
    float x[EPT], a[EPT], g[EPT];
    R::take(rx, (const T*)p.x + r * p.ld_x, t, C, x);
    R::take(ra, (const T*)p.a + r * p.ld_a, t, C, a);
    if (p.gate_mode) R::take(rg, gate_row(r), t, C, g);
    if (base + stride < rows) fetch(base + stride);
#pragma unroll
    for (int e = 0; e < EPT; ++e) g[e] = p.gate_mode ? gate_act(g[e], p.gate_act) : 1.f;
    float mean, rstd;
    if (p.post) {
      stats<R, TPR>(a, t, C, p.layer, p.eps, sm, phase, mean, rstd);
      if (live && t == 0 && p.stat) *reinterpret_cast<float2*>(p.stat + r * 4) = make_float2(mean, rstd);
#pragma unroll
      for (int e = 0; e < EPT; ++e) a[e] = (a[e] - mean) * rstd * pw[e] + pb[e];
    }
#pragma unroll
    for (int e = 0; e < EPT; ++e) x[e] = R::col(t, e) < C ? p.alpha * x[e] + sc[e] * g[e] * a[e] : 0.f;
    if (live) R::store((T*)p.y + r * (long)C, t, C, x);
    if (p.pre) {
      stats<R, TPR>(x, t, C, p.layer, p.eps, sm, phase, mean, rstd);
      if (live && t == 0 && p.stat) *reinterpret_cast<float2*>(p.stat + r * 4 + 2) = make_float2(mean, rstd);
#pragma unroll
      for (int e = 0; e < EPT; ++e) x[e] = (x[e] - mean) * rstd * qw[e] + qb[e];
      if (live) R::store((T*)p.h + r * (long)C, t, C, x);
    }
  }
}

// grid (blocks per sample, B): a workgroup's rows belong to one sample, so its partial of the sample's gate gradient is one row
// BIAS, GSUM: which column sums exist at all (24 and 8 registers a thread: an occupancy step)
template <typename T, int TPR, int EPT, bool ALIGNED, bool BIAS, bool GSUM> __global__ __launch_bounds__(threads_of(TPR)) void block_norm_bwd_kernel(tfpp_block_norm_params p) {
  constexpr int NT = threads_of(TPR), RPB = NT / TPR;
  typedef Row<T, TPR, EPT, ALIGNED> R;
  extern __shared__ float red[];  // RPB > 1: column sums of the row groups
  __shared__ float sm[4 * (NT / 64)];
  int phase = 0;
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, C = p.C;
  const float inv = 1.f / (float)C;
  float pw[EPT], pb[EPT], qw[EPT], sc[EPT];
  load_param<T, TPR, EPT, ALIGNED>(p.post_w, 1.f, t, C, pw);
  load_param<T, TPR, EPT, ALIGNED>(BIAS ? p.post_b : nullptr, 0.f, t, C, pb);
  load_param<T, TPR, EPT, ALIGNED>(p.pre_w, 1.f, t, C, qw);
  load_param<T, TPR, EPT, ALIGNED>(p.scale, 1.f, t, C, sc);
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
  typename R::Raw rx, ra, rg, rdy, rdh;
  // A row's statistics come through the scalar cache, one row ahead like the rest: its threads are whole waves, and four more vector registers would
  // cost a third of the waves of wide rows (151 -> 191 us over 16384 rows of 2048)
  typedef float stat_t __attribute__((ext_vector_type(4)));
  const int usub = __builtin_amdgcn_readfirstlane(sub);
  stat_t rst;
  auto fetch = [&](int tt) {
    const long r = (long)blockIdx.y * p.T + (tt + sub < t1 ? tt + sub : t0);
    const long ur = (long)blockIdx.y * p.T + (tt + usub < t1 ? tt + usub : t0);
    rst = *(const __attribute__((address_space(4))) stat_t*)(uintptr_t)(p.stat + ur * 4);
    R::fetch((const T*)p.x + r * p.ld_x, t, C, rx);
    R::fetch((const T*)p.a + r * p.ld_a, t, C, ra);
    if (p.dy) R::fetch((const T*)p.dy + r * p.ld_dy, t, C, rdy);
    if (p.dh) R::fetch((const T*)p.dh + r * p.ld_dh, t, C, rdh);
    if (p.gate_mode == GATE_TOKEN) R::fetch((const T*)p.gate + r * p.ld_g, t, C, rg);
  };
  if (t0 < t1) fetch(t0);
  for (int tt = t0; tt < t1; tt += RPB) {
    const bool live = tt + sub < t1;
    const long r = (long)blockIdx.y * p.T + (live ? tt + sub : t0);
    float dy[EPT], dh[EPT], x[EPT], n[EPT], g[EPT];
    R::take(rx, (const T*)p.x + r * p.ld_x, t, C, x);
    R::take(ra, (const T*)p.a + r * p.ld_a, t, C, n);
    if (p.dy) R::take(rdy, (const T*)p.dy + r * p.ld_dy, t, C, dy);
    if (p.dh) R::take(rdh, (const T*)p.dh + r * p.ld_dh, t, C, dh);
    if (p.gate_mode == GATE_TOKEN) R::take(rg, (const T*)p.gate + r * p.ld_g, t, C, g);
    const stat_t st = rst;
    if (tt + RPB < t1) fetch(tt + RPB);
#pragma unroll
    for (int e = 0; e < EPT; ++e) g[e] = p.gate_mode == GATE_TOKEN ? gate_act(g[e], p.gate_act) : gs[e];
    if (!p.dy)
#pragma unroll
      for (int e = 0; e < EPT; ++e) dy[e] = 0.f;
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
          if constexpr (BIAS) acc[1][e] += dh[e];
        }
        const bool in = R::col(t, e) < C;
        dh[e] *= qw[e];
        s[0] += in ? dh[e] : 0.f;
        s[1] += in ? dh[e] * xh : 0.f;
        x[e] = xh;
      }
      row_sums<TPR, 2>(s, sm, phase);
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
        if constexpr (GSUM) acc[5][e] += dg;
        acc[2][e] += dn * n[e];
        if constexpr (BIAS) acc[3][e] += dn;
      }
      x[e] = dg;
      const bool in = R::col(t, e) < C;
      dy[e] = dn * pw[e];
      s[0] += in ? dy[e] : 0.f;
      s[1] += in ? dy[e] * n[e] : 0.f;
    }
    if (live && p.gate_mode == GATE_TOKEN && p.dgate) R::store((T*)p.dgate + r * (long)C, t, C, x);
    if (p.post) {
      row_sums<TPR, 2>(s, sm, phase);
      const float c0 = p.layer ? s[0] * inv : 0.f, c1 = s[1] * inv;
#pragma unroll
      for (int e = 0; e < EPT; ++e) dy[e] = st.y * (dy[e] - c0 - n[e] * c1);
    }
    if (live) R::store((T*)p.da + r * (long)C, t, C, dy);
  }
  float* out = p.partial + ((long)blockIdx.y * gridDim.x + blockIdx.x) * K_SUMS * C;
#pragma unroll
  for (int k = 0; k < K_SUMS; ++k) {
    if ((!GSUM && k == 5) || (!BIAS && (k == 1 || k == 3))) continue;
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

// out[k][c] (+)= sum over the workgroups' partials, 64 columns x 16 slices of them per workgroup; y = 0 .. 4: the parameter gradients over all workgroups,
// y = 5 + b: the gate gradient of sample b over that sample's workgroups, in the gate's type
template <typename T> __global__ __launch_bounds__(1024) void block_norm_colsum_kernel(tfpp_block_norm_params p, int bps) {
  constexpr int SLICES = 16;
  __shared__ float sm[1024];
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
  if (c < C) {
    const float* src = p.partial + (long)k * C + c;
    const long step = (long)K_SUMS * C;
    long i = lo + slice;
    for (; i + 7 * SLICES < hi; i += 8 * SLICES) {  // (eight loads in flight)
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = src[(i + u * SLICES) * step];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
    for (; i < hi; i += SLICES) s += src[i * step];
  }
  sm[threadIdx.x] = s;
  __syncthreads();
  if (slice == 0 && c < C) {
#pragma unroll
    for (int w = 1; w < SLICES; ++w) s += sm[w * 64 + threadIdx.x];
    if (k < 5) out[c] = (p.accumulate >> k) & 1 ? out[c] + s : s;
    else reinterpret_cast<T*>(p.dgate)[(long)b * C + c] = ElemTraits<T>::from_f(s);
  }
}

bool has_bias(const tfpp_block_norm_params& p) { return p.post_b || p.dpost_b || p.dpre_b; }

int blocks_per_sample(const tfpp_block_norm_params& p) {
  // 8 waves a CU fill the chip at this register count (12 without the sums that few of them need); each workgroup has at least 4 rows, since its 6 rows of partials are traffic too
  const int tpr = p.C <= 512 ? 64 : (p.C <= 1024 ? 128 : (p.C <= 2048 ? 256 : 512)), rpb = tpr == 64 ? 4 : 1, waves = has_bias(p) || p.gate_mode == GATE_SAMPLE ? 8 : 12, wgs = 256 * 64 * waves / threads_of(tpr);
  long n = (wgs + p.B - 1) / p.B;
  const long most = (p.T + 4L * rpb - 1) / (4L * rpb);
  if (n > most) n = most;
  return n < 1 ? 1 : (int)n;
}

bool aligned16(const tfpp_block_norm_params& p, int vec) {
  const void* ptrs[] = {p.x, p.a, p.gate, p.y, p.h, p.dy, p.dh, p.dx, p.da, p.gate_mode == GATE_TOKEN ? p.dgate : nullptr, p.post_w, p.post_b, p.pre_w, p.pre_b, p.scale};
  for (const void* q : ptrs)
    if ((uintptr_t)q & 15) return false;
  const int64_t lds[] = {p.ld_x, p.ld_a, p.gate_mode ? p.ld_g : 0, p.dy ? p.ld_dy : 0, p.dh ? p.ld_dh : 0, p.C};
  for (int64_t l : lds)
    if (l % vec) return false;
  return true;
}

bool valid(const tfpp_block_norm_params& p, int dtype) {
  return (dtype == TFPP_F32 || dtype == TFPP_BF16) && p.C >= 1 && p.C <= 4096 && p.B >= 1 && p.T >= 1 && (long)p.B * p.T < (1l << 30) && p.x && p.a && p.gate_mode >= 0 && p.gate_mode <= 2 &&
         (!p.gate_mode || p.gate) && (p.gate_act == ACT_NONE || p.gate_act == ACT_SIGMOID || p.gate_act == ACT_TANH);
}

template <typename T, int TPR, int EPT, bool AL> void launch(const tfpp_block_norm_params& p, bool bwd, int bps, hipStream_t st) {
  constexpr int NT = threads_of(TPR), RPB = NT / TPR;
  if (bwd) {
    const size_t lds = RPB > 1 ? (size_t)EPT * NT * 4 : 0;
    const bool bias = !AL || has_bias(p), gsum = !AL || p.gate_mode == GATE_SAMPLE;
    const dim3 grid(bps, p.B);
    if (bias && gsum) hipLaunchKernelGGL((block_norm_bwd_kernel<T, TPR, EPT, AL, true, true>), grid, dim3(NT), lds, st, p);
    else if (bias) hipLaunchKernelGGL((block_norm_bwd_kernel<T, TPR, EPT, AL, true, !AL>), grid, dim3(NT), lds, st, p);
    else if (gsum) hipLaunchKernelGGL((block_norm_bwd_kernel<T, TPR, EPT, AL, !AL, true>), grid, dim3(NT), lds, st, p);
    else hipLaunchKernelGGL((block_norm_bwd_kernel<T, TPR, EPT, AL, !AL, !AL>), grid, dim3(NT), lds, st, p);
  } else {
    const long rows = (long)p.B * p.T, groups = (rows + RPB - 1) / RPB, most = 256 * 1024 / NT;  // 16 waves a CU: what fits beside 40 registers of parameters
    hipLaunchKernelGGL((block_norm_fwd_kernel<T, TPR, EPT, AL>), dim3((unsigned)(groups < most ? groups : most)), dim3(NT), 0, st, p);
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
  if (!p || !valid(*p, dtype) || !p->y || (p->pre && !p->h) || ((uintptr_t)p->stat & 15)) return TFPP_EINVAL;
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
  if (dtype == TFPP_F32) hipLaunchKernelGGL(block_norm_colsum_kernel<float>, grid, dim3(1024), 0, st, *p, bps);
  else hipLaunchKernelGGL(block_norm_colsum_kernel<bf16_t>, grid, dim3(1024), 0, st, *p, bps);
  TFPP_CHECK_LAUNCH();
  return 0;
}
