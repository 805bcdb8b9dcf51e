// Differential attention: the difference of two softmax maps with a learned weight, and the norm of each head's result.
//   P_i = softmax(scale Q_i K_i^T) (i = 1, 2)      O = (P_1 - lambda P_2) V      out = out_scale * w * O / sqrt(mean(O^2) + eps)
// Q [B, Tq, H, 2, d], K [B, Tk, Hkv, 2, d], V [B, Tk, Hkv, dv] with any strides but a contiguous last dimension; H / Hkv query heads share a key /
// value head; d <= 128, dv <= 256.  Keys are left out by kv_len (per sequence), key_mask (per key) and causality (key <= q_start + query); a query
// that sees no key gives zeros and takes no part in any gradient.  What lies at keys that no query of the sequence sees (NaN included) has no effect: they are
// zeros in the images, and their own columns in dK / dV, which may have read them, are dropped.  A key that causality hides from some queries only is read
// beside them, with a probability of zero: it has to be finite.
//
// All products are 32 x 32 x 16 MFMA tiles (bf16; fp32 runs the same code on eight 32 x 32 x 2 each).  Every score tile is computed transposed to
// where it is contracted next, so that its C fragment IS the B operand of the following product and never leaves the registers:
//   C layout: lane l, register r hold (row 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32);  registers 8 t .. 8 t + 7 are the eight contraction
//   slots of lane l for rows 16 t .. 16 t + 15 once both operands label slot e of half l / 32 as row 16 t + 8 (e / 4) + 4 (l / 32) + e % 4.
// The other operand is read in that labelling from an LDS image [row][channel] by two ds_read_b64_tr_b16 (bf16) or eight scalar reads (fp32).
// Images hold 16-byte chunks, chunk c of row r at r * NC + (c ^ swizzle(r)): row reads (32 rows, one chunk) and transpose reads (4 rows x 64
// bytes) are both free of bank conflicts.  They are filled by buffer loads into LDS (16 bytes a lane, no registers), one tile ahead of the products,
// where rows are 16-byte aligned, else element by element.
#include <cmath>

#include "common.h"
#include "../../include/tfpp.h"

namespace {
typedef __attribute__((ext_vector_type(16))) float f32x16_t;
typedef __attribute__((ext_vector_type(4))) short s16x4_t;
typedef __attribute__((address_space(3))) void lds_void_t;

constexpr float LOG2E = 1.4426950408889634f;
constexpr float NO_MAX = -1.0e30f;     // running maximum before the first visible key: finite, so that -inf scores give exp2(-inf) = 0
constexpr float MAX_SLACK = 8.f;       // the running maximum follows once it is 2^8 behind: probabilities stay below 256, exact in fp32 / bf16 range
constexpr int QB = 128;                // queries (keys) of a workgroup in the backward passes, 32 per wave

template <typename T> struct Frag8;
template <> struct Frag8<bf16_t> { uint4 v; };
template <> struct Frag8<float> { float v[8]; };

__device__ __forceinline__ void mma(const Frag8<bf16_t>& a, const Frag8<bf16_t>& b, f32x16_t& c) {
  c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a.v), __builtin_bit_cast(bf16x8_t, b.v), c, 0, 0, 0);
}
__device__ __forceinline__ void mma(const Frag8<float>& a, const Frag8<float>& b, f32x16_t& c) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[e], b.v[e], c, 0, 0, 0);
}
// C registers 8 t .. 8 t + 7 as an operand.  bf16: one rounding (2^-8 relative at most) of each probability / score gradient, as its partner operand has:
// the matrix unit takes both in one type, and a second product for what the rounding takes off would double the work with V.  It leaves outputs 2.4e-3
// off in the 2-norm where the rounding of the result alone leaves 1.7e-3, gradients 3.5e-3.
__device__ __forceinline__ void to_frag(const f32x16_t& c, int t, Frag8<bf16_t>& f) {
  f.v = make_uint4(f2bf_pack2(c[8 * t], c[8 * t + 1]), f2bf_pack2(c[8 * t + 2], c[8 * t + 3]), f2bf_pack2(c[8 * t + 4], c[8 * t + 5]),
                   f2bf_pack2(c[8 * t + 6], c[8 * t + 7]));
}
__device__ __forceinline__ void to_frag(const f32x16_t& c, int t, Frag8<float>& f) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f.v[e] = c[8 * t + e];
}

__device__ __forceinline__ unsigned long long low_bits(int n) { return n >= 64 ? ~0ull : (n <= 0 ? 0ull : (1ull << n) - 1ull); }
constexpr int pow2_at_least(int n) { return n <= 1 ? 1 : 2 * pow2_at_least((n + 1) / 2); }

struct Rows {  // which rows of a tile exist
  int count;                 // rows 0 .. count - 1 ..
  bool holes;                // .. but only those whose bit is set
  unsigned long long bits;
};

// LDS image of rows with 32 * CB channels (NC 16-byte chunks a row, a power of two)
template <typename T, int CB> struct Img {
  static constexpr int VEC = ElemTraits<T>::VEC, USED = 32 * CB / VEC, NC = pow2_at_least(USED);
  static constexpr int ROW_BYTES = NC * 16;
  __device__ static __forceinline__ int swizzle(int r) {
    if constexpr (NC >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (NC == 8) return ((r & 2) << 1) | ((r >> 2) & 3);
    else return (r >> 2) & 3;
  }
  __device__ static __forceinline__ int off(int r, int c) { return (r * NC + (c ^ swizzle(r))) * 16; }
  // Reads take a lane's byte offset for the first rows and channels (rows_at / cols_at, plus the image's place and 16-row steps, both multiples of a row)
  // and reach the other channels by an XOR with a constant: one register for a whole image.
  // Operand of 32 rows x 16 channels (16 ks ..): lane l has row l % 32, channels 16 ks + 8 (l / 32) ..
  __device__ static __forceinline__ int rows_at(int lane) { return off(lane & 31, (sizeof(T) == 2 ? 1 : 2) * (lane >> 5)); }
  __device__ static __forceinline__ void rows(const unsigned char* lds, int at, int ks, Frag8<T>& f) {
    if constexpr (sizeof(T) == 2) {
      f.v = *reinterpret_cast<const uint4*>(lds + (at ^ ks << 5));
    } else {
      const float4 a = *reinterpret_cast<const float4*>(lds + (at ^ ks << 6)), b = *reinterpret_cast<const float4*>(lds + (at ^ (ks << 6 | 16)));
      f.v[0] = a.x; f.v[1] = a.y; f.v[2] = a.z; f.v[3] = a.w; f.v[4] = b.x; f.v[5] = b.y; f.v[6] = b.z; f.v[7] = b.w;
    }
  }
  // operand of 32 channels (32 cb ..) x 16 rows, contraction over rows in the C fragments' labelling
  __device__ static __forceinline__ int cols_at(int lane) {
    const int half = lane >> 5, i = lane & 15;
    if constexpr (sizeof(T) == 2) return off(4 * half + (i >> 2), ((lane >> 4) & 1) * 2 + ((i & 3) >> 1)) + (i & 1) * 8;
    else return off(4 * half, (lane & 31) >> 2) + (lane & 3) * 4;
  }
  __device__ static __forceinline__ void cols(const unsigned char* lds, int at, int cb, Frag8<T>& f) {
    if constexpr (sizeof(T) == 2) {  // rows + 8: the swizzle's bit 1 turns over
      const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t __attribute__((address_space(3)))*)(lds + (at ^ cb << 6)));
      const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4_t __attribute__((address_space(3)))*)(lds + (at ^ (cb << 6 | 32)) + 8 * ROW_BYTES));
      const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
      f.v = make_uint4(a.x, a.y, b.x, b.y);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // (the swizzle of 4 half + k is that of 4 half XOR that of k: the bits are disjoint)
        const int k = 8 * (e >> 2) + (e & 3);
        f.v[e] = *reinterpret_cast<const float*>(lds + (at ^ (cb << 7 ^ swizzle(k) << 4)) + k * ROW_BYTES);
      }
    }
  }
  // fill ROWS rows: row r comes from base + r * ld (n channels), zeros from row `have.count` on, where a row is left out, and behind channel n.  VECTOR:
  // buffer loads into LDS, one 32-bit offset a lane (64 rows stay below 2 GB: checked by the launcher).  The descriptor ends with the last row that
  // exists, a chunk that is left out gets an offset behind it, and the hardware returns zeros for both without touching memory.
  template <int ROWS, bool VECTOR, int NT> __device__ static __forceinline__ void fill(unsigned char* img, const T* __restrict__ base, long ld, int n, Rows have, int tid) {
    constexpr int SLOTS = ROWS * NC;
    const int count = have.count < 0 ? 0 : (have.count < ROWS ? have.count : ROWS);
    if constexpr (VECTOR) {
      static_assert(NT % NC == 0 && SLOTS % 64 == 0, "a thread keeps its position in the row");
      const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
      const int ldb = (int)ld * (int)sizeof(T), r0 = tid / NC, rowb = r0 * ldb;
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, count > 0 ? (count - 1) * ldb + n * (int)sizeof(T) : 0, 0x00020000);
      auto put = [&](int u, bool ok) {
        const int c = (tid % NC) ^ swizzle(r0 + u * (NT / NC));
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_t*)(img + (u * NT + wave * 64) * 16), 16,
                                                 (ok && c * VEC < n ? rowb + c * 16 : (int)0x80000000) + u * (NT / NC) * ldb, 0, 0, 0);
      };
      if (!have.holes) {
#pragma unroll
        for (int u = 0; u * NT < SLOTS; ++u)
          if (u * NT + wave * 64 < SLOTS) put(u, true);
      } else {
#pragma unroll
        for (int u = 0; u * NT < SLOTS; ++u)
          if (u * NT + wave * 64 < SLOTS) put(u, ((have.bits >> (u * (NT / NC))) >> r0) & 1ull);
      }
    } else {
#pragma unroll 1
      for (int i = tid; i < ROWS * 32 * CB; i += NT) {
        const int r = i / (32 * CB), c = i % (32 * CB);
        T v = ElemTraits<T>::from_f(0.f);
        if (c < n && r < count && (!have.holes || ((have.bits >> r) & 1ull))) v = base[(long)r * ld + c];
        *reinterpret_cast<T*>(img + off(r, c / VEC) + (c % VEC) * sizeof(T)) = v;
      }
    }
  }
};

// operand straight from global memory: 8 channels (c ..) of one row, zeros behind channel n or where the row is left out
template <typename T, bool VECTOR> __device__ __forceinline__ void load_frag(const T* __restrict__ row, int c, int n, bool ok, Frag8<T>& f) {
  if constexpr (VECTOR) {
    if constexpr (sizeof(T) == 2) {
      f.v = ok && c < n ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const float4 a = ok && c + e < n ? *reinterpret_cast<const float4*>(row + c + e) : make_float4(0.f, 0.f, 0.f, 0.f);
        f.v[e] = a.x; f.v[e + 1] = a.y; f.v[e + 2] = a.z; f.v[e + 3] = a.w;
      }
    }
  } else if constexpr (sizeof(T) == 2) {
    unsigned u[4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const unsigned lo = ok && c + e < n ? row[c + e] : 0, hi = ok && c + e + 1 < n ? row[c + e + 1] : 0;
      u[e / 2] = lo | hi << 16;
    }
    f.v = make_uint4(u[0], u[1], u[2], u[3]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = ok && c + e < n ? row[c + e] : 0.f;
  }
}

struct Weights {  // of the heads' norm: none (null), fp32 or bf16
  const void* w;
  int is_bf16;
  __device__ __forceinline__ float operator[](int c) const { return is_bf16 ? bf2f(((const bf16_t*)w)[c]) : ((const float*)w)[c]; }
};

// Results leave through an LDS strip of the wave, two 32-channel blocks at a time: the C layout has a row in each lane, 4 channels a register quad, while
// memory wants whole rows; and the loop that stores them is ROLLED -- unrolled per register, an epilogue is thousands of instructions that every
// workgroup fetches once, 20 us of a short kernel.  Chunks of 4 floats, chunk c of row r at c ^ (r & 7).
constexpr int STRIP_BYTES = 32 * 64 * 4;
__device__ __forceinline__ int strip_at(int row, int chunk) { return row * 64 + ((chunk ^ (row & 7)) << 2); }
__device__ __forceinline__ void strip_put(float* strip, int lane, int block, const f32x16_t& o, float f) {
#pragma unroll
  for (int g = 0; g < 4; ++g)
    *reinterpret_cast<float4*>(strip + strip_at(lane & 31, block * 8 + 2 * g + (lane >> 5))) = make_float4(o[4 * g] * f, o[4 * g + 1] * f, o[4 * g + 2] * f, o[4 * g + 3] * f);
}
// channels c0 .. c0 + 32 * blocks - 1 of 32 rows; row(r): where row r starts (null: not stored); n: channels of a row; w: multiplied by the norm's weights
template <typename T, typename Row> __device__ __forceinline__ void strip_store(const float* strip, int lane, int blocks, int c0, int n, bool vec, Weights w, Row row) {
  const int per = blocks * 4, piece = lane & (per - 1), c = c0 + piece * 8;  // 8-channel pieces of a row: 4 or 8; a lane keeps its channels
  if (c >= n) return;
  float wf[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) wf[e] = w.w && c + e < n ? w[c + e] : 1.f;
#pragma unroll 1
  for (int r = lane / per; r < 32; r += 64 / per) {
    T* dst = row(r);
    if (!dst) break;  // (rows that do not exist are the last ones)
    float f[8];
    *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(strip + strip_at(r, 2 * piece));
    *reinterpret_cast<float4*>(f + 4) = *reinterpret_cast<const float4*>(strip + strip_at(r, 2 * piece + 1));
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= wf[e];
    if (vec && c + 8 <= n) {
#pragma unroll
      for (int e = 0; e < 8; e += ElemTraits<T>::VEC) store_vec<T>(dst + c + e, f + e);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < n) dst[c + e] = ElemTraits<T>::from_f(f[e]);
    }
  }
}
// all N blocks of a wave's 32 rows
template <typename T, int N, typename Row> __device__ __forceinline__ void store_rows(float* strip, int lane, const f32x16_t (&o)[N], float f, int n, bool vec, Weights w, Row row) {
#pragma unroll
  for (int b = 0; b < N; b += 2) {
    strip_put(strip, lane, 0, o[b], f);
    if (b + 1 < N) strip_put(strip, lane, 1, o[b + 1 < N ? b + 1 : b], f);
    __builtin_amdgcn_wave_barrier();  // (one wave's LDS operations complete in order)
    strip_store<T>(strip, lane, b + 1 < N ? 2 : 1, b * 32, n, vec, w, row);
    __builtin_amdgcn_wave_barrier();
  }
}

// workgroup -> (tile, batch x head).  Workgroups go round the 8 XCDs in turn: where the heads divide evenly, all tiles of a head stay on one XCD (its
// K and V are read from that XCD's L2).  Equal tiles: head after head, so that few heads share an L2 at a time; causal: tile after tile over all
// heads, the caller turning the order so that the longest start first and the short ones fill the end.
__device__ __forceinline__ void place(int heads, int tiles, bool by_tile, int& bh, int& tile) {
  const int id = blockIdx.x;
  if (by_tile) {
    bh = id % heads;
    tile = id / heads;
  } else if (heads % 8 == 0) {
    bh = (id % 8) + 8 * ((id / 8) / tiles);
    tile = (id / 8) % tiles;
  } else {
    bh = id / tiles;
    tile = id % tiles;
  }
}

// Fill the next images while the present ones are read.  The two are different memory, and the compiler has to be told: it puts a wait for ALL loads
// into LDS that are under way in front of an LDS read that may alias them, which would undo the prefetch.
// The noalias arguments become scopes on both sides when this is inlined.  The wait that IS needed stands at the top of each step.
template <typename Fill, typename Use> __device__ __forceinline__ void overlap(unsigned char* __restrict__ next, const unsigned char* __restrict__ now, Fill fill, Use use) {
  fill(next);
  use(now);
}

struct Seq {  // what a sequence's queries may see
  int len, start;  // keys 0 .. len - 1, no query sees one behind; query i sees key j <= start + i (causal)
};
__device__ __forceinline__ Seq sequence(const tfpp_diff_attn_params& p, int b) {
  Seq s;
  s.len = p.Tk;
  if (p.kv_len) {
    const int n = __builtin_amdgcn_readfirstlane(p.kv_len[b]);  // (the compiler does not know that it is the same in all lanes)
    s.len = n < 0 ? 0 : (n < p.Tk ? n : p.Tk);
  }
  const int start = p.q_start ? __builtin_amdgcn_readfirstlane(p.q_start[b]) : p.q_start_all;
  s.start = start < -p.Tq ? -p.Tq : (start < p.Tk ? start : p.Tk);  // (beyond: nothing is seen, everything is; sums with positions stay in 32 bits)
  if (p.causal && s.start + p.Tq < s.len) s.len = s.start + p.Tq;    // (what lies behind the last query's keys may be stale: slots of a cache)
  return s;
}
// bit i: key j0 + i exists and is not left out
__device__ __forceinline__ unsigned long long key_bits(const tfpp_diff_attn_params& p, int b, int j0, int len, int lane) {
  if (!p.key_mask) return low_bits(len - j0);
  const int j = j0 + lane;
  return __ballot(j < len && p.key_mask[(long)b * p.ld_mask + (j < len ? j : 0)] != 0);
}

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

template <typename T> constexpr int key_tile() { return sizeof(T) == 2 ? 64 : 32; }

// ---------------------------------------------------------------------------------------------------------------------------------
// forward.  A wave has 32 queries, lane l and l + 32 = one query.  S_i^T = K_i Q_i^T (keys x queries), running maximum and sum per query,
// O_i^T += V^T P_i^T: both maps share every V operand.  O_1 and O_2 are kept apart to the end because their sums are not known before; one pass,
// 4 d + 4 dv flop a pair.  Long sequences are bounded by a wave's own chain of scores, exponentials and value products, of which two waves a SIMD overlap
// a part: 8100 causal tokens, 8 heads of 128 / 256: 437 us (0.92 PFLOP/s of these products; one of 8192^3 by the library: 1.19), the matrix unit busy in
// 47 % of the cycles, vector issue in 42 %, LDS in 24 %.  (Clocks that have settled; the first dozen calls after a pause take up to 570 us.)  2 x 4096 causal,
// 16 heads of 64 / 128: 243 us; 12 x 320, 4 heads of 72 / 144: 24 us, 10 of them launch, first loads and epilogue.  Wide heads (split):
// O_1 and O_2 of 32 queries do not fit one wave's registers, so two waves share the queries, one map each, and meet in LDS at the end.
template <typename T, int NB> constexpr bool fwd_split() { return NB >= (sizeof(T) == 2 ? 5 : 4); }

enum { Q_HELD, Q_GLOBAL, Q_LDS };  // where a wave's queries are: registers, or read again for every tile
template <typename T, int NB, bool VECTOR, int Q, int MAPS> struct Fwd {
  static constexpr int CD = (NB + 1) / 2;
  typedef Img<T, CD> ImgK;
  typedef Img<T, NB> ImgV;
  int map0;        // the wave's (first) map
  const T* qrow;   // the lane's query, map 0 (Q_GLOBAL)
  int q_at, k_at, v_at;  // the lane's place in the images of Q (Q_LDS), K and V
  long qmap;       // from map to map
  Frag8<T> q[MAPS][Q == Q_HELD ? NB : 1];
  f32x16_t o[MAPS][NB];
  float m[MAPS], l[MAPS];  // m: both halves of a query agree; l: this half's keys

  __device__ __forceinline__ void init(int map, const T* row, long to_map, int d, int lane) {
    const int half = lane >> 5;
    map0 = map; qrow = row; qmap = to_map;
    q_at = 0; k_at = ImgK::rows_at(lane); v_at = ImgV::cols_at(lane);
    if constexpr (Q == Q_HELD)
#pragma unroll
      for (int i = 0; i < MAPS; ++i)
#pragma unroll
        for (int ks = 0; ks < NB; ++ks) load_frag<T, VECTOR>(qrow + (long)(map0 + i) * qmap, ks * 16 + half * 8, d, true, q[i][ks]);
#pragma unroll
    for (int i = 0; i < MAPS; ++i) {
      m[i] = NO_MAX; l[i] = 0.f;
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][n][r] = 0.f;
    }
  }
  // 32 keys: rows at kimg, vimg bytes into lds (kimg: the wave's first map, the other kbytes behind); qimg: the first map's queries (Q_LDS); vis: bit of
  // a key, the lane's half already shifted out
  __device__ __forceinline__ void tile(const unsigned char* lds, const unsigned char* qimg, int kimg, int kbytes, int vimg, bool masked, unsigned vis, float c, int d, int half) {
    const int kat = k_at + kimg, vat = v_at + vimg;
    f32x16_t sc[MAPS];
#pragma unroll
    for (int i = 0; i < MAPS; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[i][r] = 0.f;
#pragma unroll
    for (int i = 0; i < MAPS; ++i)
#pragma unroll
      for (int ks = 0; ks < NB; ++ks) {
        Frag8<T> a;
        ImgK::rows(lds + i * kbytes, kat, ks, a);
        if constexpr (Q == Q_LDS) ImgK::rows(qimg + i * 32 * ImgK::ROW_BYTES, q_at, ks, q[i][0]);
        if constexpr (Q == Q_GLOBAL) load_frag<T, VECTOR>(qrow + (long)(map0 + i) * qmap, ks * 16 + half * 8, d, true, q[i][0]);
        mma(a, q[i][Q == Q_HELD ? ks : 0], sc[i]);
        if (sizeof(T) == 4 || ks % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
    __builtin_amdgcn_sched_barrier(0);
    if (masked) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const bool keep = (vis >> (8 * (r >> 2) + (r & 3))) & 1u;
#pragma unroll
        for (int i = 0; i < MAPS; ++i) sc[i][r] = keep ? sc[i][r] : -INFINITY;
      }
    }
    float mx[MAPS];
    bool grew = false;
#pragma unroll
    for (int i = 0; i < MAPS; ++i) {
      mx[i] = sc[i][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mx[i] = fmaxf(mx[i], sc[i][r]);
      mx[i] *= c;
      grew = grew || mx[i] > m[i] + MAX_SLACK;
    }
    if (__any(grew)) {
#pragma unroll
      for (int i = 0; i < MAPS; ++i) {
        const float to = fmaxf(m[i], fmaxf(mx[i], other_half(mx[i])));
        const float f = exp2f(m[i] - to);
        m[i] = to;
        l[i] *= f;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[i][n][r] *= f;
      }
    }
    Frag8<T> pf[MAPS][2];
#pragma unroll
    for (int i = 0; i < MAPS; ++i) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        sc[i][r] = __builtin_amdgcn_exp2f(fmaf(sc[i][r], c, -m[i]));
        l[i] += sc[i][r];
      }
      to_frag(sc[i], 0, pf[i][0]);
      to_frag(sc[i], 1, pf[i][1]);
    }
    __builtin_amdgcn_sched_barrier(0);  // (operands loaded far ahead of their products would not fit the registers)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        Frag8<T> v;
        ImgV::cols(lds + 16 * t * ImgV::ROW_BYTES, vat, n, v);
#pragma unroll
        for (int i = 0; i < MAPS; ++i) mma(v, pf[i][t], o[i][n]);
        if (sizeof(T) == 4 || n % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
  }
};

// 1 / sum of a query's exponentials: zero without a visible key, NaN stays NaN
__device__ __forceinline__ float inverse_sum(float l) { return l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l); }
// log2 of the sum; +inf for a query without keys: exp2(score - inf) = 0 in the backward passes
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.f ? INFINITY : m + log2f(l); }

// many queries: workgroup = (batch, head, 128 queries), the waves' queries differ and the images are shared by the workgroup, one tile ahead
template <typename T, int NB> constexpr int fwd_threads() { return fwd_split<T, NB>() && sizeof(T) == 2 ? 512 : 256; }
template <typename T, int NB> constexpr int fwd_queries(int threads) { return threads / (fwd_split<T, NB>() ? 4 : 2); }
constexpr int at_least(int a, int b) { return a > b ? a : b; }
template <typename T, int NB> constexpr int fwd_lds() {
  return at_least(2 * key_tile<T>() * (2 * Img<T, (NB + 1) / 2>::ROW_BYTES + Img<T, NB>::ROW_BYTES), fwd_threads<T, NB>() / 64 * STRIP_BYTES);
}

template <typename T, int NB, bool VECTOR, int NT> __global__ __launch_bounds__(NT, 2) void diff_attn_fwd_kernel(tfpp_diff_attn_params p) {
  typedef Fwd<T, NB, VECTOR, (sizeof(T) == 2 ? VECTOR || NB < 8 : NB < 5) ? Q_HELD : Q_GLOBAL, fwd_split<T, NB>() ? 1 : 2> F;  // (wide fp32 heads do not fit the registers)
  typedef typename F::ImgK ImgK;
  typedef typename F::ImgV ImgV;
  constexpr int KT = key_tile<T>(), MAPS = fwd_split<T, NB>() ? 1 : 2, QB = fwd_queries<T, NB>(NT);
  constexpr int K_BYTES = KT * ImgK::ROW_BYTES, V_BYTES = KT * ImgV::ROW_BYTES, BUF = 2 * K_BYTES + V_BYTES;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int tiles = (p.Tq + QB - 1) / QB;
  int bh, tile;
  place(p.B * p.H, tiles, p.causal, bh, tile);
  if (p.causal) tile = tiles - 1 - tile;  // the longest rows first
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hkv);
  const Seq sq = sequence(p, b);
  const int w0 = tile * QB + (MAPS == 1 ? wave >> 1 : wave) * 32, qi = w0 + (lane & 31), qc = qi < p.Tq ? qi : p.Tq - 1;
  const T* kb = (const T*)p.k + (long)b * p.k_s[0] + (long)hk * p.k_s[2];
  const T* vb = (const T*)p.v + (long)b * p.v_s[0] + (long)hk * p.v_s[2];
  F f;
  f.init(MAPS == 1 ? wave & 1 : 0, (const T*)p.q + (long)b * p.q_s[0] + (long)qc * p.q_s[1] + (long)h * p.q_s[2], p.q_s[3], p.d, lane);
  const int last = tile * QB + QB < p.Tq ? tile * QB + QB : p.Tq;  // causal: the workgroup's last query bounds its keys
  int end = sq.len;
  if (p.causal) end = sq.start + last < end ? sq.start + last : end;
  const int steps = end > 0 ? (end + KT - 1) / KT : 0;
  const float c = p.scale * LOG2E;

  auto fill = [&](unsigned char* buf, int step, unsigned long long bits) {
    const long j0 = (long)step * KT;
    const Rows have = {sq.len - step * KT, p.key_mask != nullptr, bits};
#pragma unroll
    for (int i = 0; i < 2; ++i) ImgK::template fill<KT, VECTOR, NT>(buf + i * K_BYTES, kb + j0 * p.k_s[1] + i * p.k_s[3], p.k_s[1], p.d, have, tid);
    ImgV::template fill<KT, VECTOR, NT>(buf + 2 * K_BYTES, vb + j0 * p.v_s[1], p.v_s[1], p.dv, have, tid);
  };
  unsigned long long bits = 0;
  if (steps > 0) {
    bits = key_bits(p, b, 0, sq.len, lane);
    fill(smem, 0, bits);
  }
  for (int s = 0; s < steps; ++s) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();  // image s is complete, and every wave is past its reads of image s - 1
    const unsigned long long cur = bits;
    const bool more = s + 1 < steps;
    if (more) bits = key_bits(p, b, (s + 1) * KT, sq.len, lane);
    overlap(smem + (~s & 1) * BUF, smem + (s & 1) * BUF,
            [&](unsigned char* next) {
              if (more) fill(next, s + 1, bits);
            },
            [&](const unsigned char* now) {
              const int j0 = s * KT;
              const int seen = p.causal ? sq.start + w0 + 32 - j0 : KT;  // keys of this tile that the wave's last query sees
              if (seen <= 0 || cur == 0) return;
              const bool masked = (cur & low_bits(KT)) != low_bits(KT) || (p.causal && sq.start + w0 + 1 - j0 < KT);
              const unsigned long long mine = p.causal ? cur & low_bits(sq.start + qi + 1 - j0) : cur;
#pragma unroll 1
              for (int u = 0; u < KT / 32; ++u)
                f.tile(now, nullptr, f.map0 * K_BYTES + u * 32 * ImgK::ROW_BYTES, K_BYTES, 2 * K_BYTES + u * 32 * ImgV::ROW_BYTES, masked, (unsigned)(mine >> (u * 32)) >> (4 * half), c, p.d, half);
            });
  }

  const float lam = p.lam[p.n_lam > 1 ? h : 0];
  const long row0 = ((long)b * p.H + h) * p.Tq + w0;
  const int dvs = (p.dv + 7) & ~7, rows = p.Tq - w0;  // the wave's rows that exist
  float* strip = reinterpret_cast<float*>(smem + wave * STRIP_BYTES);
  static_assert(fwd_lds<T, NB>() >= NT / 64 * STRIP_BYTES, "the strips fit");
  __syncthreads();  // every wave is past its last image
#pragma unroll
  for (int i = 0; i < MAPS; ++i) {
    f.l[i] += other_half(f.l[i]);
    const float inv = inverse_sum(f.l[i]);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) f.o[i][n][r] *= inv;
    if (p.lse && (lane & 31) < rows && half == 0) p.lse[(long)(f.map0 + i) * p.B * p.H * p.Tq + row0 + lane] = log_sum(f.m[i], f.l[i]);
  }
  auto save = [&](void* to, const f32x16_t(&o)[NB]) {
    T* at = (T*)to + row0 * dvs;
    store_rows<T>(strip, lane, o, 1.f, dvs, true, Weights{nullptr, 0}, [&](int r) { return r < rows ? at + (long)r * dvs : nullptr; });
  };
  if constexpr (MAPS == 1) {  // O_2 of the odd waves to the even ones, in the registers' own order
    static_assert(fwd_lds<T, NB>() >= NT / 128 * NB * 16 * 64 * 4, "the exchange fits the images' LDS");
    float4* x = reinterpret_cast<float4*>(smem) + (wave >> 1) * (NB * 4 * 64) + lane;
    if (f.map0)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int g = 0; g < 4; ++g) x[(n * 4 + g) * 64] = make_float4(f.o[0][n][4 * g], f.o[0][n][4 * g + 1], f.o[0][n][4 * g + 2], f.o[0][n][4 * g + 3]);
    __syncthreads();
    if (!f.map0)
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 v = x[(n * 4 + g) * 64];
          f.o[0][n][4 * g] -= lam * v.x; f.o[0][n][4 * g + 1] -= lam * v.y; f.o[0][n][4 * g + 2] -= lam * v.z; f.o[0][n][4 * g + 3] -= lam * v.w;
        }
    __syncthreads();
    if (f.map0) {
      if (p.o2) save(p.o2, f.o[0]);
      return;
    }
  } else {
    if (p.o2) save(p.o2, f.o[MAPS - 1]);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) f.o[0][n][r] -= lam * f.o[MAPS - 1][n][r];
  }
  if (p.o1) save(p.o1, f.o[0]);  // (O and not P_1 V: rounded behind the subtraction, so that what both maps have in common is not in the rounding)
  float g = p.out_scale;
  if (p.norm) {
    float ss = 0.f;
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) ss += f.o[0][n][r] * f.o[0][n][r];
    ss += other_half(ss);
    g *= 1.f / sqrtf(ss / (float)p.dv + p.eps);
  }
  T* out = (T*)p.out + (long)b * p.o_s[0] + (long)w0 * p.o_s[1] + (long)h * p.o_s[2];
  store_rows<T>(strip, lane, f.o[0], g, p.dv, p.out_vec, Weights{p.norm_w, p.norm_w_bf16}, [&](int r) { return r < rows ? out + (long)r * p.o_s[1] : nullptr; });
}

// few queries (single tokens against a cache, short sequences): workgroup = (batch, key / value head, 32 rows, split of the keys), a row being a
// (query head of the group, query) pair, so that one read of the cache serves all heads that share it.  The WAVES take different keys, 32 at a time, from
// images of their own (no barrier in the loop), and add up in LDS.  With more than one split the sums go to `partial` and
// diff_attn_fwd_join_kernel finishes the rows: otherwise a cache would be read by as many CUs as there are heads.  Bounded by HBM where the cache is
// long: 16 sequences of 4096 to 16384 tokens, 4 heads of 64 / 128 shared by 16: 318 MB in 68 us (4.7 TB/s; a copy reaches 5.1) and 5 us for the join;
// by latency where it is short: 320 tokens, 17 us.
template <typename T, int NB> struct Few {
  static constexpr int MAPS = NB >= 5 ? 1 : 2;
  static constexpr int KEY_WAVES = MAPS == 2 ? 4 : (sizeof(T) == 2 ? 2 : 1), WAVES = KEY_WAVES * (3 - MAPS), THREADS = WAVES * 64;
  static constexpr int K_BYTES = 32 * Img<T, (NB + 1) / 2>::ROW_BYTES, V_BYTES = 32 * Img<T, NB>::ROW_BYTES, IMAGES = MAPS * K_BYTES + V_BYTES;
  static constexpr int STAGES = 2 * WAVES * IMAGES <= 128 * 1024 ? 2 : 1;
  static constexpr int BLOCK = 16 * 64;  // floats of a 32 x 32 fragment block
  static constexpr int EXCHANGE = WAVES * NB * BLOCK * 4;  // one map of every wave
  static constexpr int SUMS = WAVES * 2 * 32 * 2 * 4;      // (m, l) of every wave and map; later the rows' sums of squares
  static constexpr int QUERIES = 2 * K_BYTES;              // the 32 rows' queries, both maps
  static constexpr int LDS = at_least(at_least(STAGES * WAVES * IMAGES, EXCHANGE), WAVES * STRIP_BYTES) + QUERIES + SUMS;
  static constexpr int ROW_FLOATS = 2 * (NB * 32 + 2);     // of one row in `partial`: both maps' sums, maxima, l
};

template <typename T, int NB, bool VECTOR> __global__ __launch_bounds__((Few<T, NB>::THREADS), (sizeof(T) == 2 || NB <= 2 || NB == 5 ? 2 : 1)) void diff_attn_few_kernel(tfpp_diff_attn_params p) {
  typedef Few<T, NB> W;
  typedef Fwd<T, NB, VECTOR, Q_LDS, W::MAPS> F;
  typedef typename F::ImgK ImgK;
  typedef typename F::ImgV ImgV;
  constexpr int MAPS = W::MAPS, WAVES = W::WAVES, KW = W::KEY_WAVES;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5, col = lane & 31;
  const int group = p.H / p.Hkv, rows = group * p.Tq, tiles = (rows + 31) / 32, splits = p.splits;
  int bh = blockIdx.x / (tiles * splits);
  const int rest = blockIdx.x % (tiles * splits), tile = rest / splits, split = rest % splits;
  const int b = bh / p.Hkv, hk = bh % p.Hkv;
  const Seq sq = sequence(p, b);
  const int r = tile * 32 + col, rc = r < rows ? r : rows - 1, h = hk * group + rc / p.Tq, qi = rc % p.Tq;
  const bool live = r < rows;
  const T* kb = (const T*)p.k + (long)b * p.k_s[0] + (long)hk * p.k_s[2];
  const T* vb = (const T*)p.v + (long)b * p.v_s[0] + (long)hk * p.v_s[2];
  F f;
  f.init(MAPS == 1 ? wave & 1 : 0, nullptr, 0, p.d, lane);
  unsigned char* qimg = smem + (W::LDS - W::SUMS - W::QUERIES);
  f.q_at = ImgK::rows_at(lane);
  // the rows' queries into LDS, 16 bytes (or elements, unaligned) at a time; their rows lie in several heads, so not by `fill`
  for (int i = tid; i < 2 * 32 * ImgK::USED; i += W::THREADS) {
    const int map = i / (32 * ImgK::USED), qr = i / ImgK::USED % 32, ch = i % ImgK::USED, n = tile * 32 + qr < rows ? tile * 32 + qr : rows - 1;
    const T* src = (const T*)p.q + (long)b * p.q_s[0] + (long)(n % p.Tq) * p.q_s[1] + (long)(hk * group + n / p.Tq) * p.q_s[2] + (long)map * p.q_s[3] + ch * ImgK::VEC;
    uint4 u = make_uint4(0, 0, 0, 0);
    if constexpr (VECTOR) {
      if (ch * ImgK::VEC < p.d) u = *reinterpret_cast<const uint4*>(src);
    } else {
      float t[ImgK::VEC];
#pragma unroll
      for (int e = 0; e < ImgK::VEC; ++e) t[e] = ch * ImgK::VEC + e < p.d ? ElemTraits<T>::to_f(src[e]) : 0.f;
      u = pack16<T>(t);
    }
    *reinterpret_cast<uint4*>(qimg + map * W::K_BYTES + ImgK::off(qr, ch)) = u;
  }
  __syncthreads();
  // keys of this split: whole blocks of 32, an equal share of what the tile's rows see
  int end = sq.len;
  if (p.causal) {
    const int r1 = tile * 32 + 31 < rows ? tile * 32 + 31 : rows - 1, last = tile * 32 / p.Tq == r1 / p.Tq ? r1 % p.Tq : p.Tq - 1;
    end = sq.start + last + 1 < end ? sq.start + last + 1 : end;
  }
  const int blocks = end > 0 ? (end + 31) / 32 : 0, per = (blocks + splits - 1) / splits;
  const int first = split * per, stop = first + per < blocks ? first + per : blocks;
  const float c = p.scale * LOG2E;
  const int lim = p.causal ? sq.start + qi + 1 : end;  // keys this row sees

  auto fill = [&](unsigned char* buf, int block, unsigned bits) {
    const long j0 = (long)block * 32;
    const Rows have = {sq.len - block * 32, p.key_mask != nullptr, bits};
#pragma unroll
    for (int i = 0; i < MAPS; ++i) ImgK::template fill<32, VECTOR, 64>(buf + i * W::K_BYTES, kb + j0 * p.k_s[1] + (f.map0 + i) * p.k_s[3], p.k_s[1], p.d, have, lane);
    ImgV::template fill<32, VECTOR, 64>(buf + MAPS * W::K_BYTES, vb + j0 * p.v_s[1], p.v_s[1], p.dv, have, lane);
  };
  auto use = [&](const unsigned char* buf, int block, unsigned seen) {
    const unsigned mine = seen & (unsigned)low_bits(lim - block * 32);
    f.tile(buf, qimg + f.map0 * W::K_BYTES, 0, W::K_BYTES, MAPS * W::K_BYTES, __any(mine != ~0u), mine >> (4 * half), c, p.d, half);
  };
  const int kw = MAPS == 1 ? wave >> 1 : wave;
  unsigned char* images = smem + wave * W::STAGES * W::IMAGES;
  unsigned bits = 0;
  int stage = 0;
  if (first + kw < stop) {
    bits = (unsigned)key_bits(p, b, (first + kw) * 32, sq.len, lane);
    fill(images, first + kw, bits);
  }
  for (int k = first + kw; k < stop; k += KW) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // this wave's images are complete
    const unsigned cur = bits;
    const bool more = k + KW < stop;
    if (more) bits = (unsigned)key_bits(p, b, (k + KW) * 32, sq.len, lane);
    if constexpr (W::STAGES == 2) {
      overlap(images + (stage ^ 1) * W::IMAGES, images + stage * W::IMAGES,
              [&](unsigned char* next) {
                if (more) fill(next, k + KW, bits);
              },
              [&](const unsigned char* now) { use(now, k, cur); });
      stage ^= 1;
    } else {
      use(images, k, cur);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (every read of the image has returned before it is filled again)
      if (more) fill(images, k + KW, bits);
    }
  }

  // add the waves up: maxima and sums of all waves first, then each map's O, block by block; wave w finishes the channel blocks w, w + WAVES, ..
  float* ml = reinterpret_cast<float*>(smem + (W::LDS - W::SUMS));  // [wave][map of the wave][m, l][32]
  float4* x = reinterpret_cast<float4*>(smem);
#pragma unroll
  for (int i = 0; i < MAPS; ++i) {
    f.l[i] += other_half(f.l[i]);
    if (half == 0) {
      ml[((wave * 2 + i) * 2) * 32 + col] = f.m[i];
      ml[((wave * 2 + i) * 2 + 1) * 32 + col] = f.l[i];
    }
  }
  __syncthreads();
  float M[2], L[2];
#pragma unroll
  for (int map = 0; map < 2; ++map) {
    M[map] = NO_MAX;
    L[map] = 0.f;
#pragma unroll
    for (int w = 0; w < KW; ++w) M[map] = fmaxf(M[map], ml[(((MAPS == 1 ? 2 * w + map : w) * 2 + (MAPS == 1 ? 0 : map)) * 2) * 32 + col]);
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      const float* q = ml + (((MAPS == 1 ? 2 * w + map : w) * 2 + (MAPS == 1 ? 0 : map)) * 2) * 32 + col;
      L[map] += q[32] * exp2f(q[0] - M[map]);
    }
  }
  constexpr int MINE = (NB + WAVES - 1) / WAVES;
  f32x16_t o[2][MINE];
#pragma unroll
  for (int round = 0; round < MAPS; ++round) {
    const float g = exp2f(f.m[round] - (MAPS == 1 ? (f.map0 ? M[1] : M[0]) : M[round]));
    if (round) __syncthreads();
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[((wave * NB + n) * 4 + e) * 64 + lane] = make_float4(f.o[round][n][4 * e] * g, f.o[round][n][4 * e + 1] * g, f.o[round][n][4 * e + 2] * g, f.o[round][n][4 * e + 3] * g);
        if (e == 3) __builtin_amdgcn_sched_barrier(0);
      }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
      const int n = wave + j * WAVES;
#pragma unroll
      for (int map = 0; map < 2; ++map) {
        if (MAPS == 2 && map != round) continue;
#pragma unroll
        for (int e = 0; e < 16; ++e) o[map][j][e] = 0.f;
        if (n < NB)
#pragma unroll
          for (int w = 0; w < KW; ++w) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float4 v = x[(((MAPS == 1 ? 2 * w + map : w) * NB + n) * 4 + e) * 64 + lane];
              o[map][j][4 * e] += v.x; o[map][j][4 * e + 1] += v.y; o[map][j][4 * e + 2] += v.z; o[map][j][4 * e + 3] += v.w;
            }
            __builtin_amdgcn_sched_barrier(0);
          }
      }
    }
  }
  if (splits > 1) {
    float* out = p.partial + ((((long)split * p.B + b) * p.Hkv + hk) * rows + rc) * W::ROW_FLOATS;
    if (!live) return;
#pragma unroll
    for (int map = 0; map < 2; ++map) {
#pragma unroll
      for (int j = 0; j < MINE; ++j)
        if (wave + j * WAVES < NB)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<float4*>(out + map * NB * 32 + (wave + j * WAVES) * 32 + 8 * g + 4 * half) = make_float4(o[map][j][4 * g], o[map][j][4 * g + 1], o[map][j][4 * g + 2], o[map][j][4 * g + 3]);
      if (wave == 0 && half == 0) {
        out[2 * NB * 32 + map * 2] = M[map];
        out[2 * NB * 32 + map * 2 + 1] = L[map];
      }
    }
    return;
  }
  const float lam = p.lam[p.n_lam > 1 ? h : 0];
  const int dvs = (p.dv + 7) & ~7;
  static_assert(W::LDS - W::SUMS >= WAVES * STRIP_BYTES, "the strips fit");
  float* strip = reinterpret_cast<float*>(smem + wave * STRIP_BYTES);
  const int row0 = tile * 32;
  auto head_of = [&](int r) { return hk * group + (row0 + r) / p.Tq; };
  __syncthreads();  // every wave has read the exchange
#pragma unroll
  for (int map = 0; map < 2; ++map) {
    const float inv = inverse_sum(L[map]);
    if (p.lse && live && half == 0 && wave == 0) p.lse[((long)map * p.B + b) * p.H * p.Tq + (long)h * p.Tq + qi] = log_sum(M[map], L[map]);
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
#pragma unroll
      for (int e = 0; e < 16; ++e) o[map][j][e] *= inv;
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < MINE; ++j)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      o[0][j][e] -= lam * o[1][j][e];
      ss += o[0][j][e] * o[0][j][e];
    }
  if (p.o1)
#pragma unroll
    for (int i = 0; i < 2; ++i)  // O and O_2
#pragma unroll
      for (int j = 0; j < MINE; ++j)
        if (wave + j * WAVES < NB) {
          T* to = (T*)(i ? p.o2 : p.o1);
          strip_put(strip, lane, 0, o[i][j], 1.f);
          __builtin_amdgcn_wave_barrier();
          strip_store<T>(strip, lane, 1, (wave + j * WAVES) * 32, dvs, true, Weights{nullptr, 0},
                         [&](int r) { return row0 + r < rows ? to + (((long)b * p.H + head_of(r)) * p.Tq + (row0 + r) % p.Tq) * dvs : nullptr; });
          __builtin_amdgcn_wave_barrier();
        }
  float g = p.out_scale;
  if (p.norm) {
    ss += other_half(ss);
    __syncthreads();  // (m and l have been read)
    if (half == 0) ml[wave * 32 + col] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) ss += ml[w * 32 + col];
    g *= 1.f / sqrtf(ss / (float)p.dv + p.eps);
  }
  T* out = (T*)p.out + (long)b * p.o_s[0];
#pragma unroll
  for (int j = 0; j < MINE; ++j)
    if (wave + j * WAVES < NB) {
      strip_put(strip, lane, 0, o[0][j], g);
      __builtin_amdgcn_wave_barrier();
      strip_store<T>(strip, lane, 1, (wave + j * WAVES) * 32, p.dv, p.out_vec, Weights{p.norm_w, p.norm_w_bf16},
                     [&](int r) { return row0 + r < rows ? out + (long)((row0 + r) % p.Tq) * p.o_s[1] + (long)head_of(r) * p.o_s[2] : nullptr; });
      __builtin_amdgcn_wave_barrier();
    }
}

// the splits' sums of a row -> its result: one wave a row, channels 4 lane ..; lane s holds split s's maxima and sums (splits <= 64)
template <typename T> __global__ __launch_bounds__(256) void diff_attn_fwd_join_kernel(tfpp_diff_attn_params p, int width) {
  const int lane = threadIdx.x & 63, group = p.H / p.Hkv, rows = group * p.Tq, dvs = (p.dv + 7) & ~7, c = lane * 4;
  const long n = (long)blockIdx.x * 4 + (threadIdx.x >> 6), all = (long)p.B * p.Hkv * rows, pitch = 2 * width + 4;
  if (n >= all) return;
  const int r = (int)(n % rows), hk = (int)(n / rows % p.Hkv), b = (int)(n / rows / p.Hkv), h = hk * group + r / p.Tq, qi = r % p.Tq;
  const float* src = p.partial + n * pitch;
  const long row = ((long)b * p.H + h) * p.Tq + qi;
  float4 ml = make_float4(NO_MAX, 0.f, NO_MAX, 0.f);  // m_1, l_1, m_2, l_2
  if (lane < p.splits) ml = *reinterpret_cast<const float4*>(src + lane * all * pitch + 2 * width);
  const float M[2] = {wave_max(ml.x), wave_max(ml.z)};
  const float f[2] = {exp2f(ml.x - M[0]), exp2f(ml.z - M[1])};
  const float L[2] = {wave_sum(f[0] * ml.y), wave_sum(f[1] * ml.w)};
  float4 o[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
  __shared__ float fs[4][2][64];
  float(*mine)[64] = fs[threadIdx.x >> 6];
  mine[0][lane] = f[0];
  mine[1][lane] = f[1];
  __builtin_amdgcn_wave_barrier();
  const float* q0 = src + (c < width ? c : 0);
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float* q = q0 + s * all * pitch;
#pragma unroll
    for (int map = 0; map < 2; ++map) {
      const float w = mine[map][s];
      const float4 v = *reinterpret_cast<const float4*>(q + map * width);
      o[map].x += w * v.x; o[map].y += w * v.y; o[map].z += w * v.z; o[map].w += w * v.w;
    }
  }
  const float lam = p.lam[p.n_lam > 1 ? h : 0];
  float d[4];
#pragma unroll
  for (int map = 0; map < 2; ++map) {
    const float inv = inverse_sum(L[map]);
    if (p.lse && lane == 0) p.lse[(long)map * p.B * p.H * p.Tq + row] = log_sum(M[map], L[map]);
    const float f = c < width ? inv : 0.f;  // (the lanes behind the last channel have read channel 0)
    const float v[4] = {o[map].x * f, o[map].y * f, o[map].z * f, o[map].w * f};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      d[e] = map ? d[e] - lam * v[e] : v[e];
      if (p.o1 && map && c + e < dvs) {
        ((T*)p.o1)[row * dvs + c + e] = ElemTraits<T>::from_f(d[e]);
        ((T*)p.o2)[row * dvs + c + e] = ElemTraits<T>::from_f(v[e]);
      }
    }
  }
  float g = p.out_scale;
  if (p.norm) g *= 1.f / sqrtf(wave_sum(d[0] * d[0] + d[1] * d[1] + d[2] * d[2] + d[3] * d[3]) / (float)p.dv + p.eps);
  T* out = (T*)p.out + (long)b * p.o_s[0] + (long)qi * p.o_s[1] + (long)h * p.o_s[2];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < p.dv) out[c + e] = ElemTraits<T>::from_f(d[e] * (p.norm_w ? g * Weights{p.norm_w, p.norm_w_bf16}[c + e] : g));
}

// ---------------------------------------------------------------------------------------------------------------------------------
// backward, in three launches and a sum (nothing is accumulated by atomics: the same bits from run to run).  With u = out_scale w dout:
//   r = 1 / sqrt(mean(O^2) + eps)      dO = r u - O r^3 mean(u O)  (without the norm: dO = u)     dw = sum out_scale dout O r     dlambda = - sum dO . O_2
//   dP = dO V^T      delta_i = dO . O_i      dS_1 = P_1 (dP - delta_1)      dS_2 = -lambda P_2 (dP - delta_2)
//   dQ_i = scale dS_i K_i      dK_i = scale dS_i^T Q_i      dV = (P_1 - lambda P_2)^T dO
// 1. diff_attn_bwd_rows_kernel: dO (rounded once: it is an MFMA operand twice), delta_i from that rounded dO, as dP is, with O_1 = O + lambda O_2 of the
//    saved O and O_2 (whose rounding, 2^-8 relative at most, stays in delta_i), and partial sums of dw, dlambda from the unrounded dO.
//    The forward pass saves O, not O_1: r, dO and dw are made of it, and a difference of two saved maps would hold their roundings, |O_1| / |O| times as
//    large (64 / 128, V of mean 1, lambda 0.95: dw 1.8e-2 off, 3.4e-3 with O saved).  For bf16 also g, see dQ.
//    Bounded by HBM: 131072 rows of 128, 168 MB in 44 us (3.8 TB/s).
// grid (blocks, H); lpr lanes a row (a power of two), 8 channels a lane: 16-byte loads, 64 / lpr rows a wave at a time.  partial: [1 + dv][blocks x H], the
// sums of one value side by side.
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) { return v + __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true)); }
__device__ __forceinline__ float row_sum(float v, int lpr) {  // of lpr neighbouring lanes, in each of them; moves within 16 lanes cost no LDS round trip
  if (lpr > 1) v = dpp_add<0xB1>(v);   // lane ^ 1
  if (lpr > 2) v = dpp_add<0x4E>(v);   // lane ^ 2
  if (lpr > 4) v = dpp_add<0x141>(v);  // mirror within 8
  if (lpr > 8) v = dpp_add<0x140>(v);  // mirror within 16
  if (lpr > 16) v += __shfl_xor(v, 16, 64);
  return v;
}
template <typename T> __global__ __launch_bounds__(256) void diff_attn_bwd_rows_kernel(tfpp_diff_attn_params p, int lpr) {
  constexpr int E = 8;
  __shared__ float sm[4 * 256 + 4];  // of each wave: the columns' sums; dlambda
  const int h = blockIdx.y, lane = threadIdx.x & 63, c0 = (lane & (lpr - 1)) * E, dvs = (p.dv + 7) & ~7;
  const int rpw = 64 / lpr, slots = (int)gridDim.x * 4 * rpw;
  const long rows = (long)p.B * p.Tq;
  const float lam = p.lam[p.n_lam > 1 ? h : 0], inv_dv = 1.f / (float)p.dv;
  constexpr bool SLOPE = sizeof(T) == 2;
  float w[E], dw[E], dl = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    w[e] = c0 + e < p.dv ? p.out_scale * (p.norm_w ? Weights{p.norm_w, p.norm_w_bf16}[c0 + e] : 1.f) : 0.f;
    dw[e] = 0.f;
  }
  const long first = ((long)blockIdx.x * 4 + (threadIdx.x >> 6)) * rpw + lane / lpr;
  const long rounds = (rows + slots - 1) / slots;
  for (long k = 0; k < rounds; ++k) {  // (the same number of rounds in every lane: the shuffles below need them all)
    const long n = first + k * slots;
    const bool live = n < rows, in = live && c0 < dvs;
    const int b = live ? (int)(n / p.Tq) : 0, t = live ? (int)(n % p.Tq) : 0;
    const long row = ((long)b * p.H + h) * p.Tq + t;
    const T* dout = (const T*)p.dout + (long)b * p.do_s[0] + (long)t * p.do_s[1] + (long)h * p.do_s[2] + c0;
    float g[E], o[E], o2[E];
#pragma unroll
    for (int e = 0; e < E; ++e) g[e] = o[e] = o2[e] = 0.f;
    if (in) {
#pragma unroll
      for (int e = 0; e < E; e += ElemTraits<T>::VEC) {
        load_vec<T>((const T*)p.o1 + row * dvs + c0 + e, o + e);
        load_vec<T>((const T*)p.o2 + row * dvs + c0 + e, o2 + e);
      }
      if (p.do_vec && c0 + E <= p.dv) {
#pragma unroll
        for (int e = 0; e < E; e += ElemTraits<T>::VEC) load_vec<T>(dout + e, g + e);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c0 + e < p.dv) g[e] = ElemTraits<T>::to_f(dout[e]);
      }
    }
    float ss = 0.f, uo = 0.f, oo2 = 0.f, uo2 = 0.f, r = 1.f, a = 0.f, f = 0.f;  // (channels behind dv: V is zero there, so are O and O_2)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float u = w[e] * g[e];
      ss += o[e] * o[e];
      uo += u * o[e];
      if constexpr (SLOPE) {
        oo2 += o[e] * o2[e];
        uo2 += u * o2[e];
      }
    }
    if (p.norm) {
      ss = row_sum(ss, lpr);
      uo = row_sum(uo, lpr);
      if constexpr (SLOPE) {
        oo2 = row_sum(oo2, lpr);
        uo2 = row_sum(uo2, lpr);
      }
      r = 1.f / sqrtf(ss * inv_dv + p.eps);  // (eps > 0: checked by the launcher)
      a = r * inv_dv * uo;                   // mean(u O^), O^ = r O; every product below has O^, which is at most sqrt(dv) in size whatever r is
      f = r * inv_dv;
    }
    const float b2 = r * oo2, c2 = uo2 - 3.f * a * b2;  // O^ . O_2
    float d[E], sg[E], t1 = 0.f, t2 = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float u = w[e] * g[e], on = r * o[e];
      dw[e] += p.out_scale * g[e] * on;
      d[e] = r * (u - on * a);
      dl -= d[e] * o2[e];
      const float dr = ElemTraits<T>::to_f(ElemTraits<T>::from_f(d[e]));
      t1 += dr * (o[e] + lam * o2[e]);
      t2 += dr * o2[e];
      if constexpr (SLOPE) {
        sg[e] = -r * (f * (c2 * on + b2 * u) + a * o2[e] * r);
        dl += ElemTraits<T>::to_f(ElemTraits<T>::from_f(sg[e])) * o[e];
      }
    }
    t1 = row_sum(t1, lpr);
    t2 = row_sum(t2, lpr);
    if (in)
#pragma unroll
      for (int e = 0; e < E; e += ElemTraits<T>::VEC) {
        store_vec<T>((T*)p.d_o + row * dvs + c0 + e, d + e);
        if constexpr (SLOPE) store_vec<T>((T*)p.slope + row * dvs + c0 + e, sg + e);
      }
    if (live && c0 == 0) {
      p.delta[row] = t1;
      p.delta[(long)p.B * p.H * p.Tq + row] = t2;
    }
  }
  for (int x = lpr; x < 64; x <<= 1)  // the wave's rows
#pragma unroll
    for (int e = 0; e < E; ++e) dw[e] += __shfl_xor(dw[e], x, 64);
  if (lane < lpr)
#pragma unroll
    for (int e = 0; e < E; ++e) sm[((int)threadIdx.x >> 6) * 256 + c0 + e] = dw[e];
  dl = wave_sum(dl);
  if (lane == 0) sm[4 * 256 + (threadIdx.x >> 6)] = dl;
  __syncthreads();
  const long pitch = (long)gridDim.x * p.H, at = (long)blockIdx.x * p.H + h;
  if (threadIdx.x == 0) p.partial[at] = (sm[1024] + sm[1025]) + (sm[1026] + sm[1027]);
  const int c = threadIdx.x;
  if (c < p.dv) p.partial[(1 + c) * pitch + at] = (sm[c] + sm[256 + c]) + (sm[512 + c] + sm[768 + c]);
}

// dlambda (blocks 0 .. n_lam - 1) and dw (the blocks behind): one value per workgroup, fixed order
template <typename T> __global__ __launch_bounds__(256) void diff_attn_bwd_sum_kernel(tfpp_diff_attn_params p, int blocks, const float* rest, int rest_rows) {
  __shared__ float sm[4];
  const int x = blockIdx.x, n = blocks * p.H;
  const bool is_lam = x < p.n_lam;
  const int c = is_lam ? 0 : 1 + x - p.n_lam;
  const float* src = p.partial + (long)c * n;
  float s = 0.f;
  if (is_lam && p.n_lam > 1)
    for (int i = threadIdx.x; i < blocks; i += 256) s += src[(long)i * p.H + x];
  else
    for (int i = threadIdx.x; i < n; i += 256) s += src[i];
  if (is_lam && p.n_lam > 1)
    for (int i = threadIdx.x; i < rest_rows; i += 256) s -= rest[(long)i * p.H + x];
  else if (is_lam)
    for (long i = threadIdx.x; i < (long)rest_rows * p.H; i += 256) s -= rest[i];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x) return;
  s = (sm[0] + sm[1]) + (sm[2] + sm[3]);
  if (is_lam) p.dlam[x] = s;
  else if (p.norm_w_bf16) ((bf16_t*)p.dnorm_w)[c - 1] = f2bf(s);
  else ((float*)p.dnorm_w)[c - 1] = s;
}

// 2. dQ.  Workgroup = (batch, head, 128 queries), wave = 32 queries, as the forward pass: S_i^T = K_i Q_i^T, dP^T = V dO^T (keys x queries),
//    dQ_i^T += K_i^T dS_i^T.  The row's sum, delta_i and limits are one value a lane.  2 x 4096 causal, 16 heads of 64 / 128: 331 us, vector
//    issue in 65 % of the cycles, the matrix unit in 38 %, LDS in 17 %; 12 x 320, 4 heads of 72 / 144: 28 us.
//    bf16: dlambda = - sum f, f = dO(O) . O_2, is a sum that cancels, and the row pass has it from the saved O and O_2, which are rounded and made of
//    rounded probabilities: percents of it where the heads are few.  Here P is at hand in 32 bits, and both are put right to first order:
//      O_2 beside dO:  sum_j P_2 (dP - delta_2) = dO . (O_2 - saved O_2)
//      O inside dO:    sum_j (P_1 - lambda P_2) g . V_j - g . saved O = g . (O - saved O),  g = df/dO = - r^2 / dv ((u . O_2 - 3 a b) O^ + b u + dv a O_2)
//                      with O^ = r O, a = mean(u O^), b = O^ . O_2  (the row pass subtracts g . saved O)
//    The product with g shares the V operand of dP: 2 dv of 8 d + 4 dv flop a pair.  What is left is of second order, 1e-5 of the terms' root
//    (before: 2e-3 to 3e-2).  2 x 4096 causal: 273 -> 331 us; 12 x 320: 23 -> 28 us.
//    Wide heads: a workgroup has one map (the grid's y), dP is computed by both, and two waves fit a SIMD in place of one
//    (12 x 320 queries over 1280 keys, without g: 68 us, 82 us with both maps in a wave).  bf16 heads of 81 .. 128 hold q, dO, g and dQ in the registers of
//    one wave a SIMD (8 heads of 128 / 256 over 2 x 2048: backward 456 us; with both maps in a wave 481).
template <typename T, int NB> constexpr int dq_maps() { return NB >= (sizeof(T) == 2 ? 5 : 4) ? 1 : 2; }
template <typename T, int NB, bool VECTOR> constexpr int dq_waves() { return sizeof(T) == 2 && NB == 8 && VECTOR ? 1 : 2; }  // of a SIMD
// bf16 heads of 33 .. 64: the last fragments of a wave's g stay in LDS, which spares the registers that would go to scratch
template <typename T, int NB, bool VECTOR> constexpr int dq_stash() { return sizeof(T) == 2 && NB == 4 && VECTOR ? 4 : 0; }
template <typename T, int NB> constexpr int dq_images() { return 2 * 32 * (dq_maps<T, NB>() * Img<T, (NB + 1) / 2>::ROW_BYTES + Img<T, NB>::ROW_BYTES); }
template <typename T, int NB, bool VECTOR> constexpr int dq_lds() { return at_least(dq_images<T, NB>() + dq_stash<T, NB, VECTOR>() * 256 * 16, 4 * STRIP_BYTES); }

template <typename T, int NB, bool VECTOR> __global__ __launch_bounds__(256, (dq_waves<T, NB, VECTOR>())) void diff_attn_bwd_dq_kernel(tfpp_diff_attn_params p) {
  constexpr int KT = 32, NT = 256, CD = (NB + 1) / 2, MAPS = dq_maps<T, NB>();
  typedef Img<T, CD> ImgK;
  typedef Img<T, NB> ImgV;
  constexpr int K_BYTES = KT * ImgK::ROW_BYTES, V_BYTES = KT * ImgV::ROW_BYTES, BUF = MAPS * K_BYTES + V_BYTES;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int tiles = (p.Tq + QB - 1) / QB;
  int bh, tile;
  place(p.B * p.H, tiles, p.causal, bh, tile);
  if (p.causal) tile = tiles - 1 - tile;
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hkv), dvs = (p.dv + 7) & ~7;
  const Seq sq = sequence(p, b);
  const int w0 = tile * QB + wave * 32, qi = w0 + (lane & 31), qc = qi < p.Tq ? qi : p.Tq - 1;
  const long row = ((long)b * p.H + h) * p.Tq + qc, rows = (long)p.B * p.H * p.Tq;
  const int map0 = MAPS == 1 ? (int)blockIdx.y : 0;
  const T* kb = (const T*)p.k + (long)b * p.k_s[0] + (long)hk * p.k_s[2] + map0 * p.k_s[3];
  const T* vb = (const T*)p.v + (long)b * p.v_s[0] + (long)hk * p.v_s[2];
  constexpr bool HOLD = VECTOR ? sizeof(T) == 2 || NB < 5 : NB < 4;  // else Q and dO do not fit the registers and are read again for every tile
  const T* qrow = (const T*)p.q + (long)b * p.q_s[0] + (long)qc * p.q_s[1] + (long)h * p.q_s[2] + map0 * p.q_s[3];
  constexpr bool SLOPE = sizeof(T) == 2;
  constexpr int STASH = dq_stash<T, NB, VECTOR>(), HELD = 2 * NB - STASH;
  static_assert(!STASH || (HOLD && SLOPE), "what is put away are held fragments of g");
  Frag8<T> q[MAPS][HOLD ? NB : 1], dof[HOLD ? 2 * NB : 1], slope[HOLD && SLOPE ? HELD : 1];
  if constexpr (HOLD) {
#pragma unroll
    for (int i = 0; i < MAPS; ++i)
#pragma unroll
      for (int ks = 0; ks < NB; ++ks) load_frag<T, VECTOR>(qrow + (long)i * p.q_s[3], ks * 16 + half * 8, p.d, true, q[i][ks]);
#pragma unroll
    for (int ks = 0; ks < 2 * NB; ++ks) {
      load_frag<T, true>((const T*)p.d_o + row * dvs, ks * 16 + half * 8, dvs, true, dof[ks]);
      if constexpr (SLOPE) {
        Frag8<T> g;
        load_frag<T, true>((const T*)p.slope + row * dvs, ks * 16 + half * 8, dvs, true, g);
        if (ks < HELD) slope[ks < HELD ? ks : 0] = g;
        else if constexpr (STASH) *reinterpret_cast<uint4*>(smem + 2 * BUF + ((ks - HELD) * NT + tid) * 16) = g.v;  // (read by the lane that wrote it)
      }
    }
  }
  const bool exists = qi < p.Tq;  // (the lanes behind the last query: P = 0)
  const float lse[2] = {exists ? p.lse[map0 * rows + row] : INFINITY, exists ? p.lse[rows + row] : INFINITY}, delta[2] = {p.delta[map0 * rows + row], p.delta[rows + row]};  // (one map: the first of each)
  const float lam = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(p.lam[p.n_lam > 1 ? h : 0]))), sign = map0 ? -lam : 1.f, c = p.scale * LOG2E;
  const int last = tile * QB + QB < p.Tq ? tile * QB + QB : p.Tq;
  int end = sq.len;
  if (p.causal) end = sq.start + last < end ? sq.start + last : end;
  const int steps = end > 0 ? (end + KT - 1) / KT : 0;
  f32x16_t dq[MAPS][CD];
#pragma unroll
  for (int i = 0; i < MAPS; ++i)
#pragma unroll
    for (int n = 0; n < CD; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) dq[i][n][r] = 0.f;
  float rest = 0.f, rise = 0.f;  // sums of the last map's P_2 (dP - delta_2), of (P_1 - lambda P_2) g . V (one map a workgroup: of its P g . V)
  const int k_rows = ImgK::rows_at(lane), v_rows = ImgV::rows_at(lane), k_cols = ImgK::cols_at(lane);
  auto fill = [&](unsigned char* buf, int step, unsigned long long bits) {
    const long j0 = (long)step * KT;
    const Rows have = {sq.len - step * KT, p.key_mask != nullptr, bits};
    int tid = (int)threadIdx.x;
    if (STASH) asm volatile("" : "+v"(tid));  // (the offsets made of it are worked out again each time: kept, they would not fit the registers)
#pragma unroll
    for (int i = 0; i < MAPS; ++i) ImgK::template fill<KT, VECTOR, NT>(buf + i * K_BYTES, kb + j0 * p.k_s[1] + i * p.k_s[3], p.k_s[1], p.d, have, tid);
    ImgV::template fill<KT, VECTOR, NT>(buf + MAPS * K_BYTES, vb + j0 * p.v_s[1], p.v_s[1], p.dv, have, tid);
  };
  unsigned long long bits = 0;
  if (steps > 0) {
    bits = key_bits(p, b, 0, sq.len, lane);
    fill(smem, 0, bits);
  }
  for (int s = 0; s < steps; ++s) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const unsigned long long cur = bits & low_bits(KT);
    const bool more = s + 1 < steps;
    if (more) bits = key_bits(p, b, (s + 1) * KT, sq.len, lane);
    overlap(smem + (~s & 1) * BUF, smem + (s & 1) * BUF,
            [&](unsigned char* next) {
              if (more) fill(next, s + 1, bits);
            },
            [&](const unsigned char* now) {
    const int j0 = s * KT;
    // (no early way out for a tile that the wave's queries do not see: with accumulators in AGPRs a branch round their products costs a copy of all of
    // them at every step; such a tile is masked to zeros)
    const bool masked = cur != low_bits(KT) || (p.causal && sq.start + w0 + 1 - j0 < KT);
    const unsigned vis = (unsigned)(p.causal ? cur & low_bits(sq.start + qi + 1 - j0) : cur) >> (4 * half);
    const int vr = v_rows + MAPS * K_BYTES;
    f32x16_t sc[MAPS], dp, gv;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      dp[r] = gv[r] = 0.f;
#pragma unroll
      for (int i = 0; i < MAPS; ++i) sc[i][r] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < MAPS; ++i)
#pragma unroll
      for (int ks = 0; ks < NB; ++ks) {
        Frag8<T> a;
        ImgK::rows(now + i * K_BYTES, k_rows, ks, a);
        if constexpr (!HOLD) load_frag<T, VECTOR>(qrow + (long)i * p.q_s[3], ks * 16 + half * 8, p.d, true, q[i][0]);
        mma(a, q[i][HOLD ? ks : 0], sc[i]);
        if (STASH && ks % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (operands loaded far ahead of their products would not fit the registers)
      }
#pragma unroll
    for (int ks = 0; ks < 2 * NB; ++ks) {
      Frag8<T> a;
      ImgV::rows(now, vr, ks, a);
      if constexpr (!HOLD) load_frag<T, true>((const T*)p.d_o + row * dvs, ks * 16 + half * 8, dvs, true, dof[0]);
      mma(a, dof[HOLD ? ks : 0], dp);
      if constexpr (SLOPE) {
        if constexpr (!HOLD) load_frag<T, true>((const T*)p.slope + row * dvs, ks * 16 + half * 8, dvs, true, slope[0]);
        if (HOLD && ks >= HELD) {
          Frag8<T> g;
          if constexpr (STASH) g.v = *reinterpret_cast<const uint4*>(now + (2 - (s & 1)) * BUF + ((ks - HELD) * NT + tid) * 16);  // (an address made of `now`: see overlap)
          mma(a, g, gv);
        } else {
          mma(a, slope[HOLD ? (ks < HELD ? ks : 0) : 0], gv);
        }
      }
      if (STASH && ks % 4 == 3) __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const bool keep = !masked || ((vis >> (8 * (r >> 2) + (r & 3))) & 1u);
#pragma unroll
      for (int i = 0; i < MAPS; ++i) {
        float pr = __builtin_amdgcn_exp2f(fmaf(sc[i][r], c, -lse[i]));
        if (masked) pr = keep ? pr : 0.f;
        const float ds = pr * (dp[r] - delta[i]);
        if (i == MAPS - 1) rest += ds;
        if constexpr (SLOPE) rise += (i ? -lam * pr : pr) * gv[r];
        sc[i][r] = ds * (MAPS == 1 ? sign : (i ? -lam : 1.f));
      }
    }
#pragma unroll
    for (int i = 0; i < MAPS; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        Frag8<T> ds;
        to_frag(sc[i], t, ds);
#pragma unroll
        for (int n = 0; n < CD; ++n) {
          Frag8<T> a;
          ImgK::cols(now + i * K_BYTES + 16 * t * ImgK::ROW_BYTES, k_cols, n, a);
          mma(a, ds, dq[i][n]);
        }
      }
            });
  }
  __shared__ float sums[4];
  rest = wave_sum(MAPS == 2 ? rest + rise : (map0 ? rest - lam * rise : rise));
  if (lane == 0) sums[wave] = rest;
  __syncthreads();  // every wave is past its last image
  if (tid == 0) p.partial[(((long)map0 * tiles + tile) * p.B + b) * p.H + h] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  if (MAPS == 2 && tid == 0) p.partial[(((long)tiles + tile) * p.B + b) * p.H + h] = 0.f;  // (the place of the second map's workgroup)
  float* strip = reinterpret_cast<float*>(smem + wave * STRIP_BYTES);
#pragma unroll
  for (int i = 0; i < MAPS; ++i) {
    T* out = (T*)p.dq_out + (long)b * p.dq_s[0] + (long)w0 * p.dq_s[1] + (long)h * p.dq_s[2] + (long)(map0 + i) * p.dq_s[3];
    store_rows<T>(strip, lane, dq[i], p.scale, p.d, p.dq_vec, Weights{nullptr, 0}, [&](int r) { return w0 + r < p.Tq ? out + (long)r * p.dq_s[1] : nullptr; });
  }
}

// 3. dK, dV.  Workgroup = (batch, key / value head, 128 keys), wave = 32 keys, lane l and l + 32 = one key: S_i = Q_i K_i^T and dP = dO V^T
//    (queries x keys), dV^T += dO^T (P_1 - lambda P_2), dK_i^T += Q_i^T dS_i, over all queries of all heads that share the key / value head.
//    Wide heads: the accumulators of all three do not fit one wave's registers, so dK_1, dK_2 (PART_DK, the map in the grid's y) and dV (PART_DV) are
//    separate workgroups of one launch; S and dP are computed again (3 / 2 of the flop).  2 x 4096 causal, 4
//    heads of 64 / 128 shared by 16: 433 us and 24 us for the join, the matrix unit busy in 35 % of the cycles, LDS in 33 %, vector issue in 44 %, and its
//    two waves a SIMD wait in 44 % of theirs: the registers leave no third one.  12 x 320, 4 heads of 72 / 144: 24 us (as two launches 39).
enum { PART_ALL, PART_DK, PART_DV };
template <typename T, int NB, bool VECTOR> constexpr bool dkv_split() { return NB >= (sizeof(T) == 2 && VECTOR ? 5 : 4); }
// d = 33 .. 64, bf16: the 128 keys' V and the last 16 channels of their K stay in LDS instead of 40 registers, which lets two waves share a SIMD (256
// registers each, no AGPR copies, no scratch)
template <typename T, int NB> constexpr bool dkv_v_in_lds() { return sizeof(T) == 2 && NB == 4; }
template <typename T, int NB> constexpr int dkv_images() { return 2 * (32 * (2 * Img<T, (NB + 1) / 2>::ROW_BYTES + Img<T, NB>::ROW_BYTES) + 1024); }
template <typename T, int NB> constexpr int dkv_lds() { return at_least(dkv_images<T, NB>() + (dkv_v_in_lds<T, NB>() ? QB * Img<T, NB>::ROW_BYTES + 4 * 2 * 64 * 16 : 0), 4 * STRIP_BYTES); }

template <typename T, int NB, bool VECTOR, int PART> __device__ __forceinline__ void bwd_dkv(const tfpp_diff_attn_params& p, int y) {
  constexpr int QT = 32, NT = 256, MAPS = PART == PART_DK ? 1 : 2, CD = (NB + 1) / 2;
  typedef Img<T, CD> ImgQ;
  typedef Img<T, NB> ImgO;
  constexpr int Q_BYTES = QT * ImgQ::ROW_BYTES, O_BYTES = QT * ImgO::ROW_BYTES, BUF = 2 * Q_BYTES + O_BYTES + 1024;  // (the rows' values; images start at whole rows, <= 1 KB)
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
  const int tiles = (p.Tk + QB - 1) / QB, group = p.H / p.Hkv;
  int bh, tile;
  place(p.B * p.Hkv, tiles, p.causal, bh, tile);
  const int part = PART == PART_DK ? y >> 1 : y;  // of the queries
  const int b = bh / p.Hkv, hk = bh % p.Hkv, dvs = (p.dv + 7) & ~7;
  const Seq sq = sequence(p, b);
  const int w0 = tile * QB + wave * 32, kj = w0 + (lane & 31);
  bool seen = kj < sq.len;
  if (seen && p.key_mask) seen = p.key_mask[(long)b * p.ld_mask + kj] != 0;
  const int kc = kj < p.Tk ? kj : p.Tk - 1;
  constexpr bool V_LDS = dkv_v_in_lds<T, NB>() && PART == PART_ALL, HOLD = sizeof(T) == 2 || NB < 4, WANT_DK = PART != PART_DV, WANT_DV = PART != PART_DK;
  constexpr bool FENCE = V_LDS;  // (operands loaded far ahead of their products would not fit the registers)
  const int map0 = PART == PART_DK ? y & 1 : 0;  // wide fp32 heads do not fit the registers: K and V are read again for every tile
  const T* krow = (const T*)p.k + (long)b * p.k_s[0] + (long)kc * p.k_s[1] + (long)hk * p.k_s[2];
  const T* vrow = (const T*)p.v + (long)b * p.v_s[0] + (long)kc * p.v_s[1] + (long)hk * p.v_s[2];
  constexpr int K_HELD = V_LDS ? NB - 1 : NB;
  Frag8<T> k[MAPS][HOLD ? K_HELD : 1], v[HOLD && WANT_DK && !V_LDS ? 2 * NB : 1];
  if constexpr (HOLD) {
#pragma unroll
    for (int i = 0; i < MAPS; ++i)
#pragma unroll
      for (int ks = 0; ks < K_HELD; ++ks) load_frag<T, VECTOR>(krow + (long)(map0 + i) * p.k_s[3], ks * 16 + half * 8, p.d, true, k[i][ks]);
    if constexpr (WANT_DK && !V_LDS)
#pragma unroll
      for (int ks = 0; ks < 2 * NB; ++ks) load_frag<T, VECTOR>(vrow, ks * 16 + half * 8, p.dv, true, v[ks]);
  }
  f32x16_t dk[WANT_DK ? MAPS : 1][CD], dv[WANT_DV ? NB : 1];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
#pragma unroll
    for (int n = 0; n < CD; ++n)
#pragma unroll
      for (int i = 0; i < (WANT_DK ? MAPS : 1); ++i) dk[i][n][r] = 0.f;
#pragma unroll
    for (int n = 0; n < (WANT_DV ? NB : 1); ++n) dv[n][r] = 0.f;
  }
  const float c = p.scale * LOG2E;
  const long rows = (long)p.B * p.H * p.Tq;
  // causal: query i sees the workgroup's first key from i = first key - start on
  int q_lo = 0;
  if (p.causal && tile * QB > sq.start) q_lo = (tile * QB - sq.start) / QT * QT;
  const bool any = tile * QB < sq.len && q_lo < p.Tq;
  const int per = any ? (p.Tq - q_lo + QT - 1) / QT : 0, all = per * group;
  const int share = (all + p.dkv_splits - 1) / p.dkv_splits, first = part * share, steps = all - first < share ? all - first : share;  // (may be <= 0)

  const int q_rows = ImgQ::rows_at(lane), o_rows = ImgO::rows_at(lane), q_cols = ImgQ::cols_at(lane), o_cols = ImgO::cols_at(lane);
  // the next step's query head and first query, and where its Q, dO and row values lie: carried along, without divisions or long products in the loop
  int h_next = hk * group + (per ? first / per : 0), q_next = q_lo + (per ? first % per : 0) * QT;
  const long row0 = ((long)b * p.H + h_next) * p.Tq + q_lo;
  const T* q_head = (const T*)p.q + (long)b * p.q_s[0] + (long)q_lo * p.q_s[1] + (long)h_next * p.q_s[2];  // at the head's first step
  const T* o_head = (const T*)p.d_o + row0 * dvs;
  const float* s_head = (wave < 2 ? p.lse : p.delta) + (wave & 1) * rows + row0;  // lse_1, lse_2, delta_1, delta_2: one array a wave
  const T *q_tile = q_head + (long)(q_next - q_lo) * p.q_s[1], *o_tile = o_head + (long)(q_next - q_lo) * dvs;
  const float* s_tile = s_head + (q_next - q_lo);
  const long q_ld = p.q_s[1];
  auto fill = [&](unsigned char* buf) {
    const Rows have = {p.Tq - q_next, false, 0ull};
    int tid = (int)threadIdx.x;
    if (FENCE) asm volatile("" : "+v"(tid));  // (the offsets made of it are worked out again each time: kept, they would not fit the registers)
#pragma unroll
    for (int i = map0; i < map0 + MAPS; ++i) ImgQ::template fill<QT, VECTOR, NT>(buf + i * Q_BYTES, q_tile + i * p.q_s[3], q_ld, p.d, have, tid);
    ImgO::template fill<QT, true, NT>(buf + 2 * Q_BYTES, o_tile, dvs, dvs, have, tid);
    // queries behind the last: all zero like their Q and dO, so P = 1 but dV, dS get 0
    __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void*)s_tile, 0, have.count < QT ? have.count * 4 : QT * 4, 0x00020000),
                                             (lds_void_t*)(buf + 2 * Q_BYTES + O_BYTES + wave * 256), 4, lane * 4, 0, 0, 0);
  };
  auto advance = [&] {
    q_next += QT;
    q_tile += QT * q_ld;
    o_tile += QT * dvs;
    s_tile += QT;
    if (q_next >= p.Tq) {
      q_next = q_lo;
      ++h_next;
      q_tile = q_head += p.q_s[2];
      o_tile = o_head += (long)p.Tq * dvs;
      s_tile = s_head += p.Tq;
    }
  };
  int v_at = 0;
  uint4* stash = reinterpret_cast<uint4*>(smem + dkv_images<T, NB>() + QB * ImgO::ROW_BYTES) + wave * 2 * 64 + lane;  // (V_LDS) a lane's own operands
  if constexpr (V_LDS) {  // 32 keys a wave, filled as every other image; complete at the first step's wait
    const int place = dkv_images<T, NB>() + wave * 32 * ImgO::ROW_BYTES;
    ImgO::template fill<32, VECTOR, 64>(smem + place, (const T*)p.v + (long)b * p.v_s[0] + (long)w0 * p.v_s[1] + (long)hk * p.v_s[2], p.v_s[1], p.dv, Rows{sq.len - w0, p.key_mask != nullptr, __ballot(seen)}, lane);
    v_at = place + ImgO::rows_at(lane);
#pragma unroll
    for (int i = 0; i < MAPS; ++i) {
      Frag8<T> last;
      load_frag<T, VECTOR>(krow + (long)i * p.k_s[3], K_HELD * 16 + half * 8, p.d, true, last);
      stash[i * 64] = last.v;
    }
  }
  int h = h_next, q0 = q_next;
  float lam = 0.f;
  if (steps > 0) fill(smem);
  for (int s = 0; s < steps; ++s) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __syncthreads();
    if (s == 0 || q0 == q_lo) lam = p.lam[p.n_lam > 1 ? h : 0];
    overlap(smem + (~s & 1) * BUF, smem + (s & 1) * BUF,
            [&](unsigned char* next) {
              advance();
              if (s + 1 < steps) fill(next);
            },
            [&](const unsigned char* now) {
    const bool diag = p.causal && sq.start + q0 < w0 + 31;
    const int orow = o_rows + 2 * Q_BYTES, ocol = o_cols + 2 * Q_BYTES;
    const float* st = reinterpret_cast<const float*>(now + 2 * Q_BYTES + O_BYTES);
    // S, P, then dV += dO^T (P_1 - lambda P_2) before dP: the fewest values live at a time
    f32x16_t sc[MAPS];
#pragma unroll
    for (int i = 0; i < MAPS; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[i][r] = 0.f;
#pragma unroll
    for (int i = 0; i < MAPS; ++i)
#pragma unroll
      for (int ks = 0; ks < NB; ++ks) {
        Frag8<T> a;
        ImgQ::rows(now + (map0 + i) * Q_BYTES, q_rows, ks, a);
        if constexpr (!HOLD) load_frag<T, VECTOR>(krow + (long)(map0 + i) * p.k_s[3], ks * 16 + half * 8, p.d, true, k[i][0]);
        if constexpr (V_LDS) {
          Frag8<T> last;
          if (ks == K_HELD) last.v = stash[i * 64];
          mma(a, ks == K_HELD ? last : k[i][ks < K_HELD ? ks : 0], sc[i]);
        } else {
          mma(a, k[i][HOLD ? ks : 0], sc[i]);
        }
        if (FENCE && ks % 2 == 1) __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (FENCE) __builtin_amdgcn_sched_barrier(0);
      const int t0 = 8 * g + 4 * half;
#pragma unroll
      for (int i = 0; i < MAPS; ++i) {
        const float4 l4 = *reinterpret_cast<const float4*>(st + (map0 + i) * 64 + t0);
        const float ls[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[i][4 * g + e] = __builtin_amdgcn_exp2f(fmaf(sc[i][4 * g + e], c, -ls[e]));
        }
      }
    }
    if (diag) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const bool keep = kj <= sq.start + q0 + 8 * (r >> 2) + 4 * half + (r & 3);
#pragma unroll
        for (int i = 0; i < MAPS; ++i) sc[i][r] = keep ? sc[i][r] : 0.f;
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (WANT_DV) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        f32x16_t pd;
#pragma unroll
        for (int r = 8 * t; r < 8 * t + 8; ++r) pd[r] = fmaf(-lam, sc[MAPS - 1][r], sc[0][r]);
        Frag8<T> f;
        to_frag(pd, t, f);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          Frag8<T> a;
          ImgO::cols(now + 16 * t * ImgO::ROW_BYTES, ocol, n, a);
          mma(a, f, dv[n]);
          if (FENCE && n % 2 == 1) __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (WANT_DK) {
      f32x16_t dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < 2 * NB; ++ks) {
        Frag8<T> a;
        ImgO::rows(now, orow, ks, a);
        if constexpr (V_LDS) ImgO::rows(smem, v_at, ks, v[0]);
        else if constexpr (!HOLD) load_frag<T, VECTOR>(vrow, ks * 16 + half * 8, p.dv, true, v[0]);
        mma(a, v[HOLD && !V_LDS ? ks : 0], dp);
        if (FENCE) __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < MAPS; ++i) {
        const float sign = map0 + i ? -lam : 1.f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          if (FENCE) __builtin_amdgcn_sched_barrier(0);
          const float4 d4 = *reinterpret_cast<const float4*>(st + (2 + map0 + i) * 64 + 8 * g + 4 * half);
          const float de[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[i][4 * g + e] *= map0 + i ? sign * (dp[4 * g + e] - de[e]) : dp[4 * g + e] - de[e];
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          Frag8<T> f;
          to_frag(sc[i], t, f);
#pragma unroll
          for (int n = 0; n < CD; ++n) {
            Frag8<T> a;
            ImgQ::cols(now + (map0 + i) * Q_BYTES + 16 * t * ImgQ::ROW_BYTES, q_cols, n, a);
            mma(a, f, dk[i][n]);
          }
          if (FENCE) __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
            });
    h = h_next;
    q0 = q_next;
  }
  __syncthreads();  // every wave is past its last image
  float* strip = reinterpret_cast<float*>(smem + wave * STRIP_BYTES);
  // A key that is left out has a column of its own in every product: whatever its K and V made of it is dropped here
  if (!seen) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      if constexpr (WANT_DV)
#pragma unroll
        for (int n = 0; n < NB; ++n) dv[n][r] = 0.f;
      if constexpr (WANT_DK)
#pragma unroll
        for (int n = 0; n < CD; ++n)
#pragma unroll
          for (int i = 0; i < MAPS; ++i) dk[i][n][r] = 0.f;
    }
  }
  if (p.dkv_splits > 1) {  // fp32 sums of this part: rows of both maps' dK and dV, added by diff_attn_bwd_join_kernel
    constexpr int WIDTH = 2 * CD * 32 + NB * 32;
    float* out = p.dkv + ((((long)part * p.B + b) * p.Hkv + hk) * p.Tk + w0) * WIDTH;
    auto row = [&](int r) { return w0 + r < p.Tk ? out + (long)r * WIDTH : nullptr; };
    if constexpr (WANT_DV) store_rows<float>(strip, lane, dv, 1.f, NB * 32, true, Weights{nullptr, 0}, [&](int r) { return row(r) ? row(r) + 2 * CD * 32 : nullptr; });
    if constexpr (WANT_DK)
#pragma unroll
      for (int i = 0; i < MAPS; ++i) store_rows<float>(strip, lane, dk[i], p.scale, CD * 32, true, Weights{nullptr, 0}, [&](int r) { return row(r) ? row(r) + (map0 + i) * CD * 32 : nullptr; });
    return;
  }
  if constexpr (WANT_DV) {
    T* out = (T*)p.dv_out + (long)b * p.dv_s[0] + (long)w0 * p.dv_s[1] + (long)hk * p.dv_s[2];
    store_rows<T>(strip, lane, dv, 1.f, p.dv, p.dv_vec, Weights{nullptr, 0}, [&](int r) { return w0 + r < p.Tk ? out + (long)r * p.dv_s[1] : nullptr; });
  }
  if constexpr (WANT_DK)
#pragma unroll
    for (int i = 0; i < MAPS; ++i) {
      T* out = (T*)p.dk_out + (long)b * p.dk_s[0] + (long)w0 * p.dk_s[1] + (long)hk * p.dk_s[2] + (long)(map0 + i) * p.dk_s[3];
      store_rows<T>(strip, lane, dk[i], p.scale, p.d, p.dk_vec, Weights{nullptr, 0}, [&](int r) { return w0 + r < p.Tk ? out + (long)r * p.dk_s[1] : nullptr; });
    }
}

template <typename T, int NB, bool VECTOR> __global__ __launch_bounds__(256, (sizeof(T) == 4 || NB <= 5 ? 2 : 1)) void diff_attn_bwd_dkv_kernel(tfpp_diff_attn_params p) {
  if constexpr (dkv_split<T, NB, VECTOR>()) {
    const int y = blockIdx.y, n = 2 * p.dkv_splits;  // both maps' dK, the longer ones, start first
    if (y < n) bwd_dkv<T, NB, VECTOR, PART_DK>(p, y);
    else bwd_dkv<T, NB, VECTOR, PART_DV>(p, y - n);
  } else {
    bwd_dkv<T, NB, VECTOR, PART_ALL>(p, blockIdx.y);
  }
}

// dK, dV of one key: the parts' sums in order; one wave a (batch, key, head), 4 channels a lane
template <typename T> __global__ __launch_bounds__(256) void diff_attn_bwd_join_kernel(tfpp_diff_attn_params p, int kc, int vc) {
  const long n = (long)blockIdx.x * 4 + (threadIdx.x >> 6), all = (long)p.B * p.Hkv * p.Tk;
  if (n >= all) return;
  const int j = (int)(n % p.Tk), hk = (int)(n / p.Tk % p.Hkv), b = (int)(n / p.Tk / p.Hkv), width = 2 * kc + vc;
  const float* src = p.dkv + n * width;
  for (int c = ((int)threadIdx.x & 63) * 4; c < width; c += 256) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < p.dkv_splits; ++k) {
      const float4 v = *reinterpret_cast<const float4*>(src + k * all * width + c);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    const int map = c < 2 * kc ? c / kc : 2, ch = map < 2 ? c % kc : c - 2 * kc, limit = map < 2 ? p.d : p.dv;
    T* to = map < 2 ? (T*)p.dk_out + (long)b * p.dk_s[0] + (long)j * p.dk_s[1] + (long)hk * p.dk_s[2] + (long)map * p.dk_s[3] + ch
                    : (T*)p.dv_out + (long)b * p.dv_s[0] + (long)j * p.dv_s[1] + (long)hk * p.dv_s[2] + ch;
    if ((map < 2 ? p.dk_vec : p.dv_vec) && ch + 4 <= limit) {
      if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(to) = make_uint2(f2bf_pack2(s.x, s.y), f2bf_pack2(s.z, s.w));
      else *reinterpret_cast<float4*>(to) = s;
    } else {
      const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (ch + e < limit) to[e] = ElemTraits<T>::from_f(v[e]);
    }
  }
}

// lambda[h] = exp(lq1 . lk1) - exp(lq2 . lk2) + init of the four learned vectors of a head (one wave a head), and its gradient
__device__ __forceinline__ float vec_at(const void* p, long i, int is_bf16) { return is_bf16 ? bf2f(((const bf16_t*)p)[i]) : ((const float*)p)[i]; }
__device__ __forceinline__ void exps(const void* q1, const void* k1, const void* q2, const void* k2, int h, int d, int is_bf16, float& e1, float& e2) {
  float s1 = 0.f, s2 = 0.f;
  for (int i = threadIdx.x; i < d; i += 64) {
    const long n = (long)h * d + i;
    s1 += vec_at(q1, n, is_bf16) * vec_at(k1, n, is_bf16);
    s2 += vec_at(q2, n, is_bf16) * vec_at(k2, n, is_bf16);
  }
  e1 = expf(wave_sum(s1));
  e2 = expf(wave_sum(s2));
}
__global__ __launch_bounds__(64) void diff_lambda_fwd_kernel(const void* q1, const void* k1, const void* q2, const void* k2, float init, float* lam, int d, int is_bf16) {
  float e1, e2;
  exps(q1, k1, q2, k2, blockIdx.x, d, is_bf16, e1, e2);
  if (threadIdx.x == 0) lam[blockIdx.x] = e1 - e2 + init;
}
template <typename T> __global__ __launch_bounds__(64) void diff_lambda_bwd_kernel(const float* dlam, const T* q1, const T* k1, const T* q2, const T* k2, T* dq1, T* dk1, T* dq2,
                                                                                 T* dk2, int d) {
  typedef ElemTraits<T> E;
  float e1, e2;
  exps(q1, k1, q2, k2, blockIdx.x, d, E::DT == TFPP_BF16, e1, e2);
  const float g1 = dlam[blockIdx.x] * e1, g2 = -dlam[blockIdx.x] * e2;
  for (int i = threadIdx.x; i < d; i += 64) {
    const long n = (long)blockIdx.x * d + i;
    dq1[n] = E::from_f(g1 * E::to_f(k1[n]));
    dk1[n] = E::from_f(g1 * E::to_f(q1[n]));
    dq2[n] = E::from_f(g2 * E::to_f(k2[n]));
    dk2[n] = E::from_f(g2 * E::to_f(q2[n]));
  }
}

bool strides_vec(const int64_t* s, int n, int vec) {
  for (int i = 0; i < n; ++i)
    if (s[i] % vec) return false;
  return true;
}
bool valid(const tfpp_diff_attn_params& p, int dtype) {
  return (dtype == TFPP_F32 || dtype == TFPP_BF16) && p.q && p.k && p.v && p.lam && p.B >= 1 && p.H >= 1 && p.Hkv >= 1 && p.H % p.Hkv == 0 && p.Tq >= 1 && p.Tk >= 1 &&
         p.d >= 1 && p.d <= 128 && p.dv >= 1 && p.dv <= 256 && (p.n_lam == 1 || p.n_lam == p.H) && p.scale > 0.f && std::isfinite(p.scale) && (!p.norm || p.eps > 0.f) &&
         p.Tq < (1 << 29) && p.Tk < (1 << 29) && (long)p.B * p.H < (1l << 24);
}
// Can q, k, v be read 16 bytes at a time?  A token's stride has to hold its channels: rows that share memory (one token expanded over all, windows) would put
// what `fill` takes for zeros, the rows behind the last one, inside its buffer.
bool vector_rows(const tfpp_diff_attn_params& p, int vec) {
  if (p.q_s[1] < p.d || p.k_s[1] < p.d || p.v_s[1] < p.dv) return false;
  const int64_t far = (1 << 24) * (int64_t)vec / 16;  // 16 MB from token to token: a tile's offsets fit 32 bits
  return p.d % vec == 0 && p.dv % vec == 0 && p.q_s[1] <= far && p.k_s[1] <= far && p.v_s[1] <= far && !(((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v) & 15) && strides_vec(p.q_s, 4, vec) && strides_vec(p.k_s, 4, vec) &&
         strides_vec(p.v_s, 3, vec);
}
// the stride of a single token can be anything: one that holds its channels and is a multiple of 16 bytes
tfpp_diff_attn_params one_token(tfpp_diff_attn_params p) {
  if (p.Tq == 1) p.q_s[1] = (p.d + 7) & ~7;
  if (p.Tk == 1) {
    p.k_s[1] = (p.d + 7) & ~7;
    p.v_s[1] = (p.dv + 7) & ~7;
  }
  return p;
}
// Can an output be written 16 bytes at a time?
bool out_vector(const void* ptr, const int64_t* s, int n, int vec) { return !((uintptr_t)ptr & 15) && strides_vec(s, n, vec); }

// more than 64 KB of LDS: once for each device.  The mark is set behind the call, so that of two threads that come here first both make it.
template <typename K> int lds_limit(K* kernel, int bytes, unsigned long long* done) {
  if (bytes <= 64 * 1024) return 0;
  int dev = 0;
  (void)hipGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if (__atomic_load_n(done, __ATOMIC_ACQUIRE) & bit) return 0;
  const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return -(int)e;
  __atomic_fetch_or(done, bit, __ATOMIC_RELEASE);
  return 0;
}

template <typename K> int start(K* kernel, dim3 grid, int threads, int lds, unsigned long long* done, const tfpp_diff_attn_params& p, hipStream_t st) {
  const int rc = lds_limit(kernel, lds, done);
  if (rc) return rc;
  hipLaunchKernelGGL(kernel, grid, dim3(threads), lds, st, p);
  TFPP_CHECK_LAUNCH();
  return 0;
}

enum { STEP_FWD, STEP_FEW, STEP_DQ, STEP_DKV };
template <typename T, int NB, bool VECTOR> int launch(const tfpp_diff_attn_params& p, int step, hipStream_t st) {
  static unsigned long long done[5] = {0, 0, 0, 0, 0};
  if (step == STEP_FEW) {
    const long n = (long)p.B * p.Hkv * (((long)(p.H / p.Hkv) * p.Tq + 31) / 32) * p.splits;
    if (n > 0x7fffffffl) return TFPP_EINVAL;
    const int rc = start(diff_attn_few_kernel<T, NB, VECTOR>, dim3((unsigned)n), Few<T, NB>::THREADS, Few<T, NB>::LDS, &done[4], p, st);
    if (rc || p.splits == 1) return rc;
    const long rows = (long)p.B * p.H * p.Tq;
    hipLaunchKernelGGL(diff_attn_fwd_join_kernel<T>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, p, NB * 32);
    TFPP_CHECK_LAUNCH();
    return 0;
  }
  if (step == STEP_FWD) {
    // half the queries a workgroup where whole ones would leave CUs without any (144 or 240 workgroups: 27 or 25 us)
    constexpr int FULL = fwd_threads<T, NB>(), MOST = fwd_queries<T, NB>(FULL);
    auto groups = [&](int queries) { return (long)p.B * p.H * ((p.Tq + queries - 1) / queries); };
    if (groups(MOST) > 0x7fffffffl) return TFPP_EINVAL;
    if constexpr (VECTOR)
      if (groups(MOST) < 256) return start(diff_attn_fwd_kernel<T, NB, true, FULL / 2>, dim3((unsigned)groups(MOST / 2)), FULL / 2, fwd_lds<T, NB>(), &done[3], p, st);
    return start(diff_attn_fwd_kernel<T, NB, VECTOR, FULL>, dim3((unsigned)groups(MOST)), FULL, fwd_lds<T, NB>(), &done[0], p, st);
  }
  const long n = (long)(((step == STEP_DQ ? p.Tq : p.Tk) + QB - 1) / QB) * p.B * (step == STEP_DQ ? p.H : p.Hkv);
  if (n > 0x7fffffffl) return TFPP_EINVAL;
  if (step == STEP_DQ) return start(diff_attn_bwd_dq_kernel<T, NB, VECTOR>, dim3((unsigned)n, 3 - dq_maps<T, NB>()), 256, dq_lds<T, NB, VECTOR>(), &done[1], p, st);
  const int rc = start(diff_attn_bwd_dkv_kernel<T, NB, VECTOR>, dim3((unsigned)n, (dkv_split<T, NB, VECTOR>() ? 3 : 1) * p.dkv_splits), 256, dkv_lds<T, NB>(), &done[2], p, st);
  if (rc) return rc;
  if (p.dkv_splits > 1) {
    hipLaunchKernelGGL(diff_attn_bwd_join_kernel<T>, dim3((unsigned)(((long)p.B * p.Hkv * p.Tk + 3) / 4)), dim3(256), 0, st, p, (NB + 1) / 2 * 32, NB * 32);
    TFPP_CHECK_LAUNCH();
  }
  return 0;
}
// channels are padded to 16 NB / 32 NB: the width classes of the fusion transformers' heads (d 9, 27, 72) and the powers of two
template <typename T> int dispatch(const tfpp_diff_attn_params& p, int step, hipStream_t st) {
  const bool v = vector_rows(p, ElemTraits<T>::VEC);
  const int need = (p.d + 15) / 16 > (p.dv + 31) / 32 ? (p.d + 15) / 16 : (p.dv + 31) / 32;
#define DA_GO(NB) (v ? launch<T, NB, true>(p, step, st) : launch<T, NB, false>(p, step, st))
  if (need <= 1) return DA_GO(1);
  if (need <= 2) return DA_GO(2);
  if (need <= 4 && v) return launch<T, 4, true>(p, step, st);  // (element by element the next width serves as well)
  if (need <= 5) return DA_GO(5);
  return DA_GO(8);
#undef DA_GO
}
int padded_blocks(const tfpp_diff_attn_params& p) {  // NB of dispatch(), or more: the scratch is sized by it
  const int need = (p.d + 15) / 16 > (p.dv + 31) / 32 ? (p.d + 15) / 16 : (p.dv + 31) / 32;
  return need <= 2 ? need : (need <= 5 ? 5 : 8);
}
// Which forward kernel, and how many splits of the keys?  0: the one for many queries.
int few_splits(const tfpp_diff_attn_params& p) {
  const long wg = (long)p.B * p.H * ((p.Tq + QB - 1) / QB);
  const long group = p.H / p.Hkv, rows = group * p.Tq, base = (long)p.B * p.Hkv * ((rows + 31) / 32);
  if (p.Tq > 64 && wg > 64) return 0;  // (12 x 4 heads x 320 queries: 27 us there, 44 us here)
  // Where either kernel fills the chip, this one is for rows that fit one tile: it reads keys and values once for all heads that share them, the other one for
  // each head, with 128 queries a workgroup however few there are.  One token each, bf16: 64 x 16 heads of 64 / 128 over 4, 320 and 4096 keys, 43 and 429 us there,
  // 15 and 114 here; 128 x 8 heads of 32 / 64, not shared, 29 and 299, 25 and 231.  More tiles (32 tokens each): 46 there, 53 here.  Up to
  // 64 keys that are not shared leave waves of this one without any: 13 there, 16 here.
  if (wg >= 512 && (rows > 32 || (group == 1 && p.Tk <= 64))) return 0;
  long n = (512 + base - 1) / base, most = (p.Tk + 511) / 512;  // two workgroups a CU; at least 512 keys (4 blocks a wave) in a split
  if (n > most) n = most;
  if (n > 64) n = 64;  // (the join holds one split a lane)
  return n < 1 ? 1 : (int)n;
}
// Parts of the queries in the dK / dV pass: 1024 workgroups (two a CU and as many to follow) where there are few keys and heads, each with at least 32 tiles
// of 32 queries -- the parts' fp32 sums are written and read once more.
int dkv_parts(const tfpp_diff_attn_params& p) {
  const long wg = (long)p.B * p.Hkv * ((p.Tk + QB - 1) / QB), steps = (long)(p.H / p.Hkv) * ((p.Tq + 31) / 32);
  long n = (1024 + wg - 1) / wg;
  if (n > steps / 32) n = steps / 32;
  return n < 1 ? 1 : (n > 16 ? 16 : (int)n);
}
int row_lanes(const tfpp_diff_attn_params& p) {
  int n = 1;
  while (n * 8 < p.dv) n <<= 1;
  return n;
}
int row_blocks(const tfpp_diff_attn_params& p) {  // workgroups of the row pass for each head: two rounds of 256 / row_lanes rows, about 2048 in all at most (each writes 1 + dv sums: 4096 took 44 us in place of 33 over 8192 x 16 rows)
  const long rows = (long)p.B * p.Tq, round = 256 / row_lanes(p);
  long n = (rows + 2 * round - 1) / (2 * round), most = 2048 / p.H > 1 ? 2048 / p.H : 1;
  if (n > most) n = most;
  return (int)n;
}
int rest_rows(const tfpp_diff_attn_params& p) { return 2 * (int)((p.Tq + QB - 1) / QB) * p.B; }  // (both maps, also where one workgroup has both)
int64_t rest_floats(const tfpp_diff_attn_params& p) { return ((int64_t)rest_rows(p) * p.H + 63) & ~63ll; }  // dQ's part of dlambda, in front of the row pass's sums
int64_t row_floats(const tfpp_diff_attn_params& p) { return ((int64_t)row_blocks(p) * p.H * (1 + p.dv) + 63) & ~63ll; }
}  // namespace

extern "C" int tfpp_diff_attn_fwd(const tfpp_diff_attn_params* pp, int dtype, void* stream) {
  if (!pp || !valid(*pp, dtype) || !pp->out || (pp->o1 != nullptr) != (pp->o2 != nullptr)) return TFPP_EINVAL;
  if (((uintptr_t)pp->o1 | (uintptr_t)pp->o2 | (uintptr_t)pp->partial) & 15) return TFPP_EINVAL;  // (stored 16 bytes at a time)
  tfpp_diff_attn_params p = one_token(*pp);
  p.out_vec = out_vector(p.out, p.o_s, 3, dtype == TFPP_F32 ? 4 : 8);
  p.splits = few_splits(p);
  if (p.splits > 1 && !p.partial) return TFPP_EINVAL;
  const int step = p.splits ? STEP_FEW : STEP_FWD;
  return dtype == TFPP_F32 ? dispatch<float>(p, step, (hipStream_t)stream) : dispatch<bf16_t>(p, step, (hipStream_t)stream);
}

extern "C" int tfpp_diff_attn_fwd_partial_floats(const tfpp_diff_attn_params* p, int64_t* out) {
  if (!p || !out || p->B < 1 || p->H < 1 || p->Hkv < 1 || p->Tq < 1 || p->Tk < 1 || p->d < 1 || p->dv < 1) return TFPP_EINVAL;
  const int splits = few_splits(*p);
  *out = splits > 1 ? (int64_t)splits * p->B * p->H * p->Tq * 2 * (padded_blocks(*p) * 32 + 2) : 0;
  return 0;
}

extern "C" int tfpp_diff_attn_bwd_partial_floats(const tfpp_diff_attn_params* p, int64_t* out) {
  if (!p || !out || p->B < 1 || p->H < 1 || p->Hkv < 1 || p->Tq < 1 || p->Tk < 1 || p->d < 1 || p->dv < 1) return TFPP_EINVAL;
  const int nb = padded_blocks(*p), parts = dkv_parts(*p);
  *out = rest_floats(*p) + row_floats(*p) + (parts > 1 ? (int64_t)parts * p->B * p->Hkv * p->Tk * (2 * ((nb + 1) / 2) + nb) * 32 : 0);
  return 0;
}

extern "C" int tfpp_diff_attn_bwd(const tfpp_diff_attn_params* pp, int dtype, void* stream) {
  if (!pp || !valid(*pp, dtype)) return TFPP_EINVAL;
  tfpp_diff_attn_params p = one_token(*pp);
  if (!p.dout || !p.o1 || !p.o2 || !p.lse || !p.d_o || (dtype == TFPP_BF16 && !p.slope) || !p.delta || !p.partial || !p.dlam || !p.dq_out || !p.dk_out || !p.dv_out || (p.norm_w && !p.dnorm_w)) return TFPP_EINVAL;
  if (p.H > 65535 || (((uintptr_t)p.o1 | (uintptr_t)p.o2 | (uintptr_t)p.d_o | (dtype == TFPP_BF16 ? (uintptr_t)p.slope : 0) | (uintptr_t)p.partial) & 15)) return TFPP_EINVAL;
  const int vec = dtype == TFPP_F32 ? 4 : 8;
  p.dq_vec = out_vector(p.dq_out, p.dq_s, 4, vec);
  p.dk_vec = out_vector(p.dk_out, p.dk_s, 4, vec);
  p.dv_vec = out_vector(p.dv_out, p.dv_s, 3, vec);
  hipStream_t st = (hipStream_t)stream;
  const int blocks = row_blocks(p);
  p.dkv_splits = dkv_parts(p);
  p.dkv = p.partial + rest_floats(p) + row_floats(p);
  const int lpr = row_lanes(p);
  p.do_vec = out_vector(p.dout, p.do_s, 3, vec);
  const dim3 sums(p.n_lam + (p.norm_w ? p.dv : 0));
  tfpp_diff_attn_params pr = p;
  pr.partial += rest_floats(p);
  if (dtype == TFPP_F32) hipLaunchKernelGGL(diff_attn_bwd_rows_kernel<float>, dim3(blocks, p.H), dim3(256), 0, st, pr, lpr);
  else hipLaunchKernelGGL(diff_attn_bwd_rows_kernel<bf16_t>, dim3(blocks, p.H), dim3(256), 0, st, pr, lpr);
  TFPP_CHECK_LAUNCH();
  int rc = dtype == TFPP_F32 ? dispatch<float>(p, STEP_DQ, st) : dispatch<bf16_t>(p, STEP_DQ, st);
  if (rc) return rc;
  if (dtype == TFPP_F32) hipLaunchKernelGGL(diff_attn_bwd_sum_kernel<float>, sums, dim3(256), 0, st, pr, blocks, p.partial, rest_rows(p));
  else hipLaunchKernelGGL(diff_attn_bwd_sum_kernel<bf16_t>, sums, dim3(256), 0, st, pr, blocks, p.partial, rest_rows(p));
  TFPP_CHECK_LAUNCH();
  return dtype == TFPP_F32 ? dispatch<float>(p, STEP_DKV, st) : dispatch<bf16_t>(p, STEP_DKV, st);
}

extern "C" int tfpp_diff_lambda(const void* lq1, const void* lk1, const void* lq2, const void* lk2, float init, float* lam, int n, int d, int dtype, void* stream) {
  if (!lq1 || !lk1 || !lq2 || !lk2 || !lam || n < 1 || d < 1 || (dtype != TFPP_F32 && dtype != TFPP_BF16)) return TFPP_EINVAL;
  hipLaunchKernelGGL(diff_lambda_fwd_kernel, dim3(n), dim3(64), 0, (hipStream_t)stream, lq1, lk1, lq2, lk2, init, lam, d, dtype == TFPP_BF16);
  TFPP_CHECK_LAUNCH();
  return 0;
}

extern "C" int tfpp_diff_lambda_bwd(const float* dlam, const void* lq1, const void* lk1, const void* lq2, const void* lk2, void* dlq1, void* dlk1, void* dlq2, void* dlk2, int n,
                                    int d, int dtype, void* stream) {
  if (!dlam || !lq1 || !lk1 || !lq2 || !lk2 || !dlq1 || !dlk1 || !dlq2 || !dlk2 || n < 1 || d < 1 || (dtype != TFPP_F32 && dtype != TFPP_BF16)) return TFPP_EINVAL;
  if (dtype == TFPP_F32)
    hipLaunchKernelGGL(diff_lambda_bwd_kernel<float>, dim3(n), dim3(64), 0, (hipStream_t)stream, dlam, (const float*)lq1, (const float*)lk1, (const float*)lq2,
                       (const float*)lk2, (float*)dlq1, (float*)dlk1, (float*)dlq2, (float*)dlk2, d);
  else
    hipLaunchKernelGGL(diff_lambda_bwd_kernel<bf16_t>, dim3(n), dim3(64), 0, (hipStream_t)stream, dlam, (const bf16_t*)lq1, (const bf16_t*)lk1, (const bf16_t*)lq2,
                       (const bf16_t*)lk2, (bf16_t*)dlq1, (bf16_t*)dlk1, (bf16_t*)dlq2, (bf16_t*)dlk2, d);
  TFPP_CHECK_LAUNCH();
  return 0;
}
