// Shared pieces of the state-space sequence kernels (ssm_scan.hip, ssm_scan_bwd.hip, ssm_conv.hip, sandwich.hip).
//
// Matrix products here meet two kinds of operands: INPUTS, which are exact in their own type, and COMPUTED values (decays
// times inputs, running states, score tiles), which are 32-bit.  With bf16 inputs a computed operand is split into bf16
// parts v = p0 + p1 (+ p2): p0 = bf16(v), p1 = bf16(v - p0), ...  Two parts leave 2^-18 |v|, three 2^-27 |v|; products of
// parts are exact in the fp32 accumulator of the MFMA.  Two parts are used where the result is rounded to bf16 anyway,
// three where it stays fp32 (states, parameter gradients).  A single bf16 rounding of the computed operand would cost as
// much error again as the final rounding of the output.  With fp32 inputs every product runs on v_mfma_f32_16x16x4_f32.
//
// Fragment convention of both forms (16x16 tiles, 32 values of k a step): lane (q = lane >> 4, c = lane & 15) holds row /
// column c and eight values of k, numbers 8q .. 8q+7 (or, "perm", 4q .. 4q+3 and 16+4q .. 16+4q+3: the order in which two
// accumulator tiles hold their rows, so that a tile just computed is an operand without leaving the registers; the other
// operand is then loaded in the same order).  The accumulator holds rows 4q .. 4q+3 of column c.
#pragma once
#include "common.h"

struct SsmF8 { float v[8]; };
template <int NS> struct SsmB8 { bf16x8 p[NS]; };

// ---- accumulate a 16x16 tile over 32 values of k ----
__device__ __forceinline__ f32x4 ssm_mma1(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 ssm_mma(const bf16x8& a, const bf16x8& b, f32x4 c) { return ssm_mma1(a, b, c); }
template <int NS> __device__ __forceinline__ f32x4 ssm_mma(const SsmB8<NS>& a, const bf16x8& b, f32x4 c) {
#pragma unroll
  for (int i = NS - 1; i >= 0; --i) c = ssm_mma1(a.p[i], b, c);
  return c;
}
template <int NS> __device__ __forceinline__ f32x4 ssm_mma(const bf16x8& a, const SsmB8<NS>& b, f32x4 c) {
#pragma unroll
  for (int i = NS - 1; i >= 0; --i) c = ssm_mma1(a, b.p[i], c);
  return c;
}
// computed x computed: the products of parts whose numbers add to less than the smaller count
template <int NA, int NB> __device__ __forceinline__ f32x4 ssm_mma(const SsmB8<NA>& a, const SsmB8<NB>& b, f32x4 c) {
  constexpr int M = NA < NB ? NA : NB;
#pragma unroll
  for (int s = M - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB) c = ssm_mma1(a.p[i], b.p[s - i], c);
  return c;
}
__device__ __forceinline__ f32x4 ssm_mma(const SsmF8& a, const SsmF8& b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b.v[j], c, 0, 0, 0);
  return c;
}

// M tiles that share an operand: part by part over all of them, so that no product waits for the one before it
template <int M, int NS> __device__ __forceinline__ void ssm_mma_rows(const bf16x8 (&a)[M], const SsmB8<NS>& b, f32x4 (&c)[M]) {
#pragma unroll
  for (int i = NS - 1; i >= 0; --i)
#pragma unroll
    for (int m = 0; m < M; ++m) c[m] = ssm_mma1(a[m], b.p[i], c[m]);
}
template <int M> __device__ __forceinline__ void ssm_mma_rows(const bf16x8 (&a)[M], const bf16x8& b, f32x4 (&c)[M]) {
#pragma unroll
  for (int m = 0; m < M; ++m) c[m] = ssm_mma1(a[m], b, c[m]);
}
template <int M> __device__ __forceinline__ void ssm_mma_rows(const SsmF8 (&a)[M], const SsmF8& b, f32x4 (&c)[M]) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int m = 0; m < M; ++m) c[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[m].v[j], b.v[j], c[m], 0, 0, 0);
}
template <int M, int NS> __device__ __forceinline__ void ssm_mma_cols(const SsmB8<NS>& a, const bf16x8 (&b)[M], f32x4 (&c)[M]) {
#pragma unroll
  for (int i = NS - 1; i >= 0; --i)
#pragma unroll
    for (int m = 0; m < M; ++m) c[m] = ssm_mma1(a.p[i], b[m], c[m]);
}
template <int M, int NA, int NB> __device__ __forceinline__ void ssm_mma_cols(const SsmB8<NA>& a, const SsmB8<NB> (&b)[M], f32x4 (&c)[M]) {
  constexpr int L = NA < NB ? NA : NB;
#pragma unroll
  for (int s = L - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB) {
#pragma unroll
        for (int m = 0; m < M; ++m) c[m] = ssm_mma1(a.p[i], b[m].p[s - i], c[m]);
      }
}
template <int M> __device__ __forceinline__ void ssm_mma_cols(const SsmF8& a, const SsmF8 (&b)[M], f32x4 (&c)[M]) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int m = 0; m < M; ++m) c[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[j], b[m].v[j], c[m], 0, 0, 0);
}

// ---- operand types by input type ----
template <typename T> struct SsmOps;
template <> struct SsmOps<bf16> {
  static constexpr int PAD = 8;                      // elements behind an LDS row: rows start 16 bytes apart in the banks
  template <int NS> using Cm = SsmB8<NS>;
  using Ex = bf16x8;
  template <int NS> static constexpr int planes() { return NS; }
  template <int NS> __device__ static __forceinline__ SsmB8<NS> split(const float (&v)[8]) {
    SsmB8<NS> r;
    float rest[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) rest[j] = v[j];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      uint4 u = make_uint4(pack_bf16x2(rest[0], rest[1]), pack_bf16x2(rest[2], rest[3]), pack_bf16x2(rest[4], rest[5]), pack_bf16x2(rest[6], rest[7]));
      r.p[i] = __builtin_bit_cast(bf16x8, u);
      if (i + 1 < NS) {
        rest[0] -= bf16_lo(u.x); rest[1] -= bf16_hi(u.x); rest[2] -= bf16_lo(u.y); rest[3] -= bf16_hi(u.y);
        rest[4] -= bf16_lo(u.z); rest[5] -= bf16_hi(u.z); rest[6] -= bf16_lo(u.w); rest[7] -= bf16_hi(u.w);
      }
    }
    return r;
  }
  __device__ static __forceinline__ void widen(const bf16x8& a, float (&v)[8]) {
    const uint4 u = __builtin_bit_cast(uint4, a);
    v[0] = bf16_lo(u.x); v[1] = bf16_hi(u.x); v[2] = bf16_lo(u.y); v[3] = bf16_hi(u.y);
    v[4] = bf16_lo(u.z); v[5] = bf16_hi(u.z); v[6] = bf16_lo(u.w); v[7] = bf16_hi(u.w);
  }
};
template <> struct SsmOps<float> {
  static constexpr int PAD = 4;
  template <int NS> using Cm = SsmF8;
  using Ex = SsmF8;
  template <int NS> static constexpr int planes() { return 1; }
  template <int NS> __device__ static __forceinline__ SsmF8 split(const float (&v)[8]) {
    SsmF8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = v[j];
    return r;
  }
  __device__ static __forceinline__ void widen(const SsmF8& a, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = a.v[j];
  }
};

// ---- fragments out of LDS images (row-major, pitch in elements) ----
__device__ __forceinline__ bf16x8 ssm_row(const bf16* img, int pitch, int row, int k0) {
  return *reinterpret_cast<const bf16x8*>(img + row * pitch + k0);
}
__device__ __forceinline__ SsmF8 ssm_row(const float* img, int pitch, int row, int k0) {
  SsmF8 r;
  *reinterpret_cast<float4*>(r.v) = *reinterpret_cast<const float4*>(img + row * pitch + k0);
  *reinterpret_cast<float4*>(r.v + 4) = *reinterpret_cast<const float4*>(img + row * pitch + k0 + 4);
  return r;
}
// k in the "perm" order: k0 + 4q + 0..3 and k0 + 16 + 4q + 0..3
__device__ __forceinline__ bf16x8 ssm_row_perm(const bf16* img, int pitch, int row, int k0, int q) {
  const bf16x4 a = *reinterpret_cast<const bf16x4*>(img + row * pitch + k0 + 4 * q);
  const bf16x4 b = *reinterpret_cast<const bf16x4*>(img + row * pitch + k0 + 16 + 4 * q);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ SsmF8 ssm_row_perm(const float* img, int pitch, int row, int k0, int q) {
  SsmF8 r;
  *reinterpret_cast<float4*>(r.v) = *reinterpret_cast<const float4*>(img + row * pitch + k0 + 4 * q);
  *reinterpret_cast<float4*>(r.v + 4) = *reinterpret_cast<const float4*>(img + row * pitch + k0 + 16 + 4 * q);
  return r;
}
// transposed: lane (q, c) gets img[k0 + 8q + 0..7][col0 + c].  bf16: the transposing LDS read, in which a group of 16 lanes
// reads 4 rows x 16 columns and each lane receives one column.
__device__ __forceinline__ bf16x8 ssm_tr(const bf16* img, int pitch, int k0, int col0, int lane) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const int q = lane >> 4, c = lane & 15;
  const bf16* p = img + (k0 + 8 * q + (c >> 2)) * pitch + col0 + (c & 3) * 4;
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * pitch));
  return __builtin_shufflevector(__builtin_bit_cast(bf16x4, a), __builtin_bit_cast(bf16x4, b), 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ SsmF8 ssm_tr(const float* img, int pitch, int k0, int col0, int lane) {
  const int q = lane >> 4, c = lane & 15;
  SsmF8 r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r.v[j] = img[(k0 + 8 * q + j) * pitch + col0 + c];
  return r;
}
// computed operands kept in LDS as planes of T (bf16: NS parts; fp32: one)
template <int NS> __device__ __forceinline__ SsmB8<NS> ssm_row_planes(const bf16* img, int plane, int pitch, int row, int k0) {
  SsmB8<NS> r;
#pragma unroll
  for (int i = 0; i < NS; ++i) r.p[i] = ssm_row(img + i * plane, pitch, row, k0);
  return r;
}
template <int NS> __device__ __forceinline__ SsmF8 ssm_row_planes(const float* img, int, int pitch, int row, int k0) {
  return ssm_row(img, pitch, row, k0);
}
template <int NS> __device__ __forceinline__ SsmB8<NS> ssm_tr_planes(const bf16* img, int plane, int pitch, int k0, int col0, int lane) {
  SsmB8<NS> r;
#pragma unroll
  for (int i = 0; i < NS; ++i) r.p[i] = ssm_tr(img + i * plane, pitch, k0, col0, lane);
  return r;
}
template <int NS> __device__ __forceinline__ SsmF8 ssm_tr_planes(const float* img, int, int pitch, int k0, int col0, int lane) {
  return ssm_tr(img, pitch, k0, col0, lane);
}
// four consecutive computed values of a row into the planes
template <int NS> __device__ __forceinline__ void ssm_put4(bf16* img, int plane, int off, const float (&v)[4]) {
  float rest[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const uint2 u = make_uint2(pack_bf16x2(rest[0], rest[1]), pack_bf16x2(rest[2], rest[3]));
    *reinterpret_cast<uint2*>(img + i * plane + off) = u;
    if (i + 1 < NS) {
      rest[0] -= bf16_lo(u.x); rest[1] -= bf16_hi(u.x); rest[2] -= bf16_lo(u.y); rest[3] -= bf16_hi(u.y);
    }
  }
}
template <int NS> __device__ __forceinline__ void ssm_put4(float* img, int, int off, const float (&v)[4]) {
  *reinterpret_cast<float4*>(img + off) = make_float4(v[0], v[1], v[2], v[3]);
}

// ---- global memory, one type to fp32 and back ----
__device__ __forceinline__ float ssm_ld(const bf16* p) { return (float)*p; }
__device__ __forceinline__ float ssm_ld(const float* p) { return *p; }
__device__ __forceinline__ void ssm_st(bf16* p, float v) { *p = (bf16)v; }
__device__ __forceinline__ void ssm_st(float* p, float v) { *p = v; }
__device__ __forceinline__ void ssm_ld4(const bf16* p, float (&v)[4]) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  v[0] = bf16_lo(u.x); v[1] = bf16_hi(u.x); v[2] = bf16_lo(u.y); v[3] = bf16_hi(u.y);
}
__device__ __forceinline__ void ssm_ld4(const float* p, float (&v)[4]) {
  const float4 u = *reinterpret_cast<const float4*>(p);
  v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
}
__device__ __forceinline__ void ssm_st4(bf16* p, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}
__device__ __forceinline__ void ssm_st4(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
// four values as they lie in memory (kept in registers until they are needed)
template <typename T> struct SsmRaw4;
template <> struct SsmRaw4<bf16> {
  uint2 u;
  __device__ __forceinline__ void load(const bf16* p) { u = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void get(float (&v)[4]) const { v[0] = bf16_lo(u.x); v[1] = bf16_hi(u.x); v[2] = bf16_lo(u.y); v[3] = bf16_hi(u.y); }
  __device__ __forceinline__ void part(const bf16* p, int n) {
    bf16 t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = i < n ? p[i] : (bf16)0.f;
    __builtin_memcpy(&u, t, 8);
  }
};
template <> struct SsmRaw4<float> {
  float4 u;
  __device__ __forceinline__ void load(const float* p) { u = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void get(float (&v)[4]) const { v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w; }
  __device__ __forceinline__ void part(const float* p, int n) {
    float t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = i < n ? p[i] : 0.f;
    __builtin_memcpy(&u, t, 16);
  }
};
// four values of which the first `n` exist (n may be <= 0); `vec`: all four do and the address is aligned to them
template <typename T> __device__ __forceinline__ void ssm_ld4n(const T* p, int n, bool vec, float (&v)[4]) {
  if (vec && n >= 4) { ssm_ld4(p, v); return; }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = i < n ? ssm_ld(p + i) : 0.f;
}
template <typename T> __device__ __forceinline__ void ssm_st4n(T* p, int n, bool vec, const float (&v)[4]) {
  if (vec && n >= 4) { ssm_st4(p, v); return; }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) ssm_st(p + i, v[i]);
}
// the same where, VEC, four values exist or none does
template <bool VEC, typename T> __device__ __forceinline__ void ssm_ld4v(const T* p, int n, float (&v)[4]) {
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = 0.f;
    if (n > 0) ssm_ld4(p, v);
  } else ssm_ld4n(p, n, false, v);
}
template <bool VEC, typename T> __device__ __forceinline__ void ssm_st4v(T* p, int n, const float (&v)[4]) {
  if constexpr (VEC) {
    if (n > 0) ssm_st4(p, v);
  } else ssm_st4n(p, n, false, v);
}

__device__ __forceinline__ float ssm_exp2(float x) { return __builtin_amdgcn_exp2f(x); }   // v_exp_f32: 1 ulp, 0 below 2^-126
// exp(x) for |x| < 87 to about 2 units in the last place: 2^t with t = x log2 e in two parts (the product's rounding is made
// up for to first order); v_exp_f32 is good to one
__device__ __forceinline__ float ssm_exp(float x) {
  const float t = x * 1.44269502f;
  const float lo = fmaf(x, 1.44269502f, -t) + x * 1.92596303e-08f;
  const float e = ssm_exp2(t);
  return fmaf(e, lo * 0.693147182f, e);
}
// 1 / (1 + exp(-x)) of calls on T.  bf16: exp(-x) good to |x| 2^-24 of itself, far below the 2^-8 of their results.  fp32: to 3 units
// in the last place (exp(-x) 1.5, the sum 0.5, the reciprocal 1); under exp(-88) zero.  NaN passes through (selects, no minima).
template <typename T> __device__ __forceinline__ float ssm_sigmoid(float x) {
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(1.0f + ssm_exp2(x * -1.44269502f));
  float y = x > 87.f ? -87.f : -x;
  y = y > 88.f ? 88.f : y;
  const float s = __builtin_amdgcn_rcpf(1.0f + ssm_exp(y));
  return x < -88.f ? 0.f : s;
}
// max(x, 0) + log(1 + e), e = exp(-|x|): with s = e / (2 + e) <= 1/3 the logarithm is 2 atanh(s) = 2 (s + s^3 / 3 + s^5 / 5 ..);
// the terms up to s^15 leave 2e-9 of it, and small e keep their relative precision (steps of 1e-3 and less are common).  Below
// -87 the result is under the type's normal range: zero, so that tokens masked by -infinity or the type's lowest value do nothing
__device__ __forceinline__ float ssm_softplus(float x) {
  const float e = x < -87.f ? 0.f : ssm_exp(-fminf(fabsf(x), 87.f));
  const float s = e * __builtin_amdgcn_rcpf(2.0f + e), u = s * s;
  float p = fmaf(u, 1.0f / 15.0f, 1.0f / 13.0f);
  p = fmaf(p, u, 1.0f / 11.0f);
  p = fmaf(p, u, 1.0f / 9.0f);
  p = fmaf(p, u, 1.0f / 7.0f);
  p = fmaf(p, u, 1.0f / 5.0f);
  p = fmaf(p, u, 1.0f / 3.0f);
  p = fmaf(p, u, 1.0f);
  return x != x ? x : fmaxf(x, 0.f) + 2.0f * s * p;
}
// log2 of a token's decay exp(d A), in 64 bits (A2 = A log2 e).  Held to -1e5, which is a decay of zero as well: steps of 1e37
// would give sums outside fp32, and the difference of two infinite ones is no decay.
__device__ __forceinline__ double ssm_log_decay(float d, double A2) {
  const double l = (double)d * A2;
  return l < -1e5 ? -1e5 : l;
}

// 2^l of a sum of log decays (at most 0, but for a positive A) to two units in the last place: fp32's rounding of l, |l| 2^-25, is
// made up for to first order (a result outside the type is infinite or zero as it is)
__device__ __forceinline__ float ssm_decay(double l) {
  const float hi = (float)l, e = ssm_exp2(hi);
  return fabsf(hi) < 128.f ? fmaf(e, (float)(l - (double)hi) * 0.693147182f, e) : e;
}

// A ROWS x COLS image on its way from global memory (row stride `ld`) to LDS through the registers of a workgroup: load() is
// issued a chunk ahead of store(), so that its latency passes under the products between.  What lies outside rows x cols is
// written as zero: rows behind a sequence's end never enter a product, whatever they hold.  load() takes addresses inside
// the image for those too (no branch around a load: a merge of its result would wait for it), so rows >= 1, cols >= 1.
// VEC: 16-byte pieces are aligned and cols is a multiple of a piece.
template <typename T, int THREADS, int ROWS, int COLS, bool VEC>
struct SsmTile {
  static constexpr int V = 16 / sizeof(T), PIECES = COLS / V, N = (ROWS * PIECES + THREADS - 1) / THREADS;
  static constexpr int STEP = THREADS / PIECES;      // rows a turn of the workgroup covers
  uint4 u[N];
  __device__ __forceinline__ void load(const T* src, long ld, int rows, int cols) {
    if (VEC && rows >= ROWS && cols >= COLS && ROWS % STEP == 0) {   // a whole image: one offset a thread, the rest is uniform
      const unsigned off = ((threadIdx.x / PIECES) * (unsigned)ld + (threadIdx.x % PIECES) * V) * (unsigned)sizeof(T);
#pragma unroll
      for (int i = 0; i < N; ++i) u[i] = *reinterpret_cast<const uint4*>((const char*)(src + (long)(i * STEP) * ld) + off);
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = i * THREADS + threadIdx.x, r = e / PIECES, k = (e % PIECES) * V;
      const T* p = src + (long)min(r, rows - 1) * ld;
      if constexpr (VEC) u[i] = *reinterpret_cast<const uint4*>(p + (k < cols ? k : 0));
      else {
        T t[V];
#pragma unroll
        for (int j = 0; j < V; ++j) t[j] = p[min(k + j, cols - 1)];
        __builtin_memcpy(&u[i], t, 16);
      }
    }
  }
  __device__ __forceinline__ void store(T* img, int pitch, int rows, int cols) const {
    if (VEC && rows >= ROWS && cols >= COLS && ROWS % STEP == 0) {
      T* p = img + (threadIdx.x / PIECES) * pitch + (threadIdx.x % PIECES) * V;
#pragma unroll
      for (int i = 0; i < N; ++i) *reinterpret_cast<uint4*>(p + i * STEP * pitch) = u[i];
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = i * THREADS + threadIdx.x, r = e / PIECES, k = (e % PIECES) * V;
      if (ROWS * PIECES % THREADS != 0 && r >= ROWS) break;
      uint4 v = u[i];
      if constexpr (VEC) {
        if (r >= rows || k >= cols) v = make_uint4(0, 0, 0, 0);
      } else {
        T t[V];
        __builtin_memcpy(t, &v, 16);
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (r >= rows || k + j >= cols) t[j] = (T)0.f;
        __builtin_memcpy(&v, t, 16);
      }
      *reinterpret_cast<uint4*>(img + r * pitch + k) = v;
    }
  }
};

// inclusive sum over the 64 lanes of a wave in 64 bits, by data-parallel moves (no LDS): inside rows of 16 lanes, then a row's
// last lane into the next row, then the first half's last lane into the second half
template <int CTRL, int ROWS>
__device__ __forceinline__ double ssm_dpp_add(double v) {
  const long long b = __builtin_bit_cast(long long, v);
  const int lo = __builtin_amdgcn_update_dpp(0, (int)b, CTRL, ROWS, 0xf, true);
  const int hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xf, true);
  return v + __builtin_bit_cast(double, ((long long)hi << 32) | (unsigned)lo);
}
__device__ __forceinline__ double ssm_scan64(double v) {
  v = ssm_dpp_add<0x111, 0xf>(v);    // row_shr:1
  v = ssm_dpp_add<0x112, 0xf>(v);
  v = ssm_dpp_add<0x114, 0xf>(v);
  v = ssm_dpp_add<0x118, 0xf>(v);
  v = ssm_dpp_add<0x142, 0xa>(v);    // row_bcast:15 into rows 1 and 3
  return ssm_dpp_add<0x143, 0xc>(v); // row_bcast:31 into rows 2 and 3
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float ssm_dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, true));
}
__device__ __forceinline__ float ssm_scan64(float v) {
  v = ssm_dpp_add<0x111, 0xf>(v);
  v = ssm_dpp_add<0x112, 0xf>(v);
  v = ssm_dpp_add<0x114, 0xf>(v);
  v = ssm_dpp_add<0x118, 0xf>(v);
  v = ssm_dpp_add<0x142, 0xa>(v);
  return ssm_dpp_add<0x143, 0xc>(v);
}
__device__ __forceinline__ double ssm_last_lane(double v) {
  const long long b = __builtin_bit_cast(long long, v);
  const int lo = __builtin_amdgcn_readlane((int)b, 63), hi = __builtin_amdgcn_readlane((int)(b >> 32), 63);
  return __builtin_bit_cast(double, ((long long)hi << 32) | (unsigned)lo);
}
