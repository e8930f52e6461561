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

// ---- operand types by input type ----
template <typename T> struct SsmOps;
template <> struct SsmOps<bf16> {
  static constexpr int PAD = 8;                      // elements behind an LDS row: 16 bytes, rows start on other banks
  template <int NS> using Cm = SsmB8<NS>;
  using Ex = bf16x8;
  template <int NS> static constexpr int planes() { return NS; }
  template <int NS> __device__ static __forceinline__ SsmB8<NS> split(const float (&v)[8]) {
    SsmB8<NS> r;
    float rest[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) rest[j] = v[j];
#pragma unroll
    for (int i = 0; i < NS; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bf16 h = (bf16)rest[j];
        r.p[i][j] = h;
        if (i + 1 < NS) rest[j] -= (float)h;
      }
    return r;
  }
  __device__ static __forceinline__ void widen(const bf16x8& a, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = (float)a[j];
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

__device__ __forceinline__ float ssm_exp2(float x) { return __builtin_amdgcn_exp2f(x); }   // v_exp_f32: 1 ulp, 0 below 2^-126
__device__ __forceinline__ float ssm_sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }
__device__ __forceinline__ float ssm_softplus(float x) { return fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))); }

// A workgroup copies `rows` x `cols` elements (row stride `ld` in global memory) into an LDS image of ROWS x COLS; what lies
// outside is written as zero, so that rows behind a sequence's end never enter a product, whatever they hold.
// vec: 16-byte pieces are aligned and cols is a multiple of a piece.
template <typename T, int THREADS, int ROWS, int COLS>
__device__ __forceinline__ void ssm_stage(T* img, int pitch, const T* src, long ld, int rows, int cols, bool vec) {
  constexpr int V = 16 / sizeof(T), PIECES = COLS / V;
  for (int i = threadIdx.x; i < ROWS * PIECES; i += THREADS) {
    const int r = i / PIECES, k = (i - r * PIECES) * V;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (r < rows && k < cols) {
      const T* p = src + (long)r * ld + k;
      if (vec) u = *reinterpret_cast<const uint4*>(p);
      else {
        T t[V];
#pragma unroll
        for (int j = 0; j < V; ++j) t[j] = k + j < cols ? p[j] : (T)0.f;
        __builtin_memcpy(&u, t, 16);
      }
    }
    *reinterpret_cast<uint4*>(img + r * pitch + k) = u;
  }
}
