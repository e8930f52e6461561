// The norm behind one block and the norm before the next in one pass over the token stream:
//   h = residual + scale * gate o norm_post(y),   n = norm_pre(h)        (LayerNorm, or RMS: no centring, no bias)
// gate: none, one value per channel, per sample and channel, or per element.  Everything between is 32-bit and lives in
// registers: two rows in, two rows out.  Backward, with the rows' means and 1/std kept by the forward and h recomputed:
//   dh' = dh + norm_pre'(dn);  du = scale gate dh';  dresidual = dh';  dgate = scale u dh';  dy = norm_post'(du)
// Both passes are HBM bound.  A wave holds a row of up to 1024 columns, a workgroup of four waves a longer one.
#include "ssm_common.h"
#include "rvit_internal.h"
#include "ssm_args.h"

namespace {

template <typename T, int V>
__device__ __forceinline__ void ldv(const T* p, bool ok, float (&v)[V]) {
  if (!ok) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.f;
  } else if constexpr (V == 1) v[0] = ssm_ld(p);
  else ssm_ld4(p, v);
}
template <typename T, int V>
__device__ __forceinline__ void stv(T* p, const float (&v)[V]) {
  if constexpr (V == 1) ssm_st(p, v[0]);
  else ssm_st4(p, v);
}

// sum over the threads of a row; buf: one float per wave, two sets used in turn
template <int WPR>
__device__ __forceinline__ float row_sum(float v, float* buf, int& turn) {
  v = wave_sum(v);
  if constexpr (WPR == 1) return v;
  float* s = buf + (turn ^= 1) * WPR;
  if ((threadIdx.x & 63) == 0) s[(threadIdx.x >> 6) % WPR] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int i = 1; i < WPR; ++i) v += s[i];
  return v;
}

template <typename TY, int V>
__device__ __forceinline__ void ld_gate(const SandwichArgs& a, long row, int e, bool ok, float (&g)[V]) {
  if (a.gate_kind == 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) g[j] = 1.f;
    return;
  }
  const long at = (a.gate_kind == 1 ? 0 : a.gate_kind == 2 ? row / a.T : row) * a.E + e;
  if (a.gate_f32) ldv<float, V>((const float*)a.gate + at, ok, g);
  else ldv<TY, V>((const TY*)a.gate + at, ok, g);
}

template <typename TR, typename TY, int V, int WPR, int IT>
__global__ __launch_bounds__(256) void sandwich_fwd_kernel(SandwichArgs a) {
  __shared__ float buf[2 * WPR];
  int turn = 0;
  const int lid = threadIdx.x % (64 * WPR);
  const long row = (long)blockIdx.x * (4 / WPR) + threadIdx.x / (64 * WPR);
  if (row >= a.rows) return;     // whole waves; with WPR = 4 the whole workgroup
  const float inv = 1.0f / a.E;
  float y[IT][V], s = 0.f;
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int e = (it * 64 * WPR + lid) * V;
    ldv<TY, V>((const TY*)a.y + row * a.E + e, e < a.E, y[it]);
#pragma unroll
    for (int j = 0; j < V; ++j) s += y[it][j];
  }
  float h[IT][V];
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int e = (it * 64 * WPR + lid) * V;
    ldv<TR, V>((const TR*)a.res + row * a.E + e, e < a.E, h[it]);
  }
  const float m1 = a.rms ? 0.f : row_sum<WPR>(s, buf, turn) * inv;
  s = 0.f;
#pragma unroll
  for (int it = 0; it < IT; ++it)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = (it * 64 * WPR + lid) * V + j;
      const float d = e < a.E ? y[it][j] - m1 : 0.f;
      s = fmaf(d, d, s);
      y[it][j] = d;
    }
  const float r1 = 1.0f / sqrtf(row_sum<WPR>(s, buf, turn) * inv + a.eps);
  s = 0.f;
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int e = (it * 64 * WPR + lid) * V;
    const bool ok = e < a.E;
    float w[V], b[V], g[V];
    ldv<float, V>(a.w1 + e, ok, w);
    ldv<float, V>(a.b1 + e, ok && a.b1, b);
    ld_gate<TY, V>(a, row, e, ok, g);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      h[it][j] = fmaf(a.scale * g[j], fmaf(y[it][j] * r1, w[j], b[j]), h[it][j]);
      if (!ok) h[it][j] = 0.f;
      s += h[it][j];
    }
    if (ok) stv<TR, V>((TR*)a.h + row * a.E + e, h[it]);
  }
  const float m2 = a.rms ? 0.f : row_sum<WPR>(s, buf, turn) * inv;
  s = 0.f;
#pragma unroll
  for (int it = 0; it < IT; ++it)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = (it * 64 * WPR + lid) * V + j;
      const float d = e < a.E ? h[it][j] - m2 : 0.f;
      s = fmaf(d, d, s);
      h[it][j] = d;
    }
  const float r2 = 1.0f / sqrtf(row_sum<WPR>(s, buf, turn) * inv + a.eps);
#pragma unroll
  for (int it = 0; it < IT; ++it) {
    const int e = (it * 64 * WPR + lid) * V;
    const bool ok = e < a.E;
    float w[V], b[V], n[V];
    ldv<float, V>(a.w2 + e, ok, w);
    ldv<float, V>(a.b2 + e, ok && a.b2, b);
#pragma unroll
    for (int j = 0; j < V; ++j) n[j] = fmaf(h[it][j] * r2, w[j], b[j]);
    if (ok) stv<TY, V>((TY*)a.n + row * a.E + e, n);
  }
  if (a.stats && lid == 0) *reinterpret_cast<float4*>(a.stats + 4 * row) = make_float4(m1, r1, m2, r2);
}

// One workgroup per part of the rows; the columns' sums (dw1, db1, dw2, db2, dgate) stay in registers over its rows and leave
// as part[part][5][E], added in order by sandwich_sum_kernel: no atomics.
template <typename TR, typename TY, int V, int WPR, int IT>
__global__ __launch_bounds__(256) void sandwich_bwd_kernel(SandwichArgs a) {
  __shared__ float buf[2 * WPR];
  __shared__ float red[WPR == 1 ? 4 * 64 * IT * V : 1];
  int turn = 0;
  constexpr int GROUPS = 4 / WPR;
  const int lid = threadIdx.x % (64 * WPR), grp = threadIdx.x / (64 * WPR);
  const int part = blockIdx.x;
  long r0, r1;
  if (a.sample_parts) {
    const long b = part / a.sample_parts, k = part % a.sample_parts;
    r0 = b * a.T + k * a.part_rows;
    r1 = min(r0 + a.part_rows, (b + 1) * a.T);
  } else {
    r0 = (long)part * a.part_rows;
    r1 = min(r0 + a.part_rows, a.rows);
  }
  const float inv = 1.0f / a.E;
  float acc[5][IT][V];
#pragma unroll
  for (int k = 0; k < 5; ++k)
#pragma unroll
    for (int it = 0; it < IT; ++it)
#pragma unroll
      for (int j = 0; j < V; ++j) acc[k][it][j] = 0.f;
  for (long row = r0 + grp; row < r1; row += GROUPS) {
    const float4 st = *reinterpret_cast<const float4*>(a.stats + 4 * row);
    float y[IT][V], d[IT][V], hh[IT][V], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int e = (it * 64 * WPR + lid) * V;
      const bool ok = e < a.E;
      float w1[V], b1[V], w2[V], g[V], dn[V];
      ldv<TY, V>((const TY*)a.y + row * a.E + e, ok, y[it]);
      ldv<TR, V>((const TR*)a.res + row * a.E + e, ok, hh[it]);
      ldv<TY, V>((const TY*)a.dn + row * a.E + e, ok, dn);
      ldv<TR, V>((const TR*)a.dh + row * a.E + e, ok, d[it]);
      ldv<float, V>(a.w1 + e, ok, w1);
      ldv<float, V>(a.b1 + e, ok && a.b1, b1);
      ldv<float, V>(a.w2 + e, ok, w2);
      ld_gate<TY, V>(a, row, e, ok, g);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        y[it][j] = ok ? (y[it][j] - st.x) * st.y : 0.f;                           // normalised y
        const float h = fmaf(a.scale * g[j], fmaf(y[it][j], w1[j], b1[j]), hh[it][j]);
        hh[it][j] = ok ? (h - st.z) * st.w : 0.f;                                 // normalised h
        acc[2][it][j] = fmaf(dn[j], hh[it][j], acc[2][it][j]);
        acc[3][it][j] += dn[j];
        const float p = dn[j] * w2[j];
        s1 += p;
        s2 = fmaf(p, hh[it][j], s2);
        d[it][j] = fmaf(p, st.w, d[it][j]);
      }
    }
    s1 = a.rms ? 0.f : row_sum<WPR>(s1, buf, turn) * inv;
    s2 = row_sum<WPR>(s2, buf, turn) * inv;
    float t1 = 0.f, t2 = 0.f;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int e = (it * 64 * WPR + lid) * V;
      const bool ok = e < a.E;
      float w1[V], b1[V], g[V], dg[V];
      ldv<float, V>(a.w1 + e, ok, w1);
      ldv<float, V>(a.b1 + e, ok && a.b1, b1);
      ld_gate<TY, V>(a, row, e, ok, g);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        d[it][j] -= st.w * (s1 + hh[it][j] * s2);                                 // dh'
        const float sd = ok ? a.scale * d[it][j] : 0.f;
        dg[j] = sd * fmaf(y[it][j], w1[j], b1[j]);
        acc[4][it][j] += dg[j];
        const float du = sd * g[j];
        acc[0][it][j] = fmaf(du, y[it][j], acc[0][it][j]);
        acc[1][it][j] += du;
        hh[it][j] = du * w1[j];
        t1 += hh[it][j];
        t2 = fmaf(hh[it][j], y[it][j], t2);
      }
      if (ok) {
        stv<TR, V>((TR*)a.dres + row * a.E + e, d[it]);
        if (a.gate_kind == 3) {
          if (a.gate_f32) stv<float, V>((float*)a.dgate + row * a.E + e, dg);
          else stv<TY, V>((TY*)a.dgate + row * a.E + e, dg);
        }
      }
    }
    t1 = a.rms ? 0.f : row_sum<WPR>(t1, buf, turn) * inv;
    t2 = row_sum<WPR>(t2, buf, turn) * inv;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int e = (it * 64 * WPR + lid) * V;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = st.y * (hh[it][j] - t1 - y[it][j] * t2);
      if (e < a.E) stv<TY, V>((TY*)a.dy + row * a.E + e, o);
    }
  }
  float* out = a.part + (long)part * 5 * a.E;
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    if (k == 4 && (a.gate_kind == 0 || a.gate_kind == 3)) break;
    if constexpr (WPR == 1) {
      __syncthreads();
#pragma unroll
      for (int it = 0; it < IT; ++it)
#pragma unroll
        for (int j = 0; j < V; ++j) red[grp * 64 * IT * V + (it * 64 + lid) * V + j] = acc[k][it][j];
      __syncthreads();
      for (int e = threadIdx.x; e < a.E; e += 256) {
        constexpr int W = 64 * IT * V;
        out[(long)k * a.E + e] = (red[e] + red[W + e]) + (red[2 * W + e] + red[3 * W + e]);
      }
    } else {
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const int e = (it * 64 * WPR + lid) * V;
        if (e < a.E) stv<float, V>(out + (long)k * a.E + e, acc[k][it]);
      }
    }
  }
}

// columns of the parts, added in a fixed order: 16 threads take every 16th part of a column
__global__ __launch_bounds__(1024) void sandwich_sum_kernel(SandwichArgs a, int gate_bf16) {
  __shared__ double red[16][64];
  const int cx = threadIdx.x & 63, py = threadIdx.x >> 6;
  const int k = blockIdx.y, e = blockIdx.x * 64 + cx;
  double v = 0.0;
  if (e < a.E)
    for (int p = py; p < a.parts; p += 16) v += (double)a.part[((long)p * 5 + k) * a.E + e];
  red[py][cx] = v;
  __syncthreads();
  if (py == 0 && e < a.E) {
    for (int i = 1; i < 16; ++i) v += red[i][cx];
    float* out = k == 0 ? a.dw1 : k == 1 ? a.db1 : k == 2 ? a.dw2 : k == 3 ? a.db2 : (float*)a.dgate;
    if (k == 4 && gate_bf16) ((bf16*)out)[e] = (bf16)(float)v;
    else if (out) out[e] = (float)v;
  }
}
__global__ __launch_bounds__(256) void sandwich_sample_kernel(SandwichArgs a, int gate_bf16) {
  const long n = a.rows / a.T * a.E, i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const long b = i / a.E;
  const int e = i - b * a.E;
  double v = 0.0;
  for (int k = 0; k < a.sample_parts; ++k) v += (double)a.part[((b * a.sample_parts + k) * 5 + 4) * a.E + e];
  if (gate_bf16) ((bf16*)a.dgate)[i] = (bf16)(float)v;
  else ((float*)a.dgate)[i] = (float)v;
}

template <typename TR, typename TY, int V, int WPR, int IT>
int launch(const SandwichArgs& a, bool bwd, hipStream_t st) {
  if (bwd) {
    hipLaunchKernelGGL((sandwich_bwd_kernel<TR, TY, V, WPR, IT>), dim3(a.parts), dim3(256), 0, st, a);
    RVIT_CHECK_LAUNCH("sandwich_bwd");
    const int gb = a.gate_f32 ? 0 : (int)(sizeof(TY) == 2);
    hipLaunchKernelGGL(sandwich_sum_kernel, dim3((a.E + 63) / 64, a.gate_kind == 1 ? 5 : 4), dim3(1024), 0, st, a, gb);
    RVIT_CHECK_LAUNCH("sandwich_sum");
    if (a.gate_kind == 2) {
      const long n = a.rows / a.T * a.E;
      hipLaunchKernelGGL(sandwich_sample_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a, gb);
      RVIT_CHECK_LAUNCH("sandwich_sample");
    }
    return RVIT_OK;
  }
  constexpr int R = 4 / WPR;
  hipLaunchKernelGGL((sandwich_fwd_kernel<TR, TY, V, WPR, IT>), dim3((unsigned)((a.rows + R - 1) / R)), dim3(256), 0, st, a);
  RVIT_CHECK_LAUNCH("sandwich_fwd");
  return RVIT_OK;
}

template <typename TR, typename TY>
int launch_e(const SandwichArgs& a, bool bwd, hipStream_t st) {
  if (a.vec) {
    if (a.E <= 256) return launch<TR, TY, 4, 1, 1>(a, bwd, st);
    if (a.E <= 512) return launch<TR, TY, 4, 1, 2>(a, bwd, st);
    if (a.E <= 1024) return launch<TR, TY, 4, 1, 4>(a, bwd, st);
    if (a.E <= 2048) return launch<TR, TY, 4, 4, 2>(a, bwd, st);
    return launch<TR, TY, 4, 4, 4>(a, bwd, st);
  }
  if (a.E <= 256) return launch<TR, TY, 1, 1, 4>(a, bwd, st);
  if (a.E <= 512) return launch<TR, TY, 1, 4, 2>(a, bwd, st);
  if (a.E <= 1024) return launch<TR, TY, 1, 4, 4>(a, bwd, st);
  if (a.E <= 2048) return launch<TR, TY, 1, 4, 8>(a, bwd, st);
  return launch<TR, TY, 1, 4, 16>(a, bwd, st);
}

int go(const SandwichArgs& a, int rd, int d, bool bwd, hipStream_t st) {
  if (rd == RVIT_F32) return d == RVIT_F32 ? launch_e<float, float>(a, bwd, st) : launch_e<float, bf16>(a, bwd, st);
  return d == RVIT_F32 ? launch_e<bf16, float>(a, bwd, st) : launch_e<bf16, bf16>(a, bwd, st);
}

}  // namespace

int rvit_sandwich_fwd_impl(const SandwichArgs& a, int res_dtype, int dtype, hipStream_t st) { return go(a, res_dtype, dtype, false, st); }
int rvit_sandwich_bwd_impl(const SandwichArgs& a, int res_dtype, int dtype, hipStream_t st) { return go(a, res_dtype, dtype, true, st); }
