// The norm behind one block and the norm before the next in one pass over the token stream:
//   h = residual + scale * gate o norm_post(y),   n = norm_pre(h)        (LayerNorm, or RMS: no centring, no bias)
// gate: none, one value per channel, per sample and channel, or per element.  Everything between is 32-bit and lives in
// registers: two rows in, two rows out.  Backward, with the rows' means and 1/std kept by the forward and h recomputed:
//   dh' = dh + norm_pre'(dn);  du = scale gate dh';  dresidual = dh';  dgate = scale u dh';  dy = norm_post'(du)
// Both passes are HBM bound: at 25216 x 1024, bf16 blocks in an fp32 stream, forward 64 us (4.8 TB/s), backward 101 us (4.6 TB/s) and
// 9 us for the sums over its 1024 parts; all fp32 77 us (5.4 TB/s) and 136 us (4.6 TB/s).  Forward: a wave holds a row of up to 1024 columns, a workgroup of four waves a longer one.
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

__device__ __forceinline__ float wave_total(float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ssm_scan64(v)), 63)); }
// sums over the threads of a row (WPR waves; the 4 / WPR rows of a workgroup call it together); buf: 2 x 4 x 2 floats, two sets
// used in turn
template <int WPR>
__device__ __forceinline__ void row_sums(float& u, float& v, float* buf, int& turn) {
  u = wave_total(u);
  v = wave_total(v);
  if constexpr (WPR > 1) {
    float* s = buf + (turn ^= 1) * 8;
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) { s[w] = u; s[4 + w] = v; }
    __syncthreads();
    s += w / WPR * WPR;
    u = s[0];
    v = s[4];
#pragma unroll
    for (int i = 1; i < WPR; ++i) { u += s[i]; v += s[4 + i]; }
  }
}
template <int WPR>
__device__ __forceinline__ float row_sum(float u, float* buf, int& turn) {
  float none = 0.f;
  row_sums<WPR>(u, none, buf, turn);
  return u;
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
  __shared__ float buf[16];
  int turn = 0;
  const int lid = threadIdx.x % (64 * WPR);
  const long row = (long)blockIdx.x * (4 / WPR) + threadIdx.x / (64 * WPR);
  static_assert(WPR == 1 || WPR == 4, "a row that does not exist ends whole workgroups, or waves that meet no barrier");
  if (row >= a.rows) return;
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
template <typename T, int V> struct Raw;
template <typename T> struct Raw<T, 4> : SsmRaw4<T> {};
template <typename T> struct Raw<T, 1> {
  T u;
  __device__ __forceinline__ void load(const T* p) { u = *p; }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = (float)u; }
};

// The weights (and a gate per channel or sample) are in LDS, the next row's four inputs on their way in registers while a row is
// worked on.
template <typename TR, typename TY, int V, int WPR, int IT>
__global__ __launch_bounds__(256, IT * V > 4 ? 2 : 4) void sandwich_bwd_kernel(SandwichArgs a) {
  constexpr int W = 64 * WPR * IT * V;        // columns, padded
  __shared__ float buf[16];
  __shared__ __attribute__((aligned(16))) float sm[4 * W];      // weight and bias behind the block, weight before the next, scale x gate
  float *sw1 = sm, *sb1 = sm + W, *sw2 = sm + 2 * W, *sgt = sm + 3 * W;
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
  for (int e = threadIdx.x; e < W; e += 256) {
    const bool ok = e < a.E;
    float g[1];
    ld_gate<TY, 1>(a, a.gate_kind == 2 ? r0 : 0, e, ok && a.gate_kind != 3, g);
    sw1[e] = ok ? a.w1[e] : 0.f;
    sb1[e] = ok && a.b1 ? a.b1[e] : 0.f;
    sw2[e] = ok ? a.w2[e] : 0.f;
    sgt[e] = g[0] * a.scale;
  }
  __syncthreads();
  const float inv = 1.0f / a.E;
  float acc[5][IT][V];
#pragma unroll
  for (int k = 0; k < 5; ++k)
#pragma unroll
    for (int it = 0; it < IT; ++it)
#pragma unroll
      for (int j = 0; j < V; ++j) acc[k][it][j] = 0.f;
  Raw<TY, V> ny[IT], nn[IT];
  Raw<TR, V> nr[IT], nh[IT];
  float4 nst;
  auto fetch = [&](long row) {
    nst = *reinterpret_cast<const float4*>(a.stats + 4 * row);
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int e = (it * 64 * WPR + lid) * V;
      const long o = row * a.E + (e < a.E ? e : 0);      // (columns outside: any address of the row, dropped below)
      ny[it].load((const TY*)a.y + o);
      nr[it].load((const TR*)a.res + o);
      nn[it].load((const TY*)a.dn + o);
      nh[it].load((const TR*)a.dh + o);
    }
  };
  fetch(min(r0 + grp, r1 - 1));
  // (all rows of the workgroup take every turn: they meet in the sums.  One that is past the end counts as zero.)
  for (long base = r0; base < r1; base += GROUPS) {
    const long row = base + grp;
    const bool act = row < r1;
    // (the lane number anew for every row: the compiler would keep the weights of all its columns in registers)
    int lid = threadIdx.x % (64 * WPR);
    asm volatile("" : "+v"(lid));
    const float4 st = nst;
    float y[IT][V], d[IT][V], hh[IT][V], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int e = (it * 64 * WPR + lid) * V;
      const bool ok = e < a.E && act;
      float w1[V], b1[V], w2[V], g[V], dn[V];
      ny[it].get(y[it]);
      nr[it].get(hh[it]);
      nn[it].get(dn);
      nh[it].get(d[it]);
      ldv<float, V>(sw1 + e, true, w1);
      ldv<float, V>(sb1 + e, true, b1);
      ldv<float, V>(sw2 + e, true, w2);
      ldv<float, V>(sgt + e, true, g);
      if (a.gate_kind == 3) {
        ld_gate<TY, V>(a, row, e, ok, g);
#pragma unroll
        for (int j = 0; j < V; ++j) g[j] *= a.scale;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        y[it][j] = ok ? (y[it][j] - st.x) * st.y : 0.f;                           // normalised y
        const float h = fmaf(g[j], fmaf(y[it][j], w1[j], b1[j]), hh[it][j]);
        hh[it][j] = ok ? (h - st.z) * st.w : 0.f;                                 // normalised h
        dn[j] = ok ? dn[j] : 0.f;
        acc[2][it][j] = fmaf(dn[j], hh[it][j], acc[2][it][j]);
        acc[3][it][j] += dn[j];
        const float p = dn[j] * w2[j];
        s1 += p;
        s2 = fmaf(p, hh[it][j], s2);
        d[it][j] = fmaf(p, st.w, d[it][j]);
      }
    }
    if (base + GROUPS < r1) fetch(min(row + GROUPS, r1 - 1));
    row_sums<WPR>(s1, s2, buf, turn);
    s1 = a.rms ? 0.f : s1 * inv;
    s2 *= inv;
    float t1 = 0.f, t2 = 0.f;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int e = (it * 64 * WPR + lid) * V;
      const bool ok = e < a.E && act;
      float w1[V], b1[V], g[V], dg[V];
      ldv<float, V>(sw1 + e, true, w1);
      ldv<float, V>(sb1 + e, true, b1);
      ldv<float, V>(sgt + e, true, g);
      if (a.gate_kind == 3) {
        ld_gate<TY, V>(a, row, e, ok, g);
#pragma unroll
        for (int j = 0; j < V; ++j) g[j] *= a.scale;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        d[it][j] -= st.w * (s1 + hh[it][j] * s2);                                 // dh'
        const float dh = ok ? d[it][j] : 0.f;
        dg[j] = a.scale * dh * fmaf(y[it][j], w1[j], b1[j]);
        acc[4][it][j] += dg[j];
        const float du = dh * g[j];
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
    row_sums<WPR>(t1, t2, buf, turn);
    t1 = a.rms ? 0.f : t1 * inv;
    t2 *= inv;
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const int e = (it * 64 * WPR + lid) * V;
      float o[V];
#pragma unroll
      for (int j = 0; j < V; ++j) o[j] = st.y * (hh[it][j] - t1 - y[it][j] * t2);
      if (e < a.E && act) stv<TY, V>((TY*)a.dy + row * a.E + e, o);
    }
  }
  float* out = a.part + (long)part * 5 * a.E;
#pragma unroll
  for (int k = 0; k < 5; ++k) {
    if (k == 4 && (a.gate_kind == 0 || a.gate_kind == 3)) break;
    if constexpr (WPR < 4) {      // the groups' sums, through the weights' LDS
      __syncthreads();
#pragma unroll
      for (int it = 0; it < IT; ++it)
#pragma unroll
        for (int j = 0; j < V; ++j) sm[grp * W + (it * 64 * WPR + lid) * V + j] = acc[k][it][j];
      __syncthreads();
      for (int e = threadIdx.x; e < a.E; e += 256) {
        float v = sm[e] + sm[W + e];
        if (GROUPS == 4) v += sm[2 * W + e] + sm[3 * W + e];
        out[(long)k * a.E + e] = v;
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

// columns of the parts, added in a fixed order: 16 threads take every 16th part of a column.  Rows 0 .. 3 of the grid: the
// weights' and biases' sums; row 4 the channels' gates, or rows 4 and on, by turns, the samples' (over a sample's parts).
__global__ __launch_bounds__(1024) void sandwich_sum_kernel(SandwichArgs a, int gate_bf16) {
  __shared__ double red[16][64];
  const int cx = threadIdx.x & 63, py = threadIdx.x >> 6;
  const int e = blockIdx.x * 64 + cx;
  const bool sample = blockIdx.y >= 4 && a.gate_kind == 2;
  const int k = sample ? 4 : blockIdx.y;
  const long n = 5L * a.E, samples = sample ? a.rows / a.T : 1;
  const int parts = sample ? a.sample_parts : a.parts;
  for (long b = sample ? blockIdx.y - 4 : 0; b < samples; b += gridDim.y - 4) {
    const float* src = a.part + b * parts * n + (long)k * a.E + e;
    double v = 0.0;
    if (e < a.E) {
      int p = py;
      for (; p + 48 < parts; p += 64) {      // four loads on their way
        const float u = src[p * n], w = src[(p + 16) * n], x = src[(p + 32) * n], y = src[(p + 48) * n];
        v += ((double)u + (double)w) + ((double)x + (double)y);
      }
      for (; p < parts; p += 16) v += (double)src[p * n];
    }
    red[py][cx] = v;
    __syncthreads();
    if (py == 0 && e < a.E) {
      for (int i = 1; i < 16; ++i) v += red[i][cx];
      if (k == 4) {
        if (gate_bf16) ((bf16*)a.dgate)[b * a.E + e] = (bf16)(float)v;
        else ((float*)a.dgate)[b * a.E + e] = (float)v;
      } else {
        float* out = k == 0 ? a.dw1 : k == 1 ? a.db1 : k == 2 ? a.dw2 : a.db2;
        if (out) out[e] = (float)v;
      }
    }
    if (!sample) break;
    __syncthreads();
  }
}

template <typename TR, typename TY, int V, int WPR, int IT>
int launch_bwd(const SandwichArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((sandwich_bwd_kernel<TR, TY, V, WPR, IT>), dim3(a.parts), dim3(256), 0, st, a);
  RVIT_CHECK_LAUNCH("sandwich_bwd");
  const int gb = a.gate_f32 ? 0 : (int)(sizeof(TY) == 2);
  const long samples = a.gate_kind == 2 ? a.rows / a.T : a.gate_kind == 1;
  hipLaunchKernelGGL(sandwich_sum_kernel, dim3((a.E + 63) / 64, (unsigned)(4 + (samples < 4096 ? samples : 4096))), dim3(1024), 0, st, a, gb);
  RVIT_CHECK_LAUNCH("sandwich_sum");
  return RVIT_OK;
}
template <typename TR, typename TY, int V, int WPR, int IT>
int launch_fwd(const SandwichArgs& a, hipStream_t st) {
  constexpr int R = 4 / WPR;
  RVIT_CHECK_ARG((a.rows + R - 1) / R < (1 << 24), "sandwich_norm: %ld rows of %d columns are more than a launch can take", a.rows, a.E);
  hipLaunchKernelGGL((sandwich_fwd_kernel<TR, TY, V, WPR, IT>), dim3((unsigned)((a.rows + R - 1) / R)), dim3(256), 0, st, a);
  RVIT_CHECK_LAUNCH("sandwich_fwd");
  return RVIT_OK;
}

// Columns of a thread.  Forward: a wave takes a row of up to 1024 columns, which meets no barrier (64 us at 25216 x 1024, what
// its bytes take).  Backward: a thread keeps five sums a column over all rows, so few columns and more waves to a row.
template <typename TR, typename TY>
int launch_e(const SandwichArgs& a, bool bwd, hipStream_t st) {
  const int E = a.E;
  if (a.vec && !bwd) {
    if (E <= 256) return launch_fwd<TR, TY, 4, 1, 1>(a, st);
    if (E <= 512) return launch_fwd<TR, TY, 4, 1, 2>(a, st);
    if (E <= 1024) return launch_fwd<TR, TY, 4, 1, 4>(a, st);
    if (E <= 2048) return launch_fwd<TR, TY, 4, 4, 2>(a, st);
    return launch_fwd<TR, TY, 4, 4, 4>(a, st);
  }
  if (a.vec) {
    if (E <= 256) return launch_bwd<TR, TY, 4, 1, 1>(a, st);
    if (E <= 512) return launch_bwd<TR, TY, 4, 2, 1>(a, st);
    if (E <= 1024) return launch_bwd<TR, TY, 4, 4, 1>(a, st);
    if (E <= 2048) return launch_bwd<TR, TY, 4, 4, 2>(a, st);
    return launch_bwd<TR, TY, 4, 4, 4>(a, st);
  }
  if (!bwd) {
    if (E <= 256) return launch_fwd<TR, TY, 1, 1, 4>(a, st);
    if (E <= 512) return launch_fwd<TR, TY, 1, 4, 2>(a, st);
    if (E <= 1024) return launch_fwd<TR, TY, 1, 4, 4>(a, st);
    if (E <= 2048) return launch_fwd<TR, TY, 1, 4, 8>(a, st);
    return launch_fwd<TR, TY, 1, 4, 16>(a, st);
  }
  if (E <= 256) return launch_bwd<TR, TY, 1, 1, 4>(a, st);
  if (E <= 512) return launch_bwd<TR, TY, 1, 4, 2>(a, st);
  if (E <= 1024) return launch_bwd<TR, TY, 1, 4, 4>(a, st);
  if (E <= 2048) return launch_bwd<TR, TY, 1, 4, 8>(a, st);
  return launch_bwd<TR, TY, 1, 4, 16>(a, st);
}

int go(const SandwichArgs& a, int rd, int d, bool bwd, hipStream_t st) {
  if (rd == RVIT_F32) return d == RVIT_F32 ? launch_e<float, float>(a, bwd, st) : launch_e<float, bf16>(a, bwd, st);
  return d == RVIT_F32 ? launch_e<bf16, float>(a, bwd, st) : launch_e<bf16, bf16>(a, bwd, st);
}

}  // namespace

int rvit_sandwich_fwd_impl(const SandwichArgs& a, int res_dtype, int dtype, hipStream_t st) { return go(a, res_dtype, dtype, false, st); }
int rvit_sandwich_bwd_impl(const SandwichArgs& a, int res_dtype, int dtype, hipStream_t st) { return go(a, res_dtype, dtype, true, st); }
