// Selective state-space scan, backward.  With v' = dy silu(z) the gradient of v, and the forward's notation
// (ssm_scan.hip), a chunk's gradients follow from the state before it (kept by the forward) and the gradient dS of the
// state behind it:
//   G = C B^T, W = v' x^T, both over s <= t of the chunk
//   dx_s = d_s [ sum_t (G o E)_ts v'_t + exp(L_Q - L_s) dS B_s ] + D v'_s
//   dB_s = d_s [ sum_t (W o E)_ts C_t + exp(L_Q - L_s) dS^T x_s ]      summed over the heads of a group
//   dC_t = sum_s (W o E)_ts d_s B_s + exp(L_t) S^T v'_t                summed over the heads of a group
//   e_s  = sum_t (G W E)_ts + exp(L_Q - L_s) x_s . dS B_s              the part of dd that does not go through a decay
//   da_u = sum_{s < u <= t} M_ts + sum_{t >= u} rho_t + sum_{s < u} sigma_s + exp(L_Q) <dS, S>
//          M = G W E d_s,  rho_t = exp(L_t) C_t . S^T v'_t,  sigma_s = d_s exp(L_Q - L_s) x_s . dS B_s
//   dd = e + A da;  ddt = dd sigmoid(dt + bias);  dA = sum da d;  dD = sum v' x;  dz = dy v silu'(z)
// da is written as a sum of what really passes through token u's decay.  The shorter form, a reverse running sum over the
// whole sequence of dy . y - d e, takes the difference of two large equal parts at every token of a head that forgets fast,
// and its rounding errors add up along the sequence into dA.
// Two launches: the sweep computes dS of every chunk (from the last to the first, the gradient in registers), then every
// chunk is on its own.
#include "ssm_common.h"
#include "rvit_internal.h"
#include "ssm_args.h"

namespace {

constexpr int Q = SSM_CHUNK;

// d_t and the running log decay of a chunk, by one wave; returns the chunk's log decay (base 2, 64 bits)
template <typename T>
__device__ __forceinline__ double chunk_decay(const SsmScanArgs& f, const T* dt, long sdt, int live, double A2, float bias, int lane, float& raw,
                                              float& d, double& l2) {
  raw = lane < live ? ssm_ld(dt + lane * sdt) + bias : 0.f;
  d = lane < live ? ssm_softplus(raw) : 0.f;
  l2 = (double)d * A2;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double up = __shfl_up(l2, o, 64);
    if (lane >= o) l2 += up;
  }
  return __shfl(l2, 63, 64);
}

// ---- sweep: dS before a chunk = exp(L_Q) dS behind it + sum_t exp(L_t) v'_t C_t^T ----
template <typename T, int NP, bool OUT>
__global__ __launch_bounds__(256) void ssm_scan_bwd_state_kernel(SsmBwdArgs a) {
  using O = SsmOps<T>;
  constexpr int PN = NP + O::PAD, PV = 68, NT = NP / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* Cs = (T*)smem;
  float* Vs = (float*)(Cs + Q * PN);
  float* se = Vs + Q * PV;
  const SsmScanArgs& f = a.f;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, q = lane >> 4, c = lane & 15;
  long id = blockIdx.x;
  const int seg = id % f.nseg; id /= f.nseg;
  const int pb = id % f.pblocks; id /= f.pblocks;
  const int h = id % f.H, b = id / f.H;
  const int g = h / (f.H / f.G);
  const int len = f.lengths ? min(max(f.lengths[b], 0), f.T) : f.T;
  const int pw = min(64, f.P - pb * 64), p0 = 16 * w;
  const T* Cm = (const T*)f.Cm + b * f.scb + (long)g * f.N;
  const T* dt = (const T*)f.dt + b * f.sdb + h;
  const long hp = (long)h * f.P + pb * 64;
  const T* z = f.z ? (const T*)f.z + b * f.szb + hp : nullptr;
  const T* dy = (const T*)a.dy + b * a.syb + hp;
  const double A2 = (double)f.A[h] * 1.4426950408889634;
  const float bias = f.dt_bias ? f.dt_bias[h] : 0.f;
  f32x4 S[NT];
  const bool has_p = p0 + c < pw;
  const long srow = (((long)b * f.H + h) * f.P + pb * 64 + p0 + c) * f.N;
  const float* s0 = OUT ? (f.nseg > 1 ? f.seg_state + seg * f.seg_stride : a.dstate_out) : nullptr;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (s0 && has_p) ssm_ld4n(s0 + srow + 16 * nt + 4 * q, f.N - 16 * nt - 4 * q, f.vec_state, v);
    S[nt] = f32x4{v[0], v[1], v[2], v[3]};
  }
  double total = 0.0;
  const int c0 = seg * f.seg_chunks, c1 = min(f.nchunks, c0 + f.seg_chunks);
  for (int ch = c1 - 1; ch >= c0; --ch) {
    const int t0 = ch * Q;
    const int live = min(max(len - t0, 0), Q);
    if (live == 0) continue;
    if (OUT && has_p) {
      float* out = a.dstates + (long)ch * f.seg_stride + srow;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float v[4] = {S[nt][0], S[nt][1], S[nt][2], S[nt][3]};
        ssm_st4n(out + 16 * nt + 4 * q, f.N - 16 * nt - 4 * q, f.vec_state, v);
      }
    }
    __syncthreads();
    ssm_stage<T, 256, Q, NP>(Cs, PN, Cm + t0 * f.sct, f.sct, live, f.N, f.vec_bc);
    for (int i = threadIdx.x; i < Q * 16; i += 256) {
      const int t = i >> 4, p = (i & 15) * 4;
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (t < live && p < pw) {
        ssm_ld4n(dy + (t0 + t) * a.syt + p, pw - p, a.vec_dy, v);
        if (z) {
          float zv[4];
          ssm_ld4n(z + (t0 + t) * f.szt + p, pw - p, f.vec_z, zv);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] *= zv[j] * ssm_sigmoid(zv[j]);
        }
      }
      *reinterpret_cast<float4*>(Vs + t * PV + p) = make_float4(v[0], v[1], v[2], v[3]);
    }
    if (w == 0) {
      float raw, d;
      double l2;
      total += chunk_decay<T>(f, dt + t0 * f.sdt, f.sdt, live, A2, bias, lane, raw, d, l2);
      se[lane] = ssm_exp2((float)l2);
    }
    __syncthreads();
    const float eQ = se[Q - 1];
    if (p0 < pw) {
      typename O::template Cm<3> vw[2];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int t = 32 * ks + 8 * q + j;
          v[j] = Vs[t * PV + p0 + c] * se[t];
        }
        vw[ks] = O::template split<3>(v);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        S[nt] *= eQ;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) S[nt] = ssm_mma(ssm_tr(Cs, PN, 32 * ks, 16 * nt, lane), vw[ks], S[nt]);
      }
    }
  }
  float* out = nullptr;
  if (!OUT) {
    out = f.seg_state + seg * f.seg_stride;
    if (threadIdx.x == 0 && pb == 0) f.seg_decay[((long)seg * f.B + b) * f.H + h] = total;
  } else if (a.dstate0 && seg == 0) {
    out = a.dstate0;
  }
  if (out && has_p) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float v[4] = {S[nt][0], S[nt][1], S[nt][2], S[nt][3]};
      ssm_st4n(out + srow + 16 * nt + 4 * q, f.N - 16 * nt - 4 * q, f.vec_state, v);
    }
  }
}

// ---- the gradients of one chunk ----
// One workgroup (eight waves) per (sample, chunk, group, part of the group's heads).  B and C stay in LDS over its heads and
// the sums dB, dC over them in registers (wave: 16 states x 16 .. 64 tokens), so that shared heads cost no atomics.
template <typename T, int NP>
struct BwdLds {
  using O = SsmOps<T>;
  static constexpr int PN = NP + O::PAD, PX = 64 + O::PAD;
  static constexpr int VP = O::template planes<3>(), GP = O::template planes<2>();
  static constexpr int BS = 0, CS = BS + Q * PN, XS = CS + Q * PN, VS = XS + Q * PX, GS = VS + VP * Q * PX, WS = GS + GP * Q * PX, END = WS + GP * Q * PX;
  // floats behind: d, hi, lo, exp(L_Q - L), exp(L): 5 Q;  column sums by token tile: 2 x 4 Q;  row sums by tile: 4 Q;
  // rho by state tile: 8 Q;  sigma by channel tile: 4 Q;  <dS, S> and dD by wave: 16
  static constexpr int FLOATS = 5 * Q + 8 * Q + 4 * Q + 8 * Q + 4 * Q + 16;
  static constexpr int BYTES = END * (int)sizeof(T) + FLOATS * 4;
};

// sum over the 16 lanes of a row, in all of them (data-parallel moves inside the vector ALU, no LDS)
__device__ __forceinline__ float row16_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, true));   // row_ror:8
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xf, 0xf, true));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x122, 0xf, 0xf, true));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x121, 0xf, 0xf, true));
  return v;
}
__device__ __forceinline__ float groups_sum(float v) {   // over the four lanes with the same lane & 15
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

template <typename T, int NP>
__global__ __launch_bounds__(512) void ssm_scan_bwd_chunk_kernel(SsmBwdArgs a) {
  using O = SsmOps<T>;
  using L = BwdLds<T, NP>;
  constexpr int PN = L::PN, PX = L::PX, NT = NP / 16, CG = 8 / NT, CT = 4 / CG;   // column groups, column tiles of a wave
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* Bs = (T*)smem + L::BS;
  T* Cs = (T*)smem + L::CS;
  T* Xs = (T*)smem + L::XS;
  T* Vs = (T*)smem + L::VS;
  T* Gs = (T*)smem + L::GS;
  T* Ws = (T*)smem + L::WS;
  float* sd = (float*)((T*)smem + L::END);
  float* shi = sd + Q;
  float* slo = shi + Q;
  float* sw = slo + Q;
  float* se = sw + Q;
  float* r_e = se + Q;          // [4][Q] sum over a tile of tokens of (G W E)_ts
  float* r_z = r_e + 4 * Q;     // [4][Q] sum over a tile's t >= u of its own s < u of M_ts
  float* r_m = r_z + 4 * Q;     // [4][Q] sum over a tile's s of M_ts, by s tile and t
  float* r_rho = r_m + 4 * Q;   // [8][Q]
  float* r_sig = r_rho + 8 * Q; // [4][Q]
  float* r_w = r_sig + 4 * Q;   // [2][8]
  const SsmScanArgs& f = a.f;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, q = lane >> 4, c = lane & 15;
  long id = blockIdx.x;
  const int hs = id % a.hsplit; id /= a.hsplit;
  const int g = id % f.G; id /= f.G;
  const int ch = id % f.nchunks, b = id / f.nchunks;
  const int r = f.H / f.G, t0 = ch * Q;
  const int h0 = g * r + hs * a.hper, h1 = min(g * r + r, h0 + a.hper);
  const int len = f.lengths ? min(max(f.lengths[b], 0), f.T) : f.T;
  const int live = min(max(len - t0, 0), Q), here = min(f.T - t0, Q);
  const long ldo = (long)f.H * f.P;
  float* part = a.part + ((long)b * f.nchunks + ch) * f.H * 3;
  const int nt = w % NT, cg = w / NT;
  f32x4 accB[CT], accC[CT];
#pragma unroll
  for (int k = 0; k < CT; ++k) accB[k] = accC[k] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (live == 0) {
    for (int h = h0; h < h1; ++h) {
      for (int i = threadIdx.x; i < here * f.P; i += 512) {
        const int t = i / f.P, p = i - t * f.P;
        const long o = ((long)b * f.T + t0 + t) * ldo + (long)h * f.P + p;
        ssm_st((T*)a.dx + o, 0.f);
        if (a.dz) ssm_st((T*)a.dz + o, 0.f);
      }
      if (threadIdx.x < here) ssm_st((T*)a.ddt + ((long)b * f.T + t0 + threadIdx.x) * f.H + h, 0.f);
      if (threadIdx.x < 3) part[h * 3 + threadIdx.x] = 0.f;
    }
  } else {
    ssm_stage<T, 512, Q, NP>(Bs, PN, (const T*)f.Bm + b * f.sbb + t0 * f.sbt + (long)g * f.N, f.sbt, live, f.N, f.vec_bc);
    ssm_stage<T, 512, Q, NP>(Cs, PN, (const T*)f.Cm + b * f.scb + t0 * f.sct + (long)g * f.N, f.sct, live, f.N, f.vec_bc);
    // tiles above the diagonal that a 32-wide step reads: (0, 1) and (2, 3); they stay zero
    for (int i = threadIdx.x; i < 2 * 16 * 16; i += 512) {
      const int k = i >> 8, o = ((i >> 4 & 15) + 32 * k) * PX + 16 + 32 * k + (i & 15);
#pragma unroll
      for (int pl = 0; pl < L::GP; ++pl) { Gs[pl * Q * PX + o] = (T)0.f; Ws[pl * Q * PX + o] = (T)0.f; }
    }
    for (int h = h0; h < h1; ++h) {
      const float Ah = f.A[h], Dh = f.D ? f.D[h] : 0.f;
      float raw = 0.f, e_u = 0.f, da_u = 0.f, dD = 0.f;     // of token `lane`, in wave 0, over the channel blocks
      for (int pb = 0; pb < f.pblocks; ++pb) {
        const int pw = min(64, f.P - pb * 64);
        const long hp = (long)h * f.P + pb * 64;
        const long srow = (((long)ch * f.B + b) * f.H + h) * f.P * f.N + (long)pb * 64 * f.N;
        const float* S0 = f.states + srow;
        const float* dS = a.dstates + srow;
        // state columns of this wave's 16 states, k = channels (A operands of the products with x and v')
        float dsc[2][8], sc[2][8];
        const int n = 16 * nt + c;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int p = 32 * ks + 8 * q + j;
            const bool in = p < pw && n < f.N;
            dsc[ks][j] = in ? dS[(long)p * f.N + n] : 0.f;
            sc[ks][j] = in ? S0[(long)p * f.N + n] : 0.f;
          }
        __syncthreads();
        float dd_part = 0.f;
        for (int i = threadIdx.x; i < Q * 16; i += 512) {
          const int t = i >> 4, p = (i & 15) * 4;
          float xv[4] = {0.f, 0.f, 0.f, 0.f}, dv[4] = {0.f, 0.f, 0.f, 0.f};
          if (p < pw && t < here) {
            const long o = ((long)b * f.T + t0 + t) * ldo + hp + p;
            float dzv[4] = {0.f, 0.f, 0.f, 0.f};
            if (t < live) {
              ssm_ld4n((const T*)f.x + b * f.sxb + (t0 + t) * f.sxt + hp + p, pw - p, f.vec_x, xv);
              ssm_ld4n((const T*)a.dy + b * a.syb + (t0 + t) * a.syt + hp + p, pw - p, a.vec_dy, dv);
              if (f.z) {
                float zv[4], vv[4];
                ssm_ld4n((const T*)f.z + b * f.szb + (t0 + t) * f.szt + hp + p, pw - p, f.vec_z, zv);
                ssm_ld4n((const T*)f.v + o, pw - p, f.vec_y, vv);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const float sg = ssm_sigmoid(zv[j]);
                  dzv[j] = dv[j] * vv[j] * (sg + zv[j] * sg * (1.f - sg));
                  dv[j] *= zv[j] * sg;
                }
              }
#pragma unroll
              for (int j = 0; j < 4; ++j) dd_part += xv[j] * dv[j];
            }
            if (a.dz) ssm_st4n((T*)a.dz + o, pw - p, a.vec_out, dzv);
          }
          ssm_put4<1>(Xs, 0, t * PX + p, xv);
          ssm_put4<3>(Vs, Q * PX, t * PX + p, dv);
        }
        dd_part = wave_sum(dd_part);
        if (lane == 0) r_w[8 + w] = dd_part;
        if (w == 0 && pb == 0) {
          float d;
          double l2;
          const double end = chunk_decay<T>(f, (const T*)f.dt + b * f.sdb + t0 * f.sdt + h, f.sdt, live, (double)Ah * 1.4426950408889634,
                                            f.dt_bias ? f.dt_bias[h] : 0.f, lane, raw, d, l2);
          sd[lane] = d;
          shi[lane] = (float)l2;
          slo[lane] = (float)(l2 - (double)(float)l2);
          sw[lane] = ssm_exp2((float)(end - l2));
          se[lane] = ssm_exp2((float)l2);
        }
        __syncthreads();
        // score tiles (tt, st), st <= tt: ten of them
        for (int k = w; k < 10; k += 8) {
          const int tt = k < 1 ? 0 : k < 3 ? 1 : k < 6 ? 2 : 3, st = k - tt * (tt + 1) / 2;
          f32x4 G = {0.f, 0.f, 0.f, 0.f}, W = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < NP; ks += 32)
            G = ssm_mma(ssm_row(Bs, PN, 16 * st + c, ks + 8 * q), ssm_row(Cs, PN, 16 * tt + c, ks + 8 * q), G);
#pragma unroll
          for (int ks = 0; ks < 64; ks += 32)
            W = ssm_mma(ssm_row(Xs, PX, 16 * st + c, ks + 8 * q), ssm_row_planes<3>(Vs, Q * PX, PX, 16 * tt + c, ks + 8 * q), W);
          const int t = 16 * tt + c;
          const float thi = shi[t], tlo = slo[t];
          float gv[4], wv[4], m[4], ec[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int s = 16 * st + 4 * q + i;
            const float E = s <= t ? ssm_exp2((thi - shi[s]) + (tlo - slo[s])) : 0.f;
            const float d = sd[s];
            gv[i] = s <= t ? G[i] * E * d : 0.f;
            wv[i] = s <= t ? W[i] * E * d : 0.f;
            ec[i] = s <= t ? G[i] * W[i] * E : 0.f;
            m[i] = ec[i] * d;
          }
          ssm_put4<2>(Gs, Q * PX, t * PX + 16 * st + 4 * q, gv);
          ssm_put4<2>(Ws, Q * PX, t * PX + 16 * st + 4 * q, wv);
          // sums: of a row's tile, and of a row's part before u over the rows t >= u
          const float m4 = (m[0] + m[1]) + (m[2] + m[3]);
          const float u1 = __shfl_up(m4, 16, 64), u2 = __shfl_up(m4, 32, 64), u3 = __shfl_up(m4, 48, 64);
          float pre = (q >= 1 ? u1 : 0.f) + (q >= 2 ? u2 : 0.f) + (q >= 3 ? u3 : 0.f);
          if (q == 3) r_m[st * Q + t] = pre + m4;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int s = 16 * st + 4 * q + i;
            const float es = row16_sum(ec[i]), zs = row16_sum(s <= t ? pre : 0.f);
            pre += m[i];
            if (c == 0) { r_e[tt * Q + s] = es; r_z[tt * Q + s] = zs; }
          }
        }
        __syncthreads();
        // dx: wave = 16 channels x 32 tokens
        {
          const int pt = w & 3, p0 = 16 * pt;
          if (p0 < pw) {
            f32x4 acc[2];
            acc[0] = acc[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int m = 0; m < NP / 32; ++m) {
              float v[8];
              const int k = 32 * m + 8 * q;
              float lo[4] = {0.f, 0.f, 0.f, 0.f}, hi[4] = {0.f, 0.f, 0.f, 0.f};
              if (p0 + c < pw) {
                ssm_ld4n(dS + (long)(p0 + c) * f.N + k, f.N - k, f.vec_state, lo);
                ssm_ld4n(dS + (long)(p0 + c) * f.N + k + 4, f.N - k - 4, f.vec_state, hi);
              }
#pragma unroll
              for (int j = 0; j < 4; ++j) { v[j] = lo[j]; v[4 + j] = hi[j]; }
              const auto df = O::template split<3>(v);
#pragma unroll
              for (int k2 = 0; k2 < 2; ++k2) acc[k2] = ssm_mma(df, ssm_row(Bs, PN, 32 * (w >> 2) + 16 * k2 + c, k), acc[k2]);
            }
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
              const int st = 2 * (w >> 2) + k2, s = 16 * st + c, p = p0 + 4 * q;
              float sig = 0.f;
#pragma unroll
              for (int i = 0; i < 4; ++i) sig += ssm_ld(Xs + s * PX + p + i) * acc[k2][i];
              sig = groups_sum(sig);
              if (q == 0) r_sig[pt * Q + s] = sig;
              acc[k2] *= sw[s] * sd[s];
              for (int ks = st / 2; ks < 2; ++ks)
                acc[k2] = ssm_mma(ssm_tr_planes<2>(Vs, Q * PX, PX, 32 * ks, p0, lane), ssm_tr_planes<2>(Gs, Q * PX, PX, 32 * ks, 16 * st, lane), acc[k2]);
              if (s < here && p < pw) {
                float out[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  float v = 0.f;
#pragma unroll
                  for (int pl = L::VP - 1; pl >= 0; --pl) v += ssm_ld(Vs + pl * Q * PX + s * PX + p + i);
                  out[i] = acc[k2][i] + Dh * v;
                }
                ssm_st4n((T*)a.dx + ((long)b * f.T + t0 + s) * ldo + hp + p, pw - p, a.vec_out, out);
              }
            }
          } else if (lane < 32) {
            r_sig[pt * Q + 32 * (w >> 2) + lane] = 0.f;
          }
        }
        // dB, dC, rho, <dS, S>
        {
          const auto d0 = O::template split<2>(dsc[0]), d1 = O::template split<2>(dsc[1]);
          const auto s0 = O::template split<3>(sc[0]), s1 = O::template split<3>(sc[1]);
          float kap = 0.f;
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j) kap += dsc[ks][j] * sc[ks][j];
          kap = wave_sum(kap);
          if (lane == 0) r_w[w] = cg == 0 ? kap : 0.f;
#pragma unroll
          for (int k = 0; k < CT; ++k) {
            const int ct = cg * CT + k, t = 16 * ct + c;
            f32x4 tmp = {0.f, 0.f, 0.f, 0.f};
            tmp = ssm_mma(d0, ssm_row(Xs, PX, t, 8 * q), tmp);
            tmp = ssm_mma(d1, ssm_row(Xs, PX, t, 32 + 8 * q), tmp);
            accB[k] += tmp * (sw[t] * sd[t]);
            for (int ks = ct / 2; ks < 2; ++ks)
              accB[k] = ssm_mma(ssm_tr(Cs, PN, 32 * ks, 16 * nt, lane), ssm_tr_planes<2>(Ws, Q * PX, PX, 32 * ks, 16 * ct, lane), accB[k]);
            tmp = f32x4{0.f, 0.f, 0.f, 0.f};
            tmp = ssm_mma(s0, ssm_row_planes<3>(Vs, Q * PX, PX, t, 8 * q), tmp);
            tmp = ssm_mma(s1, ssm_row_planes<3>(Vs, Q * PX, PX, t, 32 + 8 * q), tmp);
            tmp *= se[t];
            float rho = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) rho += ssm_ld(Cs + t * PN + 16 * nt + 4 * q + i) * tmp[i];
            rho = groups_sum(rho);
            if (q == 0) r_rho[nt * Q + t] = rho;
            accC[k] += tmp;
            for (int ks = 0; ks <= ct / 2; ++ks)
              accC[k] = ssm_mma(ssm_tr(Bs, PN, 32 * ks, 16 * nt, lane), ssm_row_planes<2>(Ws, Q * PX, PX, t, 32 * ks + 8 * q), accC[k]);
          }
        }
        __syncthreads();
        if (w == 0) {     // token `lane`
          const int tl = lane >> 4;
          float e = 0.f, zz = 0.f, sg = 0.f, rho = 0.f, kap = 0.f;
          for (int tt = tl; tt < 4; ++tt) { e += r_e[tt * Q + lane]; zz += r_z[tt * Q + lane]; }
#pragma unroll
          for (int k = 0; k < 4; ++k) sg += r_sig[k * Q + lane];
#pragma unroll
          for (int k = 0; k < NT; ++k) rho += r_rho[k * Q + lane];
#pragma unroll
          for (int k = 0; k < 8; ++k) { kap += r_w[k]; dD += r_w[8 + k]; }
          sg *= sw[lane];
          e += sg;
          sg *= sd[lane];
          // rows' sums over the s tiles before u's own, over t >= u
          float rs[3], run = 0.f;
#pragma unroll
          for (int k = 0; k < 3; ++k) {
            run += k <= tl ? r_m[k * Q + lane] : 0.f;
            rs[k] = run;
          }
          float suf[4] = {rho, rs[0], rs[1], rs[2]}, pre = sg;
#pragma unroll
          for (int o = 1; o < 64; o <<= 1) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float dn = __shfl_down(suf[k], o, 64);
              if (lane + o < 64) suf[k] += dn;
            }
            const float up = __shfl_up(pre, o, 64);
            if (lane >= o) pre += up;
          }
          const float before = __shfl_up(pre, 1, 64);
          const float rows = tl == 0 ? 0.f : tl == 1 ? suf[1] : tl == 2 ? suf[2] : suf[3];
          da_u += (zz + rows) + suf[0] + (lane > 0 ? before : 0.f) + se[Q - 1] * kap;
          e_u += e;
          if (pb == f.pblocks - 1) {
            const bool ok = lane < live;
            const float ddt = ok ? (e_u + Ah * da_u) * ssm_sigmoid(raw) : 0.f;
            if (lane < here) ssm_st((T*)a.ddt + ((long)b * f.T + t0 + lane) * f.H + h, ddt);
            const float sA = wave_sum(ok ? da_u * sd[lane] : 0.f), sb = wave_sum(ddt);
            if (lane == 0) { part[h * 3] = sA; part[h * 3 + 1] = dD; part[h * 3 + 2] = sb; }
          }
        }
      }
    }
  }
  // accB, accC: states 16nt + 4q + i of token 16 ct + c
#pragma unroll
  for (int k = 0; k < CT; ++k) {
    const int t = 16 * (cg * CT + k) + c, n = 16 * nt + 4 * q;
    if (t < here && n < f.N) {
      const long o = (((long)b * f.T + t0 + t) * f.G + g) * f.N + n;
      const float vb[4] = {accB[k][0], accB[k][1], accB[k][2], accB[k][3]}, vc[4] = {accC[k][0], accC[k][1], accC[k][2], accC[k][3]};
      if (a.hsplit == 1) {
        ssm_st4n((T*)a.dB + o, f.N - n, a.vec_dbc, vb);
        ssm_st4n((T*)a.dC + o, f.N - n, a.vec_dbc, vc);
      } else {
        const long whole = (long)f.B * f.T * f.G * f.N;
        ssm_st4n(a.dbc_part + 2 * hs * whole + o, f.N - n, a.vec_dbc, vb);
        ssm_st4n(a.dbc_part + (2 * hs + 1) * whole + o, f.N - n, a.vec_dbc, vc);
      }
    }
  }
}

// dB, dC: the parts of a group's heads, added in their order
template <typename T>
__global__ __launch_bounds__(256) void ssm_dbc_sum_kernel(const float* part, T* dB, T* dC, long whole, int n) {
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < 2 * whole; i += (long)gridDim.x * 256) {
    float v = 0.f;
    for (int k = 0; k < n; ++k) v += part[(long)k * 2 * whole + i];
    if (i < whole) ssm_st(dB + i, v);
    else ssm_st(dC + i - whole, v);
  }
}

// dA, dD, ddt_bias: one workgroup per head over the chunks' parts, summed in 64 bits in a fixed order
__global__ __launch_bounds__(256) void ssm_head_sum_kernel(const float* part, float* dA, float* dD, float* db, long n, int H) {
  __shared__ double red[4][3];
  const int h = blockIdx.x;
  double v[3] = {0.0, 0.0, 0.0};
  for (long i = threadIdx.x; i < n; i += 256)
#pragma unroll
    for (int k = 0; k < 3; ++k) v[k] += (double)part[(i * H + h) * 3 + k];
#pragma unroll
  for (int k = 0; k < 3; ++k) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v[k] += __shfl_xor(v[k], o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][k] = v[k];
  }
  __syncthreads();
  if (threadIdx.x < 3) {
    const double s = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
    float* out = threadIdx.x == 0 ? dA : threadIdx.x == 1 ? dD : db;
    if (out) out[h] = (float)s;
  }
}

template <typename T, int NP>
int launch_bwd(const SsmBwdArgs& a, hipStream_t st) {
  static RvitLdsLimit lim_o, lim_s, lim_c;
  const SsmScanArgs& f = a.f;
  constexpr int sb = Q * (NP + SsmOps<T>::PAD) * (int)sizeof(T) + (Q * 68 + Q) * 4, cb = BwdLds<T, NP>::BYTES;
  if (int e = lim_o.ensure({(const void*)ssm_scan_bwd_state_kernel<T, NP, true>}, sb, "ssm_scan_bwd_state")) return e;
  if (int e = lim_s.ensure({(const void*)ssm_scan_bwd_state_kernel<T, NP, false>}, sb, "ssm_scan_bwd_state")) return e;
  if (int e = lim_c.ensure({(const void*)ssm_scan_bwd_chunk_kernel<T, NP>}, cb, "ssm_scan_bwd_chunk")) return e;
  const dim3 grid((unsigned)((long)f.B * f.H * f.pblocks * f.nseg));
  if (f.nseg > 1) {
    hipLaunchKernelGGL((ssm_scan_bwd_state_kernel<T, NP, false>), grid, dim3(256), sb, st, a);
    RVIT_CHECK_LAUNCH("ssm_scan_bwd_state");
    if (int e = rvit_ssm_join(f.seg_state, f.seg_decay, a.dstate_out, nullptr, f, 1, st)) return e;
  }
  hipLaunchKernelGGL((ssm_scan_bwd_state_kernel<T, NP, true>), grid, dim3(256), sb, st, a);
  RVIT_CHECK_LAUNCH("ssm_scan_bwd_state");
  hipLaunchKernelGGL((ssm_scan_bwd_chunk_kernel<T, NP>), dim3((unsigned)((long)f.B * f.nchunks * f.G * a.hsplit)), dim3(512), cb, st, a);
  RVIT_CHECK_LAUNCH("ssm_scan_bwd_chunk");
  const long whole = (long)f.B * f.T * f.G * f.N;
  if (a.hsplit > 1) {
    const long blocks = (2 * whole + 255) / 256;
    hipLaunchKernelGGL((ssm_dbc_sum_kernel<T>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, a.dbc_part, (T*)a.dB, (T*)a.dC,
                       whole, a.hsplit);
    RVIT_CHECK_LAUNCH("ssm_dbc_sum");
  }
  hipLaunchKernelGGL(ssm_head_sum_kernel, dim3(f.H), dim3(256), 0, st, a.part, a.dA, a.dD, a.dbias, (long)f.B * f.nchunks, f.H);
  RVIT_CHECK_LAUNCH("ssm_head_sum");
  return RVIT_OK;
}

template <typename T>
int launch_bwd_n(const SsmBwdArgs& a, hipStream_t st) {
  if (a.f.N <= 32) return launch_bwd<T, 32>(a, st);
  if (a.f.N <= 64) return launch_bwd<T, 64>(a, st);
  return launch_bwd<T, 128>(a, st);
}

}  // namespace

int rvit_ssm_scan_bwd_impl(const SsmBwdArgs& a, int dtype, hipStream_t st) {
  return dtype == RVIT_BF16 ? launch_bwd_n<bf16>(a, st) : launch_bwd_n<float>(a, st);
}
