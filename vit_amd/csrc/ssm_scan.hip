// Selective state-space scan, forward: whole sequences and single tokens.  Per sample b and head h (P channels, a state of
// P x N, B and C shared by the heads of a group)
//   d = softplus(dt + dt_bias);  S_t = exp(d_t A) S_{t-1} + d_t x_t B_t^T;  v_t = S_t C_t + D x_t;  y_t = v_t silu(z_t)
// Sequences run in chunks of 64 tokens, where the recurrence is three products on the matrix cores (L = running sum of d A
// inside the chunk, E_ts = exp(L_t - L_s) for s <= t, else 0):
//   v = (C B^T o E o d_s) x + exp(L_t) S_in C_t + D x,     S_out = exp(L_Q) S_in + sum_s exp(L_Q - L_s) d_s x_s B_s^T
// L is summed in 64 bits and kept as two floats in base-2 units: a difference of two of them keeps fp32 accuracy also where
// one token's decay is in the thousands.  Nothing is divided by a decay.
#include "ssm_common.h"
#include "rvit_internal.h"
#include "ssm_args.h"

namespace {

constexpr int Q = SSM_CHUNK;

template <typename T, int NP>
struct FwdLds {
  static constexpr int PN = NP + SsmOps<T>::PAD, PX = 64 + SsmOps<T>::PAD;
  static constexpr int GP = SsmOps<T>::template planes<2>();
  static constexpr int BS = 0, CS = BS + Q * PN, XS = CS + Q * PN, GS = XS + Q * PX, END = GS + GP * Q * PX;   // in elements of T
  static constexpr int BYTES = END * (int)sizeof(T) + 5 * Q * (int)sizeof(float);
};

// One workgroup (four waves) per (sample, head, 64 channels, segment), chunk after chunk, the state in registers: wave w
// holds S^T for channels 16w .. 16w+15, which is the A operand of exp(L_t) S C as it lies in the accumulators.
// YOUT = false: only the state a segment reaches from zero, and the segment's summed log decay (long sequences of few
// rows are cut into segments, joined by ssm_join_kernel).
template <typename T, int NP, bool YOUT>
__global__ __launch_bounds__(256) void ssm_scan_fwd_kernel(SsmScanArgs a) {
  using O = SsmOps<T>;
  using L = FwdLds<T, NP>;
  constexpr int PN = L::PN, PX = L::PX, NT = NP / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* Bs = (T*)smem + L::BS;
  T* Cs = (T*)smem + L::CS;
  T* Xs = (T*)smem + L::XS;
  T* Gs = (T*)smem + L::GS;
  float* sd = (float*)((T*)smem + L::END);   // d_t
  float* shi = sd + Q;                       // L_t in base-2 units, high and low part
  float* slo = shi + Q;
  float* sw = slo + Q;                       // exp(L_Q - L_t) d_t
  float* se = sw + Q;                        // exp(L_t)
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, q = lane >> 4, c = lane & 15;
  long id = blockIdx.x;
  const int seg = id % a.nseg; id /= a.nseg;
  const int pb = id % a.pblocks; id /= a.pblocks;
  const int h = id % a.H;
  const int b = id / a.H;
  const int g = h / (a.H / a.G);
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
  const int pw = min(64, a.P - pb * 64);           // channels of this block
  const int p0 = 16 * w;                           // this wave's first of them
  const T* x = (const T*)a.x + b * a.sxb + (long)h * a.P + pb * 64;
  const T* Bm = (const T*)a.Bm + b * a.sbb + (long)g * a.N;
  const T* Cm = (const T*)a.Cm + b * a.scb + (long)g * a.N;
  const T* dt = (const T*)a.dt + b * a.sdb + h;
  const T* z = a.z ? (const T*)a.z + b * a.szb + (long)h * a.P + pb * 64 : nullptr;
  T* y = YOUT ? (T*)a.y + ((long)b * a.T * a.H + h) * a.P + pb * 64 : nullptr;
  T* v_out = YOUT && a.v ? (T*)a.v + ((long)b * a.T * a.H + h) * a.P + pb * 64 : nullptr;
  const long ldy = (long)a.H * a.P;
  const double A2 = (double)a.A[h] * 1.4426950408889634;   // log2 e: decays in base-2 units
  const float bias = a.dt_bias ? a.dt_bias[h] : 0.f;
  const float Dh = a.D ? a.D[h] : 0.f;

  // S^T: tile nt holds states 16nt + 4q + i of channel p0 + c
  f32x4 S[NT];
  const bool has_p = p0 + c < pw;
  const long srow = (((long)b * a.H + h) * a.P + pb * 64 + p0 + c) * a.N;   // row of this lane's channel in [B,H,P,N]
  {
    const float* s0 = nullptr;
    if (YOUT) {
      if (a.nseg > 1) s0 = a.seg_state + seg * a.seg_stride + srow;          // written by the join
      else if (a.state0) s0 = a.state0 + srow;
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (s0 && has_p) ssm_ld4n(s0 + 16 * nt + 4 * q, a.N - 16 * nt - 4 * q, a.vec_state, v);
      S[nt] = f32x4{v[0], v[1], v[2], v[3]};
    }
  }
  double total = 0.0;
  const int c0 = seg * a.seg_chunks, c1 = min(a.nchunks, c0 + a.seg_chunks);
  for (int ch = c0; ch < c1; ++ch) {
    const int t0 = ch * Q;
    const int live = min(max(len - t0, 0), Q);     // tokens of this chunk that exist
    if (YOUT && a.states && has_p) {
      float* out = a.states + (long)ch * a.seg_stride + srow;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float v[4] = {S[nt][0], S[nt][1], S[nt][2], S[nt][3]};
        ssm_st4n(out + 16 * nt + 4 * q, a.N - 16 * nt - 4 * q, a.vec_state, v);
      }
    }
    if (live == 0) {                               // behind the sequence: outputs are zero, the state stays
      if (YOUT) {
        for (int i = threadIdx.x; i < Q * 64; i += 256) {
          const int t = t0 + (i >> 6), p = i & 63;
          if (t < a.T && p < pw) { ssm_st(y + t * ldy + p, 0.f); if (v_out) ssm_st(v_out + t * ldy + p, 0.f); }
        }
      }
      continue;
    }
    __syncthreads();
    ssm_stage<T, 256, Q, NP>(Bs, PN, Bm + t0 * a.sbt, a.sbt, live, a.N, a.vec_bc);
    if (YOUT) ssm_stage<T, 256, Q, NP>(Cs, PN, Cm + t0 * a.sct, a.sct, live, a.N, a.vec_bc);
    ssm_stage<T, 256, Q, 64>(Xs, PX, x + t0 * a.sxt, a.sxt, live, pw, a.vec_x);
    if (w == 0) {
      const int t = t0 + lane;
      const float d = lane < live ? ssm_softplus(ssm_ld(dt + t * a.sdt) + bias) : 0.f;
      double l2 = (double)d * A2;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const double up = __shfl_up(l2, o, 64);
        if (lane >= o) l2 += up;
      }
      const double end = __shfl(l2, 63, 64);
      sd[lane] = d;
      shi[lane] = (float)l2;
      slo[lane] = (float)(l2 - (double)(float)l2);
      sw[lane] = ssm_exp2((float)(end - l2)) * d;
      se[lane] = ssm_exp2((float)l2);
      total += end;
    }
    __syncthreads();
    const float eQ = se[Q - 1];
    if (YOUT) {
      // scores of the tokens 16w .. 16w+15 against all earlier ones, decayed, into Gs[t][s]
      const int t = 16 * w + c;
      const float thi = shi[t], tlo = slo[t];
      for (int st = 0; st <= (w | 1); ++st) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        if (st <= w) {
#pragma unroll
          for (int ks = 0; ks < NP; ks += 32)
            acc = ssm_mma(ssm_row(Bs, PN, 16 * st + c, ks + 8 * q), ssm_row(Cs, PN, t, ks + 8 * q), acc);
        }
        float val[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int s = 16 * st + 4 * q + i;
          val[i] = s <= t ? acc[i] * ssm_exp2((thi - shi[s]) + (tlo - slo[s])) * sd[s] : 0.f;
        }
        ssm_put4<2>(Gs, Q * PX, t * PX + 16 * st + 4 * q, val);
      }
      __syncthreads();
    }
    if (p0 < pw) {
      typename O::Ex xf[2];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) xf[ks] = ssm_tr(Xs, PX, 32 * ks, p0, lane);
      if (YOUT) {
        f32x4 acc[4];
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) acc[tt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int m = 0; m < NP / 32; ++m) {
          const float sv[8] = {S[2 * m][0], S[2 * m][1], S[2 * m][2], S[2 * m][3], S[2 * m + 1][0], S[2 * m + 1][1], S[2 * m + 1][2], S[2 * m + 1][3]};
          const auto sf = O::template split<2>(sv);
#pragma unroll
          for (int tt = 0; tt < 4; ++tt) acc[tt] = ssm_mma(sf, ssm_row_perm(Cs, PN, 16 * tt + c, 32 * m, q), acc[tt]);
        }
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          acc[tt] *= se[16 * tt + c];
#pragma unroll
          for (int ks = 0; ks <= tt / 2; ++ks)
            acc[tt] = ssm_mma(xf[ks], ssm_row_planes<2>(Gs, Q * PX, PX, 16 * tt + c, 32 * ks + 8 * q), acc[tt]);
          const int tl = 16 * tt + c, t = t0 + tl, p = p0 + 4 * q;
          if (t < a.T && p < pw) {
            const bool is_live = tl < live;
            float out[4], zv[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = is_live ? acc[tt][i] + Dh * ssm_ld(Xs + tl * PX + p + i) : 0.f;
            if (v_out) ssm_st4n(v_out + t * ldy + p, pw - p, a.vec_y, out);
            if (z && is_live) {
              ssm_ld4n(z + t * a.szt + p, pw - p, a.vec_z, zv);
#pragma unroll
              for (int i = 0; i < 4; ++i) out[i] *= zv[i] * ssm_sigmoid(zv[i]);
            }
            ssm_st4n(y + t * ldy + p, pw - p, a.vec_y, out);
          }
        }
      }
      // the state behind the chunk
      typename O::template Cm<3> xw[2];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        float v[8];
        O::widen(xf[ks], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= sw[32 * ks + 8 * q + j];
        xw[ks] = O::template split<3>(v);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        S[nt] *= eQ;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) S[nt] = ssm_mma(ssm_tr(Bs, PN, 32 * ks, 16 * nt, lane), xw[ks], S[nt]);
      }
    }
  }
  float* out = nullptr;
  if (!YOUT) {
    out = a.seg_state + seg * a.seg_stride + srow;
    if (threadIdx.x == 0 && pb == 0) a.seg_decay[((long)seg * a.B + b) * a.H + h] = total;
  } else if (a.state_out && seg == a.nseg - 1) {
    out = a.state_out + srow;
  }
  if (out && has_p) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float v[4] = {S[nt][0], S[nt][1], S[nt][2], S[nt][3]};
      ssm_st4n(out + 16 * nt + 4 * q, a.N - 16 * nt - 4 * q, a.vec_state, v);
    }
  }
}

// Joins the segments: in place, the state a segment reached from zero becomes the state it starts from.  `reverse` runs from
// the last segment to the first (the backward pass).  One thread per four state elements; the segments' values are loaded
// ahead of the running product.
__global__ __launch_bounds__(256) void ssm_join_kernel(float* seg_state, const double* seg_decay, const float* init, float* last,
                                                       long n, int PN, long BH, int nseg, int reverse) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const long bh = i / PN;
  float run = init ? init[i] : 0.f;
  for (int k = 0; k < nseg; ++k) {
    const int s = reverse ? nseg - 1 - k : k;
    const float own = seg_state[s * n + i];
    const float f = ssm_exp2((float)seg_decay[s * BH + bh]);
    seg_state[s * n + i] = run;
    run = f * run + own;
  }
  if (last) last[i] = run;
}

// One token per sample: the state is read once and written once, in place; HBM bound.  A workgroup takes one (sample, head);
// LN lanes share a channel (each holds 4 states a turn), so that a wave reads whole lines of the state.
template <typename T, int LN>
__global__ __launch_bounds__(256) void ssm_scan_step_kernel(SsmStepArgs a) {
  const long id = blockIdx.x;
  const int h = id % a.H, b = id / a.H;
  const int g = h / (a.H / a.G);
  const float d = ssm_softplus(ssm_ld((const T*)a.dt + b * a.sdb + h) + (a.dt_bias ? a.dt_bias[h] : 0.f));
  const float f = ssm_exp2((float)((double)d * ((double)a.A[h] * 1.4426950408889634)));
  const T* x = (const T*)a.x + b * a.sxb + (long)h * a.P;
  const T* Bm = (const T*)a.Bm + b * a.sbb + (long)g * a.N;
  const T* Cm = (const T*)a.Cm + b * a.scb + (long)g * a.N;
  const T* z = a.z ? (const T*)a.z + b * a.szb + (long)h * a.P : nullptr;
  T* y = (T*)a.y + ((long)b * a.H + h) * a.P;
  const float Dh = a.D ? a.D[h] : 0.f;
  float* S = a.state + ((long)b * a.H + h) * a.P * a.N;
  const int ln = threadIdx.x % LN;
  for (int p = threadIdx.x / LN; p < a.P; p += 256 / LN) {
    const float xv = ssm_ld(x + p), dx = d * xv;
    float acc = 0.f;
    for (int n = 4 * ln; n < a.N; n += 4 * LN) {
      float s[4], bv[4], cv[4];
      const int k = a.N - n;
      ssm_ld4n(S + (long)p * a.N + n, k, a.vec_state, s);
      ssm_ld4n(Bm + n, k, a.vec_bc, bv);
      ssm_ld4n(Cm + n, k, a.vec_bc, cv);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[i] = f * s[i] + dx * bv[i];
        acc += s[i] * cv[i];
      }
      ssm_st4n(S + (long)p * a.N + n, k, a.vec_state, s);
    }
#pragma unroll
    for (int o = 1; o < LN; o <<= 1) acc += __shfl_xor(acc, o, 64);
    if (ln == 0) {
      float v = acc + Dh * xv;
      if (z) { const float zv = ssm_ld(z + p); v *= zv * ssm_sigmoid(zv); }
      ssm_st(y + p, v);
    }
  }
}

template <typename T, int NP>
int launch_fwd(const SsmScanArgs& a, bool yout, hipStream_t st) {
  static RvitLdsLimit lim_y, lim_s;
  constexpr int bytes = FwdLds<T, NP>::BYTES;
  const void* ky = (const void*)ssm_scan_fwd_kernel<T, NP, true>;
  const void* ks = (const void*)ssm_scan_fwd_kernel<T, NP, false>;
  if (int e = yout ? lim_y.ensure({ky}, bytes, "ssm_scan_fwd") : lim_s.ensure({ks}, bytes, "ssm_scan_fwd")) return e;
  const dim3 grid((unsigned)((long)a.B * a.H * a.pblocks * a.nseg));
  if (yout) hipLaunchKernelGGL((ssm_scan_fwd_kernel<T, NP, true>), grid, dim3(256), bytes, st, a);
  else hipLaunchKernelGGL((ssm_scan_fwd_kernel<T, NP, false>), grid, dim3(256), bytes, st, a);
  RVIT_CHECK_LAUNCH("ssm_scan_fwd");
  return RVIT_OK;
}

template <typename T>
int launch_fwd_n(const SsmScanArgs& a, bool yout, hipStream_t st) {
  if (a.N <= 32) return launch_fwd<T, 32>(a, yout, st);
  if (a.N <= 64) return launch_fwd<T, 64>(a, yout, st);
  return launch_fwd<T, 128>(a, yout, st);
}

}  // namespace

int rvit_ssm_join(float* seg_state, const double* seg_decay, const float* init, float* last, const SsmScanArgs& a, int reverse, hipStream_t st) {
  const long n = (long)a.B * a.H * a.P * a.N;
  hipLaunchKernelGGL(ssm_join_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, seg_state, seg_decay, init, last, n, a.P * a.N,
                     (long)a.B * a.H, a.nseg, reverse);
  RVIT_CHECK_LAUNCH("ssm_join");
  return RVIT_OK;
}

int rvit_ssm_scan_fwd_impl(const SsmScanArgs& a, int dtype, hipStream_t st) {
  if (a.nseg > 1) {
    if (int e = dtype == RVIT_BF16 ? launch_fwd_n<bf16>(a, false, st) : launch_fwd_n<float>(a, false, st)) return e;
    if (int e = rvit_ssm_join(a.seg_state, a.seg_decay, a.state0, nullptr, a, 0, st)) return e;
  }
  return dtype == RVIT_BF16 ? launch_fwd_n<bf16>(a, true, st) : launch_fwd_n<float>(a, true, st);
}

template <typename T>
static int launch_step(const SsmStepArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((long)a.B * a.H));
  if (a.N <= 32) hipLaunchKernelGGL((ssm_scan_step_kernel<T, 8>), grid, dim3(256), 0, st, a);
  else if (a.N <= 64) hipLaunchKernelGGL((ssm_scan_step_kernel<T, 16>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((ssm_scan_step_kernel<T, 32>), grid, dim3(256), 0, st, a);
  RVIT_CHECK_LAUNCH("ssm_scan_step");
  return RVIT_OK;
}
int rvit_ssm_scan_step_impl(const SsmStepArgs& a, int dtype, hipStream_t st) {
  return dtype == RVIT_BF16 ? launch_step<bf16>(a, st) : launch_step<float>(a, st);
}
