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
  // Pitches: images with transposing reads (four rows of 32 bytes at a time) want rows 32 bytes apart in the banks, images that
  // are only read along rows 16: with 32 everywhere the score and C reads collide half as often again.
  static constexpr int SLIM = SsmOps<T>::PAD, WIDE = sizeof(T) == 2 ? 16 : 4;
  static constexpr int PB = NP + WIDE, PC = NP + SLIM, PX = 64 + WIDE, PG = 64 + SLIM;
  static constexpr int GP = SsmOps<T>::template planes<2>();
  static constexpr int BS = 0, CS = BS + Q * PB, XS = CS + Q * PC, GS = XS + Q * PX, END = GS + GP * Q * PG;   // in elements of T
  static constexpr int BYTES = END * (int)sizeof(T) + 10 * Q * (int)sizeof(float);
};

// scores of the 16 tokens of tile TILES - 1 against all up to them, decayed, times d_s, into Gs[t][s]; the tile beside the last
// is written as zero where a step over 32 tokens will read it
template <typename T, int NP, int TILES>
__device__ __forceinline__ void scores(const T* Bs, const T* Cs, T* Gs, const float* sd, int tw, int q, int c) {
  using L = FwdLds<T, NP>;
  const float *shi = sd + Q, *slo = shi + Q;
  const int t = 16 * tw + c;
  f32x4 acc[TILES];
#pragma unroll
  for (int st = 0; st < TILES; ++st) acc[st] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int ks = 0; ks < NP; ks += 32) {
    typename SsmOps<T>::Ex bf[TILES];
#pragma unroll
    for (int st = 0; st < TILES; ++st) bf[st] = ssm_row(Bs, L::PB, 16 * st + c, ks + 8 * q);
    ssm_mma_rows(bf, ssm_row(Cs, L::PC, t, ks + 8 * q), acc);
  }
  const float thi = shi[t], tlo = slo[t];
#pragma unroll
  for (int st = 0; st < TILES; ++st) {
    const int s = 16 * st + 4 * q;
    const float4 hi = *reinterpret_cast<const float4*>(shi + s), lo = *reinterpret_cast<const float4*>(slo + s), d = *reinterpret_cast<const float4*>(sd + s);
    float val[4];
    val[0] = acc[st][0] * (ssm_exp2((thi - hi.x) + (tlo - lo.x)) * d.x);
    val[1] = acc[st][1] * (ssm_exp2((thi - hi.y) + (tlo - lo.y)) * d.y);
    val[2] = acc[st][2] * (ssm_exp2((thi - hi.z) + (tlo - lo.z)) * d.z);
    val[3] = acc[st][3] * (ssm_exp2((thi - hi.w) + (tlo - lo.w)) * d.w);
    if (st == TILES - 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) val[i] = s + i <= t ? val[i] : 0.f;      // a select: what is above the diagonal may be anything
    }
    ssm_put4<2>(Gs, Q * L::PG, t * L::PG + s, val);
  }
  if (TILES & 1) {
    const float none[4] = {0.f, 0.f, 0.f, 0.f};
    ssm_put4<2>(Gs, Q * L::PG, t * L::PG + 16 * TILES + 4 * q, none);
  }
}

// One workgroup (four waves) per (sample, head, 64 channels, segment), chunk after chunk, the state in registers: wave w
// holds S^T for channels 16w .. 16w+15, which is the A operand of exp(L_t) S C as it lies in the accumulators.
// A chunk's images and decays are fetched and worked out while the chunk before it is computed.
// YOUT = false: only the state a segment (but the last) reaches from zero, and the segment's summed log decay (long sequences of few
// rows are cut into segments, joined by ssm_join_kernel).  VEC: all wide accesses are aligned and whole.
// Measured, bf16, 128 states: 32768 tokens x 16 heads x 64 (segments of 16 chunks) 111 us, the pass for states 45 us;
// [8, 2048, 24, 64] with a state kept per chunk and v in 32 bits (0.45 GB) 165 us and 40 us.  Bound by two waves a SIMD (256
// registers, 69 KB of LDS): of a wave's time vector instructions (splits, decays, the gate) fill 27 and 20 %, matrix instructions 13
// and 9 %; waits for LDS, barriers and memory 37 and 47 %, waits for the SIMD's other wave 23 %.  A second x image with two barriers a
// chunk, and one barrier in the pass for states, took the same time, as did the score tiles spread evenly over the waves; the decays
// are worked out by the wave with the fewest of them (by wave 0 of every workgroup: 8 and 4 us more).
template <typename T, int NP, bool YOUT, bool VEC>
__global__ __launch_bounds__(256, sizeof(T) == 4 && NP == 128 ? 1 : 2) void ssm_scan_fwd_kernel(SsmScanArgs a) {
  using O = SsmOps<T>;
  using L = FwdLds<T, NP>;
  constexpr int PB = L::PB, PC = L::PC, PX = L::PX, PG = L::PG, NT = NP / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* Bs = (T*)smem + L::BS;
  T* Cs = (T*)smem + L::CS;
  T* Xs = (T*)smem + L::XS;
  T* Gs = (T*)smem + L::GS;
  float* decays = (float*)((T*)smem + L::END);   // two sets, by turns: d, L (high, low), exp(L_Q - L) d, exp(L)
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, q = lane >> 4, c = lane & 15;
  long id = blockIdx.x;
  const int segs = YOUT ? a.nseg : a.nseg - 1;     // (the last one's end is nobody's start)
  const int seg = id % segs; id /= segs;
  const int pb = id % a.pblocks; id /= a.pblocks;
  const int h = id % a.H;
  const int b = id / a.H;
  const int g = h / (a.H / a.G);
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
  const int pw = min(64, a.P - pb * 64);           // channels of this block
  const int p0 = 16 * w;                           // this wave's first of them
  const int tw = (blockIdx.x & 1) ? 3 - w : w;     // this wave's token tile in the score product: later ones have more to do, so
                                                   // the two workgroups of a compute unit take them in opposite order
  const T* x = (const T*)a.x + b * a.sxb + (long)h * a.P + pb * 64;
  const T* Bm = (const T*)a.Bm + b * a.sbb + (long)g * a.N;
  const T* Cm = (const T*)a.Cm + b * a.scb + (long)g * a.N;
  const T* dt = (const T*)a.dt + b * a.sdb + h;
  const T* z = a.z ? (const T*)a.z + b * a.szb + (long)h * a.P + pb * 64 : nullptr;
  T* y = YOUT ? (T*)a.y + ((long)b * a.T * a.H + h) * a.P + pb * 64 : nullptr;
  float* v_out = YOUT && a.v ? a.v + ((long)b * a.T * a.H + h) * a.P + pb * 64 : nullptr;
  const long ldy = (long)a.H * a.P;
  const double A2 = (double)a.A[h] * 1.4426950408889634;   // log2 e: decays in base-2 units
  const float bias = a.dt_bias ? a.dt_bias[h] : 0.f;
  const float Dh = a.D ? a.D[h] : 0.f;

  // S^T: tile nt holds states 16nt + 4q + i of channel p0 + c
  f32x4 S[NT];
  const bool has_p = p0 + c < pw;
  const long srow = (((long)b * a.H + h) * a.P + pb * 64 + p0 + c) * a.N;   // row of this lane's channel in [B,H,P,N]
  const long prow = (((long)b * a.H + h) * a.pblocks + pb) * 64 * NP + (q * 64 + p0 + c) * 4;   // and in the padded copies
  auto get_state = [&](const float* in, bool padded) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (padded) ssm_ld4(in + prow + 1024 * nt, v);
      else if (has_p) ssm_ld4v<VEC>(in + srow + 16 * nt + 4 * q, a.N - 16 * nt - 4 * q, v);
      S[nt] = f32x4{v[0], v[1], v[2], v[3]};
    }
  };
  auto put_state = [&](float* out, bool padded) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float v[4] = {S[nt][0], S[nt][1], S[nt][2], S[nt][3]};
      if (padded) ssm_st4(out + prow + 1024 * nt, v);
      else if (has_p) ssm_st4v<VEC>(out + srow + 16 * nt + 4 * q, a.N - 16 * nt - 4 * q, v);
    }
  };
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) S[nt] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (YOUT && a.nseg > 1) get_state(a.seg_state + seg * a.seg_stride, true);     // written by the join
  else if (YOUT && a.state0) get_state(a.state0, false);
  double total = 0.0;
  // the wave with the fewest scores: the decays of a chunk from its dt (one token a lane)
  auto fetch_dt = [&](int ch) { return dt[(long)min(ch * Q + lane, len - 1) * a.sdt]; };
  auto decay = [&](T raw, int ch) {
    float* sd = decays + (ch & 1) * 5 * Q;
    const float d = ch * Q + lane < len ? ssm_softplus((float)raw + bias) : 0.f;
    const double l2 = ssm_scan64(ssm_log_decay(d, A2)), end = ssm_last_lane(l2);
    const float hi = (float)l2;
    sd[lane] = d;
    sd[Q + lane] = hi;
    sd[2 * Q + lane] = (float)(l2 - (double)hi);
    sd[3 * Q + lane] = ssm_decay(end - l2) * d;
    sd[4 * Q + lane] = ssm_decay(l2);
    total += end;
  };
  const int c0 = seg * a.seg_chunks, c1 = min(a.nchunks, c0 + a.seg_chunks);
  const int cl = min(c1, (len + Q - 1) / Q);       // chunks with tokens end here
  SsmTile<T, 256, Q, NP, VEC> tb, tc;
  SsmTile<T, 256, Q, 64, VEC> tx;
  auto fetch = [&](int ch) {
    const int live = min(len - ch * Q, Q);
    tb.load(Bm + (long)ch * Q * a.sbt, a.sbt, live, a.N);
    if (YOUT) tc.load(Cm + (long)ch * Q * a.sct, a.sct, live, a.N);
    tx.load(x + (long)ch * Q * a.sxt, a.sxt, live, pw);
  };
  auto put = [&](int ch) {
    const int live = min(len - ch * Q, Q);
    tb.store(Bs, PB, live, a.N);
    if (YOUT) tc.store(Cs, PC, live, a.N);
    tx.store(Xs, PX, live, pw);
  };
  T raw = (T)0.f;
  if (c0 < cl) {
    fetch(c0);
    if (tw == 0) {
      decay(fetch_dt(c0), c0);
      raw = fetch_dt(c0 + 1);
    }
    put(c0);
  }
  for (int ch = c0; ch < cl; ++ch) {
    const int t0 = ch * Q;
    const int live = min(len - t0, Q);             // tokens of this chunk that exist
    const float* sd = decays + (ch & 1) * 5 * Q;
    const float *shi = sd + Q, *slo = shi + Q, *sw = slo + Q, *se = sw + Q;
    __syncthreads();
    const bool more = ch + 1 < cl;
    if (more) fetch(ch + 1);
    if (YOUT && a.states) put_state(a.states + (long)ch * a.seg_stride, true);
    if (tw == 0 && more) {
      decay(raw, ch + 1);
      raw = fetch_dt(ch + 2);
    }
    SsmRaw4<T> zr[4];
    if (YOUT) {
      // the gate of this wave's outputs, for the end of the chunk
      const int p = p0 + 4 * q;
      if (z) {
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const T* src = z + (long)(t0 + min(16 * tt + c, live - 1)) * a.szt;
          if (VEC && a.vec_z) zr[tt].load(src + (p < pw ? p : 0));
          else zr[tt].part(src + p, pw - p);
        }
      }
      switch (tw) {
        case 0: scores<T, NP, 1>(Bs, Cs, Gs, sd, tw, q, c); break;
        case 1: scores<T, NP, 2>(Bs, Cs, Gs, sd, tw, q, c); break;
        case 2: scores<T, NP, 3>(Bs, Cs, Gs, sd, tw, q, c); break;
        default: scores<T, NP, 4>(Bs, Cs, Gs, sd, tw, q, c);
      }
      __syncthreads();
    }
    {
      const float eQ = se[Q - 1];
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
          typename O::Ex cf[4];
#pragma unroll
          for (int tt = 0; tt < 4; ++tt) cf[tt] = ssm_row_perm(Cs, PC, 16 * tt + c, 32 * m, q);
          ssm_mma_cols(O::template split<2>(sv), cf, acc);
        }
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) acc[tt] *= se[16 * tt + c];
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int tt = 2 * ks; tt < 4; ++tt)
            acc[tt] = ssm_mma(xf[ks], ssm_row_planes<2>(Gs, Q * PG, PG, 16 * tt + c, 32 * ks + 8 * q), acc[tt]);
        const int p = p0 + 4 * q;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt) {
          const int tl = 16 * tt + c, t = t0 + tl;
          float v[4], out[4], xv[4];
          ssm_ld4(Xs + tl * PX + p, xv);
#pragma unroll
          for (int i = 0; i < 4; ++i) out[i] = v[i] = acc[tt][i] + Dh * xv[i];
          if (z) {
            float zv[4];
            zr[tt].get(zv);
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] *= zv[i] * ssm_sigmoid<T>(zv[i]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {          // (a last chunk's rows behind the end)
            v[i] = tl < live ? v[i] : 0.f;
            out[i] = tl < live ? out[i] : 0.f;
          }
          if (t < a.T) {
            if (v_out) ssm_st4v<VEC>(v_out + t * ldy + p, pw - p, v);
            ssm_st4v<VEC>(y + t * ldy + p, pw - p, out);
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
      for (int nt = 0; nt < NT; ++nt) S[nt] *= eQ;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        typename O::Ex bf[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) bf[nt] = ssm_tr(Bs, PB, 32 * ks, 16 * nt, lane);
        ssm_mma_rows(bf, xw[ks], S);
      }
    }
    if (more) {
      __syncthreads();
      put(ch + 1);
    }
  }
  if (YOUT) {      // behind the sequence: outputs are zero
    const int from = max(c0, cl) * Q, to = min(c1 * Q, a.T);
    for (long i = threadIdx.x; i < (long)(to - from) * 64; i += 256) {
      const int t = from + (int)(i >> 6), p = (int)(i & 63);
      if (p < pw) { ssm_st(y + t * ldy + p, 0.f); if (v_out) v_out[t * ldy + p] = 0.f; }
    }
    if (a.state_out && seg == a.nseg - 1) put_state(a.state_out, false);
  } else {
    put_state(a.seg_state + seg * a.seg_stride, true);
    if (tw == 0 && lane == 0 && pb == 0) a.seg_decay[((long)seg * a.B + b) * a.H + h] = total;
  }
}

// Joins the segments: in place, the state a segment reached from zero becomes the state it starts from.  `reverse` runs from
// the last segment to the first (the backward pass).  `init` [B,H,P,N] (or null) is what the first one starts from.
// A thread takes four states of a channel through all segments, the next ones' on their way: its bytes in and out (192 rows of 2
// segments, 25 MB: 6.2 us, with one state a thread 12.5; 16 rows of 32 segments, 34 MB: 15 us either way).
__global__ __launch_bounds__(64) void ssm_join_kernel(float* seg_state, const double* seg_decay, const float* init, long n, int P, int N, int pblocks, int NP,
                                                      long BH, int nseg, int reverse) {
  const long i = (long)blockIdx.x * 64 + threadIdx.x;      // of the four: [BH][pblocks][NP / 4][64]
  if (i >= n / 4) return;
  const int p0 = i & 63, k = (int)(i >> 6) % (NP / 4) * 4;
  const long row = i / (16 * NP), bh = row / pblocks;
  const int p = (int)(row % pblocks) * 64 + p0;
  f32x4 run = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; ++j) run[j] = init && p < P && k + j < N ? init[(bh * P + p) * N + k + j] : 0.f;
  constexpr int AHEAD = 8;
  f32x4* st = (f32x4*)seg_state + i;
  const long step = (reverse ? -n : n) / 4;
  const long sb = reverse ? -BH : BH;
  const double* dec = seg_decay + (reverse ? (nseg - 1) * BH : 0) + bh;
  if (reverse) st += (nseg - 1) * (n / 4);
  for (int j0 = 0; j0 < nseg; j0 += AHEAD) {
    f32x4 own[AHEAD];
    float f[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      own[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      f[j] = 0.f;
      if (j0 + j < nseg - 1) {      // (of the last one nothing is needed)
        own[j] = st[(j0 + j) * step];
        f[j] = ssm_decay(dec[(j0 + j) * sb]);
      }
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (j0 + j < nseg) {
        st[(j0 + j) * step] = run;
        run = f[j] * run + own[j];
      }
  }
}

// One token per sample: the state is read once and written once, in place; HBM bound (256 samples x 32 heads x 64 x 128, 540 MB:
// 124 us, 4.4 TB/s, a copy of that size reaches 5.2; one sample: the launch).  A workgroup takes one (sample, head);
// LN lanes share a channel (each holds 4 states a turn), so that a wave reads whole lines of the state.
template <typename T, int LN>
__global__ __launch_bounds__(256) void ssm_scan_step_kernel(SsmStepArgs a) {
  const long id = blockIdx.x;
  const int h = id % a.H, b = id / a.H;
  const int g = h / (a.H / a.G);
  const float d = ssm_softplus(ssm_ld((const T*)a.dt + b * a.sdb + h) + (a.dt_bias ? a.dt_bias[h] : 0.f));
  const float f = ssm_decay(ssm_log_decay(d, (double)a.A[h] * 1.4426950408889634));
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
      if (z) { const float zv = ssm_ld(z + p); v *= zv * ssm_sigmoid<T>(zv); }
      ssm_st(y + p, v);
    }
  }
}

template <typename T, int NP, bool YOUT, bool VEC>
int launch_fwd(const SsmScanArgs& a, hipStream_t st) {
  static RvitLdsLimit lim;
  constexpr int bytes = FwdLds<T, NP>::BYTES;
  if (int e = lim.ensure({(const void*)ssm_scan_fwd_kernel<T, NP, YOUT, VEC>}, bytes, "ssm_scan_fwd")) return e;
  hipLaunchKernelGGL((ssm_scan_fwd_kernel<T, NP, YOUT, VEC>), dim3((unsigned)((long)a.B * a.H * a.pblocks * (YOUT ? a.nseg : a.nseg - 1))), dim3(256), bytes, st, a);
  RVIT_CHECK_LAUNCH("ssm_scan_fwd");
  return RVIT_OK;
}

template <typename T, int NP>
int launch_fwd_v(const SsmScanArgs& a, bool yout, hipStream_t st) {
  const bool vec = a.vec_x && a.vec_bc && a.vec_state && (!yout || a.vec_y);
  if (yout) return vec ? launch_fwd<T, NP, true, true>(a, st) : launch_fwd<T, NP, true, false>(a, st);
  return vec ? launch_fwd<T, NP, false, true>(a, st) : launch_fwd<T, NP, false, false>(a, st);
}

template <typename T>
int launch_fwd_n(const SsmScanArgs& a, bool yout, hipStream_t st) {
  if (a.N <= 32) return launch_fwd_v<T, 32>(a, yout, st);
  if (a.N <= 64) return launch_fwd_v<T, 64>(a, yout, st);
  return launch_fwd_v<T, 128>(a, yout, st);
}

}  // namespace

int rvit_ssm_join(float* seg_state, const double* seg_decay, const float* init, const SsmScanArgs& a, int reverse, hipStream_t st) {
  hipLaunchKernelGGL(ssm_join_kernel, dim3((unsigned)((a.seg_stride / 4 + 63) / 64)), dim3(64), 0, st, seg_state, seg_decay, init, a.seg_stride, a.P, a.N,
                     a.pblocks, ssm_padded_n(a.N), (long)a.B * a.H, a.nseg, reverse);
  RVIT_CHECK_LAUNCH("ssm_join");
  return RVIT_OK;
}

int rvit_ssm_scan_fwd_impl(const SsmScanArgs& a, int dtype, hipStream_t st) {
  if (a.nseg > 1) {
    if (int e = dtype == RVIT_BF16 ? launch_fwd_n<bf16>(a, false, st) : launch_fwd_n<float>(a, false, st)) return e;
    if (int e = rvit_ssm_join(a.seg_state, a.seg_decay, a.state0, a, 0, st)) return e;
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
