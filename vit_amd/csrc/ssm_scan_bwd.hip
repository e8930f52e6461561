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
// A sweep computes dS of every chunk (from the last to the first, the gradient in registers), then every chunk is on its own, and the
// sums behind the chunks end it: three launches.  Sequences cut into segments take two more (the segments' ends from nothing, the
// join); one chunk without a gradient of its end or start needs no sweep: two.
#include "ssm_common.h"
#include "rvit_internal.h"
#include "ssm_args.h"

namespace {

constexpr int Q = SSM_CHUNK;

// Everything here is linear in (v', dS), and every other chunk works on their negatives.  The matrix cores drop the low bits of
// what they align downwards, towards minus infinity; over thousands of tokens that tilts sums whose other factors are mostly
// of one sign (dA was 1e-6 of its size too low, for bf16 operands).  With the signs in turn the tilts cancel.
__device__ __forceinline__ float chunk_sign(int ch) { return ch & 1 ? -1.f : 1.f; }

// ---- sweep: dS before a chunk = exp(L_Q) dS behind it + sum_t exp(L_t) v'_t C_t^T ----
// One workgroup per (sample, head, 64 channels, segment), as the forward's.  At [8, 2048, 24, 64] x 128 states, bf16: 96 us for 0.3 GB
// (3.1 TB/s; it waits for its loads and for its stores of a state per chunk), the pass for the segments' starts 53 us.
template <typename T, int NP, bool OUT, bool VEC>
__global__ __launch_bounds__(256, 2) void ssm_scan_bwd_state_kernel(SsmBwdArgs a) {
  using O = SsmOps<T>;
  constexpr int PN = NP + O::PAD, PV = 68, NT = NP / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* Cs = (T*)smem;
  float* Vs = (float*)(Cs + Q * PN);
  float* decays = Vs + Q * PV;                // two sets of exp(L_t) with the sign of the chunk before, by turns
  const SsmScanArgs& f = a.f;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, q = lane >> 4, c = lane & 15;
  long id = blockIdx.x;
  const int segs = OUT ? f.nseg : f.nseg - 1;      // (the first one's start is nobody's end)
  const int seg = id % segs + (f.nseg - segs); id /= segs;
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
  const long prow = (((long)b * f.H + h) * f.pblocks + pb) * 64 * NP + (q * 64 + p0 + c) * 4;
  auto get_state = [&](const float* in, bool padded) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float v[4] = {0.f, 0.f, 0.f, 0.f};
      if (padded) ssm_ld4(in + prow + 1024 * nt, v);
      else if (has_p) ssm_ld4v<VEC>(in + srow + 16 * nt + 4 * q, f.N - 16 * nt - 4 * q, v);
      S[nt] = f32x4{v[0], v[1], v[2], v[3]};
    }
  };
  auto put_state = [&](float* out, bool padded) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float v[4] = {S[nt][0], S[nt][1], S[nt][2], S[nt][3]};
      if (padded) ssm_st4(out + prow + 1024 * nt, v);
      else if (has_p) ssm_st4v<VEC>(out + srow + 16 * nt + 4 * q, f.N - 16 * nt - 4 * q, v);
    }
  };
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) S[nt] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (OUT && f.nseg > 1) get_state(f.seg_state + seg * f.seg_stride, true);
  else if (OUT && a.dstate_out) get_state(a.dstate_out, false);
  double total = 0.0;
  auto fetch_dt = [&](int ch) { return dt[(long)min(max(ch, 0) * Q + lane, len - 1) * f.sdt]; };
  auto decay = [&](T raw, int ch) {
    const float d = ch * Q + lane < len ? ssm_softplus((float)raw + bias) : 0.f;
    const double l2 = ssm_scan64(ssm_log_decay(d, A2));
    decays[(ch & 1) * Q + lane] = chunk_sign(ch - 1) * ssm_decay(l2);
    total += ssm_last_lane(l2);
  };
  const int c0 = seg * f.seg_chunks, cl = min(min(f.nchunks, c0 + f.seg_chunks), (len + Q - 1) / Q);
  SsmTile<T, 256, Q, NP, VEC> tc;
  SsmRaw4<T> dr[4], zr[4];                    // four pieces of four channels of dy and z
  auto fetch = [&](int ch) {
    const int live = min(len - ch * Q, Q);
    tc.load(Cm + (long)ch * Q * f.sct, f.sct, live, f.N);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = i * 256 + threadIdx.x, p = (e & 15) * 4;
      const long t = ch * Q + min(e >> 4, live - 1);
      if (VEC) dr[i].load(dy + t * a.syt + (p < pw ? p : 0));
      else dr[i].part(dy + t * a.syt + p, pw - p);
      if (z && VEC && f.vec_z) zr[i].load(z + t * f.szt + (p < pw ? p : 0));
      else if (z) zr[i].part(z + t * f.szt + p, pw - p);
    }
  };
  auto put = [&](int ch) {
    const int live = min(len - ch * Q, Q);
    tc.store(Cs, PN, live, f.N);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = i * 256 + threadIdx.x, p = (e & 15) * 4, t = e >> 4;
      float v[4], zv[4];
      dr[i].get(v);
      if (z) zr[i].get(zv);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (z) v[j] *= zv[j] * ssm_sigmoid<T>(zv[j]);
        if (t >= live || p >= pw) v[j] = 0.f;
      }
      *reinterpret_cast<float4*>(Vs + t * PV + p) = make_float4(v[0], v[1], v[2], v[3]);
    }
  };
  // (the state behind a chunk is held with the chunk's sign)
  const float first = chunk_sign(max(cl, c0) - 1), last = chunk_sign(c0 - 1);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) S[nt] *= first;
  T raw = (T)0.f;
  if (c0 < cl) {
    fetch(cl - 1);
    if (w == 0) {
      decay(fetch_dt(cl - 1), cl - 1);
      raw = fetch_dt(cl - 2);
    }
    put(cl - 1);
  }
  for (int ch = cl - 1; ch >= c0; --ch) {
    const float* se = decays + (ch & 1) * Q;
    __syncthreads();
    const bool more = ch > c0;
    if (more) fetch(ch - 1);
    if (OUT) put_state(a.dstates + (long)ch * f.seg_stride, true);
    if (w == 0 && more) {
      decay(raw, ch - 1);
      raw = fetch_dt(ch - 2);
    }
    {
      const float eQ = -fabsf(se[Q - 1]);
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
      for (int nt = 0; nt < NT; ++nt) S[nt] *= eQ;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        typename O::Ex cf[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) cf[nt] = ssm_tr(Cs, PN, 32 * ks, 16 * nt, lane);
        ssm_mma_rows(cf, vw[ks], S);
      }
    }
    if (more) {
      __syncthreads();
      put(ch - 1);
    }
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) S[nt] *= last;
  if (!OUT) {
    put_state(f.seg_state + seg * f.seg_stride, true);
    if (threadIdx.x == 0 && pb == 0) f.seg_decay[((long)seg * f.B + b) * f.H + h] = total;
  } else if (a.dstate0 && seg == 0) {
    put_state(a.dstate0, false);
  }
}

// ---- the gradients of one chunk ----
// One workgroup (eight waves) per (sample, chunk, group, part of the group's heads).  B, C and their scores G are there once
// for all its heads, and the sums dB, dC over them stay in registers (wave: 16 states x 16 .. 64 tokens), so that shared
// heads cost no atomics and no scratch where one workgroup takes them all.  A head's inputs are fetched while the head
// before it is worked on, its states while its scores are.
// [8, 2048, 24, 64] x 128 states, bf16: 281 - 297 us for 0.75 GB (2.6 TB/s).  Its LDS and registers allow one workgroup, two waves a
// SIMD: vector instructions (three-part operands, decays, sums) are a quarter of a wave's time, so half of the SIMD's, matrix
// instructions a twelfth and a sixth, LDS is busy for 38 %; a wave waits for 43 % of its time, at the head's three barriers and for LDS,
// and another 22 % for the SIMD's other wave.  64 windows of 8 tokens: fp32 31 us, bf16 22 us.
template <typename T, int NP>
struct BwdLds {
  using O = SsmOps<T>;
  static constexpr int PN = NP + O::PAD, PX = 64 + O::PAD;
  static constexpr int VP = O::template planes<3>(), GP = O::template planes<2>();
  static constexpr int BS = 0, CS = BS + Q * PN, XS = CS + Q * PN, VS = XS + Q * PX, GS = VS + VP * Q * PX, WS = GS + GP * Q * PX, END = WS + GP * Q * PX;
  // floats behind: two sets, by turns, of d, L (high, low), exp(L_Q - L), exp(L), sigmoid: 6 Q, of sums over a token tile: 2 x
  // 4 Q, and of row sums by tile: 4 Q;  rho by state tile: 8 Q;  sigma by channel tile: 4 Q;  <dS, S> by wave, dD by wave (two
  // sets): 24
  static constexpr int SET = 18 * Q, FLOATS = 2 * SET + 8 * Q + 4 * Q + 24;
  // dS as an fp32 image where it fits: fetched once, in whole lines, a head ahead; else (fp32, 128 states) straight from memory
  // in both of its fragment layouts
  static constexpr int PS = NP + 4, DS = END * (int)sizeof(T) + FLOATS * 4;
  static constexpr bool DS_LDS = DS + Q * PS * 4 <= 160 * 1024;
  static constexpr int BYTES = DS + (DS_LDS ? Q * PS * 4 : 0);
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

template <typename T, int NP, bool VEC>
__global__ __launch_bounds__(512, 2) void ssm_scan_bwd_chunk_kernel(SsmBwdArgs a) {
  using O = SsmOps<T>;
  using L = BwdLds<T, NP>;
  constexpr int PN = L::PN, PX = L::PX, PL = Q * PX, NT = NP / 16, CG = 8 / NT, CT = 4 / CG;   // column groups, column tiles of a wave
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* Bs = (T*)smem + L::BS;
  T* Cs = (T*)smem + L::CS;
  T* Xs = (T*)smem + L::XS;
  T* Vs = (T*)smem + L::VS;
  T* Gs = (T*)smem + L::GS;
  T* Ws = (T*)smem + L::WS;
  float* sets = (float*)((T*)smem + L::END);
  float* r_rho = sets + 2 * L::SET; // [8][Q]
  float* r_sig = r_rho + 8 * Q;     // [4][Q]
  float* r_k = r_sig + 4 * Q;       // [8]
  float* r_d = r_k + 8;             // [2][8]
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
  const float sign = chunk_sign(ch);
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
    const T* gx = (const T*)f.x + b * f.sxb + t0 * f.sxt;
    const T* gdy = (const T*)a.dy + b * a.syb + t0 * a.syt;
    const T* gz = f.z ? (const T*)f.z + b * f.szb + t0 * f.szt : nullptr;
    const float* gv = f.z ? f.v + ((long)b * f.T + t0) * ldo : nullptr;
    const T* gdt = (const T*)f.dt + b * f.sdb + (long)(t0 + min(lane, live - 1)) * f.sdt;
    T* gdx = (T*)a.dx + ((long)b * f.T + t0) * ldo;
    T* gdz = a.dz ? (T*)a.dz + ((long)b * f.T + t0) * ldo : nullptr;
    // a head's x, dy, z, v: two pieces of four channels a thread, token row and row + 32
    const int row = threadIdx.x >> 4, pq = (threadIdx.x & 15) * 4;
    SsmRaw4<T> xr[2], dr[2], zr[2];
    SsmRaw4<float> vr[2];
    f32x4 dsn[NP / 32];
    T rawn = (T)0.f;
    float* Ds = (float*)(smem + L::DS);
    // (padded copies: [NP / 4][64 channels][4] of a head are one piece)
    auto padded = [&](int h, int pb) { return (long)ch * f.seg_stride + (((long)b * f.H + h) * f.pblocks + pb) * 64 * NP; };
    auto fetch = [&](int h, int pb) {
      int tid = threadIdx.x;
      asm volatile("" : "+v"(tid));
      const int row = tid >> 4, pq = (tid & 15) * 4;
      if constexpr (L::DS_LDS) {
        const f32x4* src = (const f32x4*)(a.dstates + padded(h, pb));
#pragma unroll
        for (int i = 0; i < NP / 32; ++i) dsn[i] = a.dstates ? (src + i * 512)[tid] : f32x4{0.f, 0.f, 0.f, 0.f};
      }
      const int pw = min(64, f.P - pb * 64);
      const long hp = (long)h * f.P + pb * 64;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = min(row + 32 * i, live - 1);
        if (VEC) {
          // token strides are under 2^24 here: 32-bit offsets from a uniform address
          const unsigned p = pq < pw ? pq : 0;
          auto at = [&](auto* base, long st) { return (decltype(base))((const char*)(base + hp) + ((unsigned)t * (unsigned)st + p) * (unsigned)sizeof(*base)); };
          xr[i].load(at(gx, f.sxt));
          dr[i].load(at(gdy, a.syt));
          if (gz) {
            if (f.vec_z) zr[i].load(at(gz, f.szt));
            else zr[i].part(gz + t * f.szt + hp + pq, pw - pq);
            vr[i].load(at(gv, ldo));
          }
        } else {
          xr[i].part(gx + t * f.sxt + hp + pq, pw - pq);
          dr[i].part(gdy + t * a.syt + hp + pq, pw - pq);
          if (gz) {
            zr[i].part(gz + t * f.szt + hp + pq, pw - pq);
            vr[i].part(gv + t * ldo + hp + pq, pw - pq);
          }
        }
      }
      if (w == 0 && pb == 0) rawn = gdt[h];
    };
    fetch(h0, 0);
    {
      SsmTile<T, 512, Q, NP, VEC> tb, tc;
      tb.load((const T*)f.Bm + b * f.sbb + t0 * f.sbt + (long)g * f.N, f.sbt, live, f.N);
      tc.load((const T*)f.Cm + b * f.scb + t0 * f.sct + (long)g * f.N, f.sct, live, f.N);
      tb.store(Bs, PN, live, f.N);
      tc.store(Cs, PN, live, f.N);
    }
    // tiles above the diagonal that a 32-wide step reads: (0, 1) and (2, 3); they stay zero
    for (int i = threadIdx.x; i < 2 * 16 * 16; i += 512) {
      const int k = i >> 8, o = ((i >> 4 & 15) + 32 * k) * PX + 16 + 32 * k + (i & 15);
#pragma unroll
      for (int pl = 0; pl < L::GP; ++pl) { Gs[pl * PL + o] = (T)0.f; Ws[pl * PL + o] = (T)0.f; }
    }
    __syncthreads();
    // score tiles (tt, st), st <= tt: ten of them, wave w has number w and, of waves 0 and 1, number 8 + w
    f32x4 Gt[2];
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2) {
      Gt[k2] = f32x4{0.f, 0.f, 0.f, 0.f};
      const int k = w + 8 * k2;
      if (k < 10) {
        const int tt = k < 1 ? 0 : k < 3 ? 1 : k < 6 ? 2 : 3, st = k - tt * (tt + 1) / 2;
#pragma unroll
        for (int ks = 0; ks < NP; ks += 32)
          Gt[k2] = ssm_mma(ssm_row(Bs, PN, 16 * st + c, ks + 8 * q), ssm_row(Cs, PN, 16 * tt + c, ks + 8 * q), Gt[k2]);
      }
    }
    int turn = 0, h_last = h0, pb_last = 0;
    float e_u = 0.f, da_u = 0.f, dD = 0.f;       // of token 63 - lane, in wave 7, over the channel blocks of a head
    // ddt of a head's tokens and its parts of dA, dD, dbias, by wave 7 while the others work on the next scores; the sums over
    // t >= u run along the lanes
    auto finish = [&](int h, int pb, int set) {
      const float *sd = sets + set * L::SET, *sw = sd + 3 * Q, *se = sw + Q, *ssg = se + Q, *r_e = ssg + Q, *r_z = r_e + 4 * Q, *r_m = r_z + 4 * Q;
      if (pb == 0) e_u = da_u = dD = 0.f;
      int lane = threadIdx.x & 63;
      asm volatile("" : "+v"(lane));
      const int u = 63 - lane, tl = u >> 4;
      float e = 0.f, zz = 0.f, sg = 0.f, sl = 0.f, rho = 0.f, kap = 0.f;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        const float ev = r_e[tt * Q + u], zv = r_z[tt * Q + u];
        e += tt >= tl ? ev : 0.f;
        zz += tt >= tl ? zv : 0.f;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        sg += r_sig[k * Q + u];
        sl += r_sig[k * Q + lane];
      }
#pragma unroll
      for (int k = 0; k < NT; ++k) rho += r_rho[k * Q + u];
#pragma unroll
      for (int k = 0; k < 8; ++k) { kap += r_k[k]; dD += r_d[set * 8 + k]; }
      e += sg * sw[u];
      // rows' sums over the s tiles before u's own
      float rs[3], run = 0.f;
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const float mv = r_m[k * Q + u];
        run += k <= tl ? mv : 0.f;
        rs[k] = ssm_scan64(run);
      }
      const float rows = tl == 0 ? 0.f : tl == 1 ? rs[0] : tl == 2 ? rs[1] : rs[2];
      // sigma of the tokens before u
      const float pre = ssm_scan64(sl * sw[lane] * sd[lane]);
      const float before = __shfl(pre, max(u - 1, 0), 64);
      da_u += (zz + rows) + ssm_scan64(rho) + (u > 0 ? before : 0.f) + se[Q - 1] * kap;
      e_u += e;
      if (pb == f.pblocks - 1) {
        const bool ok = u < live;
        const float ddt = ok ? sign * (e_u + f.A[h] * da_u) * ssg[u] : 0.f;
        if (u < here) ssm_st((T*)a.ddt + ((long)b * f.T + t0 + u) * f.H + h, ddt);
        const float sA = ssm_scan64(ok ? sign * da_u * sd[u] : 0.f), sb = ssm_scan64(ddt);
        if (lane == 63) { part[h * 3] = sA; part[h * 3 + 1] = sign * dD; part[h * 3 + 2] = sb; }
      }
    };
    for (int h = h0; h < h1; ++h) {
      const float Ah = f.A[h], Dh = f.D ? f.D[h] : 0.f;
      for (int pb = 0; pb < f.pblocks; ++pb, turn ^= 1) {
        const int pw = min(64, f.P - pb * 64);
        const long hp = (long)h * f.P + pb * 64;
        // (the lane number anew for every head: its many LDS offsets are cheaper to work out again than to keep in registers)
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int q = lane >> 4, c = lane & 15;
        float *sd = sets + turn * L::SET, *shi = sd + Q, *slo = shi + Q, *sw = slo + Q, *se = sw + Q, *ssg = se + Q;
        float* r_e = ssg + Q;         // [4][Q] sum over a tile of tokens of (G W E)_ts
        float* r_z = r_e + 4 * Q;     // [4][Q] sum over a tile's t >= u of its own s < u of M_ts
        float* r_m = r_z + 4 * Q;     // [4][Q] sum over a tile's s of M_ts, by s tile and t
        // x and v' into LDS, dz out
        float dd_part = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int t = row + 32 * i;
          float xv[4], dv[4], dzv[4];
          xr[i].get(xv);
          dr[i].get(dv);
          if (gz) {
            float zv[4], vv[4];
            zr[i].get(zv);
            vr[i].get(vv);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float sg = ssm_sigmoid<T>(zv[j]), zs = zv[j] * sg;
              dzv[j] = dv[j] * vv[j] * (sg + zs * (1.f - sg));
              dv[j] *= zs;
            }
          }
          const bool in = t < live && pq < pw;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            xv[j] = in && (VEC || pq + j < pw) ? xv[j] : 0.f;
            dv[j] = in && (VEC || pq + j < pw) ? dv[j] * sign : 0.f;
            dd_part += xv[j] * dv[j];
          }
          if (gdz && t < here) {
#pragma unroll
            for (int j = 0; j < 4; ++j) dzv[j] = in ? dzv[j] : 0.f;
            ssm_st4v<VEC>(gdz + t * ldo + hp + pq, pw - pq, dzv);
          }
          ssm_put4<1>(Xs, 0, t * PX + pq, xv);
          ssm_put4<3>(Vs, PL, t * PX + pq, dv);
        }
        dd_part = ssm_scan64(dd_part);
        if (lane == 63) r_d[turn * 8 + w] = dd_part;
        if (w == 0) {
          const float raw = (float)rawn + (f.dt_bias ? f.dt_bias[h] : 0.f);
          const float d = lane < live ? ssm_softplus(raw) : 0.f;
          const double l2 = ssm_scan64(ssm_log_decay(d, (double)Ah * 1.4426950408889634)), end = ssm_last_lane(l2);
          const float hi = (float)l2;
          sd[lane] = d;
          shi[lane] = hi;
          slo[lane] = (float)(l2 - (double)hi);
          sw[lane] = ssm_decay(end - l2);
          se[lane] = ssm_decay(l2);
          ssg[lane] = ssm_sigmoid<float>(raw);
        }
        if constexpr (L::DS_LDS) {
          int tid = threadIdx.x;
          asm volatile("" : "+v"(tid));
#pragma unroll
          for (int i = 0; i < NP / 32; ++i) {
            const int e = i * 512 + tid;
            *reinterpret_cast<f32x4*>(Ds + (e & 63) * L::PS + (e >> 6) * 4) = dsn[i];
          }
        }
        const int pt = w & 3, p0 = 16 * pt;
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
        // this wave's 16 states of S as columns (k = channels), for dC
        const unsigned col = (4 * nt + (c >> 2)) * 256 + 32 * q + (c & 3);
        const float* dS = a.dstates + padded(h, pb);
        float sc[2][8];
        {
          const float* S0 = f.states + padded(h, pb);
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j) sc[ks][j] = (S0 + (32 * ks + j) * 4)[col];
        }
        // score tiles
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
          const int k = w + 8 * k2;
          if (k >= 10) break;
          const int tt = k < 1 ? 0 : k < 3 ? 1 : k < 6 ? 2 : 3, st = k - tt * (tt + 1) / 2;
          const f32x4 G = Gt[k2];
          f32x4 W = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < 64; ks += 32)
            W = ssm_mma(ssm_row(Xs, PX, 16 * st + c, ks + 8 * q), ssm_row_planes<3>(Vs, PL, PX, 16 * tt + c, ks + 8 * q), W);
          const int t = 16 * tt + c, s0 = 16 * st + 4 * q;
          const float thi = shi[t], tlo = slo[t];
          float hi[4], lo[4], d[4], gv[4], wv[4], m[4], ec[4];
          ssm_ld4(shi + s0, hi);
          ssm_ld4(slo + s0, lo);
          ssm_ld4(sd + s0, d);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool on = s0 + i <= t;      // selects: what is above the diagonal may be anything
            const float E = ssm_exp2((thi - hi[i]) + (tlo - lo[i]));
            gv[i] = on ? G[i] * (E * d[i]) : 0.f;
            wv[i] = on ? W[i] * (E * d[i]) : 0.f;
            ec[i] = on ? G[i] * W[i] * E : 0.f;
            m[i] = ec[i] * d[i];
          }
          ssm_put4<2>(Gs, PL, t * PX + s0, gv);
          ssm_put4<2>(Ws, PL, t * PX + s0, wv);
          // sums: of a row's tile, and of a row's part before u over the rows t >= u
          const float m4 = (m[0] + m[1]) + (m[2] + m[3]);
          const float u1 = __shfl_up(m4, 16, 64), u2 = __shfl_up(m4, 32, 64), u3 = __shfl_up(m4, 48, 64);
          float pre = (q >= 1 ? u1 : 0.f) + (q >= 2 ? u2 : 0.f) + (q >= 3 ? u3 : 0.f);
          if (q == 3) r_m[st * Q + t] = pre + m4;
          float es[4], zs[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            es[i] = row16_sum(ec[i]);
            zs[i] = row16_sum(s0 + i <= t ? pre : 0.f);
            pre += m[i];
          }
          if (c == 0) {
            ssm_st4(r_e + tt * Q + s0, es);
            ssm_st4(r_z + tt * Q + s0, zs);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
        if (w == 7 && (h > h0 || pb > 0)) finish(h_last, pb_last, turn ^ 1);
        __syncthreads();
        {
          const bool same = pb + 1 < f.pblocks;
          if (same || h + 1 < h1) fetch(same ? h : h + 1, same ? pb + 1 : 0);
        }
        // dx: wave = 16 channels x 2 token tiles: 0 and 3, or 1 and 2
        if (p0 < pw) {
          const int st[2] = {w >> 2, 3 - (w >> 2)};
          f32x4 acc[2];
          acc[0] = acc[1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int m = 0; m < NP / 32; ++m) {
            typename O::Ex bf[2];
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) bf[k2] = ssm_row(Bs, PN, 16 * st[k2] + c, 32 * m + 8 * q);
            float v[8];      // dS, rows of this wave's channels
            if (L::DS_LDS || a.dstates) {
              const float* src = L::DS_LDS ? Ds + (p0 + c) * L::PS + 32 * m + 8 * q : dS + (8 * m + 2 * q) * 256 + (p0 + c) * 4;
              ssm_ld4(src, reinterpret_cast<float(&)[4]>(v[0]));
              ssm_ld4(src + (L::DS_LDS ? 4 : 256), reinterpret_cast<float(&)[4]>(v[4]));
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] = 0.f;
            }
            ssm_mma_cols(O::template split<3>(v), bf, acc);
          }
          const int p = p0 + 4 * q;
          float xv[2][4];
#pragma unroll
          for (int k2 = 0; k2 < 2; ++k2) {
            const int s = 16 * st[k2] + c;
            ssm_ld4(Xs + s * PX + p, xv[k2]);
            const float sig = groups_sum((xv[k2][0] * acc[k2][0] + xv[k2][1] * acc[k2][1]) + (xv[k2][2] * acc[k2][2] + xv[k2][3] * acc[k2][3]));
            if (q == 0) r_sig[pt * Q + s] = sig;
            acc[k2] *= sw[s] * sd[s];
          }
          {
            const auto vf = ssm_tr_planes<2>(Vs, PL, PX, 32, p0, lane);
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) acc[k2] = ssm_mma(vf, ssm_tr_planes<2>(Gs, PL, PX, 32, 16 * st[k2], lane), acc[k2]);
            acc[0] = ssm_mma(ssm_tr_planes<2>(Vs, PL, PX, 0, p0, lane), ssm_tr_planes<2>(Gs, PL, PX, 0, 16 * st[0], lane), acc[0]);
          }
#pragma unroll
          for (int k2 = 0; k2 < 2; ++k2) {
            const int s = 16 * st[k2] + c;
            float out[4], pv[4], v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int pl = L::VP - 1; pl >= 0; --pl) {
              ssm_ld4(Vs + pl * PL + s * PX + p, pv);
#pragma unroll
              for (int i = 0; i < 4; ++i) v[i] += pv[i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) out[i] = sign * (acc[k2][i] + Dh * v[i]);
            if (s < here) ssm_st4v<VEC>(gdx + s * ldo + hp + p, pw - p, out);
          }
        } else if (lane < 32) {
          const int st = lane < 16 ? w >> 2 : 3 - (w >> 2);
          r_sig[pt * Q + 16 * st + c] = 0.f;
        }
        __builtin_amdgcn_sched_barrier(0);
        // dB, dC, rho, <dS, S>: wave = 16 states x CT token tiles
        {
          float kap = 0.f, dsc[2][8];      // dS, columns of this wave's states
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j)
              dsc[ks][j] = L::DS_LDS ? Ds[(32 * ks + 8 * q + j) * L::PS + 16 * nt + c] : a.dstates ? (dS + (32 * ks + j) * 4)[col] : 0.f;
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int j = 0; j < 8; ++j) kap += dsc[ks][j] * sc[ks][j];
          kap = ssm_scan64(kap);
          if (lane == 63) r_k[w] = cg == 0 ? kap : 0.f;
          {
            f32x4 tb[CT];
#pragma unroll
            for (int k = 0; k < CT; ++k) tb[k] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
              typename O::Ex xf[CT];
#pragma unroll
              for (int k = 0; k < CT; ++k) xf[k] = ssm_row(Xs, PX, 16 * (cg * CT + k) + c, 32 * ks + 8 * q);
              ssm_mma_cols(O::template split<2>(dsc[ks]), xf, tb);
            }
#pragma unroll
            for (int k = 0; k < CT; ++k) {
              const int t = 16 * (cg * CT + k) + c;
              accB[k] += tb[k] * (sw[t] * sd[t]);
            }
          }
          __builtin_amdgcn_sched_barrier(0);
          {
            constexpr int CP = CT < 2 ? 1 : 2;      // two token tiles at a time: their parts fill the registers
            const auto s0 = O::template split<3>(sc[0]), s1 = O::template split<3>(sc[1]);
#pragma unroll
            for (int k = 0; k < CT; k += CP) {
              f32x4 tc[CP];
#pragma unroll
              for (int m = 0; m < CP; ++m) tc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int ks = 0; ks < 2; ++ks) {
                typename O::template Cm<3> vf[CP];
#pragma unroll
                for (int m = 0; m < CP; ++m) vf[m] = ssm_row_planes<3>(Vs, PL, PX, 16 * (cg * CT + k + m) + c, 32 * ks + 8 * q);
                ssm_mma_cols(ks ? s1 : s0, vf, tc);
              }
#pragma unroll
              for (int m = 0; m < CP; ++m) {
                const int t = 16 * (cg * CT + k + m) + c;
                tc[m] *= se[t];
                float cv[4];
                ssm_ld4(Cs + t * PN + 16 * nt + 4 * q, cv);
                const float rho = groups_sum((cv[0] * tc[m][0] + cv[1] * tc[m][1]) + (cv[2] * tc[m][2] + cv[3] * tc[m][3]));
                if (q == 0) r_rho[nt * Q + t] = rho;
                accC[k + m] += tc[m];
              }
              __builtin_amdgcn_sched_barrier(0);
            }
          }
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            const auto cf = ssm_tr(Cs, PN, 32 * ks, 16 * nt, lane);
            const auto bf = ssm_tr(Bs, PN, 32 * ks, 16 * nt, lane);
#pragma unroll
            for (int k = 0; k < CT; ++k) {
              const int ct = cg * CT + k;
              if (ct / 2 <= ks) accB[k] = ssm_mma(cf, ssm_tr_planes<2>(Ws, PL, PX, 32 * ks, 16 * ct, lane), accB[k]);
              if (ct / 2 >= ks) accC[k] = ssm_mma(bf, ssm_row_planes<2>(Ws, PL, PX, 16 * ct + c, 32 * ks + 8 * q), accC[k]);
            }
          }
        }
        __syncthreads();
        h_last = h;
        pb_last = pb;
      }
    }
    if (w == 7) finish(h_last, pb_last, turn ^ 1);
  }
  // accB, accC: states 16nt + 4q + i of token 16 ct + c
#pragma unroll
  for (int k = 0; k < CT; ++k) {
    const int t = 16 * (cg * CT + k) + c, n = 16 * nt + 4 * q;
    accB[k] *= sign;
    accC[k] *= sign;
    if (t < here) {
      const long o = (((long)b * f.T + t0 + t) * f.G + g) * f.N + n;
      const float vb[4] = {accB[k][0], accB[k][1], accB[k][2], accB[k][3]}, vc[4] = {accC[k][0], accC[k][1], accC[k][2], accC[k][3]};
      if (a.hsplit == 1) {
        ssm_st4v<VEC>((T*)a.dB + o, f.N - n, vb);
        ssm_st4v<VEC>((T*)a.dC + o, f.N - n, vc);
      } else {
        const long whole = (long)f.B * f.T * f.G * f.N;
        ssm_st4v<VEC>(a.dbc_part + 2 * hs * whole + o, f.N - n, vb);
        ssm_st4v<VEC>(a.dbc_part + (2 * hs + 1) * whole + o, f.N - n, vc);
      }
    }
  }
}

// The sums behind the chunks, in a fixed order, in one launch.  The first H workgroups: dA, dD, ddt_bias of a head from its chunks'
// parts, in 64 bits; the others (n > 1): dB, dC from the n parts of a group's heads.
template <typename T>
__global__ __launch_bounds__(256) void ssm_bwd_sum_kernel(const float* part, float* dA, float* dD, float* db, long chunks, int H, const float* dbc, T* dB, T* dC,
                                                          long whole, int n) {
  __shared__ double red[4][3];
  if ((int)blockIdx.x >= H) {
    for (long i = (long)(blockIdx.x - H) * 256 + threadIdx.x; i < 2 * whole; i += (long)(gridDim.x - H) * 256) {
      float v = 0.f;
      for (int k = 0; k < n; ++k) v += dbc[(long)k * 2 * whole + i];
      if (i < whole) ssm_st(dB + i, v);
      else ssm_st(dC + i - whole, v);
    }
    return;
  }
  const int h = blockIdx.x;
  double v[3] = {0.0, 0.0, 0.0};
  for (long i = threadIdx.x; i < chunks; i += 256)
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

template <typename T, int NP, bool VEC>
int launch_bwd(const SsmBwdArgs& a, hipStream_t st) {
  static RvitLdsLimit lim_o, lim_s, lim_c;
  const SsmScanArgs& f = a.f;
  constexpr int sb = Q * (NP + SsmOps<T>::PAD) * (int)sizeof(T) + (Q * 68 + 2 * Q) * 4, cb = BwdLds<T, NP>::BYTES;
  if (int e = lim_o.ensure({(const void*)ssm_scan_bwd_state_kernel<T, NP, true, VEC>}, sb, "ssm_scan_bwd_state")) return e;
  if (int e = lim_s.ensure({(const void*)ssm_scan_bwd_state_kernel<T, NP, false, VEC>}, sb, "ssm_scan_bwd_state")) return e;
  if (int e = lim_c.ensure({(const void*)ssm_scan_bwd_chunk_kernel<T, NP, VEC>}, cb, "ssm_scan_bwd_chunk")) return e;
  const long rows = (long)f.B * f.H * f.pblocks;
  if (f.nseg > 1) {
    hipLaunchKernelGGL((ssm_scan_bwd_state_kernel<T, NP, false, VEC>), dim3((unsigned)(rows * (f.nseg - 1))), dim3(256), sb, st, a);
    RVIT_CHECK_LAUNCH("ssm_scan_bwd_state");
    if (int e = rvit_ssm_join(f.seg_state, f.seg_decay, a.dstate_out, f, 1, st)) return e;
  }
  if (a.dstates) {
    hipLaunchKernelGGL((ssm_scan_bwd_state_kernel<T, NP, true, VEC>), dim3((unsigned)(rows * f.nseg)), dim3(256), sb, st, a);
    RVIT_CHECK_LAUNCH("ssm_scan_bwd_state");
  }
  hipLaunchKernelGGL((ssm_scan_bwd_chunk_kernel<T, NP, VEC>), dim3((unsigned)((long)f.B * f.nchunks * f.G * a.hsplit)), dim3(512), cb, st, a);
  RVIT_CHECK_LAUNCH("ssm_scan_bwd_chunk");
  const long whole = (long)f.B * f.T * f.G * f.N, blocks = a.hsplit > 1 ? (2 * whole + 255) / 256 : 0;
  hipLaunchKernelGGL((ssm_bwd_sum_kernel<T>), dim3((unsigned)(f.H + (blocks < 4096 ? blocks : 4096))), dim3(256), 0, st, a.part, a.dA, a.dD, a.dbias,
                     (long)f.B * f.nchunks, f.H, a.dbc_part, (T*)a.dB, (T*)a.dC, whole, a.hsplit);
  RVIT_CHECK_LAUNCH("ssm_bwd_sum");
  return RVIT_OK;
}

template <typename T, int NP>
int launch_bwd_v(const SsmBwdArgs& a, hipStream_t st) {
  const SsmScanArgs& f = a.f;
  const bool vec = f.vec_x && f.vec_bc && f.vec_state && (!f.z || f.vec_y) && a.vec_dy && a.vec_out && a.vec_dbc;
  return vec ? launch_bwd<T, NP, true>(a, st) : launch_bwd<T, NP, false>(a, st);
}

template <typename T>
int launch_bwd_n(const SsmBwdArgs& a, hipStream_t st) {
  if (a.f.N <= 32) return launch_bwd_v<T, 32>(a, st);
  if (a.f.N <= 64) return launch_bwd_v<T, 64>(a, st);
  return launch_bwd_v<T, 128>(a, st);
}

}  // namespace

int rvit_ssm_scan_bwd_impl(const SsmBwdArgs& a, int dtype, hipStream_t st) {
  return dtype == RVIT_BF16 ? launch_bwd_n<bf16>(a, st) : launch_bwd_n<float>(a, st);
}
