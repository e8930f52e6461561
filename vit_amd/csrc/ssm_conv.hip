// Short causal convolution per channel over the tokens of a sequence (the window in front of the selective scan), forward,
// backward and the single-token form:   u[t] = bias + sum_k w[k] x[t - K + 1 + k],  y = u or silu(u).
// HBM bound: a thread owns V channels (one 16-byte access) of a strip of tokens and slides its window through registers, so
// x is read once but for K - 1 tokens between strips (which the caches hold), and a wave reads 1 KB of a token's row.
// At 8 x 2048 x 1792: forward 29 us in bf16 (4.0 TB/s), 45 in fp32 (5.2 TB/s); backward 52 us in bf16 (3.4 TB/s) and 80 in fp32 (4.4
// TB/s), the parts' sum 4 us.  The bf16 backward pass is bound by its vector instructions: u again, silu', the window's products and
// the tests of a strip's ends keep the SIMDs busy for 80 % of it (four waves each; more tokens on their way change nothing).
#include "ssm_common.h"
#include "rvit_internal.h"
#include "ssm_args.h"

#include <type_traits>

namespace {

template <typename T, int V>
__device__ __forceinline__ void ldv(const T* p, float (&v)[V]) {
  if constexpr (V == 1) v[0] = ssm_ld(p);
  else if constexpr (V == 4) ssm_ld4(p, v);
  else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    v[0] = bf16_lo(u.x); v[1] = bf16_hi(u.x); v[2] = bf16_lo(u.y); v[3] = bf16_hi(u.y);
    v[4] = bf16_lo(u.z); v[5] = bf16_hi(u.z); v[6] = bf16_lo(u.w); v[7] = bf16_hi(u.w);
  }
}
template <typename T, int V>
__device__ __forceinline__ void stv(T* p, const float (&v)[V]) {
  if constexpr (V == 1) ssm_st(p, v[0]);
  else if constexpr (V == 4) ssm_st4(p, v);
  else *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
}
template <int V> __device__ __forceinline__ void zero(float (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = 0.f;
}
// V channels of a token as they lie in memory: fetched ahead of their use
template <typename T, int V> struct Raw {
  static constexpr int BYTES = V * sizeof(T);
  using U = typename std::conditional<BYTES == 16, uint4, typename std::conditional<BYTES == 8, uint2, typename std::conditional<BYTES == 4, uint32_t, uint16_t>::type>::type>::type;
  U u;
  __device__ __forceinline__ void load(const T* p) { u = *reinterpret_cast<const U*>(p); }
  __device__ __forceinline__ void get(float (&v)[V]) const { ldv<T, V>(reinterpret_cast<const T*>(&u), v); }
};
// token t with the kept inputs before it: t >= -(K - 1); zero where neither has it
template <typename T, int V, int K>
__device__ __forceinline__ void ldx(const SsmConvArgs& a, int b, int t, int c0, int len, float (&v)[V]) {
  if (t >= len) zero<V>(v);
  else if (t >= 0) ldv<T, V>((const T*)a.x + b * a.sxb + t * a.sxt + c0, v);
  else if (a.state && t >= 1 - K) ldv<T, V>((const T*)a.state + ((long)b * (K - 1) + (t + K - 1)) * a.C + c0, v);
  else zero<V>(v);
}
// the V x K weights of a thread lie in one piece: whole 16-byte loads where they are aligned (V > 1)
template <int V, int K>
__device__ __forceinline__ void ldw(const SsmConvArgs& a, int c0, float (&w)[K][V], float (&bias)[V]) {
  float f[V * K];
  const float* p = a.w + (long)c0 * K;
  if constexpr (V > 1) {
#pragma unroll
    for (int i = 0; i < V * K; i += 4) ssm_ld4(p + i, reinterpret_cast<float(&)[4]>(f[i]));
  } else {
#pragma unroll
    for (int i = 0; i < V * K; ++i) f[i] = p[i];
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][j] = f[j * K + k];
  }
  zero<V>(bias);
  if (a.bias) {
    if constexpr (V > 1) {
#pragma unroll
      for (int i = 0; i < V; i += 4) ssm_ld4(a.bias + c0 + i, reinterpret_cast<float(&)[4]>(bias[i]));
    } else bias[0] = a.bias[c0];
  }
}

template <typename T, int V, int K>
__global__ __launch_bounds__(256) void ssm_conv_fwd_kernel(SsmConvArgs a) {
  const int groups = a.C / V;
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  if (id >= (long)a.B * a.strips * groups) return;
  const int c0 = (int)(id % groups) * V;
  const long r = id / groups;
  const int s = r % a.strips, b = r / a.strips;
  const int len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
  const int t0 = s * a.strip, t1 = min(a.T, t0 + a.strip);
  T* y = (T*)a.y + (long)b * a.T * a.C + c0;
  float w[K][V], bias[V], win[K][V];
  ldw<V, K>(a, c0, w, bias);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) ldx<T, V, K>(a, b, t0 - (K - 1) + k, c0, len, win[k]);
  const int tl = min(t1, len);       // the strip's tokens that exist end here
  const T* x = (const T*)a.x + b * a.sxb + c0;
  constexpr int AHEAD = 4;           // tokens on their way
  Raw<T, V> next[AHEAD];
  if (t0 < tl) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) next[i].load(x + min(t0 + i, tl - 1) * a.sxt);
  }
  for (int t = t0; t < tl; t += AHEAD) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      next[i].get(win[K - 1]);
      next[i].load(x + min(t + i + AHEAD, tl - 1) * a.sxt);
      float u[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        u[j] = bias[j];
#pragma unroll
        for (int k = 0; k < K; ++k) u[j] = fmaf(w[k][j], win[k][j], u[j]);
        if (a.silu) u[j] *= ssm_sigmoid<T>(u[j]);
#pragma unroll
        for (int k = 0; k + 1 < K; ++k) win[k][j] = win[k + 1][j];
      }
      if (t + i < tl) stv<T, V>(y + (long)(t + i) * a.C, u);
    }
  }
  for (int t = max(t0, tl); t < t1; ++t) {
    float u[V];
    zero<V>(u);
    stv<T, V>(y + (long)t * a.C, u);
  }
  if (a.state_out && s == 0) {       // the last K - 1 inputs before the sequence's end
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      float v[V];
      ldx<T, V, K>(a, b, len - (K - 1) + k, c0, len, v);
      stv<T, V>((T*)a.state_out + ((long)b * (K - 1) + k) * a.C + c0, v);
    }
  }
}

// du[t] = dy silu'(u), u recomputed; dx[t] = sum_k w[k] du[t + K - 1 - k]; dw[k] = sum_t du[t] x[t - K + 1 + k]; db = sum du.
// A workgroup is 32 channel groups wide and 8 strips deep; its strips' dw, db are added in LDS in a fixed order and
// written as one part, which ssm_conv_sum_kernel adds.  (Three waves a SIMD for windows of 5 and 6: four would spill.)
template <typename T, int V, int K>
__global__ __launch_bounds__(256, V >= 4 && K >= 5 ? 3 : 4) void ssm_conv_bwd_kernel(SsmConvArgs a) {
  __shared__ float red[8][32][V];
  const int groups = a.C / V;
  const int gx = threadIdx.x & 31, sy = threadIdx.x >> 5;
  const int cblocks = (groups + 31) / 32, cx = blockIdx.x % cblocks, pi = blockIdx.x / cblocks;
  const int cg = cx * 32 + gx;
  const int sblocks = (a.strips + 7) / 8;
  const int b = pi / sblocks, s = (pi % sblocks) * 8 + sy;
  float dw[K][V], db[V];
#pragma unroll
  for (int k = 0; k < K; ++k) zero<V>(dw[k]);
  zero<V>(db);
  if (cg < groups && s < a.strips) {
    const int c0 = cg * V;
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.T) : a.T;
    const int t0 = s * a.strip, t1 = min(a.T, t0 + a.strip);
    T* dx = (T*)a.dx + (long)b * a.T * a.C + c0;
    const T* dy = (const T*)a.dy + b * a.syb + c0;
    const T* dso = a.dstate_out ? (const T*)a.dstate_out + (long)b * (K - 1) * a.C + c0 : nullptr;
    float w[K][V], bias[V], win[K][V], du[K][V];
    ldw<V, K>(a, c0, w, bias);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) ldx<T, V, K>(a, b, t0 - (K - 1) + k, c0, len, win[k]);
#pragma unroll
    for (int k = 0; k < K; ++k) zero<V>(du[k]);
    // token t enters: its du; then dx of token t - K + 1 is complete.  Tokens before the strip belong to the strip before
    // (the first strip gives them to the kept inputs).
    const T* x = (const T*)a.x + b * a.sxb + c0;
    Raw<T, V> nx, ny;                  // the next token's x and dy
    if (len > 0) {
      nx.load(x + min(t0, len - 1) * a.sxt);
      ny.load(dy + min(t0, len - 1) * a.syt);
    }
    // (K tokens a turn, the windows' places in turn: nothing moves)
    for (int tk = t0; tk < t1 + K - 1; tk += K) {
#pragma unroll
      for (int ph = 0; ph < K; ++ph) {
        const int t = tk + ph;
        if (t >= t1 + K - 1) break;
        auto at = [&](int k) { return (k + ph) % K; };      // place of token t - (K - 1) + k
        float g[V];
        zero<V>(win[at(K - 1)]);
        zero<V>(g);
        if (t < len) {
          nx.get(win[at(K - 1)]);
          ny.get(g);
          nx.load(x + min(t + 1, len - 1) * a.sxt);
          ny.load(dy + min(t + 1, len - 1) * a.syt);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (a.silu) {
            float u = bias[j];
#pragma unroll
            for (int k = 0; k < K; ++k) u = fmaf(w[k][j], win[at(k)][j], u);
            const float sg = ssm_sigmoid<T>(u);
            g[j] = t < len ? g[j] * (sg + u * sg * (1.f - sg)) : 0.f;
          }
          du[at(K - 1)][j] = g[j];
          const float own = t < t1 ? g[j] : 0.f;      // (the tokens behind the strip are another's)
          db[j] += own;
#pragma unroll
          for (int k = 0; k < K; ++k) dw[k][j] = fmaf(own, win[at(k)][j], dw[k][j]);
        }
        const int to = t - (K - 1);
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          o[j] = 0.f;
#pragma unroll
          for (int k = 0; k < K; ++k) o[j] = fmaf(w[k][j], du[at(K - 1 - k)][j], o[j]);
        }
        // du's place at(i) holds token t - (K - 1) + i, so o is dx of token `to`: complete for to >= t0, and for the kept inputs
        if (to >= t0 || s == 0) {
          if (dso && to >= len - (K - 1) && to < len) {
            float v[V];
            ldv<T, V>(dso + (long)(to - len + K - 1) * a.C, v);
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] += v[j];
          }
          if (to >= 0) stv<T, V>(dx + (long)to * a.C, o);
          else if (a.dstate) stv<T, V>((T*)a.dstate + ((long)b * (K - 1) + to + K - 1) * a.C + c0, o);
        }
      }
    }
  }
  // [part][K + 1][C]
  float* part = a.part + (long)pi * (K + 1) * a.C;
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) red[sy][gx][j] = k < K ? dw[k < K ? k : 0][j] : db[j];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * V; i += 256) {
      float v = 0.f;
#pragma unroll
      for (int y = 0; y < 8; ++y) v += red[y][i / V][i % V];
      const int c = cx * 32 * V + i;
      if (c < a.C) part[(long)k * a.C + c] = v;
    }
  }
}

// columns of the parts, added in a fixed order: 16 threads take every 16th part of a column
__global__ __launch_bounds__(1024) void ssm_conv_sum_kernel(const float* part, float* dw, float* db, int parts, int C, int K) {
  __shared__ double red[16][64];
  const long n = (long)(K + 1) * C, i = (long)blockIdx.x * 64 + (threadIdx.x & 63);
  const int py = threadIdx.x >> 6;
  double v = 0.0;
  if (i < n) {
    int p = py;
    for (; p + 48 < parts; p += 64) {      // four loads on their way
      const float a = part[p * n + i], b = part[(p + 16) * n + i], c = part[(p + 32) * n + i], d = part[(p + 48) * n + i];
      v += ((double)a + (double)b) + ((double)c + (double)d);
    }
    for (; p < parts; p += 16) v += (double)part[p * n + i];
  }
  red[py][threadIdx.x & 63] = v;
  __syncthreads();
  if (py == 0 && i < n) {
    for (int k = 1; k < 16; ++k) v += red[k][threadIdx.x];
    const int k = i / C, c = i - (long)k * C;
    if (k < K) dw[(long)c * K + k] = (float)v;
    else if (db) db[c] = (float)v;
  }
}

// one token: the kept inputs move by one, in place (a thread owns its channels of them)
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void ssm_conv_step_kernel(SsmConvArgs a) {
  const int groups = a.C / V;
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  if (id >= (long)a.B * groups) return;
  const int c0 = (int)(id % groups) * V, b = id / groups;
  T* st = (T*)a.state_out + (long)b * (K - 1) * a.C + c0;
  float w[K][V], bias[V], win[K][V];
#pragma unroll
  for (int k = 0; k < K - 1; ++k) ldv<T, V>(st + (long)k * a.C, win[k]);
  ldv<T, V>((const T*)a.x + b * a.sxb + c0, win[K - 1]);
  ldw<V, K>(a, c0, w, bias);
  float u[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    u[j] = bias[j];
#pragma unroll
    for (int k = 0; k < K; ++k) u[j] = fmaf(w[k][j], win[k][j], u[j]);
    if (a.silu) u[j] *= ssm_sigmoid<T>(u[j]);
  }
#pragma unroll
  for (int k = 0; k < K - 1; ++k) stv<T, V>(st + (long)k * a.C, win[k + 1]);
  stv<T, V>((T*)a.y + (long)b * a.C + c0, u);
}


template <typename T, int V, int K>
int launch(const SsmConvArgs& a, int what, hipStream_t st) {
  const int groups = a.C / V;
  if constexpr (V < 8) {      // (eight channels a thread: forward only, see below)
    if (what == SSM_CONV_BWD) {
      const int sblocks = (a.strips + 7) / 8;
      const long blocks = (long)((groups + 31) / 32) * a.B * sblocks;
      RVIT_CHECK_ARG(blocks < (1 << 24), "ssm_conv: more samples, tokens and channels than a backward pass can take (B=%d T=%d C=%d)", a.B, a.T, a.C);
      hipLaunchKernelGGL((ssm_conv_bwd_kernel<T, V, K>), dim3((unsigned)blocks), dim3(256), 0, st, a);
      RVIT_CHECK_LAUNCH("ssm_conv_bwd");
      hipLaunchKernelGGL(ssm_conv_sum_kernel, dim3((unsigned)(((long)(K + 1) * a.C + 63) / 64)), dim3(1024), 0, st, a.part, a.dw, a.dbias, a.B * sblocks, a.C, K);
      RVIT_CHECK_LAUNCH("ssm_conv_sum");
      return RVIT_OK;
    }
  }
  const long n = (long)a.B * (what == SSM_CONV_FWD ? a.strips : 1) * groups;
  RVIT_CHECK_ARG((n + 255) / 256 < (1 << 24), "ssm_conv: more samples, tokens and channels than a launch can take (B=%d T=%d C=%d)", a.B, a.T, a.C);
  const dim3 grid((unsigned)((n + 255) / 256));
  if (what == SSM_CONV_FWD) hipLaunchKernelGGL((ssm_conv_fwd_kernel<T, V, K>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((ssm_conv_step_kernel<T, V, K>), grid, dim3(256), 0, st, a);
  RVIT_CHECK_LAUNCH("ssm_conv");
  return RVIT_OK;
}
template <typename T, int V>
int launch_k(const SsmConvArgs& a, int what, hipStream_t st) {
  switch (a.K) {
    case 2: return launch<T, V, 2>(a, what, st);
    case 3: return launch<T, V, 3>(a, what, st);
    case 4: return launch<T, V, 4>(a, what, st);
    case 5: return launch<T, V, 5>(a, what, st);
    default: return launch<T, V, 6>(a, what, st);
  }
}

}  // namespace

int rvit_ssm_conv_impl(const SsmConvArgs& a, int dtype, int what, hipStream_t st) {
  // (bf16 backward: four channels a thread; with eight its windows and sums leave three waves a SIMD: 77 us against 55 at 8 x 2048 x 1792)
  if (dtype == RVIT_BF16) {
    if (!a.vec) return launch_k<bf16, 1>(a, what, st);
    return what == SSM_CONV_BWD ? launch_k<bf16, 4>(a, what, st) : launch_k<bf16, 8>(a, what, st);
  }
  return a.vec ? launch_k<float, 4>(a, what, st) : launch_k<float, 1>(a, what, st);
}
