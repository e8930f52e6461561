// extern "C" surface, part 3: the state-space sequence operators (ssm_conv.hip, ssm_scan.hip, ssm_scan_bwd.hip, sandwich.hip).
#include "../../include/rvit.h"
#include "common.h"
#include "rvit_internal.h"
#include "ssm_args.h"

namespace {

bool at(const void* p, unsigned a) { return (((uintptr_t)p) & (a - 1)) == 0; }
int es(int dtype) { return dtype == RVIT_BF16 ? 2 : 4; }
// Token strides under this fit a 32-bit byte offset over the tokens of a chunk, which the kernels' wide paths use (63 strides
// of fp32 and a row's columns: 63 * 4 * (2^24 - 1) + 4 * 128 < 2^32); larger ones take the paths with 64-bit offsets.
constexpr int64_t MOST = 1 << 24;
bool strides_ok(std::initializer_list<int64_t> s) {      // (unsigned there: none may be negative)
  for (int64_t v : s)
    if (v < 0) return false;
  return true;
}

// Segments of a sequence.  One workgroup walks a (sample, head, 64 channels), and a compute unit holds two of them; where there
// are too few to fill the chip the sequence is cut, at the price of a pass that only computes states.
void segments(SsmScanArgs& a) {
  a.pblocks = (a.P + 63) / 64;
  a.nchunks = (a.T + SSM_CHUNK - 1) / SSM_CHUNK;
  const long rows = (long)a.B * a.H * a.pblocks;
  long n = rows >= 512 ? 1 : 512 / rows;
  if (n > a.nchunks / 2) n = a.nchunks / 2;      // two chunks at least: a shorter one is not worth its join
  if (a.nchunks < 8) n = 1;                      // nor are three launches for one short walk
  if (n < 1) n = 1;
  a.seg_chunks = n == 1 ? a.nchunks : (int)((a.nchunks + n - 1) / n);
  a.nseg = a.seg_chunks ? (a.nchunks + a.seg_chunks - 1) / a.seg_chunks : 1;
  if (a.nseg < 1) a.nseg = 1;
  a.seg_stride = (long)a.B * a.H * a.pblocks * 64 * ssm_padded_n(a.N);
}
int64_t seg_bytes(const SsmScanArgs& a) {
  return a.nseg > 1 ? (int64_t)a.nseg * (a.seg_stride * 4 + (int64_t)a.B * a.H * 8) + 16 : 0;
}
// Parts of a group's heads in the backward pass: a compute unit holds one workgroup of its chunk kernel.
void split_heads(SsmBwdArgs& a) {
  const int r = a.f.H / a.f.G;
  const long rows = (long)a.f.B * a.f.nchunks * a.f.G;
  long n = rows >= 256 || rows < 1 ? 1 : 256 / rows;
  if (n > r) n = r;
  a.hper = (int)((r + n - 1) / n);
  a.hsplit = (r + a.hper - 1) / a.hper;
}
int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }
// (a launch has fewer than 2^32 threads; the chunk kernel has 512 a workgroup, the sums' 256)
bool bwd_fits(const SsmBwdArgs& a) {
  return (int64_t)a.f.B * a.f.nchunks * a.f.G * a.hsplit < (1 << 23) && a.f.H < (1 << 23);
}

int shape(SsmScanArgs& a, int dtype, int B, int T, int H, int P, int G, int N) {
  RVIT_CHECK_ARG(dtype == RVIT_BF16 || dtype == RVIT_F32, "ssm_scan: dtype %d", dtype);
  RVIT_CHECK_ARG(B > 0 && T >= 0 && H > 0 && P > 0 && G > 0 && H % G == 0, "ssm_scan: bad sizes B=%d T=%d H=%d P=%d G=%d", B, T, H, P, G);
  RVIT_CHECK_ARG(N > 0 && N <= SSM_MAX_N, "ssm_scan: %d states per channel (1 .. %d)", N, SSM_MAX_N);
  RVIT_CHECK_ARG((int64_t)B * H * ((P + 63) / 64) < (1 << 24) && (int64_t)B * ((T + 63) / 64) * H < (1 << 30) && T < (1 << 28),
                 "ssm_scan: too many rows");
  RVIT_CHECK_ARG(P < (1 << 24), "ssm_scan: %d channels a head (under 2^24)", P);
  a.B = B; a.T = T; a.H = H; a.P = P; a.G = G; a.N = N;
  segments(a);
  return RVIT_OK;
}

int inputs(SsmScanArgs& a, int dtype, const void* x, int64_t sxb, int64_t sxt, const void* dt, int64_t sdb, int64_t sdt, const float* A,
           const void* Bm, int64_t sbb, int64_t sbt, const void* Cm, int64_t scb, int64_t sct, const float* D, const void* z, int64_t szb,
           int64_t szt, const float* dt_bias, const int* lengths) {
  RVIT_CHECK_ARG(A && (a.T == 0 || (x && dt && Bm && Cm)), "ssm_scan: null pointer");
  RVIT_CHECK_ARG(strides_ok({sxb, sxt, sdb, sdt, sbb, sbt, scb, sct, szb, szt}), "ssm_scan: negative stride");
  a.x = x; a.dt = dt; a.A = A; a.Bm = Bm; a.Cm = Cm; a.D = D; a.z = z; a.dt_bias = dt_bias; a.lengths = lengths;
  a.sxb = sxb; a.sxt = sxt; a.sdb = sdb; a.sdt = sdt; a.sbb = sbb; a.sbt = sbt; a.scb = scb; a.sct = sct; a.szb = szb; a.szt = szt;
  const int V = 16 / es(dtype);
  a.vec_x = at(x, 16) && sxt < MOST && sbt < MOST && sct < MOST && (int64_t)a.H * a.P < MOST && sxb % V == 0 && sxt % V == 0 && a.P % V == 0;
  a.vec_bc = at(Bm, 16) && at(Cm, 16) && sbb % V == 0 && sbt % V == 0 && scb % V == 0 && sct % V == 0 && a.N % V == 0;
  a.vec_z = at(z, 4 * es(dtype)) && szt < MOST && szb % 4 == 0 && szt % 4 == 0 && a.P % 4 == 0;
  return RVIT_OK;
}

void take_segments(SsmScanArgs& a, char*& ws) {
  if (a.nseg <= 1) return;
  a.seg_decay = (double*)ws;
  ws += round16((int64_t)a.nseg * a.B * a.H * 8);
  a.seg_state = (float*)ws;
  ws += round16((int64_t)a.nseg * a.seg_stride * 4);
}

}  // namespace

extern "C" {

int rvit_ssm_scan_plan(int64_t* fwd_bytes, int64_t* state_floats, int64_t* bwd_bytes, int B, int T, int H, int P, int G, int N) {
  SsmBwdArgs a = {};
  if (int e = shape(a.f, RVIT_F32, B, T, H, P, G, N)) return e;
  split_heads(a);
  RVIT_CHECK_ARG(!bwd_bytes || bwd_fits(a), "ssm_scan: more samples, chunks of 64 tokens and groups than a backward pass can take (B=%d T=%d G=%d H=%d)", B, T, G, H);
  if (fwd_bytes) *fwd_bytes = seg_bytes(a.f) + 16;
  if (state_floats) *state_floats = (int64_t)a.f.nchunks * a.f.seg_stride;
  if (bwd_bytes)
    *bwd_bytes = seg_bytes(a.f) + 64 + round16((int64_t)a.f.nchunks * a.f.seg_stride * 4) + round16((int64_t)B * a.f.nchunks * H * 12) +
                 (a.hsplit > 1 ? round16((int64_t)a.hsplit * 2 * B * T * G * N * 4) : 0);
  return RVIT_OK;
}

int rvit_ssm_scan_fwd(const void* x, int64_t sxb, int64_t sxt, const void* dt, int64_t sdb, int64_t sdt, const float* A, const void* Bm,
                      int64_t sbb, int64_t sbt, const void* Cm, int64_t scb, int64_t sct, const float* D, const void* z, int64_t szb, int64_t szt,
                      const float* dt_bias, const float* state0, const int* lengths, void* y, float* v, float* state_out, float* states,
                      void* workspace, int64_t workspace_bytes, int dtype, int B, int T, int H, int P, int G, int N, void* stream) {
  SsmScanArgs a = {};
  if (int e = shape(a, dtype, B, T, H, P, G, N)) return e;
  if (int e = inputs(a, dtype, x, sxb, sxt, dt, sdb, sdt, A, Bm, sbb, sbt, Cm, scb, sct, D, z, szb, szt, dt_bias, lengths)) return e;
  RVIT_CHECK_ARG(T == 0 || y, "ssm_scan_fwd: null output");
  RVIT_CHECK_ARG(!workspace || at(workspace, 16), "ssm_scan_fwd: workspace alignment");
  RVIT_CHECK_ARG(seg_bytes(a) == 0 || (workspace && workspace_bytes >= seg_bytes(a) + 16), "ssm_scan_fwd: workspace of %lld bytes, %lld needed",
                 (long long)workspace_bytes, (long long)seg_bytes(a) + 16);
  a.state0 = state0; a.y = y; a.v = v; a.state_out = state_out; a.states = states;
  a.vec_y = at(y, 4 * es(dtype)) && at(v, 16) && P % 4 == 0;
  a.vec_state = N % 4 == 0 && at(state0, 16) && at(state_out, 16);
  RVIT_CHECK_ARG(at(states, 16), "ssm_scan_fwd: states alignment");
  char* ws = (char*)workspace;
  take_segments(a, ws);
  return rvit_ssm_scan_fwd_impl(a, dtype, (hipStream_t)stream);
}

int rvit_ssm_scan_bwd(const void* x, int64_t sxb, int64_t sxt, const void* dt, int64_t sdb, int64_t sdt, const float* A, const void* Bm,
                      int64_t sbb, int64_t sbt, const void* Cm, int64_t scb, int64_t sct, const float* D, const void* z, int64_t szb, int64_t szt,
                      const float* dt_bias, const int* lengths, const float* v, const float* states, const void* dy, int64_t syb, int64_t syt,
                      const float* dstate_out, void* dx, void* ddt, float* dA, void* dB, void* dC, float* dD, void* dz, float* ddt_bias,
                      float* dstate0, void* workspace, int64_t workspace_bytes, int dtype, int B, int T, int H, int P, int G, int N, void* stream) {
  SsmBwdArgs a = {};
  if (int e = shape(a.f, dtype, B, T, H, P, G, N)) return e;
  if (int e = inputs(a.f, dtype, x, sxb, sxt, dt, sdb, sdt, A, Bm, sbb, sbt, Cm, scb, sct, D, z, szb, szt, dt_bias, lengths)) return e;
  RVIT_CHECK_ARG(T > 0, "ssm_scan_bwd: no tokens");
  RVIT_CHECK_ARG(strides_ok({syb, syt}), "ssm_scan_bwd: negative stride");
  RVIT_CHECK_ARG(states && dy && dx && ddt && dA && dB && dC && (!z || (v && dz)), "ssm_scan_bwd: null pointer");
  split_heads(a);
  int64_t need = 0;
  if (int e = rvit_ssm_scan_plan(nullptr, nullptr, &need, B, T, H, P, G, N)) return e;
  RVIT_CHECK_ARG(workspace && at(workspace, 16) && workspace_bytes >= need, "ssm_scan_bwd: workspace of %lld bytes, %lld needed",
                 (long long)workspace_bytes, (long long)need);
  a.f.v = (float*)v; a.f.states = (float*)states;
  a.dy = dy; a.syb = syb; a.syt = syt; a.dstate_out = dstate_out;
  a.dx = dx; a.dz = z ? dz : nullptr; a.ddt = ddt; a.dB = dB; a.dC = dC; a.dA = dA; a.dD = dD; a.dbias = ddt_bias; a.dstate0 = dstate0;
  a.f.vec_y = at(v, 16) && P % 4 == 0;
  a.f.vec_state = N % 4 == 0 && at(dstate_out, 16) && at(dstate0, 16);
  RVIT_CHECK_ARG(at(states, 16), "ssm_scan_bwd: states alignment");
  a.vec_dy = at(dy, 4 * es(dtype)) && syt < MOST && syb % 4 == 0 && syt % 4 == 0 && P % 4 == 0;
  a.vec_out = at(dx, 4 * es(dtype)) && at(dz, 4 * es(dtype)) && P % 4 == 0;
  a.vec_dbc = at(dB, 4 * es(dtype)) && at(dC, 4 * es(dtype)) && N % 4 == 0;
  char* ws = (char*)workspace;
  take_segments(a.f, ws);
  // (of one chunk without a gradient of its end there is nothing to sweep: dS is zero)
  a.dstates = a.f.nchunks == 1 && !dstate_out && !dstate0 ? nullptr : (float*)ws;
  ws += round16((int64_t)a.f.nchunks * a.f.seg_stride * 4);
  a.part = (float*)ws;
  ws += round16((int64_t)B * a.f.nchunks * H * 12);
  a.dbc_part = (float*)ws;
  return rvit_ssm_scan_bwd_impl(a, dtype, (hipStream_t)stream);
}

int rvit_ssm_scan_step(const void* x, int64_t sxb, const void* dt, int64_t sdb, const float* A, const void* Bm, int64_t sbb, const void* Cm,
                       int64_t scb, const float* D, const void* z, int64_t szb, const float* dt_bias, float* state, void* y, int dtype, int B,
                       int H, int P, int G, int N, void* stream) {
  SsmScanArgs s = {};
  if (int e = shape(s, dtype, B, 1, H, P, G, N)) return e;
  RVIT_CHECK_ARG(x && dt && A && Bm && Cm && state && y, "ssm_scan_step: null pointer");
  RVIT_CHECK_ARG(strides_ok({sxb, sdb, sbb, scb, szb}), "ssm_scan_step: negative stride");
  SsmStepArgs a = {};
  a.x = x; a.dt = dt; a.A = A; a.Bm = Bm; a.Cm = Cm; a.D = D; a.z = z; a.dt_bias = dt_bias; a.state = state; a.y = y;
  a.sxb = sxb; a.sdb = sdb; a.sbb = sbb; a.scb = scb; a.szb = szb;
  a.B = B; a.H = H; a.P = P; a.G = G; a.N = N;
  const unsigned v = 4 * es(dtype);
  a.vec_bc = at(Bm, v) && at(Cm, v) && sbb % 4 == 0 && scb % 4 == 0 && N % 4 == 0;
  a.vec_state = at(state, 16) && N % 4 == 0;
  return rvit_ssm_scan_step_impl(a, dtype, (hipStream_t)stream);
}

}  // extern "C"

namespace {

int conv_args(SsmConvArgs& a, int dtype, const void* x, int64_t sxb, int64_t sxt, const float* w, const float* bias, int B, int T, int C, int K, int silu) {
  RVIT_CHECK_ARG(dtype == RVIT_BF16 || dtype == RVIT_F32, "ssm_conv: dtype %d", dtype);
  RVIT_CHECK_ARG(B > 0 && T > 0 && C > 0 && K >= 2 && K <= 6, "ssm_conv: bad sizes B=%d T=%d C=%d K=%d (K: 2 .. 6)", B, T, C, K);
  RVIT_CHECK_ARG((int64_t)B * C < (1 << 30) && T < (1 << 28), "ssm_conv: too many rows");
  RVIT_CHECK_ARG(x && w, "ssm_conv: null pointer");
  RVIT_CHECK_ARG(strides_ok({sxb, sxt}), "ssm_conv: negative stride");
  a.x = x; a.sxb = sxb; a.sxt = sxt; a.w = w; a.bias = bias; a.B = B; a.T = T; a.C = C; a.K = K; a.silu = silu;
  const int V = 16 / es(dtype);
  a.vec = at(x, 16) && at(w, 16) && at(bias, 16) && sxb % V == 0 && sxt % V == 0 && C % V == 0;
  return RVIT_OK;
}
// tokens of a thread: long strips reread less, short ones fill the chip
void strips(SsmConvArgs& a, int dtype) {
  const int V = a.vec ? 16 / es(dtype) : 1;
  a.strip = 16;
  while (a.strip > 4 && (int64_t)a.B * ((a.T + a.strip - 1) / a.strip) * (a.C / V) < 256 * 1024) a.strip /= 2;
  a.strips = (a.T + a.strip - 1) / a.strip;
}
// the backward pass: workgroups of eight strips, each of which leaves a part of dw
void bwd_strips(int& strip, int& n, int64_t B, int64_t T, int64_t C) {
  int64_t s = 32;
  while (s > 4 && B * ((T + 8 * s - 1) / (8 * s)) * ((C + 255) / 256) < 512) s /= 2;
  strip = (int)s;
  n = (int)((T + s - 1) / s);
}

}  // namespace

extern "C" {

int rvit_ssm_conv_fwd(const void* x, int64_t sxb, int64_t sxt, const float* w, const float* bias, const void* state, const int* lengths, void* y,
                      void* state_out, int dtype, int B, int T, int C, int K, int silu, void* stream) {
  SsmConvArgs a = {};
  if (int e = conv_args(a, dtype, x, sxb, sxt, w, bias, B, T, C, K, silu)) return e;
  RVIT_CHECK_ARG(y && (!state || state != state_out), "ssm_conv_fwd: null output, or the kept inputs in place");
  a.state = state; a.lengths = lengths; a.y = y; a.state_out = state_out;
  a.vec = a.vec && at(state, 16) && at(y, 16) && at(state_out, 16);
  strips(a, dtype);
  return rvit_ssm_conv_impl(a, dtype, SSM_CONV_FWD, (hipStream_t)stream);
}

int rvit_ssm_conv_bwd_workspace(int64_t* bytes, int B, int T, int C, int K) {
  RVIT_CHECK_ARG(B > 0 && T > 0 && C > 0 && K >= 2 && K <= 6 && bytes, "ssm_conv: bad sizes B=%d T=%d C=%d K=%d (K: 2 .. 6)", B, T, C, K);
  int strip, n;
  bwd_strips(strip, n, B, T, C);
  const int64_t wide = C % 4 ? 32 : 128;      // channels of a workgroup: 32 accesses of one or (aligned) four
  const int64_t blocks = (int64_t)B * ((n + 7) / 8) * ((C + wide - 1) / wide);
  RVIT_CHECK_ARG(blocks < (1 << 24) && (int64_t)(K + 1) * C < (1 << 28), "ssm_conv: more samples, tokens and channels than a backward pass can take (B=%d T=%d C=%d)",
                 B, T, C);
  *bytes = (int64_t)B * ((n + 7) / 8) * (K + 1) * C * 4;
  return RVIT_OK;
}

int rvit_ssm_conv_bwd(const void* x, int64_t sxb, int64_t sxt, const float* w, const float* bias, const void* state, const int* lengths,
                      const void* dy, int64_t syb, int64_t syt, const void* dstate_out, void* dx, float* dw, float* dbias, void* dstate,
                      void* workspace, int64_t workspace_bytes, int dtype, int B, int T, int C, int K, int silu, void* stream) {
  SsmConvArgs a = {};
  if (int e = conv_args(a, dtype, x, sxb, sxt, w, bias, B, T, C, K, silu)) return e;
  RVIT_CHECK_ARG(strides_ok({syb, syt}), "ssm_conv_bwd: negative stride");
  int64_t need = 0;
  if (int e = rvit_ssm_conv_bwd_workspace(&need, B, T, C, K)) return e;
  RVIT_CHECK_ARG(dy && dx && dw && workspace && at(workspace, 16) && workspace_bytes >= need, "ssm_conv_bwd: null pointer, or workspace of %lld bytes, %lld needed",
                 (long long)workspace_bytes, (long long)need);
  a.state = state; a.lengths = lengths; a.dy = dy; a.syb = syb; a.syt = syt; a.dstate_out = dstate_out; a.dx = dx; a.dw = dw; a.dbias = dbias;
  a.dstate = dstate; a.part = (float*)workspace;
  const int V = 16 / es(dtype);
  a.vec = a.vec && at(state, 16) && at(dy, 16) && syb % V == 0 && syt % V == 0 && at(dstate_out, 16) && at(dx, 16) && at(dstate, 16);
  bwd_strips(a.strip, a.strips, B, T, C);
  return rvit_ssm_conv_impl(a, dtype, SSM_CONV_BWD, (hipStream_t)stream);
}

int rvit_ssm_conv_step(const void* x, int64_t sxb, const float* w, const float* bias, void* state, void* y, int dtype, int B, int C, int K, int silu,
                       void* stream) {
  SsmConvArgs a = {};
  if (int e = conv_args(a, dtype, x, sxb, 0, w, bias, B, 1, C, K, silu)) return e;
  RVIT_CHECK_ARG(state && y, "ssm_conv_step: null pointer");
  a.state_out = state; a.y = y;
  a.vec = a.vec && at(state, 16) && at(y, 16);
  return rvit_ssm_conv_impl(a, dtype, SSM_CONV_STEP, (hipStream_t)stream);
}

}  // extern "C"

namespace {

int sandwich_args(SandwichArgs& a, const void* res, int res_dtype, const void* y, int dtype, const void* gate, int gate_kind, int gate_dtype, float scale,
                  const float* w1, const float* b1, const float* w2, const float* b2, float eps, int rms, int64_t rows, int T, int E) {
  RVIT_CHECK_ARG((res_dtype == RVIT_BF16 || res_dtype == RVIT_F32) && (dtype == RVIT_BF16 || dtype == RVIT_F32), "sandwich_norm: dtype");
  RVIT_CHECK_ARG(rows > 0 && rows < (1ll << 31) && E > 0 && E <= 4096, "sandwich_norm: rows=%lld E=%d (E: 1 .. 4096)", (long long)rows, E);
  RVIT_CHECK_ARG(res && y && w1 && w2, "sandwich_norm: null pointer");
  RVIT_CHECK_ARG(gate_kind >= 0 && gate_kind <= 3 && (gate_kind == 0 || (gate && (gate_dtype == RVIT_F32 || gate_dtype == dtype))), "sandwich_norm: gate");
  RVIT_CHECK_ARG(gate_kind != 2 || (T > 0 && rows % T == 0), "sandwich_norm: a gate per sample needs rows that are whole samples (T=%d)", T);
  a.res = res; a.y = y; a.gate = gate; a.w1 = w1; a.b1 = b1; a.w2 = w2; a.b2 = b2; a.rows = rows; a.E = E; a.T = T > 0 ? T : 1;
  a.gate_kind = gate_kind; a.gate_f32 = gate_dtype == RVIT_F32; a.rms = rms; a.scale = scale; a.eps = eps;
  a.vec = E % 4 == 0 && at(res, 16) && at(y, 16) && at(gate, 16) && at(w1, 16) && at(b1, 16) && at(w2, 16) && at(b2, 16);
  return RVIT_OK;
}
void sandwich_parts(SandwichArgs& a) {
  const int want = 1024;      // four workgroups per compute unit
  if (a.gate_kind == 2) {
    const int64_t samples = a.rows / a.T;
    int64_t per = (want + samples - 1) / samples;
    if (per > (a.T + 3) / 4) per = (a.T + 3) / 4;
    a.part_rows = (int)((a.T + per - 1) / per);
    a.sample_parts = (a.T + a.part_rows - 1) / a.part_rows;
    a.parts = (int)(samples * a.sample_parts);
  } else {
    int64_t n = (a.rows + 3) / 4 < want ? (a.rows + 3) / 4 : want;
    a.part_rows = (int)((a.rows + n - 1) / n);
    a.parts = (int)((a.rows + a.part_rows - 1) / a.part_rows);
    a.sample_parts = 0;
  }
}

}  // namespace

extern "C" {

int rvit_sandwich_norm_fwd(const void* residual, int res_dtype, const void* y, int dtype, const void* gate, int gate_kind, int gate_dtype, float scale,
                           const float* post_w, const float* post_b, const float* pre_w, const float* pre_b, float eps, int rms, void* h, void* n,
                           float* stats, int64_t rows, int T, int E, void* stream) {
  SandwichArgs a = {};
  if (int e = sandwich_args(a, residual, res_dtype, y, dtype, gate, gate_kind, gate_dtype, scale, post_w, post_b, pre_w, pre_b, eps, rms, rows, T, E)) return e;
  RVIT_CHECK_ARG(h && n && at(stats, 16), "sandwich_norm_fwd: null output, or stats unaligned");
  a.h = h; a.n = n; a.stats = stats;
  a.vec = a.vec && at(h, 16) && at(n, 16);
  return rvit_sandwich_fwd_impl(a, res_dtype, dtype, (hipStream_t)stream);
}

int rvit_sandwich_norm_bwd_workspace(int64_t* bytes, int64_t rows, int T, int E, int gate_kind) {
  RVIT_CHECK_ARG(rows > 0 && rows < (1ll << 31) && E > 0 && E <= 4096 && bytes && (gate_kind != 2 || (T > 0 && rows % T == 0)), "sandwich_norm: bad sizes");
  SandwichArgs a = {};
  a.rows = rows; a.T = T > 0 ? T : 1; a.E = E; a.gate_kind = gate_kind;
  sandwich_parts(a);
  RVIT_CHECK_ARG(a.parts < (1 << 24), "sandwich_norm: %d samples with gates are more than a backward pass can take", a.parts);
  *bytes = (int64_t)a.parts * 5 * E * 4;
  return RVIT_OK;
}

int rvit_sandwich_norm_bwd(const void* residual, int res_dtype, const void* y, int dtype, const void* gate, int gate_kind, int gate_dtype, float scale,
                           const float* post_w, const float* post_b, const float* pre_w, const float* pre_b, float eps, int rms, const float* stats,
                           const void* dh, const void* dn, void* dresidual, void* dy, void* dgate, float* dpost_w, float* dpost_b, float* dpre_w,
                           float* dpre_b, void* workspace, int64_t workspace_bytes, int64_t rows, int T, int E, void* stream) {
  SandwichArgs a = {};
  if (int e = sandwich_args(a, residual, res_dtype, y, dtype, gate, gate_kind, gate_dtype, scale, post_w, post_b, pre_w, pre_b, eps, rms, rows, T, E)) return e;
  int64_t need = 0;
  if (int e = rvit_sandwich_norm_bwd_workspace(&need, rows, T, E, gate_kind)) return e;
  RVIT_CHECK_ARG(stats && at(stats, 16) && dh && dn && dresidual && dy && (gate_kind == 0 || dgate) && dpost_w && dpre_w, "sandwich_norm_bwd: null pointer");
  RVIT_CHECK_ARG(workspace && at(workspace, 16) && workspace_bytes >= need, "sandwich_norm_bwd: workspace of %lld bytes, %lld needed",
                 (long long)workspace_bytes, (long long)need);
  a.stats = (float*)stats; a.dh = dh; a.dn = dn; a.dres = dresidual; a.dy = dy; a.dgate = dgate; a.dw1 = dpost_w; a.db1 = dpost_b; a.dw2 = dpre_w;
  a.db2 = dpre_b; a.part = (float*)workspace;
  a.vec = a.vec && at(dh, 16) && at(dn, 16) && at(dresidual, 16) && at(dy, 16) && at(dgate, 16);
  sandwich_parts(a);
  return rvit_sandwich_bwd_impl(a, res_dtype, dtype, (hipStream_t)stream);
}

}  // extern "C"
