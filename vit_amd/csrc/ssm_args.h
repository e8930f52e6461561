// Argument blocks of the state-space kernels.  Strides are in elements; [H,P] and [G,N] are packed inside a token.
#pragma once
#include "common.h"

constexpr int SSM_CHUNK = 64;     // tokens of a chunk
constexpr int SSM_MAX_N = 128;    // states per channel: the widest operand images in LDS
static inline int ssm_padded_n(int N) { return N <= 32 ? 32 : N <= 64 ? 64 : 128; }

struct SsmScanArgs {
  const void *x, *dt, *Bm, *Cm, *z;
  const float *A, *D, *dt_bias, *state0;
  const int* lengths;
  void* y;
  float* v;              // v before the gate, kept for the backward pass (or null): in 32 bits, as dz = dy v silu'(z) of bf16 calls would
                         // else be rounded twice
  float* state_out;      // [B,H,P,N] or null
  // Inner copies of states are padded to pblocks * 64 channels x NP states (NP: N up to 32, 64 or 128; what is added is zero) and
  // lie as [B, H, pblocks, NP / 4, 64, 4], so that a wave's piece of its 16 x 16 tiles is four runs of 256 bytes.  (With rows
  // of NP, 16 runs of 64: the sweeps that store a state per chunk took 86 and 173 us instead of 78 and 156 at
  // [8, 2048, 24, 64] x 128 states.)
  float* states;         // [nchunks] of them: the state before every chunk, kept for the backward pass (or null)
  float* seg_state;      // [nseg]    (nseg > 1)
  double* seg_decay;     // [nseg][B,H], base-2
  long sxb, sxt, sdb, sdt, sbb, sbt, scb, sct, szb, szt;
  long seg_stride;       // floats of one padded copy
  int B, T, H, P, G, N, pblocks, nchunks, seg_chunks, nseg;
  bool vec_x, vec_bc, vec_z, vec_y, vec_state;   // wide accesses are aligned
};

struct SsmBwdArgs {
  SsmScanArgs f;               // the forward's inputs, v and states
  const void* dy;
  const float* dstate_out;     // gradient of the returned state (or null)
  void *dx, *dz;               // [B,T,H,P], packed
  void *ddt;                   // [B,T,H]
  void *dB, *dC;               // [B,T,G,N]
  float *dA, *dD, *dbias;      // [H]
  float* dstate0;              // [B,H,P,N] or null
  float* dstates;              // [nchunks], padded: gradient of the state behind every chunk (null: zero)
  float* dbc_part;             // [hsplit][2][B,T,G,N] (hsplit > 1)
  float* part;                 // [B * nchunks][H][3]: dA, dD, dbias of a chunk
  long syb, syt;
  int hsplit, hper;            // heads of a group are taken by hsplit workgroups, hper each
  bool vec_dy, vec_out, vec_dbc;
};

struct SsmStepArgs {
  const void *x, *dt, *Bm, *Cm, *z;
  const float *A, *D, *dt_bias;
  float* state;
  void* y;
  long sxb, sdb, sbb, scb, szb;
  int B, H, P, G, N;
  bool vec_bc, vec_state;
};

struct SsmConvArgs {
  const void *x, *state, *dy, *dstate_out;
  const float *w, *bias;
  const int* lengths;
  void *y, *state_out, *dx, *dstate;
  float *dw, *dbias, *part;
  long sxb, sxt, syb, syt;
  int B, T, C, K, silu, strips, strip;
  bool vec;
};

int rvit_ssm_scan_fwd_impl(const SsmScanArgs& a, int dtype, hipStream_t st);
int rvit_ssm_scan_bwd_impl(const SsmBwdArgs& a, int dtype, hipStream_t st);
int rvit_ssm_scan_step_impl(const SsmStepArgs& a, int dtype, hipStream_t st);
int rvit_ssm_join(float* seg_state, const double* seg_decay, const float* init, const SsmScanArgs& a, int reverse, hipStream_t st);
enum { SSM_CONV_FWD = 0, SSM_CONV_BWD = 1, SSM_CONV_STEP = 2 };
int rvit_ssm_conv_impl(const SsmConvArgs& a, int dtype, int what, hipStream_t st);

struct SandwichArgs {
  const void *res, *y, *gate, *dh, *dn;
  const float *w1, *b1, *w2, *b2;    // norm behind the block (1) and before the next (2)
  void *h, *n;
  float* stats;                      // [rows][4]: mean, 1/std of y; mean, 1/std of h
  void *dres, *dy, *dgate;
  float *dw1, *db1, *dw2, *db2, *part;
  long rows;
  int E, T;                          // T: rows of a sample (gate per sample)
  int gate_kind;                     // 0 none, 1 per channel, 2 per sample, 3 per element
  int gate_f32, rms;
  float scale, eps;
  int parts, part_rows, sample_parts;   // backward: workgroups, rows of each, workgroups of a sample (gate per sample; else 0)
  bool vec;
};
int rvit_sandwich_fwd_impl(const SandwichArgs& a, int res_dtype, int dtype, hipStream_t st);
int rvit_sandwich_bwd_impl(const SandwichArgs& a, int res_dtype, int dtype, hipStream_t st);
