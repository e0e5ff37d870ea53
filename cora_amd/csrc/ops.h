// ops.h -- parameter blocks of the stand-alone operators (op_rotary.hip, op_attention.hip, op_ortho.hip); the C entry
// points that check the caller's arguments and fill them are in op_api.hip.
#pragma once
#include "common.h"

enum OpType { OP_F32 = 0, OP_BF16 = 1, OP_F16 = 2 };
inline int op_bytes(int dtype) { return dtype == OP_F32 ? 4 : 2; }

// ---- rotary positions ----------------------------------------------------------------------------
struct RotaryP {
  const void* x; void* y;
  const int* pos;               // [pos_rows, n_axes]
  long long rows, pos_rows;     // row r turns by pos[r % pos_rows]
  long long xr, xh, yr, yh;     // strides of x and y in elements: row, head
  int heads, d, n_axes, pairs;  // pairs: half the channels that turn
  int interleaved, copy;        // copy: the channels past the last axis are copied (y is not x)
  float sign;                   // +1 forward, -1 backward
  double turn[64];              // pair -> turns per unit of position, theta^(-2 i / n) / (2 pi)
  unsigned char axis[64], c0[64], c1[64];   // pair -> axis, its two channels
};
int launch_rotary(const RotaryP& p, int dtype, hipStream_t st);

// ---- attention over packed sequences -------------------------------------------------------------
struct AttnP {
  const void *q, *k, *v, *o, *dout;
  void *out, *dq, *dk, *dv;
  float* lse;                   // [heads, rows]
  float* delta;                 // backward workspace [2, heads, rows]: -rowsum(dout out), -lse (log2; fp16: 14 more)
  float* partial;               // [parts, 2, rows, kv_heads, d]: dk and dv of each part, if parts > 1
  int parts;                    // ranges the queries of a key tile are cut into (attention_parts)
  const int* cu;                // [nseq + 1] first rows, or null: nseq sequences of seqlen rows each
  long long rows;
  long long qr, qh, kr, kh, vr, vh, orow, oh, dor, doh, dqr, dqh, dkr, dkh, dvr, dvh;   // element strides
  int nseq, seqlen, heads, kv_heads, d, block;   // block: causal block, 0 = bidirectional
  float scale;
};
int attention_parts(int dtype, long long rows, int nseq, int heads, int kv_heads, int block);
int launch_attention_fwd(const AttnP& p, int dtype, hipStream_t st);
int launch_attention_bwd(const AttnP& p, int dtype, hipStream_t st);

// ---- orthogonalisation of updates ----------------------------------------------------------------
constexpr int ORTHO_GROUPS = 16, ORTHO_STEPS = 32, ORTHO_PARTS = 256;
struct OrthoG {                 // a stack of equal matrices; m = min(rows, cols), n = max
  const void* x; void* y;
  long long xm, xr, ym, yr;     // strides in elements: matrix, row
  int count, rows, cols, m, n, ldn, ldm, first;   // ldn, ldm: n, m rounded up to 64; first: matrices of the groups before
  int sn, sm;                   // row strides of the n and m columns wide planes: odd multiples of 128 bytes (op_ortho.hip)
  long long ws;                 // first 16-bit element of its matrices in the workspace
};
struct OrthoP {
  OrthoG g[ORTHO_GROUPS];
  int ngroups, matrices;
  unsigned short* ws;           // planes of 16-bit halves (op_ortho.hip)
  double* parts;                // [matrices, ORTHO_PARTS] partial sums of squares
  float eps;
};
struct OrthoCoef { int steps; float c[3 * ORTHO_STEPS]; };
bool ortho_is_small(const OrthoG& g);   // worked on by one workgroup, in LDS
size_t ortho_ws_bytes(OrthoP& p);   // sets the groups' ws offsets
void ortho_place(OrthoP& p, void* ws);  // the workspace's two parts (256-byte aligned)
int launch_ortho(const OrthoP& p, int dtype, int steps, const float* coef, hipStream_t st);
int ortho_bad_step(int steps, const float* coef);   // first step whose coefficients leave the iterates' range, -1: none

// ---- orthogonalised momentum (ctx.hip's weight step) -----------------------------------------------
// u = momentum of the scaled, clipped gradient over n elements
struct MuonP {
  const float* g; float* mu; float* u; float* w; long long n;
  const double* sumsq; float gscale, clip, beta; int nesterov;
  const float* hyp; float wd, size;   // apply: w -= hyp[0] (size u + wd w)
};
void launch_muon_momentum(const MuonP& p, hipStream_t st);
void launch_muon_apply(const MuonP& p, hipStream_t st);
// fills what both operators' callers inside the library share
void fill_rotary(RotaryP& p, int n_axes, const int* axes_dim, double theta, bool interleaved);
void fill_stack(OrthoP& p, const float* x, float* y, int count, int rows, int cols);
size_t attention_ws_bytes(int dtype, long long rows, int nseq, int heads, int kv_heads, int d, int block);
void attention_ws(AttnP& p, int dtype, void* ws);   // places delta, partial and parts
