// op_ortho.hip -- orthogonalisation of weight updates by Newton-Schulz products (gfx950).
//
// X_0 = G / (|G|_F + eps), transposed if G is tall so that X is m x n with m <= n; every step
//   A = X X^T,  P = a I + b A + c A^2,  X <- P X,
// which moves each singular value s of X to a s + b s^3 + c s^5.  A and A^2 are symmetric: only their lower tiles are
// computed, and stored twice.
//
// Number format.  With the usual coefficients small singular directions grow by 3.4 a step, 500 in five, and an error made
// in X grows with them; bf16 (2^-9) or plain fp16 (2^-12) iterates end several percent off.  fp32 matrix products run at a
// sixteenth of the 16-bit rate.  So every matrix is kept as two fp16 halves, x = hi + lo, 22 bits, and a product takes three
// fp16 matrix instructions (hi hi + hi lo + lo hi, fp32 sums): fp32-grade at a third of the 16-bit rate.  fp16 has few
// exponents, but all iterates have singular values of at most a few units, so a fixed power of two places them: X is
// stored times 2^12 (entries of a large matrix are near 1 / sqrt(m n)), A and P times 2^6 (what matters of them is their
// size next to a ~ 3); the caller's coefficients are refused where the iterates could leave these ranges.
// For bf16 results the two large products save instructions where the error does not grow: A from the upper halves of X
// alone (one instruction), and P X with the upper half of P = b A + c A^2 (two), a X being added in fp32; A^2 keeps all
// three, since at singular values near 1 an error of A^2 is amplified.  The result is then 1e-3 (rms) off the exact
// iterates before its own rounding of 1.7e-3, against 2.5e-3 with one instruction throughout.
#include "op_tile.h"
#include "ops.h"

namespace {

typedef _Float16 half;
typedef half h16x4 __attribute__((ext_vector_type(4)));
constexpr float SX = 4096.f, SA = 64.f;

// workspace of one matrix, in halves: X hi, X lo, Y hi, Y lo (m x ldn each), A hi, A lo, P hi, P lo (m x ldm each)
__device__ __forceinline__ half* plane_x(const OrthoP& p, const OrthoG& g, int mat, int which) {
  return (half*)p.ws + g.ws + (long long)mat * (4LL * g.m * g.ldn + 4LL * g.m * g.ldm) + (long long)which * g.m * g.ldn;
}
__device__ __forceinline__ half* plane_a(const OrthoP& p, const OrthoG& g, int mat, int which) {
  return plane_x(p, g, mat, 4) + (long long)which * g.m * g.ldm;
}

__device__ __forceinline__ void split2(float v, half& hi, half& lo) { hi = (half)v; lo = (half)(v - (float)hi); }

// partial sums of squares in 64 bits: part z of a matrix takes every ORTHO_PARTS-th row
template <typename T>
__global__ __launch_bounds__(256) void ortho_sumsq(const OrthoP p) {
  __shared__ double sh[4];
  const int id = blockIdx.x, part = blockIdx.y;
  int gi = 0;
  while (gi + 1 < p.ngroups && id >= p.g[gi + 1].first) ++gi;
  const OrthoG& g = p.g[gi];
  const T* x = (const T*)g.x + (long long)(id - g.first) * g.xm;
  double s = 0.0;
  for (int r = part; r < g.rows; r += ORTHO_PARTS)
    for (int c = threadIdx.x; c < g.cols; c += 256) { const double v = (double)(float)x[(long long)r * g.xr + c]; s += v * v; }
  s = block_sum_256(s, sh);
  if (threadIdx.x == 0) p.parts[(long long)id * ORTHO_PARTS + part] = s;
}

// X_0: scale, transpose if tall, split; 64 x 64 pieces, columns [n, ldn) zero
template <typename T>
__global__ __launch_bounds__(256) void ortho_load(const OrthoP p) {
  __shared__ float t[64][65];
  const int id = blockIdx.y;
  int gi = 0;
  while (gi + 1 < p.ngroups && id >= p.g[gi + 1].first) ++gi;
  const OrthoG& g = p.g[gi];
  const int mat = id - g.first, tn = g.ldn / 64, tm = g.ldm / 64;
  if ((int)blockIdx.x >= tn * tm) return;
  const int i0 = blockIdx.x / tn * 64, j0 = blockIdx.x % tn * 64;
  double s = 0.0;
  for (int k = 0; k < ORTHO_PARTS; ++k) s += p.parts[(long long)id * ORTHO_PARTS + k];
  const double f = (double)SX / (sqrt(s) + (double)p.eps);
  const bool tall = g.rows > g.cols;
  const T* x = (const T*)g.x + (long long)mat * g.xm;
  const int a = threadIdx.x & 63, b = threadIdx.x >> 6;
  for (int k = b; k < 64; k += 4) {                       // source rows along b
    const int r = (tall ? j0 : i0) + k, c = (tall ? i0 : j0) + a;
    const float v = r < g.rows && c < g.cols ? (float)((double)(float)x[(long long)r * g.xr + c] * f) : 0.f;
    if (tall) t[a][k] = v; else t[k][a] = v;
  }
  __syncthreads();
  half* hi = plane_x(p, g, mat, 0); half* lo = plane_x(p, g, mat, 1);
  for (int k = b; k < 64; k += 4)
    if (i0 + k < g.m) {
      half vh, vl;
      split2(t[k][a], vh, vl);
      const long long o = (long long)(i0 + k) * g.ldn + j0 + a;
      hi[o] = vh; lo[o] = vl;
    }
}

// One product for all matrices.  STEP 0: A = X X^T; 1: P = a I + b A + c A A; 2: X' = P X (last: to the caller's matrix).
// Tile 128 x 128, four waves of 64 x 64, slabs of 32: the first operand gives the output's columns, the second its rows
// (op_tile.h), so a lane holds four neighbouring columns of one output row.
template <typename T, int STEP, bool FULL>
__global__ __launch_bounds__(256, 2) void ortho_product(const OrthoP p, const int cur, const int last, const float ca, const float cb, const float cc) {
  constexpr int TK = 32;
  typedef Tile<half, TK> LR; typedef Tile<half, 128> LC;
  typedef Op<half> O;
  __shared__ __attribute__((aligned(16))) half Bs[2][128 * TK];   // rows of the output (second operand): hi, lo
  __shared__ __attribute__((aligned(16))) half As[2][128 * TK];   // columns of the output (first operand)
  int gi = 0, id = blockIdx.x, per = 0;
  for (;; ++gi) {                                          // group of this tile
    if (gi == p.ngroups) return;
    const int tm = (p.g[gi].m + 127) / 128, tn = (p.g[gi].ldn + 127) / 128;
    per = STEP == 2 ? tm * tn : tm * (tm + 1) / 2;
    if (id < per * p.g[gi].count) break;
    id -= per * p.g[gi].count;
  }
  const OrthoG& g = p.g[gi];
  const int mat = id / per, tl = id % per;
  int ti, tj;
  if (STEP == 2) { const int tm = (g.m + 127) / 128; ti = tl % tm; tj = tl / tm; }
  else {
    ti = (int)((sqrtf(8.f * tl + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > tl) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= tl) ++ti;
    tj = tl - ti * (ti + 1) / 2;
  }
  const int ld = STEP == 0 ? g.ldn : g.ldm;                // contraction length
  const half* bh = STEP == 0 ? plane_x(p, g, mat, cur) : plane_a(p, g, mat, STEP == 1 ? 0 : 2);
  const half* bl = STEP == 0 ? plane_x(p, g, mat, cur + 1) : plane_a(p, g, mat, STEP == 1 ? 1 : 3);
  const half* ah = STEP == 2 ? plane_x(p, g, mat, cur) : bh;
  const half* al = STEP == 2 ? plane_x(p, g, mat, cur + 1) : bl;
  constexpr bool BLO = FULL || STEP == 1, ALO = FULL || STEP != 0;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5;
  const int r0 = ti * 128, c0 = tj * 128;

  uint4 vb[2][2], va[2][2];
  auto load = [&](int k0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int q = i * 256 + (int)threadIdx.x;
      const uint4 z = make_uint4(0u, 0u, 0u, 0u);
      { const int r = r0 + q / 4, c = k0 + 8 * (q & 3);
        const long long o = (long long)r * ld + c;
        vb[0][i] = r < g.m ? *reinterpret_cast<const uint4*>(bh + o) : z;
        if (BLO) vb[1][i] = r < g.m ? *reinterpret_cast<const uint4*>(bl + o) : z; }
      if (STEP != 2) {
        const int r = c0 + q / 4, c = k0 + 8 * (q & 3);
        const long long o = (long long)r * ld + c;
        va[0][i] = r < g.m ? *reinterpret_cast<const uint4*>(ah + o) : z;
        if (ALO) va[1][i] = r < g.m ? *reinterpret_cast<const uint4*>(al + o) : z;
      } else {
        const int r = k0 + q / 16, c = c0 + 8 * (q & 15);
        const long long o = (long long)r * g.ldn + c;
        const bool ok = r < g.m && c < g.ldn;
        va[0][i] = ok ? *reinterpret_cast<const uint4*>(ah + o) : z;
        if (ALO) va[1][i] = ok ? *reinterpret_cast<const uint4*>(al + o) : z;
      }
    }
  };
  auto store = [&]() {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int q = i * 256 + (int)threadIdx.x;
      *reinterpret_cast<uint4*>(Bs[0] + LR::at(q / 4, q & 3)) = vb[0][i];
      if (BLO) *reinterpret_cast<uint4*>(Bs[1] + LR::at(q / 4, q & 3)) = vb[1][i];
      const int o = STEP != 2 ? LR::at(q / 4, q & 3) : LC::at(q / 16, q & 15);
      *reinterpret_cast<uint4*>(As[0] + o) = va[0][i];
      if (ALO) *reinterpret_cast<uint4*>(As[1] + o) = va[1][i];
    }
  };
  // second operand in contraction order 16 s + 8 h + 0 .. 7, as row_frag gives it
  auto col = [&](const half* t, int s, int ct) {
    const int i = lane & 15, row = 16 * s + 8 * h + (i >> 2), ch = ct + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
    s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS3 s16x4*)(t + LC::at(row, ch / 8) + (ch & 7)));
    s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS3 s16x4*)(t + LC::at(row + 4, ch / 8) + (ch & 7)));
    s16x8 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
    return __builtin_bit_cast(h16x8, v);
  };
  const int wr = 64 * (w >> 1), wc = 64 * (w & 1);
  f32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  load(0);
  for (int k0 = 0; k0 < ld; k0 += TK) {
    __syncthreads();
    store();
    __syncthreads();
    if (k0 + TK < ld) load(k0 + TK);
#pragma unroll
    for (int s = 0; s < TK / 16; ++s) {
      h16x8 b0[2], b1[2], a0[2], a1[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        b0[i] = LR::row_frag(Bs[0], wr + 32 * i, s, lane);
        if (BLO) b1[i] = LR::row_frag(Bs[1], wr + 32 * i, s, lane);
        a0[i] = STEP != 2 ? LR::row_frag(As[0], wc + 32 * i, s, lane) : col(As[0], s, wc + 32 * i);
        if (ALO) a1[i] = STEP != 2 ? LR::row_frag(As[1], wc + 32 * i, s, lane) : col(As[1], s, wc + 32 * i);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          acc[i][j] = O::mma(a0[j], b0[i], acc[i][j]);
          if (ALO) acc[i][j] = O::mma(a1[j], b0[i], acc[i][j]);
          if (BLO) acc[i][j] = O::mma(a0[j], b1[i], acc[i][j]);
        }
    }
  }
  const bool mirror = STEP != 2 && ti != tj;
  half *oh, *ol;
  if (STEP == 0) { oh = plane_a(p, g, mat, 0); ol = plane_a(p, g, mat, 1); }
  else if (STEP == 1) { oh = plane_a(p, g, mat, 2); ol = plane_a(p, g, mat, 3); }
  else { oh = plane_x(p, g, mat, 2 - cur); ol = plane_x(p, g, mat, 3 - cur); }
  const int lo_out = STEP == 2 ? g.ldn : g.ldm;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = r0 + wr + 32 * i + (lane & 31), c = c0 + wc + 32 * j + 8 * q + 4 * h;
        // rows behind the matrix are zero: their mirror images fill the columns up to ldm
        if (r >= (STEP == 2 ? g.m : g.ldm) || c >= lo_out) continue;
        const bool in = r < g.m;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e];
        if (STEP == 0) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] *= SA / (SX * SX);
        } else if (STEP == 1 && in) {
          const h16x4 xh = *reinterpret_cast<const h16x4*>(bh + (long long)r * g.ldm + c);
          const h16x4 xl = *reinterpret_cast<const h16x4*>(bl + (long long)r * g.ldm + c);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            v[e] = __builtin_fmaf(cc / SA, v[e], cb * ((float)xh[e] + (float)xl[e])) + (FULL && r == c + e ? ca * SA : 0.f);
        } else if (STEP == 2) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] *= 1.f / SA;
          if (!FULL) {
            const h16x4 xh = *reinterpret_cast<const h16x4*>(ah + (long long)r * g.ldn + c);
            const h16x4 xl = *reinterpret_cast<const h16x4*>(al + (long long)r * g.ldn + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(ca, (float)xh[e] + (float)xl[e], v[e]);
          }
        }
        if (STEP == 2 && last) {
          T* y = (T*)g.y + (long long)mat * g.ym;
          const bool tall = g.rows > g.cols;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < g.n) y[tall ? (long long)(c + e) * g.yr + r : (long long)r * g.yr + c + e] = (T)(v[e] * (1.f / SX));
          continue;
        }
        h16x4 vh, vl;
#pragma unroll
        for (int e = 0; e < 4; ++e) { half a, b; split2(v[e], a, b); vh[e] = a; vl[e] = b; }
        if (in) {
          *reinterpret_cast<h16x4*>(oh + (long long)r * lo_out + c) = vh;
          *reinterpret_cast<h16x4*>(ol + (long long)r * lo_out + c) = vl;
        }
        if (mirror) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c + e < g.m) { oh[(long long)(c + e) * lo_out + r] = vh[e]; ol[(long long)(c + e) * lo_out + r] = vl[e]; }
        }
      }
}

template <typename T, bool FULL> int run(const OrthoP& p, int steps, const float* coef, hipStream_t st) {
  int load_tiles = 0;
  long long sym = 0, full = 0;
  for (int i = 0; i < p.ngroups; ++i) {
    const OrthoG& g = p.g[i];
    const int t = g.ldn / 64 * (g.ldm / 64), tm = (g.m + 127) / 128, tn = (g.ldn + 127) / 128;
    if (t > load_tiles) load_tiles = t;
    sym += (long long)g.count * tm * (tm + 1) / 2;
    full += (long long)g.count * tm * tn;
  }
  ortho_sumsq<T><<<dim3(p.matrices, ORTHO_PARTS), 256, 0, st>>>(p);
  ortho_load<T><<<dim3(load_tiles, p.matrices), 256, 0, st>>>(p);
  for (int s = 0; s < steps; ++s) {
    const int cur = 2 * (s & 1), last = s == steps - 1;
    const float a = coef[3 * s], b = coef[3 * s + 1], c = coef[3 * s + 2];
    ortho_product<T, 0, FULL><<<dim3((unsigned)sym), 256, 0, st>>>(p, cur, 0, a, b, c);
    ortho_product<T, 1, FULL><<<dim3((unsigned)sym), 256, 0, st>>>(p, cur, 0, a, b, c);
    ortho_product<T, 2, FULL><<<dim3((unsigned)full), 256, 0, st>>>(p, cur, last, a, b, c);
  }
  return hipGetLastError() != hipSuccess;
}

}  // namespace

size_t ortho_ws_bytes(OrthoP& p) {
  long long at = 0;
  for (int i = 0; i < p.ngroups; ++i) {
    p.g[i].ws = at;
    at += (long long)p.g[i].count * (4LL * p.g[i].m * p.g[i].ldn + 4LL * p.g[i].m * p.g[i].ldm);
  }
  return (size_t)at * 2 + (size_t)p.matrices * ORTHO_PARTS * sizeof(double) + 256;
}

int launch_ortho(const OrthoP& p, int dtype, int steps, const float* coef, hipStream_t st) {
  return dtype == OP_F32 ? run<float, true>(p, steps, coef, st)
                         : dtype == OP_BF16 ? run<__bf16, false>(p, steps, coef, st) : run<half, true>(p, steps, coef, st);
}
