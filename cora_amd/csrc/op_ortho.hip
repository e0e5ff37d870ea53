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
// For bf16 results of large matrices the products with X take one instruction: A from the upper halves of X, and B X with
// the upper halves of X and of B = b A + c A^2, while a X is added in fp32 from both halves, so that what the iteration
// amplifies most is never rounded to 11 bits; A^2 keeps all three, since at singular values near 1 its errors are
// amplified.  The result is then 1.1e-3 (rms) off the exact iterates before its own rounding of 1.7e-3; with A^2 from upper
// halves too it is 2e-3, and with X itself in 11 bits 2.5e-3.
#include "op_tile.h"
#include "ops.h"

#include <atomic>

namespace {

typedef _Float16 half;
typedef half h16x4 __attribute__((ext_vector_type(4)));
constexpr float SX = 4096.f, SA = 64.f;

// workspace of one matrix, in halves: X hi, X lo, Y hi, Y lo (m rows of stride sn each), A hi, A lo, P hi, P lo (stride sm).
// Strides are odd multiples of 128 bytes: with a power of two the rows of a tile all lie in one channel of the L2 cache.
__device__ __forceinline__ half* plane_x(const OrthoP& p, const OrthoG& g, int mat, int which) {
  return (half*)p.ws + g.ws + (long long)mat * (4LL * g.m * (g.sn + g.sm)) + (long long)which * g.m * g.sn;
}
__device__ __forceinline__ half* plane_a(const OrthoP& p, const OrthoG& g, int mat, int which) {
  return plane_x(p, g, mat, 4) + (long long)which * g.m * g.sm;
}

__device__ __forceinline__ void split2(float v, half& hi, half& lo) { hi = (half)v; lo = (half)(v - (float)hi); }

// partial sums of squares in 64 bits: part z of a matrix takes every ORTHO_PARTS-th run of 256 vectors
template <typename T>
__global__ __launch_bounds__(256) void ortho_sumsq(const OrthoP p) {
  constexpr int V = 16 / (int)sizeof(T);
  typedef T vec __attribute__((ext_vector_type(V)));
  __shared__ double sh[4];
  const int id = blockIdx.x, part = blockIdx.y;
  int gi = 0;
  while (gi + 1 < p.ngroups && id >= p.g[gi + 1].first) ++gi;
  const OrthoG& g = p.g[gi];
  const T* x = (const T*)g.x + (long long)(id - g.first) * g.xm;
  const unsigned cols = g.cols, total = (unsigned)g.rows * cols;      // at most 2^30
  const long long xr = g.xr;
  const bool packed = xr == cols;
  double s = 0.0;
  if ((uintptr_t)x % 16 == 0 && xr % V == 0 && cols % V == 0) {
#pragma unroll 4
    for (unsigned e = (part * 256 + threadIdx.x) * V; e < total; e += ORTHO_PARTS * 256 * V) {
      const unsigned r = packed ? 0 : e / cols, c = packed ? e : e - r * cols;
      const vec v = *reinterpret_cast<const vec*>(x + r * xr + c);
#pragma unroll
      for (int i = 0; i < V; ++i) s += (double)(float)v[i] * (double)(float)v[i];
    }
  } else
#pragma unroll 4
    for (unsigned e = part * 256 + threadIdx.x; e < total; e += ORTHO_PARTS * 256) {
      const unsigned r = e / cols, c = e - r * cols;
      const double v = (double)(float)x[r * xr + c];
      s += v * v;
    }
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
#pragma unroll
  for (int i = 0; i < ORTHO_PARTS / 64; ++i) s += p.parts[(long long)id * ORTHO_PARTS + 64 * i + (threadIdx.x & 63)];
  s = wave_sum_d(s);
  const double f = (double)SX / (sqrt(s) + (double)p.eps);
  const bool tall = g.rows > g.cols;
  const T* x = (const T*)g.x + (long long)mat * g.xm;
  const int a = threadIdx.x & 63, b = threadIdx.x >> 6;
#pragma unroll 4
  for (int k = b; k < 64; k += 4) {                       // source rows along b
    const int r = (tall ? j0 : i0) + k, c = (tall ? i0 : j0) + a;
    const float v = r < g.rows && c < g.cols ? (float)((double)(float)x[(long long)r * g.xr + c] * f) : 0.f;
    if (tall) t[a][k] = v; else t[k][a] = v;
  }
  __syncthreads();
  half* hi = plane_x(p, g, mat, 0); half* lo = plane_x(p, g, mat, 1);
#pragma unroll
  for (int k = threadIdx.x >> 4; k < 64; k += 16)
    if (i0 + k < g.m) {
      h16x4 vh, vl;
#pragma unroll
      for (int e = 0; e < 4; ++e) { half u, v; split2(t[k][4 * (threadIdx.x & 15) + e], u, v); vh[e] = u; vl[e] = v; }
      const long long o = (long long)(i0 + k) * g.sn + j0 + 4 * (threadIdx.x & 15);
      *reinterpret_cast<h16x4*>(hi + o) = vh;
      *reinterpret_cast<h16x4*>(lo + o) = vl;
    }
}

// ---- matrices that fit one compute unit's LDS ----------------------------------------------------
// All steps of one matrix in one workgroup of 8 waves: X, then A and P in A's place, as two fp16 planes each in LDS; 32 x 32
// tiles, three instructions a product for every type.  What a step costs is the chain of its three products, the splitting
// of their results into halves and 5 barriers: 2.5 us at 64 x 64, 4.4 at 64 x 256, 9.7 at 128 x 128 (16 x 16 tiles on 16 waves:
// 2.4, 4.9, 14).  Against the tiled path this saves 2 + 3 steps launches: the 6-block model's 36 updates 38 us instead of 156.
// Rows are padded to a stride of 80 bytes mod 256 (the 16 rows of a row read start 16 bytes apart mod 256, the 4 rows of a
// transposing read 80 apart) or, where that does not fit, to 16 mod 256.
constexpr int SMALL_LDS = 160 * 1024 - 256;
struct SmallDim { int mp, np, sx, sa, bytes; };           // padded sizes, row strides in halves, LDS bytes
__host__ __device__ constexpr SmallDim small_dim(int m, int n) {
  SmallDim d = {};
  d.mp = (m + 31) / 32 * 32; d.np = (n + 31) / 32 * 32;
  for (int want = 80; want >= 16; want -= 64) {
    d.sx = d.np + ((want - 2 * d.np) & 255) / 2; d.sa = d.mp + ((want - 2 * d.mp) & 255) / 2;
    d.bytes = 4 * d.mp * (d.sx + d.sa);
    if (d.bytes <= SMALL_LDS) break;
  }
  return d;
}
static_assert(small_dim(97, 128).bytes <= SMALL_LDS && small_dim(97, 129).bytes > SMALL_LDS, "4 row tiles: never more than 16 tiles of X");

// the steps, for matrices of RT row tiles and X of at most 8 XT tiles
template <int RT, int XT>
__device__ __forceinline__ void small_steps(half* lds, const SmallDim d, const OrthoCoef& co) {
  constexpr int MP = 32 * RT, NZ = (RT * RT + 7) / 8;      // tiles of A per wave
  typedef Op<half> O;
  const int np = d.np, sx = d.sx, sa = d.sa, units = np / 32 * RT;
  half *xh = lds, *xl = xh + MP * sx, *ah = xl + MP * sx, *al = ah + MP * sa;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r32 = lane & 31, h = lane >> 5;
  // 32 x 16 operand pieces: lane holds index l & 31, contraction 8 (l >> 5) + 0 .. 7
  auto row = [&](const half* t, int stride, int i0, int k0) {
    return *reinterpret_cast<const h16x8*>(t + (i0 + r32) * stride + k0 + 8 * h);
  };
  auto col = [&](const half* t, int k0, int j0) {
    const int i = lane & 15;
    const half* q = t + (k0 + 8 * h + (i >> 2)) * sx + j0 + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
    s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS3 s16x4*)q);
    s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS3 s16x4*)(q + 4 * sx));
    s16x8 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
    return __builtin_bit_cast(h16x8, v);
  };
  auto zero = [](f32x16& v) {
#pragma unroll
    for (int r = 0; r < 16; ++r) v[r] = 0.f;
  };
  // hi hi + (hi lo + lo hi) over `len` values (a multiple of 32) of the contraction; the operands of the next 32 are under way
  // while the current ones are multiplied.  The small products have a sum of their own: the large one then takes a third of
  // the roundings (16 x 1000, 3 steps: error 7.2e-7 -> 4.6e-7).
  auto product = [&](f32x16& acc, int len, auto first, auto second) {
    f32x16 rest;
    zero(acc); zero(rest);
    h16x8 a[4], b[4];
    auto get = [&](h16x8 (&p)[4], h16x8 (&q)[4], int k) {
#pragma unroll
      for (int e = 0; e < 4; ++e) { p[e] = first(e & 1, k + 16 * (e >> 1)); q[e] = second(e & 1, k + 16 * (e >> 1)); }
    };
    get(a, b, 0);
#pragma unroll 1
    for (int k = 32; k <= len; k += 32) {
      h16x8 an[4], bn[4];
      get(an, bn, k < len ? k : 0);
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        acc = O::mma(a[e], b[e], acc); rest = O::mma(a[e + 1], b[e], rest); rest = O::mma(a[e], b[e + 1], rest);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) { a[e] = an[e]; b[e] = bn[e]; }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[r] += rest[r];
  };
  // a lane's four times four columns of its row, times f, split
  auto put = [&](half* hi, half* lo, int o, const f32x16& v, float f) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      h16x4 vh, vl;
#pragma unroll
      for (int e = 0; e < 4; ++e) { half a, b; split2(v[4 * q + e] * f, a, b); vh[e] = a; vl[e] = b; }
      *reinterpret_cast<h16x4*>(hi + o + 8 * q) = vh;
      *reinterpret_cast<h16x4*>(lo + o + 8 * q) = vl;
    }
  };
  for (int step = 0; step < co.steps; ++step) {
    const float ca = co.c[3 * step], cb = co.c[3 * step + 1], cc = co.c[3 * step + 2];
    f32x16 pt[NZ];
    __syncthreads();
#pragma unroll
    for (int z = 0; z < NZ; ++z) {                         // A = X X^T
      const int t = w + 8 * z, i = 32 * (t / RT), j = 32 * (t % RT);
      if (t >= RT * RT) continue;
      product(pt[z], np, [&](int lo, int k) { return row(lo ? xl : xh, sx, j, k); }, [&](int lo, int k) { return row(lo ? xl : xh, sx, i, k); });
      put(ah, al, (i + r32) * sa + j + 4 * h, pt[z], SA / (SX * SX));
    }
    __syncthreads();
#pragma unroll
    for (int z = 0; z < NZ; ++z) {                         // P = a I + b A + c A A
      const int t = w + 8 * z, i = 32 * (t / RT), j = 32 * (t % RT);
      if (t >= RT * RT) continue;
      product(pt[z], MP, [&](int lo, int k) { return row(lo ? al : ah, sa, j, k); }, [&](int lo, int k) { return row(lo ? al : ah, sa, i, k); });
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = i + r32, c = j + 8 * q + 4 * h;
        const h16x4 vh = *reinterpret_cast<const h16x4*>(ah + r * sa + c), vl = *reinterpret_cast<const h16x4*>(al + r * sa + c);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          pt[z][4 * q + e] = __builtin_fmaf(cc / SA, pt[z][4 * q + e], cb * ((float)vh[e] + (float)vl[e])) + (r == c + e ? ca * SA : 0.f);
      }
    }
    __syncthreads();
#pragma unroll
    for (int z = 0; z < NZ; ++z) {
      const int t = w + 8 * z, i = 32 * (t / RT), j = 32 * (t % RT);
      if (t < RT * RT) put(ah, al, (i + r32) * sa + j + 4 * h, pt[z], 1.f);
    }
    __syncthreads();
    f32x16 xt[XT];
#pragma unroll
    for (int z = 0; z < XT; ++z) {                         // X <- P X: row tile u % RT of columns 32 (u / RT) ..
      const int u = w + 8 * z, i = 32 * (u % RT), j = 32 * (u / RT);
      if (u >= units) continue;
      product(xt[z], MP, [&](int lo, int k) { return col(lo ? xl : xh, k, j); }, [&](int lo, int k) { return row(lo ? al : ah, sa, i, k); });
    }
    __syncthreads();                                       // X has been read
#pragma unroll
    for (int z = 0; z < XT; ++z) {
      const int u = w + 8 * z;
      if (u < units) put(xh, xl, (32 * (u % RT) + r32) * sx + 32 * (u / RT) + 4 * h, xt[z], 1.f / SA);
    }
  }
}

template <typename T, int RT, int XT>
__global__ __launch_bounds__(512) void ortho_small(const OrthoP p, const OrthoCoef co) {
  extern __shared__ __attribute__((aligned(16))) half lds[];
  __shared__ double red[8];
  const int id = blockIdx.x;
  int gi = 0;
  while (gi + 1 < p.ngroups && id >= p.g[gi + 1].first) ++gi;
  const OrthoG& g = p.g[gi];
  const SmallDim d = small_dim(g.m, g.n);
  const int rows = g.rows, cols = g.cols, sx = d.sx, tid = threadIdx.x;
  const bool tall = rows > cols;
  const T* x = (const T*)g.x + (long long)(id - g.first) * g.xm;
  const long long xr = g.xr;
  unsigned short *xh = (unsigned short*)lds, *xl = xh + d.mp * sx;

  // The matrix goes to its place with its bits halved between the planes and is scaled and split there once its norm is
  // known.  Loops are kept short: a workgroup lives for some 10 us and fetches its code cold.
  for (int i = tid; i < d.mp * sx / 4; i += 512) reinterpret_cast<uint4*>(lds)[i] = make_uint4(0u, 0u, 0u, 0u);   // both planes
  __syncthreads();
  // four neighbouring elements a lane where rows allow it, else one; eight of them under way at a time
  double s = 0.0;
  typedef T vec4 __attribute__((ext_vector_type(4)));
  const bool wide = cols % 4 == 0 && xr % 4 == 0 && (uintptr_t)x % sizeof(vec4) == 0;
  const int per = wide ? 4 : 1, cv = cols / per;           // vectors a row
  const int dr = 512 / cv, dc = 512 - dr * cv;             // vector tid + 512 i: its row and column step by these
  int r = tid / cv, c = tid - r * cv;
  while (r < rows) {
    float v[8][4]; int o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o[i] = -1;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = 0.f;
      if (r < rows) {
        if (wide) {
          const vec4 t = *reinterpret_cast<const vec4*>(x + r * xr + 4 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[i][e] = (float)t[e];
        } else v[i][0] = (float)x[r * xr + c];
        o[i] = tall ? per * c * sx + r : r * sx + per * c;
      }
      r += dr; c += dc;
      if (c >= cv) { c -= cv; ++r; }
    }
    const int de = tall ? sx : 1;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s += (double)v[i][e] * (double)v[i][e];
        if (o[i] >= 0 && e < per) {
          const unsigned u = __float_as_uint(v[i][e]);
          xh[o[i] + e * de] = (unsigned short)(u >> 16); xl[o[i] + e * de] = (unsigned short)u;
        }
      }
  }
  s = wave_sum_d(s);
  if ((tid & 63) == 0) red[tid >> 6] = s;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += red[i];
  const double f = (double)SX / (sqrt(s) + (double)p.eps);
  for (int i = tid; i < d.mp * sx / 4; i += 512) {
    const ushort4 uh = reinterpret_cast<ushort4*>(xh)[i], ul = reinterpret_cast<ushort4*>(xl)[i];
    const unsigned u[4] = {(unsigned)uh.x << 16 | ul.x, (unsigned)uh.y << 16 | ul.y, (unsigned)uh.z << 16 | ul.z, (unsigned)uh.w << 16 | ul.w};
    h16x4 vh, vl;
#pragma unroll
    for (int e = 0; e < 4; ++e) { half a, b; split2((float)((double)__uint_as_float(u[e]) * f), a, b); vh[e] = a; vl[e] = b; }
    reinterpret_cast<h16x4*>(xh)[i] = vh; reinterpret_cast<h16x4*>(xl)[i] = vl;
  }
  small_steps<RT, XT>(lds, d, co);
  __syncthreads();
  T* y = (T*)g.y + (long long)(id - g.first) * g.ym;
  const long long yr = g.yr;
  const int er = 512 / cols, ec = 512 - er * cols;
  r = tid / cols; c = tid - r * cols;
  while (r < rows) {
    const int o = tall ? c * sx + r : r * sx + c;
    y[r * yr + c] = (T)(((float)lds[o] + (float)lds[d.mp * sx + o]) * (1.f / SX));
    r += er; c += ec;
    if (c >= cols) { c -= cols; ++r; }
  }
}

// One product for all matrices.  STEP 0: A = X X^T; 1: P = a I + b A + c A A; 2: X' = P X (last: to the caller's
// matrix). Tile TS x TS: 64 with four waves of 32 x 32, for matrices that give few tiles; 128 with four waves of 64 x
// 64, two workgroups a compute unit (the symmetric products of few wide matrices); or 256 with eight waves of 128 x 64,
// which halves what a flop reads from L2 (the 128 tile's 43 bytes a cycle and compute unit exceed it).  The first
// operand gives the output's columns, the second its rows (op_tile.h), so a lane holds four neighbouring columns of one
// output row.  Slabs go from global memory straight into one of two LDS buffers while the other is worked on; a lane
// fetches the 16-byte piece that belongs at its place of the swizzled tile.  Rows outside a matrix arrive as zeros,
// columns behind it as whatever follows (the columns up to ldn and ldm are stored as zeros, what lies behind gives
// nothing that is stored).
constexpr int threads_of(int ts) { return ts == 256 ? 512 : 256; }
template <typename T, int STEP, bool FULL, int TS>
__global__ __launch_bounds__(threads_of(TS), 2) void ortho_product(const OrthoP p, const int cuts, const int cur, const int last, const float ca, const float cb, const float cc) {
  constexpr bool LO = FULL || STEP == 1;                  // both halves of both operands
  constexpr int NPL = LO ? 4 : 2, PB1 = 1, PA0 = LO ? 2 : 1, PA1 = LO ? 3 : 0;    // planes: B hi, (B lo,) A hi, (A lo)
  constexpr int TK = LO && TS > 64 ? 32 : 64, NW = threads_of(TS) / 64, NI = TS * TK / 512 / NW;   // slab, waves, requests of a wave and plane
  constexpr int NB = TS / 64, NA = TS / (NW / 2) / 32, CW = 32 * NA;       // row and column tiles of a wave, its columns
  typedef Tile<half, TK> LR; typedef Tile<half, TS> LC;
  typedef Op<half> O;
  __shared__ __attribute__((aligned(16))) half buf0[NPL][TS * TK];
  __shared__ __attribute__((aligned(16))) half buf1[NPL][TS * TK];
  // Workgroups go round robin over the 8 XCDs; each matrix' tiles are cut into `cuts` runs and the runs dealt to the XCDs, so
  // that the tiles that read the same rows share one XCD's L2.
  const int xcd = blockIdx.x & 7;
  int gi = 0, k = blockIdx.x >> 3, per, run, mat, tl;
  for (;; ++gi) {
    if (gi == p.ngroups) return;
    const int tm = (p.g[gi].m + TS - 1) / TS, tn = (p.g[gi].ldn + TS - 1) / TS;
    per = STEP == 2 ? tm * tn : tm * (tm + 1) / 2;
    run = (per + cuts - 1) / cuts;
    const int off = (xcd - p.g[gi].first * cuts) & 7, have = (p.g[gi].count * cuts - off + 7) >> 3;
    if (k < have * run) {
      const int unit = off + 8 * (k / run);
      mat = unit / cuts;
      tl = unit % cuts * run + k % run;
      break;
    }
    k -= max(have, 0) * run;
  }
  if (tl >= per) return;
  const OrthoG& g = p.g[gi];
  const int m = g.m, ldn = g.ldn, ldm = g.ldm, sn = g.sn, sm = g.sm;
  int ti, tj;
  if (STEP == 2) { const int tm = (m + TS - 1) / TS; ti = tl % tm; tj = tl / tm; }
  else {
    ti = (int)((sqrtf(8.f * tl + 1.f) - 1.f) * 0.5f);
    while (ti * (ti + 1) / 2 > tl) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= tl) ++ti;
    tj = tl - ti * (ti + 1) / 2;
  }
  const int ld = STEP == 0 ? ldn : ldm, sk = STEP == 0 ? sn : sm;   // contraction length, stride of the planes along it
  const half* bh = STEP == 0 ? plane_x(p, g, mat, cur) : plane_a(p, g, mat, STEP == 1 ? 0 : 2);
  const half* bl = STEP == 0 ? plane_x(p, g, mat, cur + 1) : plane_a(p, g, mat, STEP == 1 ? 1 : 3);
  const half* ah = STEP == 2 ? plane_x(p, g, mat, cur) : bh;
  const half* al = STEP == 2 ? plane_x(p, g, mat, cur + 1) : bl;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int r0 = ti * TS, c0 = tj * TS;

  // wave w fills chunks w, w + NW, .. (64 pieces each) of every plane.  A lane's piece is at a constant offset; the slab's
  // start goes into the descriptor (64-bit pointers kept for every request cost the 256 tile its accumulators' registers).
  int at[2][NI];                                           // B, A
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int q = (NW * i + w) * 64 + lane, r = q / (TK / 8), c = (q % (TK / 8)) ^ LR::swz(r);
    at[0][i] = (int)(2u * ((unsigned)(r0 + r) * sk + 8 * c));       // planes have less than 2^32 bytes
    at[1][i] = (int)(2u * ((unsigned)(c0 + r) * sk + 8 * c));
    if (STEP == 2) {
      const int rk = q / (TS / 8), ck = c0 + 8 * ((q % (TS / 8)) ^ LC::swz(rk));
      at[1][i] = 2 * (rk * sn + ck);
    }
  }
  auto fetch = [&](half (&dst)[NPL][TS * TK], int k0) {
#pragma unroll
    for (int pl = 0; pl < NPL; ++pl) {
      [[maybe_unused]] const half* base = pl == 0 ? bh : (LO && pl == PB1) ? bl : pl == PA0 ? ah : al;
      const long long from = STEP == 2 && pl >= PA0 ? (long long)k0 * sn : k0;
      [[maybe_unused]] const long long bytes = 2 * ((STEP == 2 && pl >= PA0 ? (long long)m * sn : (long long)m * sk) - from);
#pragma unroll
      for (int i = 0; i < NI; ++i)
        REQUEST(base + from, k0 < ld && bytes > 0 ? (int)(unsigned)bytes : 0, dst[pl] + (NW * i + w) * 512, 16, at[pl >= PA0][i]);
    }
    __builtin_amdgcn_sched_barrier(0);                     // the requests leave before the work on the other buffer starts
  };
  // first operand from a tile of contraction rows x columns, in contraction order 16 s + 8 h + 0 .. 7 as row_frag gives it
  auto col = [&](const half* t, int s, int ct) {
    const int i = lane & 15, row = 16 * s + 8 * h + (i >> 2), ch = ct + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
    s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS3 s16x4*)(t + LC::at(row, ch / 8) + (ch & 7)));
    s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS3 s16x4*)(t + LC::at(row + 4, ch / 8) + (ch & 7)));
    s16x8 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
    return __builtin_bit_cast(h16x8, v);
  };
  const int wr = (TS / 2) * (w / (NW / 2)), wc = CW * (w % (NW / 2));
  f32x16 acc[NB][NA];
#pragma unroll
  for (int i = 0; i < NB; ++i)
#pragma unroll
    for (int j = 0; j < NA; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  // The 64 tile sums 512 products at a time: a matrix of few rows has long ones (8 x 3000, 5 steps: error 2.3e-6 -> 9e-7), and
  // there the 16 registers are free.
  constexpr bool PARTS = TS == 64;
  static_assert(!PARTS || NA * NB == 1, "one tile a wave");
  [[maybe_unused]] f32x16 total;
#pragma unroll
  for (int r = 0; r < 16; ++r) total[r] = 0.f;
  auto bank = [&] {
#pragma unroll
    for (int r = 0; r < 16; ++r) { total[r] += acc[0][0][r]; acc[0][0][r] = 0.f; }
  };
  auto work = [&](half (&t)[NPL][TS * TK]) {
#pragma unroll
    for (int s = 0; s < TK / 16; ++s) {
      h16x8 a0[NA], a1[NA], b0 = LR::row_frag(t[0], wr, s, lane), b1 = LO ? LR::row_frag(t[PB1], wr, s, lane) : b0;
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        a0[i] = STEP != 2 ? LR::row_frag(t[PA0], wc + 32 * i, s, lane) : col(t[PA0], s, wc + 32 * i);
        if (LO) a1[i] = STEP != 2 ? LR::row_frag(t[PA1], wc + 32 * i, s, lane) : col(t[PA1], s, wc + 32 * i);
      }
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const h16x8 c0 = b0, c1 = b1;
        if (i + 1 < NB) {
          b0 = LR::row_frag(t[0], wr + 32 * (i + 1), s, lane);
          if (LO) b1 = LR::row_frag(t[PB1], wr + 32 * (i + 1), s, lane);
        }
#pragma unroll
        for (int j = 0; j < NA; ++j) {
          acc[i][j] = O::mma(a0[j], c0, acc[i][j]);
          if (LO) acc[i][j] = O::mma(a1[j], c0, acc[i][j]);
          if (LO) acc[i][j] = O::mma(a0[j], c1, acc[i][j]);
        }
        if (TS == 256) __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  // two slabs a turn; an odd number ends with a slab of zeros (a second exit from the loop makes the compiler keep two
  // copies of the accumulators)
  const int slabs = ld / TK;                               // ld is a multiple of 64
  fetch(buf0, 0);
  for (int k = 0; k < slabs; k += 2) {
    arrive_barrier();                                      // buf0 has arrived, buf1 is no longer read
    fetch(buf1, (k + 1) * TK);
    work(buf0);
    arrive_barrier();
    if (k + 2 < slabs) fetch(buf0, (k + 2) * TK);
    work(buf1);
    if (PARTS && (k & 6) == 6) bank();
  }
  if (PARTS) { bank(); acc[0][0] = total; }
  // Epilogue, 32 rows x CW columns of a wave at a time through its own piece of LDS, so that every row is read and written as
  // whole 128-byte lines (stored as the matrix unit leaves them, 16 bytes a row and instruction, P X of the wide layers
  // took 404 us instead of 244).  Place of the four columns 4 k of row r: k ^ (r mod CW / 4).
  const bool mirror = STEP != 2 && ti != tj, tall = g.rows > g.cols;
  half *oh, *ol;
  if (STEP == 0) { oh = plane_a(p, g, mat, 0); ol = plane_a(p, g, mat, 1); }
  else if (STEP == 1) { oh = plane_a(p, g, mat, 2); ol = plane_a(p, g, mat, 3); }
  else { oh = plane_x(p, g, mat, 2 - cur); ol = plane_x(p, g, mat, 3 - cur); }
  const int cols = STEP == 2 ? ldn : ldm, so = STEP == 2 ? sn : sm;
  T* y = (T*)g.y + (long long)mat * g.ym;
  constexpr int VT = 16 / (int)sizeof(T);                  // 16-byte pieces of the caller's rows
  const bool vec = !tall && (uintptr_t)y % 16 == 0 && g.yr % VT == 0;
  static_assert(sizeof buf0 >= NW * CW * 128, "the first buffer holds every wave's piece");
  float* mine = reinterpret_cast<float*>(&buf0[0][0]) + w * (CW * 32);
  auto place = [&](int r, int c4) { return mine + r * CW + ((c4 ^ (r & (CW / 4 - 1))) << 2); };
  __syncthreads();                                         // the slabs are no longer read
#pragma unroll
  for (int i = 0; i < NB; ++i) {
#pragma unroll
    for (int j = 0; j < NA; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f32x4*>(place(lane & 31, 8 * j + 2 * q + h)) =
            f32x4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int z = 0; z < CW / 16; ++z) {
      const int lr = 512 / CW * z + lane / (CW / 8), k4 = 2 * (lane % (CW / 8));
      const int r = r0 + wr + 32 * i + lr, c = c0 + wc + 4 * k4;
      // A and P: rows behind the matrix are zero, their mirror images fill the columns up to ldm
      const bool in = r < m, some = r < (STEP == 2 ? m : ldm) && c < cols;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; e += 4) {
        const f32x4 f = *reinterpret_cast<const f32x4*>(place(lr, k4 + e / 4));
#pragma unroll
        for (int x = 0; x < 4; ++x) v[e + x] = in && (STEP == 2 || c + e + x < m) ? f[x] : 0.f;
      }
      if (STEP == 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= SA / (SX * SX);
      } else if (STEP == 1) {
        if (in && some) {
          const h16x8 xh = *reinterpret_cast<const h16x8*>(bh + (long long)r * sm + c);
          const h16x8 xl = *reinterpret_cast<const h16x8*>(bl + (long long)r * sm + c);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            v[e] = __builtin_fmaf(cc / SA, v[e], cb * ((float)xh[e] + (float)xl[e])) + (FULL && r == c + e ? ca * SA : 0.f);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= 1.f / SA;
        if (!FULL && some) {
          const h16x8 xh = *reinterpret_cast<const h16x8*>(ah + (long long)r * sn + c);
          const h16x8 xl = *reinterpret_cast<const h16x8*>(al + (long long)r * sn + c);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(ca, (float)xh[e] + (float)xl[e], v[e]);
        }
      }
      if ((STEP == 2 && last && tall) || mirror) {         // the transpose is read from LDS below
#pragma unroll
        for (int e = 0; e < 8; e += 4) *reinterpret_cast<f32x4*>(place(lr, k4 + e / 4)) = f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]};
      }
      if (!some || !in) continue;
      if (STEP == 2 && last) {
        if (tall) continue;
        T* row = y + (long long)r * g.yr + c;
        if (vec && c + 8 <= g.n) {
          typedef T vecT __attribute__((ext_vector_type(VT)));
#pragma unroll
          for (int e = 0; e < 8; e += VT) {
            vecT t;
#pragma unroll
            for (int x = 0; x < VT; ++x) t[x] = (T)(v[e + x] * (1.f / SX));
            *reinterpret_cast<vecT*>(row + e) = t;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < g.n) row[e] = (T)(v[e] * (1.f / SX));
        }
      } else {
        h16x8 vh, vl;
#pragma unroll
        for (int e = 0; e < 8; ++e) { half a, b; split2(v[e], a, b); vh[e] = a; vl[e] = b; }
        *reinterpret_cast<h16x8*>(oh + (long long)r * so + c) = vh;
        *reinterpret_cast<h16x8*>(ol + (long long)r * so + c) = vl;
      }
    }
    __builtin_amdgcn_wave_barrier();
    if ((STEP == 2 && last && tall) || mirror) {
      const int lr = lane & 31, r = r0 + wr + 32 * i + lr;
#pragma unroll 4
      for (int k = 0; k < CW / 2; ++k) {                   // two columns at a time, 32 rows each
        const int lc = 2 * k + h, c = c0 + wc + lc;
        const float v = place(lr, lc >> 2)[lc & 3];
        if (STEP == 2) {
          if (r < m && c < g.n) y[(long long)c * g.yr + r] = (T)(v * (1.f / SX));
        } else if (r < ldm && c < m) {
          half a, b;
          split2(v, a, b);
          oh[(long long)c * so + r] = a; ol[(long long)c * so + r] = b;
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// workgroups of a launch over `tiles(group)` tiles a matrix cut into `cuts` runs: the fullest XCD's, eight times
template <typename F> unsigned grid_of(const OrthoP& p, int cuts, F tiles) {
  long long most = 0;
  for (int x = 0; x < 8; ++x) {
    long long n = 0;
    for (int i = 0; i < p.ngroups; ++i) {
      const int per = tiles(p.g[i]), run = (per + cuts - 1) / cuts, off = (x - p.g[i].first * cuts) & 7;
      const long long have = ((long long)p.g[i].count * cuts - off + 7) >> 3;
      if (have > 0) n += have * run;
    }
    if (n > most) most = n;
  }
  return (unsigned)(8 * most);
}

// TS: tile of P X; the symmetric products, which have far fewer tiles, take 256 only where there are two per compute unit
template <typename T, bool FULL, int TS> int run_tiled(const OrthoP& p, int steps, const float* coef, hipStream_t st) {
  int load_tiles = 0, cuts = 1;
  for (int i = 0; i < p.ngroups; ++i) {
    const int t = p.g[i].ldn / 64 * (p.g[i].ldm / 64);
    if (t > load_tiles) load_tiles = t;
  }
  while (cuts < 8 && p.matrices * cuts < 64) cuts *= 2;
  auto sym = [&](int ts) { return grid_of(p, cuts, [=](const OrthoG& g) { const int tm = (g.m + ts - 1) / ts; return tm * (tm + 1) / 2; }); };
  const unsigned sym_ts = sym(TS), sym_128 = sym(128);
  const bool wide = TS == 64 || sym_ts >= 512;
  // P X of the 64 class: 128 where that still gives two workgroups a compute unit (36 x 384 x 384 and 12 x 384 x 1536: 37 us, 47 with 64)
  long long full_128 = 0;
  for (int i = 0; i < p.ngroups; ++i) full_128 += (long long)p.g[i].count * ((p.g[i].m + 127) / 128) * ((p.g[i].ldn + 127) / 128);
  auto full = [&](int ts) { return grid_of(p, cuts, [=](const OrthoG& g) { return (g.m + ts - 1) / ts * ((g.ldn + ts - 1) / ts); }); };
  ortho_sumsq<T><<<dim3(p.matrices, ORTHO_PARTS), 256, 0, st>>>(p);
  ortho_load<T><<<dim3(load_tiles, p.matrices), 256, 0, st>>>(p);
  for (int s = 0; s < steps; ++s) {
    const int cur = 2 * (s & 1), last = s == steps - 1;
    const float a = coef[3 * s], b = coef[3 * s + 1], c = coef[3 * s + 2];
    if (wide) {
      ortho_product<T, 0, FULL, TS><<<dim3(sym_ts), threads_of(TS), 0, st>>>(p, cuts, cur, 0, a, b, c);
      ortho_product<T, 1, FULL, TS><<<dim3(sym_ts), threads_of(TS), 0, st>>>(p, cuts, cur, 0, a, b, c);
    } else {
      ortho_product<T, 0, FULL, 128><<<dim3(sym_128), 256, 0, st>>>(p, cuts, cur, 0, a, b, c);
      ortho_product<T, 1, FULL, 128><<<dim3(sym_128), 256, 0, st>>>(p, cuts, cur, 0, a, b, c);
    }
    if (TS == 64 && full_128 >= 512) ortho_product<T, 2, FULL, 128><<<dim3(full(128)), 256, 0, st>>>(p, cuts, cur, last, a, b, c);
    else ortho_product<T, 2, FULL, TS><<<dim3(full(TS)), threads_of(TS), 0, st>>>(p, cuts, cur, last, a, b, c);
  }
  return hipGetLastError() != hipSuccess;
}

template <typename T, int RT, int XT> int run_small(const OrthoP& p, const OrthoCoef& co, hipStream_t st) {
  static std::atomic<unsigned long long> ready{0};          // devices; marked when done, as two threads may come here at once
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return 1;
  const unsigned long long bit = dev < 64 ? 1ULL << dev : 0;
  if (!(ready.load(std::memory_order_acquire) & bit)) {
    if (hipFuncSetAttribute((const void*)ortho_small<T, RT, XT>, hipFuncAttributeMaxDynamicSharedMemorySize, SMALL_LDS) != hipSuccess) return 1;
    ready.fetch_or(bit, std::memory_order_release);
  }
  int bytes = 0;
  for (int i = 0; i < p.ngroups; ++i) { const int b = small_dim(p.g[i].m, p.g[i].n).bytes; if (b > bytes) bytes = b; }
  ortho_small<T, RT, XT><<<dim3(p.matrices), 512, bytes, st>>>(p, co);
  return hipGetLastError() != hipSuccess;
}

// How a stack is worked on: in one workgroup with 1 to 4 row tiles of 32 (+ 8, up to 3 of them: more than 16 tiles of X), or with tiles:
// 64, or 256 for m >= 1024, and for bf16 results (+ 1) of m >= 256 with fewer instructions a product (below that it
// costs precision and saves nothing)
int class_of(const OrthoG& g, bool bf16) {
  if (ortho_is_small(g)) return (g.m + 31) / 32 + ((g.m + 31) / 32 * ((g.n + 31) / 32) > 16 ? 8 : 0);
  return (g.m >= 1024 ? 256 : 64) + (bf16 && g.m >= 256);
}
OrthoP only(const OrthoP& p, bool bf16, int cls) {
  OrthoP q = p;
  q.ngroups = 0; q.matrices = 0;
  for (int i = 0; i < p.ngroups; ++i)
    if (class_of(p.g[i], bf16) == cls) {
      q.g[q.ngroups] = p.g[i];
      q.g[q.ngroups++].first = q.matrices;
      q.matrices += p.g[i].count;
    }
  return q;
}

template <typename T> int run(const OrthoP& p, int steps, const float* coef, hipStream_t st) {
  constexpr bool BF16 = __is_same(T, __bf16);
  OrthoCoef co;
  co.steps = steps;
  for (int i = 0; i < 3 * steps; ++i) co.c[i] = coef[i];
  for (int cls : {256 + BF16, 64 + 1, 64, 8 + 3, 8 + 2, 8 + 1, 4, 3, 2, 1}) {
    const OrthoP q = only(p, BF16, cls);
    if (!q.ngroups) continue;
    // 256 tiles need half the compute units to have one: 5 steps of 2 x 2048 x 8192 fp32 in 5.0 ms with 64, 4.2 with 128, 4.0
    // with 256; of 1 x 2048 x 2048 868, 878, 1194 us; of 36 x 384 x 384 357, 375, 438 us; of 1 x 768 x 768 221, 401, 542 us
    long long wide = 0;
    for (int i = 0; i < q.ngroups; ++i) wide += (long long)q.g[i].count * ((q.g[i].m + 255) / 256) * ((q.g[i].n + 255) / 256);
    const int rc = cls >= 256 ? (wide >= 128 ? run_tiled<T, !BF16, 256>(q, steps, coef, st) : run_tiled<T, !BF16, 64>(q, steps, coef, st)) :
                   cls == 64 + 1 ? run_tiled<T, !BF16, 64>(q, steps, coef, st) : cls == 64 ? run_tiled<T, true, 64>(q, steps, coef, st) :
                   cls == 11 ? run_small<T, 3, 5>(q, co, st) :
                   cls == 10 ? run_small<T, 2, 5>(q, co, st) : cls == 9 ? run_small<T, 1, 5>(q, co, st) :
                   cls == 4 ? run_small<T, 4, 2>(q, co, st) : cls == 3 ? run_small<T, 3, 2>(q, co, st) :
                   cls == 2 ? run_small<T, 2, 2>(q, co, st) : run_small<T, 1, 2>(q, co, st);
    if (rc) return rc;
  }
  return 0;
}

}  // namespace

bool ortho_is_small(const OrthoG& g) { return g.m <= 128 && small_dim(g.m, g.n).bytes <= SMALL_LDS; }

size_t ortho_ws_bytes(OrthoP& p) {
  long long at = 0;
  for (int i = 0; i < p.ngroups; ++i) {
    p.g[i].ws = at;
    if (!ortho_is_small(p.g[i])) at += (long long)p.g[i].count * (4LL * p.g[i].m * (p.g[i].sn + p.g[i].sm));
  }
  return (size_t)at * 2 + (size_t)p.matrices * ORTHO_PARTS * sizeof(double) + 256;
}

int launch_ortho(const OrthoP& p, int dtype, int steps, const float* coef, hipStream_t st) {
  return dtype == OP_F32 ? run<float>(p, steps, coef, st) : dtype == OP_BF16 ? run<__bf16>(p, steps, coef, st) : run<half>(p, steps, coef, st);
}

// ---- orthogonalised momentum: what goes in and what comes out, one pass each, bound by memory -------
namespace {
__global__ __launch_bounds__(256) void muon_momentum_kernel(const MuonP p) {
  float cm = 1.f;                                          // clip_by_global_norm, as adamw_kernel
  if (p.clip > 0.f) {
    const double gn = sqrt(p.sumsq[0]);
    if (!(gn < (double)p.clip)) cm = (float)((double)p.clip / gn);
  }
  const float gmul = p.gscale * cm;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < p.n; i += (long long)gridDim.x * 256) {
    const float g = p.g[i] * gmul, m = __builtin_fmaf(p.beta, p.mu[i], g);
    p.mu[i] = m;
    p.u[i] = p.nesterov ? __builtin_fmaf(p.beta, m, g) : m;
  }
}
__global__ __launch_bounds__(256) void muon_apply_kernel(const MuonP p) {
  const float lr = p.hyp[0];
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < p.n; i += (long long)gridDim.x * 256) {
    const float w = p.w[i];
    p.w[i] = w - lr * (p.size * p.u[i] + p.wd * w);
  }
}
unsigned muon_blocks(long long n) { const long long b = (n + 255) / 256; return (unsigned)(b > 2048 ? 2048 : b); }
}  // namespace
void launch_muon_momentum(const MuonP& p, hipStream_t st) { muon_momentum_kernel<<<muon_blocks(p.n), 256, 0, st>>>(p); }
void launch_muon_apply(const MuonP& p, hipStream_t st) { muon_apply_kernel<<<muon_blocks(p.n), 256, 0, st>>>(p); }
