// op_rotary.hip -- rotary positions over several axes (time, height, width), forward and backward (gfx950).
//
// Axis a owns n_a consecutive channels of every head; its pair i (of n_a / 2) turns by the angle pos_a theta^(-2 i / n_a):
//   (u, v) -> (u cos - v sin, u sin + v cos)
// with u, v neighbours (interleaved) or n_a / 2 channels apart.  The map is orthogonal, so the backward pass is the same
// kernel with the opposite sign.  Channels behind the last axis pass through.
//
// The angle of a far position loses its fraction in 32 bits (position 1e6 times a frequency near 1 is off by 0.06), so
// turns = pos * (theta^(-2 i / n) / 2 pi) and the reduction to a quarter turn are done in 64 bits; sine and cosine of what
// is left, in [-pi/4, pi/4], are taken in 32.  A thread does this once for its channels of a row and then walks the heads,
// which share the angles: the kernel is bound by reading and writing x.  bf16, 3.4 GB in and out, packed rows: 690 us, the
// rate of a large copy (4.9 TB/s; with the passing channels in a loop of their own 1150 us).  fp32, 2 x 8 MB: 6 us.
#include "ops.h"

namespace {

// cos, sin of 2 pi turns
__device__ __forceinline__ void turn_cs(double turns, float sign, float& c, float& s) {
  const double t4 = 4.0 * turns, q = rint(t4);
  const float f = 0.5f * (float)(t4 - q);               // [-1/4, 1/4] half turns
  const int k = (int)(q - 4.0 * floor(0.25 * q));       // quarter turns mod 4, exact for any position
  float fs, fc;
  sincospif(f, &fs, &fc);
  const float a = (k & 1) ? fs : fc, b = (k & 1) ? fc : fs;
  c = (k == 1 || k == 2) ? -a : a;
  s = ((k >= 2) ? -b : b) * sign;
}

template <typename T, int V> struct VecOf { typedef T type __attribute__((ext_vector_type(V))); };
template <typename T> struct VecOf<T, 1> { struct type { T v; __device__ T& operator[](int) { return v; } }; };

// INTER: V neighbouring channels (V / 2 pairs, V even) a thread; else V first and the V second channels of V pairs.  V = 1
// takes any layout.  Threads of channels that pass through move one (INTER) or two vectors in the same loop.
template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryP p, const long long row0, const int units, const int hchunk) {
  constexpr int NPAIR = INTER ? V / 2 : V;
  typedef typename VecOf<T, V>::type vec;
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x, row = row0 + id / units;
  if (row >= p.rows) return;
  const int u = (int)(id % units);
  const int h0 = blockIdx.y * hchunk, h1 = min(p.heads, h0 + hchunk);
  const int turning = p.pairs / NPAIR;
  const bool turns = u < turning;
  const T* x = (const T*)p.x + row * p.xr + h0 * p.xh;
  T* y = (T*)p.y + row * p.yr + h0 * p.yh;
  float cs[NPAIR], sn[NPAIR];
  int ca, cb;
  if (turns) {
    const int* pos = p.pos + (row % p.pos_rows) * p.n_axes;
#pragma unroll
    for (int i = 0; i < NPAIR; ++i) {
      const int pr = u * NPAIR + i;
      turn_cs((double)pos[p.axis[pr]] * p.turn[pr], p.sign, cs[i], sn[i]);
    }
    ca = INTER ? u * V : p.c0[u * NPAIR];
    cb = INTER ? 0 : p.c1[u * NPAIR];
  } else {
#pragma unroll
    for (int i = 0; i < NPAIR; ++i) cs[i] = sn[i] = 0.f;
    ca = 2 * p.pairs + (u - turning) * (INTER ? V : 2 * V);
    cb = min(ca + V, p.d - V);
  }
#pragma unroll 4
  for (int h = h0; h < h1; ++h, x += p.xh, y += p.yh) {
    if (INTER) {
      vec a = *reinterpret_cast<const vec*>(x + ca);
#pragma unroll
      for (int i = 0; i < NPAIR; ++i) {
        const float ua = (float)a[2 * i], ub = (float)a[(2 * i + 1) % V];
        if (turns) {
          a[2 * i] = (T)(ua * cs[i] - ub * sn[i]);
          a[(2 * i + 1) % V] = (T)(ua * sn[i] + ub * cs[i]);
        }
      }
      *reinterpret_cast<vec*>(y + ca) = a;
    } else {
      vec a = *reinterpret_cast<const vec*>(x + ca), b = *reinterpret_cast<const vec*>(x + cb);
#pragma unroll
      for (int i = 0; i < NPAIR; ++i) {
        const float ua = (float)a[i], ub = (float)b[i];
        if (turns) {
          a[i] = (T)(ua * cs[i] - ub * sn[i]);
          b[i] = (T)(ua * sn[i] + ub * cs[i]);
        }
      }
      *reinterpret_cast<vec*>(y + ca) = a;
      *reinterpret_cast<vec*>(y + cb) = b;
    }
  }
}

// vectors of V channels fit: every address is a multiple of their size, and none crosses the border between turning and
// passing channels (halves: between an axis' halves)
template <typename T> bool fits(const RotaryP& p, int v) {
  if (p.interleaved && v < 2) return false;
  const int bytes = v * (int)sizeof(T);
  if (p.d % v || 2 * p.pairs % v || ((uintptr_t)p.x | (uintptr_t)p.y) % bytes || p.xr % v || p.xh % v || p.yr % v || p.yh % v) return false;
  if (p.interleaved) return true;
  if (p.pairs % v) return false;
  for (int i = 0; i < p.pairs; i += v)
    if (p.c0[i] % v || p.c1[i] % v || p.c0[i + v - 1] != p.c0[i] + v - 1 || p.axis[i + v - 1] != p.axis[i]) return false;
  return true;
}
template <typename T, int V, bool INTER> int go(const RotaryP& p, hipStream_t st) {
  const int rest = p.copy ? p.d - 2 * p.pairs : 0;
  const int units = INTER ? (2 * p.pairs + rest) / V : p.pairs / V + (rest + 2 * V - 1) / (2 * V);
  const long long blocks = (p.rows * units + 255) / 256;
  // few rows: the heads are split over the grid until there are about four workgroups per compute unit
  int split = 1;
  while (split < p.heads && blocks * split < 1024) split *= 2;
  const int hchunk = (p.heads + split - 1) / split;
  const long long per = ((1LL << 32) - 256) / units;        // rows of a launch, which has fewer than 2^32 threads along x
  for (long long row0 = 0; row0 < p.rows; row0 += per) {
    const long long rows = p.rows - row0 < per ? p.rows - row0 : per;
    rotary_kernel<T, V, INTER><<<dim3((unsigned)((rows * units + 255) / 256), (unsigned)((p.heads + hchunk - 1) / hchunk)), 256, 0, st>>>(p, row0, units, hchunk);
    if (hipGetLastError() != hipSuccess) return 1;
  }
  return 0;
}
// the widest vectors that fit: 16, 8 or 4 bytes
template <typename T> int run(const RotaryP& p, hipStream_t st) {
  constexpr int V = 16 / (int)sizeof(T);
  if (fits<T>(p, V)) return p.interleaved ? go<T, V, true>(p, st) : go<T, V, false>(p, st);
  if (fits<T>(p, V / 2)) return p.interleaved ? go<T, V / 2, true>(p, st) : go<T, V / 2, false>(p, st);
  if constexpr (V == 8)
    if (fits<T>(p, 2)) return p.interleaved ? go<T, 2, true>(p, st) : go<T, 2, false>(p, st);
  return go<T, 1, false>(p, st);
}

}  // namespace

int launch_rotary(const RotaryP& p, int dtype, hipStream_t st) {
  return dtype == OP_F32 ? run<float>(p, st) : dtype == OP_BF16 ? run<__bf16>(p, st) : run<_Float16>(p, st);
}
