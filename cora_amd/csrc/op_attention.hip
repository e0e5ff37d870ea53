// op_attention.hip -- attention over packed sequences of different lengths, forward and backward (gfx950).
//
// Rows of q, k and v are tokens; sequence s owns rows cu[s] .. cu[s+1]-1.  With causal block b token i of a sequence sees
// tokens j < lim(i) = min(n, (floor(i / b) + 1) b) of it, without one lim(i) = n.  Query head h reads key head h / (H / Hkv).
//   t_ij = scale q_i k_j;  lse_i = log sum_j exp t_ij;  p_ij = exp(t_ij - lse_i);  o_i = sum_j p_ij v_j
//   delta_i = do_i . o_i;  ds_ij = p_ij (do_i . v_j - delta_i);  dq_i = scale sum_j ds_ij k_j
//   dk_j = scale sum_i ds_ij q_i;  dv_j = sum_i p_ij do_i          (sums over the query heads of the key head's group too)
//
// Every product runs on 32 x 32 matrix tiles whose FIRST operand comes from LDS and whose second operand is the wave's own
// (registers), so that the tile's column -- one per lane pair (l, l + 32) -- is the wave's own row: its query in the
// forward and dq kernels, its key in the dk/dv kernel.  Row statistics are then per-lane scalars and a row reduction is
// one exchange between the lane halves.  The score tile leaves the matrix unit as the second operand of the next product
// (rows 16 s + {4 h .. 4 h + 3, 8 + 4 h ..} of lane half h): the contraction order is free, so the first operand of that
// product is fetched in the same order and the probabilities never pass through LDS.
// fp32 operands use v_mfma_f32_32x32x2_f32, 16-bit ones v_mfma_f32_32x32x16_*; a "chunk" is what one 16-byte register
// piece per lane covers of the contraction: 8 channels in fp32, 16 in 16 bits.
// All sums, statistics and accumulators are fp32.  The probabilities (and ds) of 16-bit operands are rounded to the
// operands' type before their product, as the matrix unit takes them; their row sum is taken before that rounding.
//
// No atomics: every output element is summed by one wave in a fixed order, so results repeat bit for bit.
#include "op_tile.h"
#include "ops.h"

namespace {

// Staging of R rows x D channels through registers: load() issues the global reads of the next tile, store() puts them
// into LDS after the current one has been used.  Rows >= nvalid and channels >= d are zero.
template <typename T, int D, int R, int NT>
struct Stage {
  static constexpr int NP = D / Op<T>::E, N = R * NP, NI = (N + NT - 1) / NT;
  uint4 v[NI];
  __device__ __forceinline__ void load(const T* base, long long stride, int nvalid, int d) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int id = i * NT + (int)threadIdx.x, r = id / NP, c = id % NP;
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if ((N % NT == 0 || id < N) && r < nvalid && c * Op<T>::E < d)
        v[i] = *reinterpret_cast<const uint4*>(base + r * stride + c * Op<T>::E);
    }
  }
  __device__ __forceinline__ void store(T* lds) const {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int id = i * NT + (int)threadIdx.x, r = id / NP, c = id % NP;
      if (N % NT == 0 || id < N) *reinterpret_cast<uint4*>(lds + Tile<T, D>::at(r, c)) = v[i];
    }
  }
};

// Which rows work item `slot` has: tile `tile` (of TR rows) of the sequence with rows [b, b + n).  Sequence s starts at slot
// floor(cu[s] / TR) + s; as ceil(n / TR) <= floor((c + n) / TR) - floor(c / TR) + 1 its tiles fit before the next
// sequence's, so rows / TR + nseq slots hold every tile of any packing, found by bisection without a table and without
// reading lengths on the host.  Bounds outside [0, rows] are cut, so a broken table reads and writes no other memory.
__device__ __forceinline__ bool locate(const AttnP& p, int slot, int TR, long long& b, int& n, int& tile) {
  if (!p.cu) {
    const int per = (p.seqlen + TR - 1) / TR;
    const int s = slot / per;
    if (s >= p.nseq) return false;
    b = (long long)s * p.seqlen; n = p.seqlen; tile = slot - s * per;
    return true;
  }
  const int rows = (int)p.rows;
  auto first = [&](int s) { int c = p.cu[s]; c = c < 0 ? 0 : (c > rows ? rows : c); return c; };
  int lo = 0, hi = p.nseq;                       // the last sequence whose first slot is <= slot
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first(mid) / TR + mid <= slot) lo = mid; else hi = mid;
  }
  const int c0 = first(lo), c1 = first(lo + 1);
  b = c0; n = c1 - c0; tile = slot - (c0 / TR + lo);
  return n > 0 && tile >= 0 && (long long)tile * TR < n;
}

constexpr float NO_EXP = -1e30f;   // exponent of a row of zeros (attn_bwd_q)
__device__ __forceinline__ float half_max(float v) { return fmaxf(v, __shfl_xor(v, 32, 64)); }
__device__ __forceinline__ float half_sum(float v) { return v + __shfl_xor(v, 32, 64); }
// row of accumulator register r of lane half h in a 32 x 32 tile
__device__ __forceinline__ int acc_row(int r, int h) { return (r & 3) + 8 * (r >> 2) + 4 * h; }

template <typename T> __device__ __forceinline__ void store4(T* dst, const float a, const float b, const float c, const float e) {
  typedef T v4 __attribute__((ext_vector_type(4)));
  v4 v; v[0] = (T)a; v[1] = (T)b; v[2] = (T)c; v[3] = (T)e;
  *reinterpret_cast<v4*>(dst) = v;
}
// D / 32 tiles of (channels x own rows), times f, to the lane's own row
template <typename T, int D> __device__ __forceinline__ void store_own(T* row, const f32x16 (&acc)[D / 32], float f, int d, int h) {
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int ch = 32 * dt + 8 * g + 4 * h;
      if (ch < d) store4<T>(row + ch, acc[dt][4 * g] * f, acc[dt][4 * g + 1] * f, acc[dt][4 * g + 2] * f, acc[dt][4 * g + 3] * f);
    }
}

// query heads of one key head next to each other in the block order (they read the same keys and values)
__device__ __forceinline__ int head_of(int i, int heads, int kv) { return (i % kv) * (heads / kv) + i / kv; }

// ---- forward -------------------------------------------------------------------------------------
template <typename T, int D>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 1 : 2) void attn_fwd(const AttnP p) {
  typedef Op<T> O; typedef Tile<T, D> L; typedef typename O::frag frag;
  constexpr int KT = sizeof(T) == 4 ? 32 : 64, QT = 128, NC = D / O::CH, NS = KT / O::CH;
  __shared__ __attribute__((aligned(16))) T Ks[2][KT * D];
  __shared__ __attribute__((aligned(16))) T Vs[2][KT * D];
  long long b; int n, tile;
  if (!locate(p, blockIdx.x / p.heads, QT, b, n, tile)) return;
  tile = (n + QT - 1) / QT - 1 - tile;                      // causal: the tiles with most keys start first
  const int head = head_of(blockIdx.x % p.heads, p.heads, p.kv_heads), kv = head / (p.heads / p.kv_heads);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5;
  const int qw = tile * QT + 32 * w, qi = qw + (lane & 31);  // the wave's first query, the lane's
  const bool own = qi < n;
  auto limit = [&](int i) { return p.block ? (int)min((long long)n, ((long long)(i / p.block) + 1) * p.block) : n; };
  const int lim = own ? limit(qi) : 0;
  const int wave_end = qw < n ? limit(min(qw + 31, n - 1)) : 0;      // keys the wave needs
  const int wave_min = limit(min(qw, n - 1));                        // keys every query of it sees
  const int end = limit(min(tile * QT + QT, n) - 1);                 // keys the workgroup needs

  const T* kb = (const T*)p.k + b * p.kr + (long long)kv * p.kh;
  const T* vb = (const T*)p.v + b * p.vr + (long long)kv * p.vh;
  const T* qrow = (const T*)p.q + (b + qi) * p.qr + (long long)head * p.qh;
  frag qf[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) qf[c] = L::own_frag(qrow, own, c, p.d, lane);

  f32x16 acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  float m = -INFINITY, l = 0.f;                             // running maximum (log2 units) and sum
  const float sl2 = p.scale * CORA_LOG2E;

  Stage<T, D, KT, 256> sk, sv;
  sk.load(kb, p.kr, end, p.d); sv.load(vb, p.vr, end, p.d);
  sk.store(Ks[0]); sv.store(Vs[0]);
  __syncthreads();
  for (int j0 = 0, cur = 0; j0 < end; j0 += KT, cur ^= 1) {
    const bool more = j0 + KT < end;
    if (more) {
      sk.load(kb + (long long)(j0 + KT) * p.kr, p.kr, end - j0 - KT, p.d);
      sv.load(vb + (long long)(j0 + KT) * p.vr, p.vr, end - j0 - KT, p.d);
    }
    if (j0 < wave_end) {
      f32x16 s[KT / 32];
      float mx = -INFINITY;
#pragma unroll
      for (int t = 0; t < KT / 32; ++t) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) s[t] = O::mma(L::row_frag(Ks[cur], 32 * t, c, lane), qf[c], s[t]);
      }
      if (j0 + KT > wave_min) {
#pragma unroll
        for (int t = 0; t < KT / 32; ++t)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (j0 + 32 * t + acc_row(r, h) >= lim) s[t][r] = -INFINITY;
      }
#pragma unroll
      for (int t = 0; t < KT / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[t][r]);
      mx = half_max(mx) * sl2;
      const float mn = fmaxf(m, mx);
      if (__any(mn > m)) {
        const float al = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        l *= al;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[i][r] *= al;
        m = mn;
      }
      const float mb = m == -INFINITY ? 0.f : m;            // a row that has seen nothing yet
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < KT / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], sl2, -mb));
          sum += s[t][r];
        }
      l += sum;
#pragma unroll
      for (int k = 0; k < NS; ++k) {
        const frag pf = O::pack(s[k * O::CH / 32], k % (32 / O::CH));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] = O::mma(L::col_frag(Vs[cur], k, i, lane), pf, acc[i]);
      }
    }
    if (more) { sk.store(Ks[cur ^ 1]); sv.store(Vs[cur ^ 1]); }
    __syncthreads();
  }
  l = half_sum(l);
  if (own) {
    store_own<T, D>((T*)p.out + (b + qi) * p.orow + (long long)head * p.oh, acc, 1.f / l, p.d, h);
    if (h == 0) p.lse[(long long)head * p.rows + b + qi] = (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
  }
}

// ---- backward: dq (and the row constants the dk/dv kernel reads) ---------------------------------
// fp16 holds nothing below 2^-24, and ds ~ p do / sqrt(n) of an unscaled loss lies there.  Every query row of do therefore
// enters with a power of two 2^-e that brings its largest element to [1, 2); e is kept beside delta for the other kernel.
template <typename T, int D>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 1 : 2) void attn_bwd_q(const AttnP p) {
  typedef Op<T> O; typedef Tile<T, D> L; typedef typename O::frag frag;
  constexpr bool F16 = sizeof(T) == 2 && O::CH == 16 && __is_same(T, _Float16);
  constexpr int KT = sizeof(T) == 4 ? 32 : 64, QT = 128, NC = D / O::CH;
  __shared__ __attribute__((aligned(16))) T Ks[2][KT * D];
  __shared__ __attribute__((aligned(16))) T Vs[2][KT * D];
  long long b; int n, tile;
  if (!locate(p, blockIdx.x / p.heads, QT, b, n, tile)) return;
  tile = (n + QT - 1) / QT - 1 - tile;
  const int head = head_of(blockIdx.x % p.heads, p.heads, p.kv_heads), kv = head / (p.heads / p.kv_heads);
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5;
  const int qw = tile * QT + 32 * w, qi = qw + (lane & 31);
  const bool own = qi < n;
  auto limit = [&](int i) { return p.block ? (int)min((long long)n, ((long long)(i / p.block) + 1) * p.block) : n; };
  const int lim = own ? limit(qi) : 0;
  const int wave_end = qw < n ? limit(min(qw + 31, n - 1)) : 0;
  const int wave_min = limit(min(qw, n - 1));
  const int end = limit(min(tile * QT + QT, n) - 1);

  const T* kb = (const T*)p.k + b * p.kr + (long long)kv * p.kh;
  const T* vb = (const T*)p.v + b * p.vr + (long long)kv * p.vh;
  Stage<T, D, KT, 256> sk, sv;
  sk.load(kb, p.kr, end, p.d); sv.load(vb, p.vr, end, p.d);

  const long long row = b + qi;
  frag qf[NC], df[NC];
  float delta = 0.f, big = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    qf[c] = L::own_frag((const T*)p.q + row * p.qr + (long long)head * p.qh, own, c, p.d, lane);
    df[c] = L::own_frag((const T*)p.dout + row * p.dor + (long long)head * p.doh, own, c, p.d, lane);
    const frag of = L::own_frag((const T*)p.o + row * p.orow + (long long)head * p.oh, own, c, p.d, lane);
#pragma unroll
    for (int i = 0; i < O::E; ++i) { delta = __builtin_fmaf((float)df[c][i], (float)of[i], delta); big = fmaxf(big, fabsf((float)df[c][i])); }
  }
  delta = half_sum(delta);
  float dscale = 1.f, back = p.scale;
  if (F16) {
    big = half_max(big);
    const int e = big > 0.f && big < INFINITY ? __builtin_amdgcn_frexp_expf(big) - 1 : 0;
    dscale = __builtin_amdgcn_ldexpf(1.f, -e); back = __builtin_amdgcn_ldexpf(p.scale, e);
    if (own && h == 0) p.delta[((long long)p.heads + head) * p.rows + row] = big > 0.f ? (float)e : NO_EXP;
  }
  const float lse2 = own ? p.lse[(long long)head * p.rows + row] * CORA_LOG2E : 0.f;
  if (own && h == 0) p.delta[(long long)head * p.rows + row] = delta;
  const float sl2 = p.scale * CORA_LOG2E;

  f32x16 acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  sk.store(Ks[0]); sv.store(Vs[0]);
  __syncthreads();
  for (int j0 = 0, cur = 0; j0 < end; j0 += KT, cur ^= 1) {
    const bool more = j0 + KT < end;
    if (more) {
      sk.load(kb + (long long)(j0 + KT) * p.kr, p.kr, end - j0 - KT, p.d);
      sv.load(vb + (long long)(j0 + KT) * p.vr, p.vr, end - j0 - KT, p.d);
    }
    if (j0 < wave_end) {
#pragma unroll
      for (int t = 0; t < KT / 32; ++t) {
        f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          s = O::mma(L::row_frag(Ks[cur], 32 * t, c, lane), qf[c], s);
          dp = O::mma(L::row_frag(Vs[cur], 32 * t, c, lane), df[c], dp);
        }
        const bool edge = j0 + 32 * t + 32 > wave_min;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], sl2, -lse2)) * (dp[r] - delta);
          if (F16) pr *= dscale;
          s[r] = edge && j0 + 32 * t + acc_row(r, h) >= lim ? 0.f : pr;
        }
#pragma unroll
        for (int k = 0; k < 32 / O::CH; ++k) {
          const frag pf = O::pack(s, k);
#pragma unroll
          for (int i = 0; i < D / 32; ++i) acc[i] = O::mma(L::col_frag(Ks[cur], t * (32 / O::CH) + k, i, lane), pf, acc[i]);
        }
      }
    }
    if (more) { sk.store(Ks[cur ^ 1]); sv.store(Vs[cur ^ 1]); }
    __syncthreads();
  }
  if (own) store_own<T, D>((T*)p.dq + row * p.dqr + (long long)head * p.dqh, acc, back, p.d, h);
}

// ---- backward: dk and dv -------------------------------------------------------------------------
// A workgroup owns 128 keys of one key head and walks the queries that see any of them, head after head of its group.
template <typename T, int D>
__global__ __launch_bounds__(256, 1) void attn_bwd_kv(const AttnP p) {
  typedef Op<T> O; typedef Tile<T, D> L; typedef typename O::frag frag;
  constexpr bool F16 = sizeof(T) == 2 && O::CH == 16 && __is_same(T, _Float16);
  constexpr int QT = sizeof(T) == 4 ? 32 : 64, KB = 128, NC = D / O::CH;
  __shared__ __attribute__((aligned(16))) T Qs[2][QT * D];
  __shared__ __attribute__((aligned(16))) T Ds[2][QT * D];
  __shared__ float cl[2][QT], cd[2][QT], ce[2][QT];     // per staged query: lse (log2), delta, exponent of its do scale
  __shared__ int lm[2][QT];                             // and the keys it sees
  long long b; int n, tile;
  if (!locate(p, blockIdx.x / p.kv_heads, KB, b, n, tile)) return;
  const int kv = blockIdx.x % p.kv_heads, group = p.heads / p.kv_heads;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, h = lane >> 5;
  const int k0 = tile * KB, kw = k0 + 32 * w, ki = kw + (lane & 31);
  const bool own = ki < n;
  const int qbeg = p.block ? k0 / p.block * p.block / QT * QT : 0;    // the first staged query that sees key k0 is behind it
  const int ntile = (n - qbeg + QT - 1) / QT, total = ntile * group;

  frag kf[NC], vf[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    kf[c] = L::own_frag((const T*)p.k + (b + ki) * p.kr + (long long)kv * p.kh, own, c, p.d, lane);
    vf[c] = L::own_frag((const T*)p.v + (b + ki) * p.vr + (long long)kv * p.vh, own, c, p.d, lane);
  }
  f32x16 ak[D / 32], av[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) { ak[i][r] = 0.f; av[i][r] = 0.f; }
  const float sl2 = p.scale * CORA_LOG2E;
  float ecur = NO_EXP;                                  // F16: exponent ak is scaled by

  Stage<T, D, QT, 256> sq, sd;
  float rl = 0.f, rd = 0.f, re = 0.f; int rm = 0;
  auto load = [&](int it) {
    const int head = kv * group + it / ntile, q0 = qbeg + (it % ntile) * QT;
    sq.load((const T*)p.q + (b + q0) * p.qr + (long long)head * p.qh, p.qr, n - q0, p.d);
    sd.load((const T*)p.dout + (b + q0) * p.dor + (long long)head * p.doh, p.dor, n - q0, p.d);
    const int i = q0 + (int)threadIdx.x;
    if (threadIdx.x < QT) {
      const bool ok = i < n;
      const long long at = (long long)head * p.rows + b + i;
      rl = ok ? p.lse[at] * CORA_LOG2E : INFINITY;      // exp2(. - inf) = 0: rows behind the sequence add nothing
      rd = ok ? p.delta[at] : 0.f;
      rm = ok ? (p.block ? (int)min((long long)n, ((long long)(i / p.block) + 1) * p.block) : n) : 0;
      if (F16) re = ok ? p.delta[(long long)p.heads * p.rows + at] : NO_EXP;
    }
  };
  auto store = [&](int s) {
    sq.store(Qs[s]); sd.store(Ds[s]);
    if (threadIdx.x < QT) { cl[s][threadIdx.x] = rl; cd[s][threadIdx.x] = rd; lm[s][threadIdx.x] = rm; if (F16) ce[s][threadIdx.x] = re; }
  };
  load(0); store(0);
  __syncthreads();
  for (int it = 0, cur = 0; it < total; ++it, cur ^= 1) {
    const bool more = it + 1 < total;
    if (more) load(it + 1);
    const int q0 = qbeg + (it % ntile) * QT;
    if (kw < n) {
      if (F16) {
        float e = ce[cur][lane & (QT - 1)];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) e = fmaxf(e, __shfl_xor(e, o, 64));
        if (e > ecur) {                                 // larger gradients than before: bring the sum to their scale
          const float f = ecur == NO_EXP ? 0.f : __builtin_amdgcn_exp2f(ecur - e);
#pragma unroll
          for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) ak[i][r] *= f;
          ecur = e;
        }
      }
      const float ds = F16 && ecur != NO_EXP ? __builtin_amdgcn_exp2f(-ecur) : 1.f;
#pragma unroll
      for (int t = 0; t < QT / 32; ++t) {
        if (q0 + 32 * t >= n) break;
        f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          s = O::mma(L::row_frag(Qs[cur], 32 * t, c, lane), kf[c], s);
          dp = O::mma(L::row_frag(Ds[cur], 32 * t, c, lane), vf[c], dp);
        }
        const bool edge = p.block && lm[cur][32 * t] < kw + 32;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int q = 32 * t + acc_row(r, h);
          float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], sl2, -cl[cur][q]));
          float g = pr * (dp[r] - cd[cur][q]);
          if (F16) g *= ds;
          const bool hide = edge && ki >= lm[cur][q];
          s[r] = hide ? 0.f : pr;
          dp[r] = hide ? 0.f : g;
        }
#pragma unroll
        for (int k = 0; k < 32 / O::CH; ++k) {
          const frag pf = O::pack(s, k), gf = O::pack(dp, k);
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            av[i] = O::mma(L::col_frag(Ds[cur], t * (32 / O::CH) + k, i, lane), pf, av[i]);
            ak[i] = O::mma(L::col_frag(Qs[cur], t * (32 / O::CH) + k, i, lane), gf, ak[i]);
          }
        }
      }
    }
    if (more) store(cur ^ 1);
    __syncthreads();
  }
  if (own) {
    const float f = F16 && ecur != NO_EXP ? p.scale * __builtin_amdgcn_exp2f(ecur) : p.scale;
    store_own<T, D>((T*)p.dk + (b + ki) * p.dkr + (long long)kv * p.dkh, ak, f, p.d, h);
    store_own<T, D>((T*)p.dv + (b + ki) * p.dvr + (long long)kv * p.dvh, av, 1.f, p.d, h);
  }
}

long long slots(const AttnP& p, int tr) {
  return p.cu ? p.rows / tr + p.nseq : (long long)p.nseq * ((p.seqlen + tr - 1) / tr);
}
template <typename T, int D> int fwd(const AttnP& p, hipStream_t st) {
  attn_fwd<T, D><<<dim3((unsigned)(slots(p, 128) * p.heads)), 256, 0, st>>>(p);
  return hipGetLastError() != hipSuccess;
}
template <typename T, int D> int bwd(const AttnP& p, hipStream_t st) {
  attn_bwd_q<T, D><<<dim3((unsigned)(slots(p, 128) * p.heads)), 256, 0, st>>>(p);
  if (hipGetLastError() != hipSuccess) return 1;
  attn_bwd_kv<T, D><<<dim3((unsigned)(slots(p, 128) * p.kv_heads)), 256, 0, st>>>(p);
  return hipGetLastError() != hipSuccess;
}
template <typename T> int fwd_d(const AttnP& p, hipStream_t st) {
  return p.d <= 32 ? fwd<T, 32>(p, st) : p.d <= 64 ? fwd<T, 64>(p, st) : p.d <= 96 ? fwd<T, 96>(p, st) : fwd<T, 128>(p, st);
}
template <typename T> int bwd_d(const AttnP& p, hipStream_t st) {
  return p.d <= 32 ? bwd<T, 32>(p, st) : p.d <= 64 ? bwd<T, 64>(p, st) : p.d <= 96 ? bwd<T, 96>(p, st) : bwd<T, 128>(p, st);
}

}  // namespace

int launch_attention_fwd(const AttnP& p, int dtype, hipStream_t st) {
  return dtype == OP_F32 ? fwd_d<float>(p, st) : dtype == OP_BF16 ? fwd_d<__bf16>(p, st) : fwd_d<_Float16>(p, st);
}
int launch_attention_bwd(const AttnP& p, int dtype, hipStream_t st) {
  return dtype == OP_F32 ? bwd_d<float>(p, st) : dtype == OP_BF16 ? bwd_d<__bf16>(p, st) : bwd_d<_Float16>(p, st);
}
