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
// All sums, statistics and accumulators are fp32; fp32's are taken 32 rows at a time (sum_apart).  The probabilities (and ds) of 16-bit
// operands are rounded to the operands' type before their product, as the matrix unit takes them, or given in two pieces (FINE, at
// bwd); their row sum is taken before that rounding (lse is exact to fp32).  fp16's enter times powers of two (fit_half).
//
// No atomics: every output element is summed by one wave in a fixed order, so results repeat bit for bit.
#include "op_tile.h"
#include "ops.h"

namespace {

// Staging of R rows x D channels straight from global memory into an LDS tile by NW waves.  A wave's request fills 64
// consecutive 16-byte places; each lane asks for the piece that belongs there (Tile::swz).  The buffer descriptor ends
// with the last valid row, and the pieces of channels >= d ask for an address past any end: both arrive as zeros.
template <typename T, int D, int R, int NW>
struct Fetch {
  static constexpr int NP = D / Op<T>::E, NI = R * NP / 64 / NW;
  static_assert(R * NP % (64 * NW) == 0, "whole requests");
  int at[NI], stride, width;
  __device__ __forceinline__ Fetch(long long row_stride, int d, int w, int lane) : stride((int)row_stride * (int)sizeof(T)), width(d * (int)sizeof(T)) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int id = (i * NW + w) * 64 + lane, r = id / NP, c = (id % NP) ^ Tile<T, D>::swz(r);
      at[i] = c * 16 < width ? r * stride + c * 16 : (int)0x80000000;
    }
  }
  __device__ __forceinline__ void operator()(const T* rows, int nvalid, T* lds, int w) const {
    [[maybe_unused]] const int bytes = nvalid > 0 ? (min(nvalid, R) - 1) * stride + width : 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) REQUEST(rows, bytes, lds + (i * NW + w) * 64 * Op<T>::E, 16, at[i]);
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

// The same for causal walks, the longest first over all sequences: a long tile that starts last would keep the chip waiting.
// Work item i in the order of falling `tile`, where a sequence of T tiles has 0 .. T - 1: N(t) = sum over the sequences of
// max(0, T - t) items have tile t or more, so t is found by bisection and the sequence by its rank among those with T > t.
// One sequence a lane, so up to 64 of them; more keep their own order.  Worth its 1 to 2 us a workgroup where not all
// workgroups run at once (longest_first; LDS: bytes of a workgroup).  Forward, us, own order / longest first: fp32, 16 x 1024
// tokens, 1 head 54 / 40; packed clips, bf16, 12 heads of 64 102 / 94; all at once, bf16, 9 sequences, 2 heads 17.9 / 20.3.
template <int LDS> __device__ __forceinline__ bool longest_first(const AttnP& p) {
  return p.block && gridDim.x > (LDS <= 80 * 1024 ? 512 : 256);
}
__device__ __forceinline__ bool locate_longest(const AttnP& p, int i, int TR, long long& b, int& n, int& tile) {
  if (!p.cu || p.nseq > 64) {
    if (!locate(p, i, TR, b, n, tile)) return false;
    const int T = (n + TR - 1) / TR;
    if (!p.cu) { tile = T - 1 - i / p.nseq; b = (long long)(i % p.nseq) * n; }
    else tile = T - 1 - tile;
    return true;
  }
  const int rows = (int)p.rows, lane = threadIdx.x & 63;
  auto first = [&](int s) { int c = p.cu[s]; return c < 0 ? 0 : (c > rows ? rows : c); };
  int c0 = 0, len = 0;
  if (lane < p.nseq) { c0 = first(lane); len = max(0, first(lane + 1) - c0); }
  const int T = (len + TR - 1) / TR;
  auto sum = [](int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return __builtin_amdgcn_readfirstlane(v);
  };
  int hi = T;                                     // the largest T
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) hi = max(hi, __shfl_xor(hi, o, 64));
  if (i >= sum(T)) return false;
  int lo = 0, above = 0;                          // N(lo) > i >= N(hi) = above
  hi = __builtin_amdgcn_readfirstlane(hi);
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1, c = sum(max(0, T - mid));
    if (c > i) lo = mid; else { hi = mid; above = c; }
  }
  const unsigned long long in = __ballot(T > lo);
  const int rank = __popcll(in & ((1ULL << lane) - 1));
  const int s = max(0, __ffsll((long long)__ballot(T > lo && rank == i - above)) - 1);
  b = __builtin_amdgcn_readlane(c0, s); n = __builtin_amdgcn_readlane(len, s); tile = lo;
  return (long long)tile * TR < n;                // a broken table may give no such tile
}

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

// the keys a sequence's token i sees end here
__device__ __forceinline__ int limit(int i, int n, int block) {
  return block ? (int)min((long long)n, ((long long)(i / block) + 1) * block) : n;
}

// The tiles a workgroup walks pass through two LDS buffers, each an object of its own so that the compiler sees that the
// requests for one do not touch what is read from the other.  Between two barriers the next tile is under way while the
// current one is worked on.  (One exit only: a second one makes the compiler keep two copies of the accumulators.)
#define WALK(COUNT, FETCH, WORK)                                                   \
  FETCH(0, 0);                                                                     \
  for (int it_ = 0; it_ < (COUNT); it_ += 2) {                                     \
    arrive_barrier();                                                              \
    if (it_ + 1 < (COUNT)) FETCH(it_ + 1, 1);                                      \
    __builtin_amdgcn_sched_barrier(0);                                             \
    WORK(it_, 0);                                                                  \
    arrive_barrier();                                                              \
    if (it_ + 2 < (COUNT)) FETCH(it_ + 2, 0);                                      \
    __builtin_amdgcn_sched_barrier(0);                                             \
    if (it_ + 1 < (COUNT)) WORK(it_ + 1, 1);                                       \
  }

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
// What a mask hides must not count, even if it is not finite: hidden scores are replaced, but in the product behind them 0 times
// infinity would.  A tile of which some rows of the workgroup do not see all is therefore searched first (each lane its own
// 16-byte pieces, as it requested them): elements that are not finite become zeros, and mark(piece) makes the score
// of their row NaN, so that whoever sees the row comes out as NaN in all channels.
template <typename T, int D, int R, int NW, typename M> __device__ __forceinline__ void quarantine(T* t, int w, int lane, const M& mark) {
  constexpr unsigned INF = sizeof(T) == 4 ? 0x7f800000u : __is_same(T, __bf16) ? 0x7f80u : 0x7c00u;     // the exponent's bits
#pragma unroll 1
  for (int i = 0; i < R * D / Op<T>::E / 64 / NW; ++i) {
    const int id = (i * NW + w) * 64 + lane;
    u32x4& at = reinterpret_cast<u32x4*>(t)[id];          // a vector type, which may alias the elements that others read
    u32x4 v = at;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      unsigned keep = ~0u;
      if ((v[e] & INF) == INF) keep = sizeof(T) == 4 ? 0u : 0xffff0000u;
      if (sizeof(T) == 2 && (v[e] >> 16 & INF) == INF) keep &= 0xffffu;
      bad |= keep != ~0u;
      v[e] &= keep;
    }
    if (bad) { at = v; mark(id); }
  }
}
// the waves' LDS writes are done; requests under way stay under way.  WAVE: only the wave's own, whose buffer no other wave reads
template <bool WAVE = false> __device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  if (!WAVE) __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Queries of a workgroup and its walk over keys.  SPLIT = false: NW waves of 32 queries each share every staged tile of KT
// keys.  SPLIT = true, for few rows: NW waves share the same 32 queries, wave w walks the key tiles w, w + NW, .. through
// buffers of its own, and the waves' results are joined in LDS at the end (join_own).
template <typename T, int D, int NW, bool SPLIT> struct Walk {
  static constexpr int KT = sizeof(T) == 4 || SPLIT ? 32 : 64, QT = SPLIT ? 32 : 32 * NW;
  static constexpr int TILE = KT * D, BUF = SPLIT ? NW * TILE : TILE, FW = SPLIT ? 1 : NW;    // elements; waves that fetch a tile
};

// Sum over the waves of a workgroup of their accumulators, into wave 0, in halving steps.  lds: NW / 2 * D * 32 floats,
// no longer used for anything else.
template <int D, int NW>
__device__ __forceinline__ void join_own(f32x16 (&acc)[D / 32], float* lds, int w, int lane) {
#pragma unroll
  for (int o = NW / 2; o >= 1; o /= 2) {
    float* at = lds + (w % o) * (D * 32) + lane * 4;
    __syncthreads();
    if (w >= o && w < 2 * o)
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(at + (4 * i + g) * 256) = f32x4{acc[i][4 * g], acc[i][4 * g + 1], acc[i][4 * g + 2], acc[i][4 * g + 3]};
    __syncthreads();
    if (w < o)
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 v = *reinterpret_cast<const f32x4*>(at + (4 * i + g) * 256);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][4 * g + e] += v[e];
        }
  }
}

// Issue order of the block it stands in: READS reads of LDS first, then N times M matrix instructions followed by PER more reads.
// Left alone the compiler reads an operand right before its use, and where few waves share a SIMD nothing else hides
// the way from LDS: dk/dv of 16-bit types at 128 channels 2.9 ms, so 2.7; the fp32 forward pass 77 us, so 73 (sizes as below; without a
// profiler, which adds 2 to 4 us).
// The 16-bit forward pass and dq, whose tiles are longer, gain nothing or lose.
template <int READS, int PER, int N, int GROUP, int M = 1> __device__ __forceinline__ void feed() {
  __builtin_amdgcn_sched_group_barrier(0x100, READS, GROUP);
#pragma unroll
  for (int c = 0; c < N; ++c) { __builtin_amdgcn_sched_group_barrier(0x8, M, GROUP); __builtin_amdgcn_sched_group_barrier(0x100, PER, GROUP); }
}

// acc += (tile of rows)^T w with a sum of its own for the 32 rows.  For fp32: added one after the other, two products an instruction, the
// terms of a long walk leave thousands of roundings in one growing sum.  Taken by dk and dv, and by out and dq of heads up to 64
// (wider heads have as large errors in their scores).  Against 64 bits, one sum / sums apart: 8 x 2048 tokens, 8 of 2 heads of 64,
// causal, dk 1.1e-6 / 4.8e-7, dq 5.7e-7 / 4.5e-7, out 4.0e-7 / 2.6e-7.  Time, us: forward 310 / 311, backward 1190 / 1155 (fewer registers
// are held); 64 x 196 tokens, 8 heads of 48, 73 / 75 and 246 / 244; backward of heads of 80 and 128 3 and 2 % longer.
template <typename T, int D> __device__ __forceinline__ void sum_apart(const T* tile, const f32x16& w, int t, int i, int lane, f32x16& acc) {
  f32x16 part;
#pragma unroll
  for (int r = 0; r < 16; ++r) part[r] = 0.f;
#pragma unroll
  for (int c = 0; c < 32 / Op<T>::CH; ++c) part = Op<T>::mma(Tile<T, D>::col_frag(tile, t * (32 / Op<T>::CH) + c, i, lane), Op<T>::pack(w, c), part);
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] += part[r];
}

// fp16 holds 2^-24 .. 2^16, and ds ~ p do / sqrt(n) of an unscaled loss lies below.  A tile of ds, whose column is the lane's own
// row, therefore enters its product times 2^-e, and so do the sums acc: times mul here, or (IN) it comes so.  Every lane has an e of its own: small values of a
// row keep their bits whatever the other rows hold.  Kept while the column's largest value comes out in 2^-8 .. 2^15 (what fp16 then
// rounds by 2^-25 is 2^-17 of it), else set so that it is in 2^4 .. 2^5: e is hardly ever changed, and costs a search of the tile.
// The probabilities of dk/dv, 1 / n where all keys are alike, enter times 2^14: fp16 then holds them with 11 bits down to 2^-28.
constexpr int P_EXP = 14;
constexpr int LEAST_EXP = -30;     // ds below 2^-38 gives nothing in fp16 results; the sums times 2^30 stay finite
template <bool IN, int N> __device__ __forceinline__ void fit_half(f32x16& ds, f32x16 (&acc)[N], int& e, float& mul) {
  float big = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r) big = fmaxf(big, fabsf(ds[r]));
  if (!IN) big *= mul;
  // a lane pair shares a column: it is too small if both halves are, and not both empty
  unsigned long long small = __ballot(big < 0x1p-8f && e > LEAST_EXP), none = __ballot(big == 0.f);
  small &= small >> 32; none &= none >> 32;
  if ((unsigned)(small & ~none) || __any(big > 0x1p15f)) {
    big = half_max(big);
    int to = e;
    if (big < INFINITY && (big > 0x1p15f || (big > 0.f && big < 0x1p-8f)))
      to = min(max(__builtin_amdgcn_frexp_expf(big) - 5 + e, LEAST_EXP), 90);
    const float f = __builtin_amdgcn_ldexpf(1.f, e - to);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] *= f;
    if (IN)
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] *= f;
    e = to;
    mul = __builtin_amdgcn_ldexpf(1.f, -to);
  }
  if (!IN)
#pragma unroll
    for (int r = 0; r < 16; ++r) ds[r] *= mul;
}

// ---- forward -------------------------------------------------------------------------------------
// Bound by the matrix units and, as close behind, by LDS: every matrix instruction (32 cycles of a SIMD in 16 bits) takes 1 KB
// from LDS, which four SIMDs reading at once is all that LDS gives (128 bytes a cycle).  One workgroup per 128 queries, two to
// a compute unit; or, for few rows, four waves that share 32 queries (the rule and its figures are at run below).  Measured, causal
// bf16: 16384 tokens x 16 heads of 128 1.05 ms, 1050 TFLOP/s (a large library product: 1133); fp32 64 images of 196 tokens x 8 heads of 48
// 75 us: padding (196 queries to 256, 196 keys to 224, in the second product 48 channels to 64), two rounds of workgroups, and matrix
// units that are busy 64 % of the cycles in which their compute unit has waves (dq 66 %, dk/dv 68 %).
// The running maximum m only has to keep exp2 in range, so it is raised (and the sums
// scaled) when a score exceeds it by 8 in log2 units, not at every new maximum: the sums then carry factors up to 2^8.
// Each row goes by its own scores, so its result does not depend on which other rows share its tile.
template <typename T, int D, int DK, int NW, bool SPLIT>
__global__ __launch_bounds__(64 * NW, SPLIT || (sizeof(T) == 4 && D > 64) ? 1 : DK == 48 ? 3 : 2) void attn_fwd(const AttnP p) {
  typedef Op<T> O; typedef Tile<T, D> L; typedef typename O::frag frag;
  typedef Walk<T, D, NW, SPLIT> W;
  constexpr int KT = W::KT, QT = W::QT, NC = DK / O::CH, NS = KT / O::CH;
  __shared__ __attribute__((aligned(16))) T ks0[W::BUF];
  __shared__ __attribute__((aligned(16))) T vs0[W::BUF];
  __shared__ __attribute__((aligned(16))) T ks1[W::BUF];
  __shared__ __attribute__((aligned(16))) T vs1[W::BUF];
  long long b; int n, tile;
  if (!(longest_first<4 * W::BUF * sizeof(T)>(p) ? locate_longest(p, blockIdx.x / p.heads, QT, b, n, tile) : locate(p, blockIdx.x / p.heads, QT, b, n, tile))) return;
  const int head = head_of(blockIdx.x % p.heads, p.heads, p.kv_heads), kv = head / (p.heads / p.kv_heads);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int qw = tile * QT + (SPLIT ? 0 : 32 * w), qi = qw + (lane & 31);  // the wave's first query, the lane's
  const bool own = qi < n;
  const int lim = own ? limit(qi, n, p.block) : 0;
  const int wave_end = qw < n ? limit(min(qw + 31, n - 1), n, p.block) : 0;      // keys the wave needs
  const int wave_min = limit(min(qw, n - 1), n, p.block);                        // keys every query of it sees
  const int all_min = limit(tile * QT, n, p.block);                              // keys every query of the workgroup sees
  const int end = limit(min(tile * QT + QT, n) - 1, n, p.block);                 // keys the workgroup needs

  const T* kb = (const T*)p.k + b * p.kr + (long long)kv * p.kh;
  const T* vb = (const T*)p.v + b * p.vr + (long long)kv * p.vh;
  const int fw = SPLIT ? 0 : w, mine = SPLIT ? w * W::TILE : 0;    // the wave's share of the requests, its place in a buffer
  const Fetch<T, D, KT, W::FW> fk(p.kr, p.d, fw, lane), fv(p.vr, p.d, fw, lane);
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

  auto fetch = [&](int it, T* k, T* v) {
    const int j0 = (SPLIT ? it * NW + w : it) * KT;
    fk(kb + j0 * p.kr, end - j0, k + mine, fw);
    fv(vb + j0 * p.vr, end - j0, v + mine, fw);
  };
  auto work = [&](int it, T* k, T* v) {
    const int j0 = (SPLIT ? it * NW + w : it) * KT;
    k += mine; v += mine;
    if (j0 + KT > all_min && j0 < end && p.block) {
      quarantine<T, D, KT, W::FW>(v, fw, lane, [&](int id) { k[id * Op<T>::E] = (T)NAN; });
      lds_barrier<SPLIT>();
    }
    if (j0 >= wave_end) return;
    f32x16 s[KT / 32];
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < KT / 32; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) s[t] = O::mma(L::row_frag(k, 32 * t, c, lane), qf[c], s[t]);
    }
    if (sizeof(T) == 4) feed<3, 1, NC, 0, 4>();
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
    if (__any(mx > m + 8.f)) {
      const float mn = mx > m + 8.f ? mx : m, al = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= al;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= al;
      m = mn;
    }
    const float mb = m == -INFINITY ? 0.f : m;              // a row that has seen nothing yet
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < KT / 32; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[t][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][r], sl2, -mb));
        sum += s[t][r];
      }
    l += sum;
    if constexpr (sizeof(T) == 4 && D <= 64) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i) sum_apart<T, D>(v, s[0], 0, i, lane, acc[i]);
    } else
#pragma unroll
    for (int c = 0; c < NS; ++c) {
      const frag pf = O::pack(s[c * O::CH / 32], c % (32 / O::CH));
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] = O::mma(L::col_frag(v, c, i, lane), pf, acc[i]);
    }
  };
#define FETCH(it, buf) fetch(it, buf ? ks1 : ks0, buf ? vs1 : vs0)
#define WORK(it, buf) work(it, buf ? ks1 : ks0, buf ? vs1 : vs0)
  WALK(SPLIT ? (end + NW * KT - 1) / (NW * KT) : (end + KT - 1) / KT, FETCH, WORK)
#undef FETCH
#undef WORK
  l = half_sum(l);
  if constexpr (SPLIT) {                                    // one maximum for all waves, then their sums add up
    __shared__ float ml[2][NW][32];
    if (h == 0) { ml[0][w][lane & 31] = m; ml[1][w][lane & 31] = l; }
    __syncthreads();
    float mt = ml[0][0][lane & 31];
#pragma unroll
    for (int o = 1; o < NW; ++o) mt = fmaxf(mt, ml[0][o][lane & 31]);
    l = 0.f;
#pragma unroll
    for (int o = 0; o < NW; ++o) {
      const float mo = ml[0][o][lane & 31];                 // -infinity: nothing seen (l = 0), or nothing but NaN (l = NaN)
      l += ml[1][o][lane & 31] * (mo == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(mo - mt));
    }
    const float al = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mt);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] *= al;
    join_own<D, NW>(acc, reinterpret_cast<float*>(ks0), w, lane);
    if (w) return;
    m = mt;
  }
  if (!own) return;
  store_own<T, D>((T*)p.out + (b + qi) * p.orow + (long long)head * p.oh, acc, 1.f / l, p.d, h);
  if (h == 0) p.lse[(long long)head * p.rows + b + qi] = (m + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

// ---- backward: dq (and the row constants the dk/dv kernel reads) ---------------------------------
// Three products where the forward pass has two, bound like it: 16384 tokens x 16 heads of 128, causal bf16, 1.5 ms, 1100 TFLOP/s.
// q k and do v are computed here and in the dk/dv kernel: seven products instead of five, but no atomics and no ds in memory.
// The row constants are -delta, from which the product do v starts, and -lse (log2 units).  (Starting q k from -lse / scale saves
// nothing and triples the error of fp32 gradients: the sum is then rounded at the size of lse / scale.)
// FINE: ds enters its product in two pieces of the 16-bit type, so that its rounding does not count (the rule is at bwd).
template <typename T, int D, int DK, int NW, bool SPLIT, bool FINE>
__global__ __launch_bounds__(64 * NW, SPLIT || (sizeof(T) == 4 && D > 64) ? 1 : sizeof(T) == 2 && D == 64 ? 3 : 2) void attn_bwd_q(const AttnP p) {
  typedef Op<T> O; typedef Tile<T, D> L; typedef typename O::frag frag;
  constexpr bool F16 = __is_same(T, _Float16);
  typedef Walk<T, D, NW, SPLIT> W;
  constexpr int KT = W::KT, QT = W::QT, NC = DK / O::CH;
  __shared__ __attribute__((aligned(16))) T ks0[W::BUF];
  __shared__ __attribute__((aligned(16))) T vs0[W::BUF];
  __shared__ __attribute__((aligned(16))) T ks1[W::BUF];
  __shared__ __attribute__((aligned(16))) T vs1[W::BUF];
  long long b; int n, tile;
  if (!(longest_first<4 * W::BUF * sizeof(T)>(p) ? locate_longest(p, blockIdx.x / p.heads, QT, b, n, tile) : locate(p, blockIdx.x / p.heads, QT, b, n, tile))) return;
  const int head = head_of(blockIdx.x % p.heads, p.heads, p.kv_heads), kv = head / (p.heads / p.kv_heads);
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int qw = tile * QT + (SPLIT ? 0 : 32 * w), qi = qw + (lane & 31);
  const bool own = qi < n;
  const int lim = own ? limit(qi, n, p.block) : 0;
  const int wave_end = qw < n ? limit(min(qw + 31, n - 1), n, p.block) : 0;
  const int wave_min = limit(min(qw, n - 1), n, p.block), all_min = limit(tile * QT, n, p.block);
  const int end = limit(min(tile * QT + QT, n) - 1, n, p.block);

  const T* kb = (const T*)p.k + b * p.kr + (long long)kv * p.kh;
  const T* vb = (const T*)p.v + b * p.vr + (long long)kv * p.vh;
  const int fw = SPLIT ? 0 : w, mine = SPLIT ? w * W::TILE : 0;    // the wave's share of the requests, its place in a buffer
  const Fetch<T, D, KT, W::FW> fk(p.kr, p.d, fw, lane), fv(p.vr, p.d, fw, lane);
  const long long row = b + qi, at = (long long)head * p.rows + row, plane = (long long)p.heads * p.rows;
  frag qf[NC], df[NC];
  float delta = 0.f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    qf[c] = L::own_frag((const T*)p.q + row * p.qr + (long long)head * p.qh, own, c, p.d, lane);
    df[c] = L::own_frag((const T*)p.dout + row * p.dor + (long long)head * p.doh, own, c, p.d, lane);
    const frag of = L::own_frag((const T*)p.o + row * p.orow + (long long)head * p.oh, own, c, p.d, lane);
#pragma unroll
    for (int i = 0; i < O::E; ++i) delta = __builtin_fmaf((float)df[c][i], (float)of[i], delta);
  }
  delta = half_sum(delta);
  [[maybe_unused]] int ex = 0;                              // F16: acc and ds are scaled by mul = 2^-ex
  [[maybe_unused]] float mul = 1.f;
  const float lse2 = own ? p.lse[at] * CORA_LOG2E : 0.f, sl2 = p.scale * CORA_LOG2E;
  // A row that sees the first key tile only takes delta from the tile itself, sum_j p_ij (do_i v_j): the rounding of out to
  // 16 bits, which delta otherwise inherits, counts most in rows that see few keys.
  const bool whole = sizeof(T) == 2 && lim <= KT;
  if (own && h == 0 && (!SPLIT || w == 0)) { if (!whole) p.delta[at] = -delta; p.delta[plane + at] = (F16 ? P_EXP : 0) - lse2; }

  f32x16 acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;

  auto fetch = [&](int it, T* k, T* v) {
    const int j0 = (SPLIT ? it * NW + w : it) * KT;
    fk(kb + j0 * p.kr, end - j0, k + mine, fw);
    fv(vb + j0 * p.vr, end - j0, v + mine, fw);
  };
  auto work = [&](int it, T* k, T* v) {
    const int j0 = (SPLIT ? it * NW + w : it) * KT;
    k += mine; v += mine;
    if (j0 + KT > all_min && j0 < end && p.block) {
      quarantine<T, D, KT, W::FW>(k, fw, lane, [&](int id) { v[id * Op<T>::E] = (T)NAN; });
      lds_barrier<SPLIT>();
    }
    if (j0 >= wave_end) return;
    if (sizeof(T) == 2 && j0 == 0 && wave_min <= KT) {
      float sum = 0.f;
#pragma unroll 1
      for (int t = 0; t < KT / 32; ++t) {
        f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          s = O::mma(L::row_frag(k, 32 * t, c, lane), qf[c], s);
          dp = O::mma(L::row_frag(v, 32 * t, c, lane), df[c], dp);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * t + acc_row(r, h) < lim) sum = __builtin_fmaf(__builtin_amdgcn_exp2f(__builtin_fmaf(s[r], sl2, -lse2)), dp[r], sum);
      }
      sum = half_sum(sum);
      if (whole) {
        delta = sum;
        if (own && h == 0) p.delta[at] = -delta;
      }
    }
#pragma unroll
    for (int t = 0; t < KT / 32; ++t) {
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = -delta; }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        s = O::mma(L::row_frag(k, 32 * t, c, lane), qf[c], s);
        dp = O::mma(L::row_frag(v, 32 * t, c, lane), df[c], dp);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], sl2, F16 ? -lse2 - (float)ex : -lse2)) * dp[r];
      if (j0 + 32 * t + 32 > wave_min) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (j0 + 32 * t + acc_row(r, h) >= lim) s[r] = 0.f;
      }
      if constexpr (F16) fit_half<true>(s, acc, ex, mul);
      if constexpr (sizeof(T) == 4 && D <= 64) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) sum_apart<T, D>(k, s, t, i, lane, acc[i]);
      } else
#pragma unroll
      for (int c = 0; c < 32 / O::CH; ++c) {
        const frag pf = O::pack(s, c);
        [[maybe_unused]] frag rf;
        if constexpr (FINE) rf = O::rest(s, c, pf);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const frag kf = L::col_frag(k, t * (32 / O::CH) + c, i, lane);
          acc[i] = O::mma(kf, pf, acc[i]);
          if constexpr (FINE) acc[i] = O::mma(kf, rf, acc[i]);
        }
      }
    }
  };
#define FETCH(it, buf) fetch(it, buf ? ks1 : ks0, buf ? vs1 : vs0)
#define WORK(it, buf) work(it, buf ? ks1 : ks0, buf ? vs1 : vs0)
  WALK(SPLIT ? (end + NW * KT - 1) / (NW * KT) : (end + KT - 1) / KT, FETCH, WORK)
#undef FETCH
#undef WORK
  float f = F16 ? __builtin_amdgcn_ldexpf(p.scale, ex) : p.scale;
  if constexpr (SPLIT) {                                    // the waves' exponents differ
    if constexpr (F16) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= f;
      f = 1.f;
    }
    join_own<D, NW>(acc, reinterpret_cast<float*>(ks0), w, lane);
    if (w) return;
  }
  if (own) store_own<T, D>((T*)p.dq + row * p.dqr + (long long)head * p.dqh, acc, f, p.d, h);
}

// ---- backward: dk and dv -------------------------------------------------------------------------
// A workgroup owns 32 NW keys of one key head and walks the queries that see any of them, head after head of its group.
// With p.parts > 1 that walk is cut into as many ranges, one per workgroup (blockIdx.y), whose sums go to the workspace in
// fp32 and are added in order by attn_bwd_sum: few workgroups with long walks would leave most of the chip idle.
// Four products.  The two accumulators and the own keys and values fill the registers: at 128 channels one wave per SIMD, and
// vector work (exp, masks, packing) is not hidden behind another wave's matrix instructions: 2.65 ms, 830 TFLOP/s at the size above.
// Staged rows behind the sequence are zeros, or pieces of its last rows where rows repeat or overlap (a stride below the
// row's length); their -lse is set to -infinity, so their p and ds are zero whatever is there.
template <typename T, int D, int DK, int NW, bool FINE>
__global__ __launch_bounds__(64 * NW, (sizeof(T) == 4 && D > 64) || D == 128 ? 1 : 2) void attn_bwd_kv(const AttnP p) {
  typedef Op<T> O; typedef Tile<T, D> L; typedef typename O::frag frag;
  constexpr bool F16 = __is_same(T, _Float16);
  constexpr int QT = sizeof(T) == 4 ? 32 : 64, KB = 32 * NW, NC = DK / O::CH;
  __shared__ __attribute__((aligned(16))) T qs0[QT * D];
  __shared__ __attribute__((aligned(16))) T ds0[QT * D];
  __shared__ __attribute__((aligned(16))) T qs1[QT * D];
  __shared__ __attribute__((aligned(16))) T ds1[QT * D];
  __shared__ __attribute__((aligned(16))) float cs0[2][64];   // per staged query: -delta, -lse (log2; fp16: 14 more)
  __shared__ __attribute__((aligned(16))) float cs1[2][64];
  long long b; int n, tile;
  // here already with more than one workgroup a compute unit, which two then share: 16 x 1024 as above 178 / 141 us the whole pass
  const bool longest = p.block && gridDim.x * gridDim.y > 256;
  if (!(longest ? locate_longest(p, blockIdx.x / p.kv_heads, KB, b, n, tile) : locate(p, blockIdx.x / p.kv_heads, KB, b, n, tile))) return;
  if (longest) tile = (n + KB - 1) / KB - 1 - tile;         // the first keys have the longest walks
  const int kv = blockIdx.x % p.kv_heads, group = p.heads / p.kv_heads;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const int k0 = tile * KB, kw = k0 + 32 * w, ki = kw + (lane & 31);
  const bool own = ki < n;
  const int qmin = p.block ? ki / p.block * p.block : 0;              // the first query that sees the lane's key
  const int wave_max = p.block ? (kw + 31) / p.block * p.block : 0;   // the first that sees all keys of the wave
  const int all_max = p.block ? (min(k0 + KB, n) - 1) / p.block * p.block : 0;     // .. all keys of the workgroup
  const int qbeg = p.block ? k0 / p.block * p.block / QT * QT : 0;    // the first tile with a query that sees key k0
  const int ntile = (n - qbeg + QT - 1) / QT, total = ntile * group;
  const int it0 = (int)((long long)total * blockIdx.y / p.parts), it1 = (int)((long long)total * (blockIdx.y + 1) / p.parts);

  const Fetch<T, D, QT, NW> into_q(p.qr, p.d, w, lane), into_d(p.dor, p.d, w, lane);
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
  [[maybe_unused]] int ex = 0;                          // F16: ak and ds are scaled by mul = 2^-ex
  [[maybe_unused]] float mul = 1.f;
  [[maybe_unused]] const long long plane = (long long)p.heads * p.rows;

  int fhead = kv * group + it0 / ntile, fq = it0 % ntile, wq = fq;       // the next tile to fetch and to work on (counted: a division per tile is 6 % of the time)
  auto fetch = [&](int, T* q, T* d, float (&cs)[2][64]) {
    const int q0 = qbeg + fq * QT, head = fhead;
    if (++fq == ntile) { fq = 0; ++fhead; }
    into_q((const T*)p.q + (b + q0) * p.qr + (long long)head * p.qh, n - q0, q, w);
    into_d((const T*)p.dout + (b + q0) * p.dor + (long long)head * p.doh, n - q0, d, w);
    // constants: one request of 64 floats each (fp32 stages 32 queries and asks for 32 more than it needs)
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (w == k % NW) REQUEST(p.delta + k * plane + (long long)head * p.rows + b + q0, 4 * min(n - q0, 64), cs[k], 4, 4 * lane);
  };
  auto work = [&](int, T* qt, T* dt_, float (&cs)[2][64]) {
    const int q0 = qbeg + wq * QT;
    if (++wq == ntile) wq = 0;
    const bool edge = q0 < all_max, tail = q0 + QT > n;
    if (tail && w == 0 && lane >= n - q0) cs[1][lane] = -INFINITY;
    if (edge) {
      auto mark = [&](int id) { cs[1][id / (D / O::E)] = NAN; };
      quarantine<T, D, QT, NW>(qt, w, lane, mark);
      quarantine<T, D, QT, NW>(dt_, w, lane, mark);
    }
    if (edge || tail) lds_barrier();
    if (kw >= n) return;
#pragma unroll D == 128 ? 1 : 2
    for (int t = 0; t < QT / 32; ++t) {
      f32x16 s, dp;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 c1 = *reinterpret_cast<const f32x4*>(&cs[0][32 * t + 8 * g + 4 * h]);
#pragma unroll
        for (int i = 0; i < 4; ++i) { s[4 * g + i] = 0.f; dp[4 * g + i] = c1[i]; }
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        s = O::mma(L::row_frag(qt, 32 * t, c, lane), kf[c], s);
        dp = O::mma(L::row_frag(dt_, 32 * t, c, lane), vf[c], dp);
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 c0 = *reinterpret_cast<const f32x4*>(&cs[1][32 * t + 8 * g + 4 * h]);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[4 * g + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * g + i], sl2, c0[i]));
      }
      if (sizeof(T) == 2) feed<12, 1, 2 * NC, 0>();
      if (q0 + 32 * t < wave_max) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (q0 + 32 * t + acc_row(r, h) < qmin) { s[r] = 0.f; dp[r] = 0.f; }       // p = 0 does not hide an infinite do v
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] *= s[r];
      if constexpr (F16) fit_half<false>(dp, ak, ex, mul);
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          sum_apart<T, D>(dt_, s, t, i, lane, av[i]);
          sum_apart<T, D>(qt, dp, t, i, lane, ak[i]);
        }
      } else
#pragma unroll
      for (int c = 0; c < 32 / O::CH; ++c) {
        const frag pf = O::pack(s, c), gf = O::pack(dp, c);
        [[maybe_unused]] frag pr, gr;
        if constexpr (FINE) { pr = O::rest(s, c, pf); gr = O::rest(dp, c, gf); }
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
          const frag df = L::col_frag(dt_, t * (32 / O::CH) + c, i, lane), qf = L::col_frag(qt, t * (32 / O::CH) + c, i, lane);
          av[i] = O::mma(df, pf, av[i]);
          ak[i] = O::mma(qf, gf, ak[i]);
          if constexpr (FINE) { av[i] = O::mma(df, pr, av[i]); ak[i] = O::mma(qf, gr, ak[i]); }
        }
      }
      if (sizeof(T) == 2 && !FINE) feed<8, 2, D / 8, 1>();
    }
  };
#define FETCH(it, buf) fetch(it, buf ? qs1 : qs0, buf ? ds1 : ds0, buf ? cs1 : cs0)
#define WORK(it, buf) work(it, buf ? qs1 : qs0, buf ? ds1 : ds0, buf ? cs1 : cs0)
  if (it1 > it0) { WALK(it1 - it0, FETCH, WORK) }
#undef FETCH
#undef WORK
  if (own) {
    const float f = F16 ? __builtin_amdgcn_ldexpf(p.scale, ex - P_EXP) : p.scale, fv = F16 ? __builtin_amdgcn_ldexpf(1.f, -P_EXP) : 1.f;
    if (p.parts > 1) {
      const long long half = p.rows * p.kv_heads * p.d;
      float* dst = p.partial + 2 * half * blockIdx.y + ((b + ki) * p.kv_heads + kv) * p.d;
      store_own<float, D>(dst, ak, f, p.d, h);
      store_own<float, D>(dst + half, av, fv, p.d, h);
      return;
    }
    store_own<T, D>((T*)p.dk + (b + ki) * p.dkr + (long long)kv * p.dkh, ak, f, p.d, h);
    store_own<T, D>((T*)p.dv + (b + ki) * p.dvr + (long long)kv * p.dvh, av, fv, p.d, h);
  }
}

// dk and dv from the parts' sums; a thread takes four channels of a row.  Bound by reading 8 parts bytes per element.
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_sum(const AttnP p) {
  const long long half = p.rows * p.kv_heads * p.d, e = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (e >= half) return;
  const int ch = (int)(e % p.d);
  const long long rh = e / p.d, row = rh / p.kv_heads;
  const int kv = (int)(rh - row * p.kv_heads);
  // rows of no sequence stay as they are
  const long long lo = p.cu ? p.cu[0] : 0, hi = p.cu ? p.cu[p.nseq] : (long long)p.nseq * p.seqlen;
  if (row < lo || row >= hi) return;
  const float* src = p.partial + (blockIdx.y ? half : 0) + e;
  f32x4 s = *reinterpret_cast<const f32x4*>(src);
  for (int i = 1; i < p.parts; ++i) s += *reinterpret_cast<const f32x4*>(src + 2 * half * i);
  T* dst = blockIdx.y ? (T*)p.dv + row * p.dvr + (long long)kv * p.dvh : (T*)p.dk + row * p.dkr + (long long)kv * p.dkh;
  store4<T>(dst + ch, s[0], s[1], s[2], s[3]);
}

long long slots(const AttnP& p, int tr) {
  return p.cu ? p.rows / tr + p.nseq : (long long)p.nseq * ((p.seqlen + tr - 1) / tr);
}
template <typename T, int D, int DK, int NW, bool SPLIT> int fwd(const AttnP& p, hipStream_t st) {
  attn_fwd<T, D, DK, NW, SPLIT><<<dim3((unsigned)(slots(p, Walk<T, D, NW, SPLIT>::QT) * p.heads)), 64 * NW, 0, st>>>(p);
  return hipGetLastError() != hipSuccess;
}
// FINE: the rounding of ds and p to 16 bits is as large as the results' own; both together are 1.41 times that, 1.48 with the
// rounding of out in delta.  Small calls (all gradients), where few terms make up a result, and narrow heads (dq), where delta counts
// more, come to 1.5 .. 1.8 times; there ds and p enter the products in two pieces.  dq, dk, dv against 64 bits, in errors of the
// plain form, one piece / two, bf16: 46 tokens, 2 heads of 16, causal, 1.67 1.48 1.29 / 1.03 1.02 1.00; 2258 + 257 tokens, 4 heads of 16, dq
// 1.53 / 1.08; 906 random calls with this rule: 1.50 at most.  Backward pass, us: 10 x 100 tokens, 4 heads of 16, 10.6 / 11.6; 8 x 512, 8
// heads of 24 (dq alone), causal, 28.6 / 31.2.  With no need for it: dq of heads of 32 426 for 352 (8 x 2048 tokens, 16 heads, fp16); 702 + 223
// tokens, 2 heads of 80, causal, with the forward pass 59 for 51.
template <typename T, int D, int DK, int NW, bool SPLIT, bool FINE> int bwd_q(const AttnP& p, hipStream_t st) {
  attn_bwd_q<T, D, DK, NW, SPLIT, FINE><<<dim3((unsigned)(slots(p, Walk<T, D, NW, SPLIT>::QT) * p.heads)), 64 * NW, 0, st>>>(p);
  return hipGetLastError() != hipSuccess;
}
template <typename T, int D, int DK, bool FINE> int bwd_kv(const AttnP& p, hipStream_t st) {
  attn_bwd_kv<T, D, DK, 4, FINE><<<dim3((unsigned)(slots(p, 128) * p.kv_heads), (unsigned)p.parts), 256, 0, st>>>(p);
  return hipGetLastError() != hipSuccess;
}
template <typename T, int D, int DK, int NW, bool SPLIT> int bwd(const AttnP& p, hipStream_t st) {
  constexpr bool HALF = sizeof(T) == 2;
  const bool small = HALF && p.rows * p.heads <= (p.d <= 24 ? 4096 : 1024);
  if constexpr (HALF && (SPLIT || D == 32)) {                // small calls are split
    if (small || p.d <= 24 ? bwd_q<T, D, DK, NW, SPLIT, true>(p, st) : bwd_q<T, D, DK, NW, SPLIT, false>(p, st)) return 1;
  } else if (bwd_q<T, D, DK, NW, SPLIT, false>(p, st)) return 1;
  if (small ? bwd_kv<T, D, DK, HALF>(p, st) : bwd_kv<T, D, DK, false>(p, st)) return 1;
  if (p.parts == 1) return 0;
  attn_bwd_sum<T><<<dim3((unsigned)((p.rows * p.kv_heads * p.d / 4 + 255) / 256), 2), 256, 0, st>>>(p);
  return hipGetLastError() != hipSuccess;
}
// Forward and dq, few rows: with W = rows * heads / 32 waves of queries and 1024 SIMDs, splitting the keys over the waves of
// a workgroup pays up to W = 512 where two such workgroups fit a compute unit (D <= 64), to 256 above, and to twice that
// for causal walks over long sequences, whose last tiles keep the rest waiting.  Forward, us, split / not:
//   fp32 D 64:  16 x 1024 tokens x 1 head (W 512) 60 / 82;  4 x 1024 x 8 (W 1024) 102 / 81;  1 x 4096 x 8 causal 199 / 292
//   bf16 D 128: 1 x 4096 x 2 (W 256) 46 / 80;  16 x 1024 x 1 (W 512) 33 / 26;  1 x 16384 x 1 causal (W 512) 176 / 288
template <typename T, int D, int DK, bool BWD> int run(const AttnP& p, hipStream_t st) {
  constexpr int NS = sizeof(T) == 4 && D > 64 ? 2 : 4;      // waves whose buffers fit LDS
  const long long w = p.rows * p.heads / 32, most = (D <= 64 ? 512 : 256) * (p.block && p.rows / p.nseq >= 2048 ? 2 : 1);
  if (w <= most) { if constexpr (BWD) return bwd<T, D, DK, NS, true>(p, st); else return fwd<T, D, DK, NS, true>(p, st); }
  if constexpr (BWD) return bwd<T, D, DK, 4, false>(p, st); else return fwd<T, D, DK, 4, false>(p, st);
}
// D: channels of the tiles and of the results, 32 at a time; DK: channels of the score products.  In fp32, which the matrix unit
// bounds, 16 of padding are left out there: 64 images of 196 tokens, 8 heads of 48, forward / dq / dk and dv 77 / 108 / 144 us under a profiler,
// with all 64 channels 88 / 125 / 159.  In 16 bits it gives nothing (fp16, heads of 80 as 80 or 96 channels: 80 / 101 / 144, 78 / 104 / 143).
template <typename T, bool BWD> int run_d(const AttnP& p, hipStream_t st) {
  if constexpr (sizeof(T) == 4)
    if (p.d > 32 && p.d <= 48) return run<T, 64, 48, BWD>(p, st);
  return p.d <= 32 ? run<T, 32, 32, BWD>(p, st) : p.d <= 64 ? run<T, 64, 64, BWD>(p, st) : p.d <= 96 ? run<T, 96, 96, BWD>(p, st) : run<T, 128, 128, BWD>(p, st);
}
template <bool BWD> int run_t(const AttnP& p, int dtype, hipStream_t st) {
  return dtype == OP_F32 ? run_d<float, BWD>(p, st) : dtype == OP_BF16 ? run_d<__bf16, BWD>(p, st) : run_d<_Float16, BWD>(p, st);
}

}  // namespace

// dk/dv: parts until there is a workgroup per compute unit, and four where the walks are causal and long; a part keeps at
// least 256 queries (fp32 128).  Whole backward pass, us, 1 / 2 / 4 parts:
//   fp32 D 64: 16 x 1024 tokens x 1 head 212 / 159 / 161;  4 x 1024 x 8: 250 / 253 / 263;  1 x 4096 x 8 causal 810 / 772 / 644
//   bf16 D 64: 1 x 4096 x 2: 108 / 79 / 66;  16 x 1024 x 4: 78 / 100 / 120;  12 packed clips of very different lengths, 12 of 4 heads,
//   causal, with the forward pass 450 / 397 / 406
int attention_parts(int dtype, long long rows, int nseq, int heads, int kv_heads, int block) {
  if (nseq < 1) return 1;
  const long long blocks = (rows / 128 + nseq) * kv_heads, walk = rows / nseq * (heads / kv_heads);
  long long parts = ((block && walk >= 4096 ? 1024 : 256) + blocks - 1) / blocks;
  const long long most = walk / (dtype == OP_F32 ? 128 : 256);
  if (parts > most) parts = most;
  return parts < 1 ? 1 : parts > 8 ? 8 : (int)parts;
}
int launch_attention_fwd(const AttnP& p, int dtype, hipStream_t st) { return run_t<false>(p, dtype, st); }
int launch_attention_bwd(const AttnP& p, int dtype, hipStream_t st) { return run_t<true>(p, dtype, st); }
