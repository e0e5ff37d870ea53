// op_api.hip -- C entry points of the stand-alone operators (include/cora_hip.h): argument checks, then one launch set.
#include "../../include/cora_hip.h"
#include "ops.h"

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <vector>

void cora_note_error(const char* msg) noexcept;   // ctx.hip

namespace {

int refuse(const char* fmt, ...) {
  char buf[320];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  cora_note_error(buf);
  return -1;
}

// the caller's current device is left as it was
struct OnDevice {
  int prev = -1; bool ok = false;
  explicit OnDevice(int device) {
    if (hipGetDevice(&prev) != hipSuccess) { prev = -1; (void)hipGetLastError(); return; }
    ok = prev == device || hipSetDevice(device) == hipSuccess;
    if (!ok) (void)hipGetLastError();
    else (void)hipGetLastError();                     // an error of an earlier call of the caller is not this launch's
    if (prev == device) prev = -1;
  }
  ~OnDevice() { if (prev >= 0) (void)hipSetDevice(prev); }
};

// rows x heads x d elements at strides (row, head) do not overlap each other
bool disjoint(long long rows, long long heads, long long d, long long sr, long long sh) {
  if (sr < 0 || sh < 0) return false;
  if (rows <= 1 && heads <= 1) return true;
  if (rows <= 1) return sh >= d;
  if (heads <= 1) return sr >= d;
  return (sh >= d && sr >= (heads - 1) * sh + d) || (sr >= d && sh >= (rows - 1) * sr + d);
}
// n0 x n1 pieces of w bytes, s0 and s1 bytes apart
struct Span {
  long long at, n0, s0, n1, s1, w;
  long long end() const { return at + (n0 - 1) * s0 + (n1 - 1) * s1 + w; }
  bool gapless() const {
    const bool swap = n1 <= 1 || (n0 > 1 && s0 < s1);
    const long long a = swap ? s0 : s1, na = swap ? n0 : n1, b = swap ? s1 : s0, nb = swap ? n1 : n0;
    const long long inner = (na - 1) * a + w;
    return (na <= 1 || a <= w) && (nb <= 1 || b <= inner);
  }
};
Span bytes(const void* p, long long n) { return Span{(long long)(uintptr_t)p, 1, 0, 1, 0, n}; }
// Do they share memory?  Decided where one of the two strides agrees, as views of one buffer do, and where neither has gaps; what
// this leaves open (interleaved pieces of different strides) is the caller's to know.
bool meet(Span a, Span b) {
  if (a.at >= b.end() || b.at >= a.end()) return false;
  if (a.gapless() && b.gapless()) return true;
  auto same = [](long long na, long long sa, long long nb, long long sb) { return na <= 1 || nb <= 1 || sa == sb; };
  const bool one = same(a.n0, a.s0, b.n0, b.s0), two = same(a.n1, a.s1, b.n1, b.s1);
  if (!one && !two) return false;
  if (!one || (two && a.n0 + b.n0 < a.n1 + b.n1))             // dimension 0 is solved for, dimension 1 tried out
    for (Span* s : {&a, &b}) { const long long n = s->n0, st = s->s0; s->n0 = s->n1; s->s0 = s->s1; s->n1 = n; s->s1 = st; }
  const long long r = a.n0 > 1 ? a.s0 : b.s0;
  auto hit = [&](long long o) {                               // is there a d with -a.w < o + d r < b.w?
    long long lo = -(b.n0 - 1), hi = a.n0 - 1;
    if (r == 0) return -a.w < o && o < b.w;
    auto floor_div = [](long long x, long long y) { return x / y - (x % y < 0); };
    const long long first = floor_div(-a.w - o, r) + 1, last = -floor_div(o - b.w, r) - 1;
    if (first > lo) lo = first;
    if (last < hi) hi = last;
    return lo <= hi;
  };
  if (same(a.n1, a.s1, b.n1, b.s1)) {
    const long long st = a.n1 > 1 ? a.s1 : b.s1;
    for (long long k = -(b.n1 - 1); k < a.n1; ++k)
      if (hit(a.at - b.at + k * st)) return true;
  } else if (a.n1 * b.n1 <= 4096)
    for (long long i = 0; i < a.n1; ++i)
      for (long long j = 0; j < b.n1; ++j)
        if (hit(a.at + i * a.s1 - b.at - j * b.s1)) return true;
  return false;
}
bool bad_dtype(int dtype) { return dtype < CORA_F32 || dtype > CORA_F16; }

int check_attention(const cora_attention_args* a, AttnP* p, const char* who, bool backward) {
  if (!a) return refuse("%s: null argument", who);
  if (bad_dtype(a->dtype)) return refuse("%s: dtype must be CORA_F32, CORA_BF16 or CORA_F16", who);
  if (a->heads < 1 || a->kv_heads < 1 || a->heads > 65535 || a->heads % a->kv_heads)
    return refuse("%s: heads (%d) must be a positive multiple of kv_heads (%d)", who, a->heads, a->kv_heads);
  const int v = 16 / op_bytes(a->dtype);
  if (a->head_dim < 1 || a->head_dim > 128 || a->head_dim % v)
    return refuse("%s: head_dim %d must be a multiple of %d and at most 128", who, a->head_dim, v);
  if (a->rows < 0 || a->rows >= (1LL << 31)) return refuse("%s: rows must be below 2^31", who);
  if (a->n_seq < 0) return refuse("%s: n_seq is negative", who);
  if (a->causal_block < 0) return refuse("%s: causal_block is negative", who);
  if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return refuse("%s: scale must be positive and finite", who);
  if (!a->cu_seqlens && a->n_seq > 0 && (a->seq_len < 1 || (long long)a->n_seq * a->seq_len > a->rows))
    return refuse("%s: n_seq * seq_len must be at most rows, seq_len at least 1", who);
  if (a->rows == 0 || a->n_seq == 0) return 1;                                  // nothing to do
  struct Ref { const char* name; const void* ptr; long long row, head; int heads; bool out, bwd; };
  const Ref refs[] = {
    {"q", a->q, a->q_row, a->q_head, a->heads, false, false}, {"k", a->k, a->k_row, a->k_head, a->kv_heads, false, false},
    {"v", a->v, a->v_row, a->v_head, a->kv_heads, false, false}, {"out", a->out, a->out_row, a->out_head, a->heads, !backward, false},
    {"dout", a->dout, a->dout_row, a->dout_head, a->heads, false, true}, {"dq", a->dq, a->dq_row, a->dq_head, a->heads, true, true},
    {"dk", a->dk, a->dk_row, a->dk_head, a->kv_heads, true, true}, {"dv", a->dv, a->dv_row, a->dv_head, a->kv_heads, true, true}};
  for (const Ref& r : refs) {
    if (r.bwd && !backward) continue;
    if (!r.ptr) return refuse("%s: %s is NULL", who, r.name);
    if ((uintptr_t)r.ptr % 16 || r.row % v || r.head % v || r.row < 0 || r.head < 0)
      return refuse("%s: %s must be 16-byte aligned with non-negative strides that are multiples of 16 bytes", who, r.name);
    if (r.row >= (1LL << 24)) return refuse("%s: the row stride of %s must be below 2^24 elements", who, r.name);
    if (r.out && !disjoint(a->rows, r.heads, a->head_dim, r.row, r.head)) return refuse("%s: rows or heads of %s overlap", who, r.name);
  }
  if (!a->lse || (uintptr_t)a->lse % 4 || (a->cu_seqlens && (uintptr_t)a->cu_seqlens % 4))
    return refuse("%s: lse is NULL, or lse or cu_seqlens is not 4-byte aligned", who);
  // workgroups of up to 256 threads, fewer than 2^32 threads: one per 128 rows of a sequence and head (32 where there are few rows)
  const long long tiles = a->cu_seqlens ? a->rows / 128 + a->n_seq : a->n_seq * (((long long)a->seq_len + 127) / 128);
  if ((tiles + 1024) * a->heads >= (1LL << 24)) return refuse("%s: too many tiles for one launch", who);
  if (backward) {
    if (!a->workspace || (uintptr_t)a->workspace % 16 || a->workspace_bytes < cora_attention_workspace(a))
      return refuse("%s: workspace is NULL, not 16-byte aligned or smaller than cora_attention_workspace says (%zu bytes)", who,
                    cora_attention_workspace(a));
  }
  for (const Ref& r : refs)
    for (const Ref& s : refs)
      if (r.out && &r != &s && (backward || !s.bwd) && r.ptr == s.ptr) return refuse("%s: %s is %s", who, r.name, s.name);
  const long long eb = op_bytes(a->dtype);
  auto span = [&](const Ref& r) { return Span{(long long)(uintptr_t)r.ptr, a->rows, r.row * eb, r.heads, r.head * eb, a->head_dim * eb}; };
  struct Flat { const char* name; Span s; bool out; } flat[] = {
    {"lse", bytes(a->lse, 4LL * a->heads * a->rows), !backward}, {"cu_seqlens", bytes(a->cu_seqlens, a->cu_seqlens ? 4LL * (a->n_seq + 1) : 0), false},
    {"workspace", bytes(a->workspace, backward ? (long long)cora_attention_workspace(a) : 0), backward}};
  for (const Ref& r : refs) {
    if (r.bwd && !backward) continue;
    if (r.out)
      for (const Ref& s : refs)
        if (&r != &s && (backward || !s.bwd) && meet(span(r), span(s))) return refuse("%s: %s overlaps %s", who, r.name, s.name);
    for (const Flat& f : flat)
      if (f.s.w && (r.out || f.out) && meet(span(r), f.s)) return refuse("%s: %s overlaps %s", who, r.name, f.name);
  }
  for (const Flat& f : flat)
    for (const Flat& g : flat)
      if (&f != &g && f.out && f.s.w && g.s.w && meet(f.s, g.s)) return refuse("%s: %s overlaps %s", who, f.name, g.name);
  memset(p, 0, sizeof *p);
  p->q = a->q; p->k = a->k; p->v = a->v; p->out = a->out; p->o = a->out; p->lse = a->lse;
  p->dout = a->dout; p->dq = a->dq; p->dk = a->dk; p->dv = a->dv; p->cu = a->cu_seqlens;
  p->rows = a->rows;
  p->qr = a->q_row; p->qh = a->q_head; p->kr = a->k_row; p->kh = a->k_head; p->vr = a->v_row; p->vh = a->v_head;
  p->orow = a->out_row; p->oh = a->out_head; p->dor = a->dout_row; p->doh = a->dout_head;
  p->dqr = a->dq_row; p->dqh = a->dq_head; p->dkr = a->dk_row; p->dkh = a->dk_head; p->dvr = a->dv_row; p->dvh = a->dv_head;
  p->nseq = a->n_seq; p->seqlen = a->seq_len; p->heads = a->heads; p->kv_heads = a->kv_heads; p->d = a->head_dim;
  p->block = a->causal_block; p->scale = a->scale;
  if (backward) attention_ws(*p, a->dtype, a->workspace);
  return 0;
}

OrthoG& add_stack(OrthoP& p, int count, int rows, int cols) {
  OrthoG& g = p.g[p.ngroups++];
  g.count = count; g.rows = rows; g.cols = cols;
  g.m = rows < cols ? rows : cols; g.n = rows < cols ? cols : rows;
  g.ldn = (g.n + 63) / 64 * 64; g.ldm = (g.m + 63) / 64 * 64;
  g.sn = g.ldn | 64; g.sm = g.ldm | 64;
  g.first = p.matrices;
  p.matrices += count;
  return g;
}

// a launch has fewer than 2^32 threads, 256 a tile (and some idle ones)
constexpr long long ORTHO_TILES = 1LL << 22;
long long tiles_64(const cora_matrices& s) { return ((long long)s.rows + 63) / 64 * ((s.cols + 63) / 64) * s.count; }

// up to ORTHO_GROUPS stacks from stacks[i0]; returns how many were taken
int take_stacks(const cora_matrices* stacks, int i0, int n, OrthoP* p) {
  p->ngroups = 0; p->matrices = 0;
  int i = i0;
  long long tiles = 0;
  for (; i < n && p->ngroups < ORTHO_GROUPS; ++i) {
    const cora_matrices& s = stacks[i];
    if (s.count == 0) continue;
    tiles += tiles_64(s);
    if (p->matrices + s.count > 65535 || (p->ngroups && tiles >= ORTHO_TILES)) break;
    OrthoG& g = add_stack(*p, s.count, s.rows, s.cols);
    g.x = s.x; g.y = s.y; g.xm = s.x_mat; g.xr = s.x_row; g.ym = s.y_mat; g.yr = s.y_row;
  }
  return i - i0;
}

int check_stacks(int dtype, const cora_matrices* s, int n, const char* who) {
  if (bad_dtype(dtype)) return refuse("%s: dtype must be CORA_F32, CORA_BF16 or CORA_F16", who);
  if (n < 0 || (n > 0 && !s)) return refuse("%s: null argument", who);
  for (int i = 0; i < n; ++i) {
    if (s[i].count < 0 || s[i].count > 65535 || s[i].rows < 1 || s[i].cols < 1 || s[i].rows > 32768 || s[i].cols > 32768)
      return refuse("%s: stack %d: count must be 0 .. 65535, rows and cols 1 .. 32768", who, i);
    if (tiles_64(s[i]) >= ORTHO_TILES) return refuse("%s: stack %d: too many tiles for one launch", who, i);
  }
  return 0;
}

}  // namespace

// the iterates' formats hold singular values up to 8 and products up to 1000: follow the interval of singular values
int ortho_bad_step(int steps, const float* coef) {
  float sv[257];
  for (int i = 0; i <= 256; ++i) sv[i] = i / 256.f;
  for (int s = 0; s < steps; ++s)
    for (float& x : sv) {
      const float l = x * x, g = coef[3 * s + 1] * l + coef[3 * s + 2] * l * l, f = coef[3 * s] + g;   // g: of b A + c A^2 alone
      x = fabsf(x * f);
      if (!(fabsf(f) <= 1000.f) || !(fabsf(g) <= 1000.f) || !(x <= 8.f) || !(fabsf(coef[3 * s]) <= 1000.f)) return s;
    }
  return -1;
}

void fill_rotary(RotaryP& p, int n_axes, const int* axes_dim, double theta, bool interleaved) {
  int c = 0, k = 0;
  for (int i = 0; i < n_axes; ++i) {
    const int n = axes_dim[i];
    for (int j = 0; j < n / 2; ++j, ++k) {
      p.axis[k] = (unsigned char)i;
      p.c0[k] = (unsigned char)(c + (interleaved ? 2 * j : j));
      p.c1[k] = (unsigned char)(c + (interleaved ? 2 * j + 1 : j + n / 2));
      p.turn[k] = std::pow(theta, -2.0 * j / n) / 6.283185307179586476925286766559;
    }
    c += n;
  }
  p.n_axes = n_axes; p.pairs = k; p.interleaved = interleaved;
}

void fill_stack(OrthoP& p, const float* x, float* y, int count, int rows, int cols) {
  OrthoG& g = add_stack(p, count, rows, cols);
  g.x = x; g.y = y; g.xr = g.yr = cols; g.xm = g.ym = (long long)rows * cols;
}

void ortho_place(OrthoP& p, void* ws) {
  p.parts = (double*)ws;
  p.ws = (unsigned short*)((char*)ws + ((size_t)p.matrices * ORTHO_PARTS * sizeof(double) + 255) / 256 * 256);
}

static size_t constants_bytes(long long rows, int heads) { return ((size_t)rows * heads * 2 * sizeof(float) + 15) / 16 * 16; }
size_t attention_ws_bytes(int dtype, long long rows, int nseq, int heads, int kv_heads, int d, int block) {
  const int parts = attention_parts(dtype, rows, nseq, heads, kv_heads, block);
  return constants_bytes(rows, heads) + (parts > 1 ? (size_t)parts * 2 * sizeof(float) * (size_t)rows * (size_t)kv_heads * (size_t)d : 0);
}
void attention_ws(AttnP& p, int dtype, void* ws) {
  p.parts = attention_parts(dtype, p.rows, p.nseq, p.heads, p.kv_heads, p.block);
  p.delta = (float*)ws;
  p.partial = (float*)((char*)ws + constants_bytes(p.rows, p.heads));
}

extern "C" {

int cora_rotary(const cora_rotary_args* a, int device, void* hip_stream) {
  const char* who = "cora_rotary";
  if (!a) return refuse("%s: null argument", who);
  if (bad_dtype(a->dtype)) return refuse("%s: dtype must be CORA_F32, CORA_BF16 or CORA_F16", who);
  if (a->heads < 1 || a->heads > 65535 || a->head_dim < 2) return refuse("%s: heads must be 1 .. 65535, head_dim at least 2", who);
  if (a->n_axes < 1 || a->n_axes > 4) return refuse("%s: n_axes must be 1 .. 4", who);
  int sum = 0;
  for (int i = 0; i < a->n_axes; ++i) {
    if (a->axes_dim[i] < 2 || a->axes_dim[i] % 2 || a->axes_dim[i] > 128) return refuse("%s: axes_dim[%d] = %d must be positive, even and at most 128", who, i, a->axes_dim[i]);
    sum += a->axes_dim[i];
  }
  if (sum > a->head_dim || sum > 128) return refuse("%s: the axes take %d channels, head_dim is %d (and at most 128 may turn)", who, sum, a->head_dim);
  if (!(a->theta > 0.0) || !std::isfinite(a->theta)) return refuse("%s: theta must be positive and finite", who);
  if (a->rows < 0 || a->pos_rows < 1) return refuse("%s: rows is negative or pos_rows not positive", who);
  if (a->rows == 0) return 0;
  if (!a->x || !a->y || !a->pos) return refuse("%s: x, y or pos is NULL", who);
  const int eb = op_bytes(a->dtype);
  if ((uintptr_t)a->x % eb || (uintptr_t)a->y % eb || (uintptr_t)a->pos % 4) return refuse("%s: a pointer is not aligned to its element size", who);
  if (a->x_row < 0 || a->x_head < 0) return refuse("%s: negative stride", who);
  if (!disjoint(a->rows, a->heads, a->head_dim, a->y_row, a->y_head)) return refuse("%s: rows or heads of y overlap", who);
  if (a->x == a->y && ((a->rows > 1 && a->x_row != a->y_row) || (a->heads > 1 && a->x_head != a->y_head)))
    return refuse("%s: in place, x and y need the same strides", who);
  if (a->rows > (1LL << 39) / a->head_dim) return refuse("%s: too many rows for one launch", who);
  const Span y{(long long)(uintptr_t)a->y, a->rows, a->y_row * eb, a->heads, a->y_head * eb, (long long)a->head_dim * eb};
  if (a->x != a->y && meet(y, Span{(long long)(uintptr_t)a->x, a->rows, a->x_row * eb, a->heads, a->x_head * eb, y.w})) return refuse("%s: y overlaps x", who);
  if (meet(y, bytes(a->pos, a->pos_rows * a->n_axes * 4))) return refuse("%s: y overlaps pos", who);
  RotaryP p;
  memset(&p, 0, sizeof p);
  p.x = a->x; p.y = a->y; p.pos = a->pos; p.rows = a->rows; p.pos_rows = a->pos_rows;
  p.xr = a->x_row; p.xh = a->x_head; p.yr = a->y_row; p.yh = a->y_head;
  p.heads = a->heads; p.d = a->head_dim; p.copy = a->x != a->y; p.sign = a->backward ? -1.f : 1.f;
  fill_rotary(p, a->n_axes, a->axes_dim, a->theta, a->interleaved != 0);
  OnDevice dev(device);
  if (!dev.ok) return refuse("%s: device %d is not available", who, device);
  if (launch_rotary(p, a->dtype, (hipStream_t)hip_stream)) { refuse("%s: launch failed", who); return -3; }
  return 0;
}

size_t cora_attention_workspace(const cora_attention_args* a) {
  if (!a || a->heads < 1 || a->kv_heads < 1 || a->head_dim < 1 || a->rows < 1 || a->n_seq < 0) return 16;
  return attention_ws_bytes(a->dtype, a->rows, a->n_seq, a->heads, a->kv_heads, a->head_dim, a->causal_block);
}

int cora_attention(const cora_attention_args* a, int device, void* hip_stream) {
  AttnP p;
  if (int rc = check_attention(a, &p, "cora_attention", false)) return rc > 0 ? 0 : rc;
  OnDevice dev(device);
  if (!dev.ok) return refuse("cora_attention: device %d is not available", device);
  if (launch_attention_fwd(p, a->dtype, (hipStream_t)hip_stream)) { refuse("cora_attention: launch failed"); return -3; }
  return 0;
}

int cora_attention_backward(const cora_attention_args* a, int device, void* hip_stream) {
  AttnP p;
  if (int rc = check_attention(a, &p, "cora_attention_backward", true)) return rc > 0 ? 0 : rc;
  OnDevice dev(device);
  if (!dev.ok) return refuse("cora_attention_backward: device %d is not available", device);
  if (launch_attention_bwd(p, a->dtype, (hipStream_t)hip_stream)) { refuse("cora_attention_backward: launch failed"); return -3; }
  return 0;
}

size_t cora_orthogonalize_workspace(int dtype, const cora_matrices* stacks, int n_stacks) {
  if (check_stacks(dtype, stacks, n_stacks, "cora_orthogonalize_workspace")) return 0;
  size_t most = 256;
  OrthoP p;
  for (int i = 0; i < n_stacks;) {                     // batches of stacks take turns in one workspace
    i += take_stacks(stacks, i, n_stacks, &p);
    const size_t b = ortho_ws_bytes(p);
    if (b > most) most = b;
  }
  return most;
}

int cora_orthogonalize(int dtype, const cora_matrices* stacks, int n_stacks, int steps, const float* coef, float eps,
                       void* workspace, size_t workspace_bytes, int device, void* hip_stream) {
  const char* who = "cora_orthogonalize";
  if (int rc = check_stacks(dtype, stacks, n_stacks, who)) return rc;
  if (steps < 1 || steps > ORTHO_STEPS || !coef) return refuse("%s: steps must be 1 .. %d, coef not NULL", who, ORTHO_STEPS);
  if (!(eps >= 0.f) || !std::isfinite(eps)) return refuse("%s: eps must be finite and not negative", who);
  const int bad = ortho_bad_step(steps, coef);
  if (bad >= 0) return refuse("%s: coefficients of step %d drive singular values of [0, 1] out of range", who, bad);
  bool any = false;
  for (int i = 0; i < n_stacks; ++i) {
    const cora_matrices& s = stacks[i];
    if (s.count == 0) continue;
    any = true;
    const int eb = op_bytes(dtype);
    if (!s.x || !s.y || (uintptr_t)s.x % eb || (uintptr_t)s.y % eb) return refuse("%s: stack %d: x or y is NULL or not aligned to its element size", who, i);
    if (s.x_row < 0 || s.x_mat < 0) return refuse("%s: stack %d: negative stride", who, i);
    if (!disjoint(s.rows, s.count, s.cols, s.y_row, s.count > 1 ? s.y_mat : (long long)s.rows * (s.y_row > s.cols ? s.y_row : s.cols)) ||
        (s.rows > 1 && s.y_row < s.cols))
      return refuse("%s: stack %d: rows or matrices of y overlap", who, i);
    if (s.x == s.y && ((s.rows > 1 && s.x_row != s.y_row) || (s.count > 1 && s.x_mat != s.y_mat)))
      return refuse("%s: stack %d: in place, x and y need the same strides", who, i);
  }
  if (!any) return 0;
  const long long eb = op_bytes(dtype);
  auto x_of = [&](const cora_matrices& s) { return Span{(long long)(uintptr_t)s.x, s.count, s.x_mat * eb, s.rows, s.x_row * eb, s.cols * eb}; };
  auto y_of = [&](const cora_matrices& s) { return Span{(long long)(uintptr_t)s.y, s.count, s.y_mat * eb, s.rows, s.y_row * eb, s.cols * eb}; };
  // in the order of their addresses only neighbours need to be compared
  struct Item { Span s; int stack; bool y; };
  std::vector<Item> all;
  try {
    all.reserve(2 * (size_t)n_stacks);
  } catch (...) { return refuse("%s: out of host memory", who); }
  for (int i = 0; i < n_stacks; ++i)
    if (stacks[i].count) { all.push_back({x_of(stacks[i]), i, false}); all.push_back({y_of(stacks[i]), i, true}); }
  std::sort(all.begin(), all.end(), [](const Item& a, const Item& b) { return a.s.at < b.s.at; });
  for (size_t k = 0; k < all.size(); ++k)
    for (size_t l = k + 1; l < all.size() && all[l].s.at < all[k].s.end(); ++l) {
      if (!all[k].y && !all[l].y) continue;
      const bool first = all[k].y && (!all[l].y || all[k].stack < all[l].stack);
      const Item &y = first ? all[k] : all[l], &o = first ? all[l] : all[k];
      if (y.s.at == o.s.at) {
        if (y.stack != o.stack) return refuse("%s: y of stack %d is x or y of stack %d", who, y.stack, o.stack);
      } else if (meet(y.s, o.s)) return refuse("%s: y of stack %d overlaps %c of stack %d", who, y.stack, o.y ? 'y' : 'x', o.stack);
    }
  const size_t need = cora_orthogonalize_workspace(dtype, stacks, n_stacks);
  if (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < need)
    return refuse("%s: workspace is NULL, not 256-byte aligned or smaller than %zu bytes", who, need);
  for (int i = 0; i < n_stacks; ++i)
    if (stacks[i].count && (meet(bytes(workspace, (long long)need), x_of(stacks[i])) || meet(bytes(workspace, (long long)need), y_of(stacks[i]))))
      return refuse("%s: the workspace overlaps stack %d", who, i);
  OnDevice dev(device);
  if (!dev.ok) return refuse("%s: device %d is not available", who, device);
  for (int i = 0; i < n_stacks;) {
    OrthoP p;
    i += take_stacks(stacks, i, n_stacks, &p);
    if (!p.ngroups) continue;
    p.eps = eps;
    ortho_ws_bytes(p);
    ortho_place(p, workspace);
    if (launch_ortho(p, dtype, steps, coef, (hipStream_t)hip_stream)) { refuse("%s: launch failed", who); return -3; }
  }
  return 0;
}

}  // extern "C"
