// op_tile.h -- matrix-unit operand types and the LDS tile layout shared by the stand-alone operators (gfx950).
#pragma once
#include "common.h"

typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

#define LDS3 __attribute__((address_space(3)))

// Direct requests of 16 or 4 bytes a lane: the lane's bytes at base + at go to lds + 16 (4) * lane, zeros where at is behind
// `bytes`.  (The host pass has no buffer descriptor type and silently drops kernels that name one.)
#ifdef __HIP_DEVICE_COMPILE__
#define REQUEST(base, bytes, lds, n, at) \
  __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc((void*)(base), 0, bytes, 0x00020000), (LDS3 void*)(lds), n, at, 0, 0, 0)
#else
#define REQUEST(base, bytes, lds, n, at) (void)0
#endif

template <typename T> struct Op;
template <> struct Op<float> {
  typedef f32x4 frag;
  static constexpr int CH = 8, E = 4;     // contraction values per chunk, per lane piece
  static __device__ __forceinline__ f32x16 mma(const frag a, const frag b, f32x16 c) {
#pragma unroll
    for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[t], b[t], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ frag pack(const f32x16& c, int s) {
    frag f;
#pragma unroll
    for (int t = 0; t < 4; ++t) f[t] = c[4 * s + t];
    return f;
  }
};
template <> struct Op<__bf16> {
  typedef b16x8 frag;
  static constexpr int CH = 16, E = 8;
  static __device__ __forceinline__ f32x16 mma(const frag a, const frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ frag pack(const f32x16& c, int s) {
    frag f;
#pragma unroll
    for (int t = 0; t < 8; ++t) f[t] = (__bf16)c[8 * s + t];
    return f;
  }
  // what pack left of the values, in the same type
  static __device__ __forceinline__ frag rest(const f32x16& c, int s, const frag& p) {
    frag f;
#pragma unroll
    for (int t = 0; t < 8; ++t) f[t] = (__bf16)(c[8 * s + t] - (float)p[t]);
    return f;
  }
};
template <> struct Op<_Float16> {
  typedef h16x8 frag;
  static constexpr int CH = 16, E = 8;
  static __device__ __forceinline__ f32x16 mma(const frag a, const frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ frag pack(const f32x16& c, int s) {
    frag f;
#pragma unroll
    for (int t = 0; t < 8; ++t) f[t] = (_Float16)c[8 * s + t];
    return f;
  }
  static __device__ __forceinline__ frag rest(const f32x16& c, int s, const frag& p) {
    frag f;
#pragma unroll
    for (int t = 0; t < 8; ++t) f[t] = (_Float16)(c[8 * s + t] - (float)p[t]);
    return f;
  }
};

// A tile of R rows x D channels in LDS, rows of D elements without padding; the 16-byte piece c of row r sits at place
// c ^ swz(r), which keeps both reads of a wave off each other's banks: 16 consecutive rows at one piece (row_frag), and
// 4 consecutive rows x 64 bytes (col_frag of 16-bit types) or two rows 4 apart x 128 bytes (fp32).
template <typename T, int D> struct Tile {
  static constexpr int E = Op<T>::E, CH = Op<T>::CH, NP = D / E;   // pieces per row
  static __device__ __forceinline__ int swz(int r) {
    if (sizeof(T) == 4) {
      if (D == 64 || D == 128) return (r & 3) | (((r >> 3) & 1) << 2) | (((r >> 2) & 1) << 3);
      return (r >> 1) & 7;
    }
    const int hi = D >= 128 ? (r & 3) : (D == 64 ? ((r >> 1) & 1) : 0);
    return ((r >> 2) & 3) | (hi << 2);
  }
  static __device__ __forceinline__ int at(int r, int c) { return r * D + ((c ^ swz(r)) * E); }   // element offset of a piece

  // first operand "row r of the tile x chunk c": lane l holds its piece of row r0 + (l & 31)
  static __device__ __forceinline__ typename Op<T>::frag row_frag(const T* t, int r0, int c, int lane) {
    return *reinterpret_cast<const typename Op<T>::frag*>(t + at(r0 + (lane & 31), 2 * c + (lane >> 5)));
  }
  // first operand "channel 32 dt + (l & 31) of the tile's transpose x chunk s of rows", rows in the order a score tile
  // leaves the matrix unit
  static __device__ __forceinline__ typename Op<T>::frag col_frag(const T* t, int s, int dt, int lane) {
    typename Op<T>::frag f;
    if constexpr (sizeof(T) == 4) {
      const int ch = 32 * dt + (lane & 31);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = t[at(8 * s + 4 * (lane >> 5) + i, ch / 4) + (ch & 3)];
    } else {
      // ds_read_b64_tr_b16: in each group of 16 lanes, lane i gives the address of row i / 4, channels 4 (i % 4) .. + 3 of a
      // 4 x 16 block and receives channel i of its 4 rows
      const int i = lane & 15, g16 = (lane >> 4) & 1, h = lane >> 5;
      const int row = 16 * s + 4 * h + (i >> 2), ch = 32 * dt + 16 * g16 + 4 * (i & 3);
      s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS3 s16x4*)(t + at(row, ch / 8) + (ch & 7)));
      s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS3 s16x4*)(t + at(row + 8, ch / 8) + (ch & 7)));
      s16x8 v;
#pragma unroll
      for (int j = 0; j < 4; ++j) { v[j] = a[j]; v[4 + j] = b[j]; }
      f = __builtin_bit_cast(typename Op<T>::frag, v);
    }
    return f;
  }
  // one lane's piece of an own row straight from global memory (second operand); zero outside
  static __device__ __forceinline__ typename Op<T>::frag own_frag(const T* row, bool ok, int c, int d, int lane) {
    const int ch = c * CH + (lane >> 5) * E;
    typename Op<T>::frag f;
    if (ok && ch < d) f = *reinterpret_cast<const typename Op<T>::frag*>(row + ch);
    else
#pragma unroll
      for (int i = 0; i < E; ++i) f[i] = (T)0.f;
    return f;
  }
};

// Barrier behind which the direct requests into LDS of every wave of the workgroup have arrived.  The wait is explicit: a
// workgroup barrier alone orders LDS and global accesses of the waves, but does not wait for requests still under way.
__device__ __forceinline__ void arrive_barrier() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}
