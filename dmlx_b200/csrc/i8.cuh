// Rows and weights in 8-bit integers: how they lie in memory, and how a row becomes one (i8.cu multiplies them, residual_norm.cu makes rows too).
//
// Both are [tile of 128 rows][block of 128 columns][row][128 bytes], a block 16 KiB in one piece: what a stage of the matmul kernels takes with one bulk copy.
// The 16-byte chunks of a row are permuted by the row's place in its group of eight (the 128-byte swizzle that the MMAs read).  Columns behind the last are
// zero.  Rows behind the last hold whatever they held: their products go nowhere.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "dmlx_b200.h"
#include "ptx.cuh"

constexpr int kI8Tile = 128;              // rows of a tile
constexpr int kI8Chunk = 128;             // columns of a block
constexpr int kI8Block = kI8Tile * kI8Chunk;
constexpr int kI8MaxK = 131072;           // 127 * 128 * 131072 < 2^31: a sum fits 32 bits whatever it is made of

struct I8RowsDev {
  signed char* q;  // [row tile][chunks][128][128], swizzled
  float* scale;    // [row]
};

struct b200_i8_rows {
  int max_rows = 0, max_k = 0, max_hidden = 0;
  int rows = -1, k = 0;                 // what it holds; -1: nothing yet
  I8RowsDev x{}, hidden{};
  // [max_rows][h_stride]: the feed-forward block's inner rows until their largest is known.  In bf16 the products behind them were 1e-2 off (what is
  // rounded twice goes to another of 255 numbers one time in twenty, and a rounded largest moves a row's every step).
  float* h = nullptr;
  int h_stride = 0;
  float* most = nullptr;                // [max_rows][their groups of 32 channels]: the largest magnitude in each
};

struct b200_i8_weight {
  int n = 0, k = 0, tiles = 0, chunks = 0;
  bool gated = false;                   // tiles alternate: 128 channels of the gate, the same 128 of up
  signed char* q = nullptr;             // [tile][chunks][128][128], swizzled
  float* scale = nullptr;               // [tiles * 128]
};

// Rows in memory, as one call gives them: `bytes` of each, `stride` bytes apart.
struct RowsAt {
  const void* p;
  long long rows, stride, bytes;
};
// Whether two of them share a byte.  Rows of one buffer side by side (the same stride, other columns) do not.
inline bool rows_overlap(const RowsAt& a, const RowsAt& b) {
  if (!a.p || !b.p || a.rows <= 0 || b.rows <= 0) return false;
  const long long d = (long long)((uintptr_t)b.p - (uintptr_t)a.p), end_a = (a.rows - 1) * a.stride + a.bytes, end_b = (b.rows - 1) * b.stride + b.bytes;
  if (d >= end_a || -d >= end_b) return false;
  if (a.rows == 1 && b.rows == 1) return true;
  const long long stride = a.rows > 1 ? a.stride : b.stride;
  if (stride <= 0 || (a.rows > 1 && b.rows > 1 && a.stride != b.stride)) return true;  // (may be: no layout that a tensor's columns have)
  const long long off = (d % stride + stride) % stride;
  return off < a.bytes || off + b.bytes > stride;
}

inline int i8_chunks(int k) { return (k + kI8Chunk - 1) / kI8Chunk; }

#ifdef __CUDACC__
// Where column c of a row lies.
__device__ __forceinline__ size_t i8_at(int row, int c, int chunks) {
  const int r = row % kI8Tile;
  return ((size_t)(row / kI8Tile) * chunks + c / kI8Chunk) * kI8Block + r * kI8Chunk + ((((c % kI8Chunk) >> 4) ^ (r & 7)) << 4) + (c & 15);
}

// A row's numbers as multiples of most / 127, most = its largest magnitude.  The quotient 127 x / most is rounded to the nearest, halves to the even, as if
// it were exact: its product with the rounded 127 / most is at most 127 * 2^-24 off, and where that could decide, the division is made.  (For x of bf16
// 127 x is exact, and the division rounds correctly: halves are numbers of f32, so it can reach one but not cross it, and nothing is left to chance.)
struct I8Scale {
  float most, inv;
  bool plain;  // else all zeros: a row of nothing, or one without numbers
  static __device__ __forceinline__ I8Scale of(float m) { return I8Scale{m, __fdiv_rn(127.0f, m), m > 0.f && m < __int_as_float(0x7f800000)}; }
  __device__ __forceinline__ float step() const { return __fdiv_rn(most, 127.0f); }
  // The eight numbers in eight bytes.  (1.5 * 2^23 added leaves the nearest whole number in the low bits.)
  __device__ __forceinline__ uint2 quantize(const float (&v)[8]) const {
    if (!plain) return make_uint2(0u, 0u);
    constexpr float kWhole = 12582912.0f, kNearHalf = 0.49999f;
    uint32_t q[8];
    float d[8], off = 0.f;  // distances to the whole numbers, the largest
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float r = fmaf(v[e], inv, kWhole);
      d[e] = fmaf(v[e], inv, kWhole - r);
      off = fmaxf(off, fabsf(d[e]));
      q[e] = __float_as_uint(r);
    }
    if (!(off < kNearHalf) || !(inv < 1e38f)) {  // (or 127 / most is no f32)
      const float down = most > 1e30f ? 0.00390625f : 1.0f;  // (127 times the largest numbers is none either)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (!(fabsf(d[e]) < kNearHalf) || !(inv < 1e38f)) q[e] = (uint32_t)(int)rintf(__fdiv_rn(127.0f * (v[e] * down), most * down));
    }
    return make_uint2(__byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410));
  }
};

// Eight neighbouring numbers of a row as they lie in memory, those behind the last as zeros.
template <typename T>
struct Eight { uint4 r[sizeof(T) / 2]; };

// N times eight numbers of a row of n, at columns at(0), at(1), ..., multiples of eight; fit: the row starts on 16 bytes.  Elsewhere the 16-byte pieces that
// hold the numbers are fetched and shifted into place (rows of 5003 bf16 and f32 one number at a time took three times as long).  All loads are on
// their way before the first is looked at; what lies at a row's ends, where a piece would reach beyond it, is fetched number by number behind them.
// The row may begin at column lo.
template <typename T, int N, class At>
__device__ __forceinline__ void load_eights(Eight<T> (&e)[N], const T* p, int n, bool fit, At at, int lo = 0) {
  constexpr int R = sizeof(T) / 2, kWords = 4 * R;
  const uint32_t off = fit ? 0u : (uint32_t)(reinterpret_cast<uintptr_t>(p) & 15);
  const int before = (int)(off / sizeof(T));  // numbers of the first piece that come ahead
  const uint4* pieces = reinterpret_cast<const uint4*>(p - before);
  uint4 last[N];
  auto whole = [&](int c) { return c - before >= lo && (fit ? c + 8 <= n : c - before + 8 + 16 / (int)sizeof(T) <= n); };
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int c = at(k);
    const bool here = whole(c);
    const uint4* from = pieces + (size_t)(c / 8) * R;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      e[k].r[i] = make_uint4(0u, 0u, 0u, 0u);
      if (here) e[k].r[i] = from[i];
    }
    last[k] = make_uint4(0u, 0u, 0u, 0u);
    if (!fit && here) last[k] = from[R];
  }
  if (!fit) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      uint32_t w[kWords + 4];
#pragma unroll
      for (int i = 0; i <= R; ++i) {
        const uint4 q = i < R ? e[k].r[i < R ? i : 0] : last[k];
        w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w;
      }
#pragma unroll
      for (int i = 0; i < kWords + 2; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
      for (int i = 0; i < kWords + 1; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (off & 2) * 8);
      }
#pragma unroll
      for (int i = 0; i < R; ++i) e[k].r[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    }
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int c = at(k);
    if (whole(c) || c >= n) continue;
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i >= lo && c + i < n ? p[c + i] : T(0.f);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(v[4 * i + j]);
        else w[j] = (uint32_t)__bfloat16_as_ushort(v[2 * j]) | (uint32_t)__bfloat16_as_ushort(v[2 * j + 1]) << 16;
      }
      e[k].r[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}
template <typename T>
__device__ __forceinline__ Eight<T> load_eight(const T* p, int c, int n, bool fit, int lo = 0) {
  Eight<T> e[1];
  load_eights(e, p, n, fit, [&](int) { return c; }, lo);
  return e[0];
}
__device__ __forceinline__ void widen(const Eight<__nv_bfloat16>& e, float (&v)[8]) {
  const uint32_t w[4] = {e.r[0].x, e.r[0].y, e.r[0].z, e.r[0].w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = ptx::bf16_lo(w[i]);
    v[2 * i + 1] = ptx::bf16_hi(w[i]);
  }
}
__device__ __forceinline__ void widen(const Eight<float>& e, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    v[4 * i] = __uint_as_float(e.r[i].x); v[4 * i + 1] = __uint_as_float(e.r[i].y);
    v[4 * i + 2] = __uint_as_float(e.r[i].z); v[4 * i + 3] = __uint_as_float(e.r[i].w);
  }
}
// The largest magnitude of m and eight numbers, as bits: what is no number is the largest of all.
__device__ __forceinline__ uint32_t most_of(uint32_t m, const Eight<__nv_bfloat16>& e) {
  const uint4& r = e.r[0];
  const uint32_t a = __vmaxu2(__vmaxu2(r.x & 0x7fff7fffu, r.y & 0x7fff7fffu), __vmaxu2(r.z & 0x7fff7fffu, r.w & 0x7fff7fffu));
  return max(m, max(a << 16, a & 0xffff0000u));
}
__device__ __forceinline__ uint32_t most_of(uint32_t m, const Eight<float>& e) {
#pragma unroll
  for (int i = 0; i < 2; ++i) m = max(max(max(m, e.r[i].x & 0x7fffffffu), max(e.r[i].y & 0x7fffffffu, e.r[i].z & 0x7fffffffu)), e.r[i].w & 0x7fffffffu);
  return m;
}

// Eight neighbouring columns, the first a multiple of eight.
__device__ __forceinline__ void i8_store8(signed char* q, int row, int c, int chunks, const I8Scale& s, const float (&v)[8]) {
  *reinterpret_cast<uint2*>(q + i8_at(row, c, chunks)) = s.quantize(v);
}
#endif
