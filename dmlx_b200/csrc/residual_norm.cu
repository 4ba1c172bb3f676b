// The norms behind and before a block with its gate and its factor on the residual, in one pass over the rows:
//   p = y r(y) w_post (or y), times the gate or its sigmoid;  h' = h + scale p;  x = h' r(h') w_norm (or h'),  r(v) = 1 / sqrt(mean(v^2) + eps).
//
// A row waits in registers, a block of threads for it (a warp where it is short), and two rounds of sums: |y|^2, then |h'|^2 together with the
// largest |h' w_norm|, from which the 8-bit form's step follows without a third (r > 0, and rounding keeps the order).  x is made of h' before its rounding.
// f32 in between, one rounding for each result.  Everything a row needs is asked for before its first sum.
//
// Bound by what it reads and writes: 8192 rows of 4096 bf16 with a gate for each take 55 to 57 us in a graph, 6 TB/s (the gate behind the first sum 64, weights too 75); one row 2.2
// us, a launch's latency; 333 rows of 5003, f32 beside bf16, 7.1 to 7.7 (number by number 18).  Into 8-bit rows: 8192 of 4096 55.8 (235 MB, 36 at the rate of a copy: the 8 bits
// take the arithmetic), one 2.5; 333 of 5003 7.6 and 3000 45.6, whose columns are dealt out from the first and whose loads are shifted into place therefore.
#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "common.h"
#include "i8.cuh"
#include "launch.cuh"
#include "ptx.cuh"
#include "rows.cuh"

namespace {

struct ResidualNormArgs {
  const void *h, *y;
  const __nv_bfloat16 *gate, *post_w, *norm_w;
  void* h_out;
  __nv_bfloat16* x_out;
  I8RowsDev q;
  long long h_stride, y_stride, gate_stride, h_out_stride, x_out_stride;
  int rows, n, chunks, sigmoid;
  int shift;  // columns may be dealt out from ahead of the first: no 8-bit rows, which want them from the first, and room for a vector more
  float scale, eps;
};

// The lanes' numbers, eight for each, neighbouring lanes' next to one another, to a row of n from column c of each lane on.  Where rows do not start on 16
// bytes a lane's numbers behind the first boundary and the next lane's ahead of it are a piece; a warp's ends go one by one.  (All lanes of the warp.)
template <typename T>
__device__ __forceinline__ void store_eight(T* p, int c, int n, bool fit, const float (&v)[8], int lo = 0) {
  constexpr int kWords = 2 * (int)sizeof(T);
  uint32_t w[kWords + 4];
#pragma unroll
  for (int i = 0; i < kWords; ++i) {
    if constexpr (sizeof(T) == 4) {
      w[i] = __float_as_uint(v[i]);
    } else {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
  if (fit) {
    if (c >= lo && c + 8 <= n) {
#pragma unroll
      for (int i = 0; i < kWords / 4; ++i) reinterpret_cast<uint4*>(p + c)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i >= lo && c + i < n) st(p + c + i, v[i]);
    return;
  }
  const uint32_t off = (16u - (uint32_t)(reinterpret_cast<uintptr_t>(p + c) & 15)) & 15;  // bytes up to the first boundary
  const int head = (int)(off / sizeof(T)), lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[kWords + i] = __shfl_down_sync(0xffffffffu, w[i], 1);
#pragma unroll
  for (int i = 0; i < kWords + 2; ++i) w[i] = off & 8 ? w[i + 2] : w[i];
#pragma unroll
  for (int i = 0; i < kWords + 1; ++i) w[i] = off & 4 ? w[i + 1] : w[i];
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], (off & 2) * 8);
  }
  const bool pieces = (lane < 31 || head == 0) && c + head >= lo && c + head + 8 <= n;
  if (pieces) {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) reinterpret_cast<uint4*>(p + c + head)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  }
  const bool before = lane == 0 || c + head > n || c - 8 + head < lo;  // the lane ahead has not taken this one's first
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c + i >= lo && c + i < n && (i < head ? before : !pieces)) st(p + c + i, v[i]);
}

// Where all rows start on 16 bytes and are whole vectors (FIT), a row's sum of squares is made in an order that its columns alone set, so that what shares its batch changes
// no bit of it, though a thread has two vectors in place of one where the batch is larger: eight columns one after the other; 32 such vectors as a tree over lanes; these
// groups as a tree too, lane l those of l and l + 32.  (With more vectors every batch has as many to a thread, and its sum comes first.)  Elsewhere bits go by where the row
// lies: a vector may go on in the next lane, and in the next warp (an order by columns took 8.4 us in place of 7.0 for 333 rows of 5003, 181 in place of 153 for 3000 of 16383).

// Eight more columns' squares.
__device__ __forceinline__ float squares(float sum, const float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) sum = fmaf(v[e], v[e], sum);
  return sum;
}
// The row's sum of what each of its threads, a block's (or a warp's) all, has.
template <bool WARP>
__device__ __forceinline__ float sum_of(float* part, float v) {
  v = warp_sum(v);
  if constexpr (!WARP) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = warp_sum(lane < (blockDim.x >> 5) ? part[lane] : 0.f);
  }
  return v;
}
// The same of two vectors a thread, each a tree of its own (both at a time: half of the lanes go on with one, half with the other).
__device__ __forceinline__ float sum_of_two(float* part, float a, float b) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const bool second = lane >= 16;
  float v = (second ? b : a) + __shfl_xor_sync(0xffffffffu, second ? a : b, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((lane & 15) == 0) part[(threadIdx.x >> 5) + (second ? warps : 0)] = v;
  __syncthreads();
  v = lane < 2 * warps ? part[lane] : 0.f;
  if (warps > 16 && lane + 32 < 2 * warps) v += part[lane + 32];
  return warp_sum(v);
}

// The sigmoid of a gate of bf16, for an h' of type T.  In f32 2^t, t = z log2(e), takes log2(e) in two parts, the first of 16 bits, so that its product with z is exact, the
// rest's a factor 1 + d: t's rounding alone would be 2^-19 of the result at |z| of 30.  (8192 rows of 4096, f32, 70.7 us as without that, 78.4 with expf and a division; 3000
// of 16384 133, 126 and 142.)
template <typename T>
__device__ __forceinline__ float gate_sigmoid(float z) {
  if constexpr (sizeof(T) == 2) return sigmoid_for<T>(z);
  constexpr float kHigh = 47274.0f / 32768.0f, kLow = 4.8884952e-6f;  // log2(e) = kHigh + kLow / ln(2)
  const float d = fmaxf(-kLow * z, -1.0f);  // (z = inf: p = 0)
  float p;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(-kHigh * z));
  return __fdividef(1.0f, 1.0f + fmaf(p, d, p));
}

// NV vectors of eight columns for each thread.  WARP: a warp for a row.  FIT: all rows start on 16 bytes and are whole vectors.  (1024 threads with 32 numbers each have 64
// registers: half of a row's y is still in its 16 bits while h comes.)
template <typename H, typename Y, typename O, int NV, bool WARP, bool FIT>
__global__ void __launch_bounds__(WARP ? 256 : 1024) residual_norm_kernel(const __grid_constant__ ResidualNormArgs a) {
  after_previous();
  // A row's vectors one after the other, or behind all stores: 8192 rows of 4096 bf16 57.8 and 54.8 us, 3000 f32 rows of 16384 119 and 127.
  constexpr bool kTwo = FIT && NV == 2 && !WARP, kBehind = kTwo && sizeof(H) + sizeof(Y) == 4;
  constexpr int kSums = kTwo ? 2 : 1;
  __shared__ float part[3][kTwo ? 64 : 32];
  const int threads = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int row = WARP ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.rows) return;
  auto column = [&](int u) { return (t + u * threads) * 8; };
  // Where rows do not start on 16 bytes, the columns are dealt out from a boundary of h_out ahead of its row (`lo` columns that are not there), and so are on
  // boundaries of all that lies like it.
  const int lo = FIT || !a.shift ? 0 : (int)((reinterpret_cast<uintptr_t>((O*)a.h_out + (size_t)row * a.h_out_stride) / sizeof(O)) % 8);
  const int n = a.n + lo;
  const H* h = (const H*)a.h + (size_t)row * a.h_stride - lo;
  const Y* y = (const Y*)a.y + (size_t)row * a.y_stride - lo;
  const __nv_bfloat16 *gate = a.gate ? a.gate + (size_t)row * a.gate_stride - lo : nullptr, *post_w = a.post_w ? a.post_w - lo : nullptr, *norm_w = a.norm_w ? a.norm_w - lo : nullptr;
  O* h_out = (O*)a.h_out + (size_t)row * a.h_out_stride - lo;
  __nv_bfloat16* x_out = a.x_out ? a.x_out + (size_t)row * a.x_out_stride - lo : nullptr;
  auto fits = [](const void* p) { return FIT || (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  Eight<Y> yr[NV];
  Eight<H> hr[NV];
  load_eights(yr, y, n, fits(y), column, lo);
  load_eights(hr, h, n, fits(h), column, lo);
  Eight<__nv_bfloat16> gr[NV <= 2 ? NV : 1];
  if constexpr (NV <= 2) {
    if (gate) load_eights(gr, gate, n, fits(gate), column, lo);
  }
  Eight<__nv_bfloat16> pr[NV <= 2 ? NV : 1], nr[NV == 1 ? NV : 1] = {};
  if constexpr (NV <= 2) {
    if (post_w) load_eights(pr, post_w, n, fits(post_w), column, lo);
  }
  if constexpr (NV == 1) {
    if (norm_w) load_eights(nr, norm_w, n, fits(norm_w), column, lo);
  }
  float ry = 1.f;
  if (a.post_w) {
    if constexpr (kBehind) {
      float v[NV][8];
#pragma unroll
      for (int u = 0; u < NV; ++u) widen(yr[u], v[u]);
      ry = sum_of_two(part[0], squares(0.f, v[0]), squares(0.f, v[NV - 1]));
    } else {
      float ss[kSums] = {};
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        float v[8];
        widen(yr[u], v);
        ss[u % kSums] = squares(ss[u % kSums], v);
      }
      if constexpr (kTwo) ry = sum_of_two(part[0], ss[0], ss[kSums - 1]);
      else ry = sum_of<WARP>(part[0], ss[0]);
    }
    ry = rsqrtf(ry / (float)a.n + a.eps);
  }
  float x[NV][8], ss[kSums] = {};
  uint32_t most = 0u;
  auto weigh = [&](int u) {
    float w[8];
    if (a.norm_w) {
      widen(NV == 1 ? nr[0] : load_eight(norm_w, column(u), n, fits(norm_w), lo), w);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[u][e] *= w[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(x[u][e]) & 0x7fffffffu);
  };
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int c = column(u);
    float p[8], w[8];
    widen(yr[u], p);
    if (a.post_w) {
      widen(NV <= 2 ? pr[NV <= 2 ? u : 0] : load_eight(post_w, c, n, fits(post_w), lo), w);
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = p[e] * ry * w[e];
    }
    if (a.gate) {
      widen(NV <= 2 ? gr[NV <= 2 ? u : 0] : load_eight(gate, c, n, fits(gate), lo), w);
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] *= a.sigmoid ? gate_sigmoid<O>(w[e]) : w[e];
    }
    widen(hr[u], w);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[u][e] = fmaf(a.scale, p[e], w[e]);
      if constexpr (!kBehind) ss[u % kSums] = fmaf(x[u][e], x[u][e], ss[u % kSums]);  // (behind the last column all is zero)
    }
    store_eight(h_out, c, n, fits(h_out), x[u], lo);
    if constexpr (!kBehind) weigh(u);
  }
  if (!a.x_out && !a.q.q) return;
  if constexpr (kBehind) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      ss[u] = squares(0.f, x[u]);
      weigh(u);
    }
  }
  float r = 1.f;
  most = __reduce_max_sync(0xffffffffu, most);
  if constexpr (!WARP) {
    if ((t & 31) == 0) part[2][t >> 5] = __uint_as_float(most);
  }
  if constexpr (kTwo) r = sum_of_two(part[1], ss[0], ss[kSums - 1]);
  else if (a.norm_w || !WARP) r = sum_of<WARP>(part[1], ss[0]);
  r = a.norm_w ? rsqrtf(r / (float)a.n + a.eps) : 1.f;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[u][e] *= r;
    if (x_out) store_eight(x_out, column(u), n, fits(x_out), x[u], lo);
  }
  if (!a.q.q) return;
  if constexpr (!WARP) most = __reduce_max_sync(0xffffffffu, (t & 31) < (threads >> 5) ? __float_as_uint(part[2][t & 31]) : 0u);
  const I8Scale s = I8Scale::of(__uint_as_float(most) * r);
  if (t == 0) a.q.scale[row] = s.step();
#pragma unroll
  for (int u = 0; u < NV; ++u)
    if (column(u) < a.chunks * kI8Chunk) i8_store8(a.q.q, row, column(u), a.chunks, s, x[u]);
}

template <typename H, typename Y, typename O, bool FIT>
b200_status launch(const ResidualNormArgs& a, cudaStream_t s) {
  const int vectors = std::max(a.chunks * (kI8Chunk / 8), a.shift ? (a.n + 14) / 8 : 0);  // (up to seven columns ahead of the first)
  if (vectors <= 32 * 2) {
    const int warps = a.rows >= 8 * b200_sm_count() ? 8 : 1;
    const unsigned grid = (unsigned)((a.rows + warps - 1) / warps);
    if (vectors <= 32) launch_after(residual_norm_kernel<H, Y, O, 1, true, FIT>, grid, warps * 32, 0, s, a);
    else launch_after(residual_norm_kernel<H, Y, O, 2, true, FIT>, grid, warps * 32, 0, s, a);
  } else {
    // Few rows: more threads, each with fewer loads to wait for, while all of them run at once (200 rows of 4096 3.2 us with one vector a thread, 3.4 with two; 600
    // 6.8 and 5.7; 64 of 8192 3.2 and 3.5, 200 5.9 and 4.6).
    const int nv = vectors <= 1024 && (long long)a.rows * vectors <= 864ll * b200_sm_count() ? 1 : vectors <= 2048 ? 2 : 4;
    const int threads = (vectors + 32 * nv - 1) / (32 * nv) * 32;
    if (nv == 1) launch_after(residual_norm_kernel<H, Y, O, 1, false, FIT>, a.rows, threads, 0, s, a);
    else if (nv == 2) launch_after(residual_norm_kernel<H, Y, O, 2, false, FIT>, a.rows, threads, 0, s, a);
    else launch_after(residual_norm_kernel<H, Y, O, 4, false, FIT>, a.rows, threads, 0, s, a);
  }
  B200_LAUNCH_CHECK();
  return B200_OK;
}

template <typename H, typename Y>
b200_status launch_any(const ResidualNormArgs& a, bool out_f32, bool fit, cudaStream_t s) {
  if (out_f32) return fit ? launch<H, Y, float, true>(a, s) : launch<H, Y, float, false>(a, s);
  return fit ? launch<H, Y, __nv_bfloat16, true>(a, s) : launch<H, Y, __nv_bfloat16, false>(a, s);
}

constexpr int kMostColumns = 32768;  // 1024 threads of four vectors

}  // namespace

extern "C" b200_status b200_residual_norm(const b200_residual_norm_shape* shape, const void* d_h, int64_t h_stride, const void* d_y, int64_t y_stride,
                                          const void* d_gate, int64_t gate_stride, const void* d_post_weight, const void* d_norm_weight, int32_t rows, void* d_h_out,
                                          int64_t h_out_stride, void* d_x_out, int64_t x_out_stride, b200_i8_rows* q_out, void* stream) {
  if (!shape || rows < 0) { b200_set_error("residual norm: no shape, or %d rows", rows); return B200_ERR_INVALID_ARGUMENT; }
  const int n = shape->n;
  if (n <= 0 || n > kMostColumns) { b200_set_error("residual norm: rows of %d columns (at most %d)", n, kMostColumns); return B200_ERR_UNSUPPORTED; }
  if (!(shape->eps >= 0.f)) { b200_set_error("residual norm: eps %g", (double)shape->eps); return B200_ERR_INVALID_ARGUMENT; }
  if (shape->h_out < B200_H_OUT_AS_H || shape->h_out > B200_H_OUT_F32) { b200_set_error("residual norm: h_out of type %d", shape->h_out); return B200_ERR_INVALID_ARGUMENT; }
  const bool out_f32 = shape->h_out == B200_H_OUT_AS_H ? shape->h_f32 != 0 : shape->h_out == B200_H_OUT_F32;
  const int h_size = shape->h_f32 ? 4 : 2, y_size = shape->y_f32 ? 4 : 2, out_size = out_f32 ? 4 : 2;
  auto holds = [&](const void* p, int64_t stride, int size) { return p && ((uintptr_t)p & (size - 1)) == 0 && (rows <= 1 || stride >= n); };
  if (rows > 0 && (!holds(d_h, h_stride, h_size) || !holds(d_y, y_stride, y_size) || !holds(d_h_out, h_out_stride, out_size) || (d_x_out && !holds(d_x_out, x_out_stride, 2)) ||
                   (d_gate && gate_stride != 0 && !holds(d_gate, gate_stride, 2)) || (((uintptr_t)d_gate | (uintptr_t)d_post_weight | (uintptr_t)d_norm_weight) & 1) != 0)) {
    b200_set_error("residual norm: rows of %d columns, each on a number's boundary, strides that hold a row", n);
    return B200_ERR_INVALID_ARGUMENT;
  }
  auto at = [&](const void* p, int64_t stride, int size) { return RowsAt{p, stride ? rows : 1, stride * size, (long long)n * size}; };
  const RowsAt h_out = at(d_h_out, h_out_stride, out_size), x_out = at(d_x_out, x_out_stride, 2);
  bool over = rows_overlap(h_out, x_out) || (rows_overlap(h_out, at(d_h, h_stride, h_size)) && (d_h_out != d_h || out_size != h_size || (rows > 1 && h_out_stride != h_stride))) ||
              rows_overlap(x_out, at(d_h, h_stride, h_size));
  for (const RowsAt& in : {at(d_y, y_stride, y_size), at(d_gate, gate_stride, 2), at(d_post_weight, 0, 2), at(d_norm_weight, 0, 2)})
    over = over || rows_overlap(h_out, in) || rows_overlap(x_out, in);
  if (rows > 0 && over) {
    b200_set_error("residual norm: h_out is h itself or lies apart from all else, and so does x");
    return B200_ERR_INVALID_ARGUMENT;
  }
  if (q_out && (rows > q_out->max_rows || n > q_out->max_k)) {
    b200_set_error("residual norm: %d rows of %d columns, the 8-bit rows are for %d of %d", rows, n, q_out->max_rows, q_out->max_k);
    return B200_ERR_CAPACITY;
  }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  if (q_out) { q_out->rows = rows; q_out->k = n; }
  if (rows == 0) return B200_OK;
  ResidualNormArgs a{};
  a.h = d_h; a.y = d_y; a.gate = (const __nv_bfloat16*)d_gate; a.post_w = (const __nv_bfloat16*)d_post_weight; a.norm_w = (const __nv_bfloat16*)d_norm_weight;
  a.h_out = d_h_out; a.x_out = (__nv_bfloat16*)d_x_out;
  if (q_out) a.q = q_out->x;
  a.h_stride = h_stride; a.y_stride = y_stride; a.gate_stride = gate_stride; a.h_out_stride = h_out_stride; a.x_out_stride = x_out_stride;
  a.rows = rows; a.n = n; a.chunks = i8_chunks(n); a.sigmoid = shape->gate_sigmoid != 0; a.scale = shape->scale; a.eps = shape->eps;
  auto fits = [&](const void* p, int64_t stride, int size) { return ((uintptr_t)p & 15) == 0 && (rows <= 1 || stride * size % 16 == 0); };
  const bool fit = n % 8 == 0 && fits(d_h, h_stride, h_size) && fits(d_y, y_stride, y_size) && fits(d_gate, gate_stride, 2) && fits(d_post_weight, 0, 2) &&
                   fits(d_norm_weight, 0, 2) && fits(d_h_out, h_out_stride, out_size) && fits(d_x_out, x_out_stride, 2);
  a.shift = !fit && !q_out && (n + 14) / 8 <= kMostColumns / 8;
  cudaStream_t s = (cudaStream_t)stream;
  if (shape->h_f32) return shape->y_f32 ? launch_any<float, float>(a, out_f32, fit, s) : launch_any<float, __nv_bfloat16>(a, out_f32, fit, s);
  return shape->y_f32 ? launch_any<__nv_bfloat16, float>(a, out_f32, fit, s) : launch_any<__nv_bfloat16, __nv_bfloat16>(a, out_f32, fit, s);
}
