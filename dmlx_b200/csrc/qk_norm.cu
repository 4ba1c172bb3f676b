// Norm of every query and key head and the rotation behind it, in one pass over the rows; into pages as well.
//
// n = x / sqrt(mean(x^2) + eps) * w over a head's D numbers, then the first rot_dim of them rotate in pairs by position * theta^(-2 i / rot_dim).
// Everything between the load and the store is f32, and there is one rounding at the end.  The angle of a far position does not fit f32 (position
// 2^20 has 4 bits left behind the point of a turn), so it is kept in turns: position * (frequency / 2 pi) in f64, its whole turns dropped, and
// what is left goes to sincospif, which is exact about the 2 pi.
//
// A head is D / 8 lanes of eight neighbouring elements, so a warp takes 512 bytes (32 / (D / 8) heads) at once.  A pair (i, i + rot_dim / 2) lies
// in two lanes at the same place, which a shuffle brings together; a pair (2 i, 2 i + 1) lies in one.  A warp has its row's cosines and sines in
// registers for all the heads it takes, and takes as many of them as the number of rows allows (few rows: one load each).
#include <cuda_bf16.h>
#include <math.h>

#include <cmath>

#include <algorithm>

#include "common.h"
#include "kv_pool.cuh"
#include "launch.cuh"
#include "ptx.cuh"
#include "rows.cuh"

namespace {

constexpr int kMostPairs = 128;  // rot_dim / 2 of the widest head
constexpr int kWarps = 8;
constexpr int kAhead = 4;        // loads of 512 bytes that a warp has in flight

struct NormRopeArgs {
  const __nv_bfloat16 *q, *k, *v;
  int q_stride, k_stride, v_stride;
  const __nv_bfloat16 *q_weight, *k_weight;
  const int *positions, *row_seq;
  __nv_bfloat16 *q_out, *k_out;
  int q_out_stride, k_out_stride;
  int rows, hq, hkv, rot, interleaved, parts;  // parts: warps that share a row
  float eps;
  KvDev d;
  int layer;
  double turns[kMostPairs];  // frequency / (2 pi) of each pair
};

// PAGES: k goes into the row's page, and so does v.
template <int D, bool PAGES>
__global__ void __launch_bounds__(kWarps * 32) qk_norm_rope_kernel(const __grid_constant__ NormRopeArgs a) {
  after_previous();
  constexpr int LANES = D / 8, HEADS = 32 / LANES;  // lanes of a head; heads of a load
  __shared__ double turns[kMostPairs];
  if ((int)threadIdx.x < a.rot / 2) turns[threadIdx.x] = a.turns[threadIdx.x];
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = blockIdx.x * kWarps + (threadIdx.x >> 5);
  const int row = warp / a.parts, part = warp - row * a.parts;
  if (row >= a.rows) return;
  const int at = (lane % LANES) * 8, sub = lane / LANES;  // this lane's elements of a head; its head of a load
  const int pos = a.positions[row];

  float cs[8], sn[8];  // of this lane's elements; interleaved: of its four pairs
  const int half = a.rot / 2;
  const bool turns_here = at < a.rot, second = !a.interleaved && at >= half;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    cs[e] = 1.f; sn[e] = 0.f;
    if (!turns_here || (a.interleaved && e >= 4)) continue;
    const double t = (double)pos * turns[a.interleaved ? at / 2 + e : (second ? at - half : at) + e];
    sincospif((float)(2.0 * (t - rint(t))), &sn[e], &cs[e]);
    if (second) sn[e] = -sn[e];
  }
  const int partner = (lane & ~(LANES - 1)) | (!turns_here || a.interleaved ? lane & (LANES - 1) : (second ? at - half : at + half) / 8);

  float wq[8], wk[8];
  auto weights = [&](const __nv_bfloat16* w, float (&f)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 1.f;
    if (!w) return;
    const uint4 u = *reinterpret_cast<const uint4*>(w + at);
    const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) { f[2 * e] = ptx::bf16_lo(x[e]); f[2 * e + 1] = ptx::bf16_hi(x[e]); }
  };
  weights(a.q_weight, wq);
  weights(a.k_weight, wk);

  // a step whose reservation failed has no page for this row: nothing of it is written there (the error word is set)
  size_t tile = 0;  // elements from the pool's start to this row in head 0 of its page
  bool have_page = false;
  if constexpr (PAGES) {
    const int seq = a.row_seq[row], page_idx = pos / a.d.page_size;
    have_page = pos >= 0 && seq >= 0 && seq < a.d.max_seqs && page_idx < a.d.seq_pages[seq];
    if (have_page) {
      const int page = a.d.block_table[(size_t)seq * a.d.max_pages_per_seq + page_idx];
      tile = (((size_t)a.layer * a.d.n_pages + page) * a.hkv * a.d.page_size + (pos - page_idx * a.d.page_size)) * (size_t)D;
    }
  }
  const int heads = a.hq + (PAGES ? 2 : 1) * a.hkv;
  for (int h0 = part * HEADS; h0 < heads; h0 += kAhead * a.parts * HEADS) {
    uint4 in[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int h = h0 + u * a.parts * HEADS + sub;
      in[u] = make_uint4(0, 0, 0, 0);
      if (h >= heads) continue;
      const __nv_bfloat16* src = h < a.hq ? a.q + (size_t)row * a.q_stride + (size_t)h * D
                                 : h < a.hq + a.hkv ? a.k + (size_t)row * a.k_stride + (size_t)(h - a.hq) * D
                                                    : a.v + (size_t)row * a.v_stride + (size_t)(h - a.hq - a.hkv) * D;
      in[u] = *reinterpret_cast<const uint4*>(src + at);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int h = h0 + u * a.parts * HEADS + sub;
      if (h0 + u * a.parts * HEADS >= heads) break;  // (the whole warp)
      const uint32_t w[4] = {in[u].x, in[u].y, in[u].z, in[u].w};
      float x[8], ss = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[2 * e] = ptx::bf16_lo(w[e]);
        x[2 * e + 1] = ptx::bf16_hi(w[e]);
        ss = fmaf(x[2 * e], x[2 * e], fmaf(x[2 * e + 1], x[2 * e + 1], ss));
      }
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss * (1.0f / D) + a.eps);
      const bool is_q = h < a.hq;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] * r * (is_q ? wq[e] : wk[e]);
      float y[8];
      if (a.interleaved) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[2 * e] = x[2 * e] * cs[e] - x[2 * e + 1] * sn[e];
          y[2 * e + 1] = x[2 * e] * sn[e] + x[2 * e + 1] * cs[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float other = __shfl_sync(0xffffffffu, x[e], partner);
          y[e] = x[e] * cs[e] - other * sn[e];
        }
      }
      if (!turns_here) {  // (0 times an infinite neighbour would not be 0)
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = x[e];
      }
      uint4 out;
      uint32_t* o = reinterpret_cast<uint32_t*>(&out);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(y[2 * e], y[2 * e + 1]);
        o[e] = *reinterpret_cast<const uint32_t*>(&p);
      }
      if (h >= heads) continue;
      if (is_q) {
        *reinterpret_cast<uint4*>(a.q_out + (size_t)row * a.q_out_stride + (size_t)h * D + at) = out;
      } else if constexpr (PAGES) {
        const bool is_v = h >= a.hq + a.hkv;
        const int head = h - a.hq - (is_v ? a.hkv : 0);
        __nv_bfloat16* pool = (__nv_bfloat16*)(is_v ? a.d.v_pool : a.d.k_pool) + tile + (size_t)head * a.d.page_size * D + at;
        if (have_page) *reinterpret_cast<uint4*>(pool) = is_v ? in[u] : out;
      } else {
        *reinterpret_cast<uint4*>(a.k_out + (size_t)row * a.k_out_stride + (size_t)(h - a.hq) * D + at) = out;
      }
    }
  }
}

// The checks and the tables that both entry points share.
b200_status fill(NormRopeArgs& a, const char* who, const b200_norm_rope* s, const void* d_q, const void* d_k, int32_t q_stride, int32_t k_stride,
                 const void* d_q_weight, const void* d_k_weight, const int32_t* d_positions, int32_t rows, void* d_q_out, int32_t q_out_stride) {
  if (!s) { b200_set_error("%s: no shape", who); return B200_ERR_INVALID_ARGUMENT; }
  if (s->head_dim != 64 && s->head_dim != 128 && s->head_dim != 256) { b200_set_error("%s: head_dim %d (64, 128 or 256)", who, s->head_dim); return B200_ERR_UNSUPPORTED; }
  if (s->rot_dim < 0 || s->rot_dim > s->head_dim || s->rot_dim % 16 != 0) {
    b200_set_error("%s: rot_dim %d is no multiple of 16 up to head_dim %d", who, s->rot_dim, s->head_dim);
    return B200_ERR_UNSUPPORTED;
  }
  if (s->n_q_heads < 0 || s->n_kv_heads < 0 || s->n_q_heads > 4096 || s->n_kv_heads > 4096 || rows < 0) { b200_set_error("%s: %d rows of %d and %d heads", who, rows, s->n_q_heads, s->n_kv_heads); return B200_ERR_INVALID_ARGUMENT; }
  if (s->rot_dim > 0 && !(s->theta > 0.0 && std::isfinite(s->theta))) { b200_set_error("%s: theta %g", who, s->theta); return B200_ERR_INVALID_ARGUMENT; }
  if (!(s->eps >= 0.f)) { b200_set_error("%s: eps %g", who, (double)s->eps); return B200_ERR_INVALID_ARGUMENT; }
  auto rows_fit = [&](const void* p, int stride, int heads) { return heads == 0 || (p && ((uintptr_t)p & 15) == 0 && stride % 8 == 0 && stride >= heads * s->head_dim); };
  if (rows > 0 && (!d_positions || !rows_fit(d_q, q_stride, s->n_q_heads) || !rows_fit(d_q_out, q_out_stride, s->n_q_heads) || !rows_fit(d_k, k_stride, s->n_kv_heads) ||
                   ((uintptr_t)d_q_weight & 15) != 0 || ((uintptr_t)d_k_weight & 15) != 0)) {
    b200_set_error("%s: rows and weights start on 16 bytes, strides are multiples of 8 elements and hold all heads", who);
    return B200_ERR_INVALID_ARGUMENT;
  }
  a.q = (const __nv_bfloat16*)d_q; a.k = (const __nv_bfloat16*)d_k; a.q_stride = q_stride; a.k_stride = k_stride;
  a.q_weight = (const __nv_bfloat16*)d_q_weight; a.k_weight = (const __nv_bfloat16*)d_k_weight;
  a.positions = d_positions; a.rows = rows; a.hq = s->n_q_heads; a.hkv = s->n_kv_heads;
  a.rot = s->rot_dim; a.interleaved = s->interleaved != 0; a.eps = s->eps;
  a.q_out = (__nv_bfloat16*)d_q_out; a.q_out_stride = q_out_stride;
  for (int i = 0; i < s->rot_dim / 2; ++i) a.turns[i] = pow(s->theta, -2.0 * i / s->rot_dim) / (2.0 * M_PI);
  return B200_OK;
}

template <bool PAGES>
b200_status launch(NormRopeArgs& a, int head_dim, cudaStream_t s) {
  const int heads = a.hq + (PAGES ? 2 : 1) * a.hkv, loads = (heads * head_dim + 255) / 256;
  // 32 warps per SM take the row's loads between them; with more rows than that a warp has whole rows
  const int want = 32 * b200_sm_count();
  a.parts = std::min(loads, std::max(1, (want + a.rows - 1) / a.rows));
  const long long warps = (long long)a.rows * a.parts;
  const unsigned grid = (unsigned)((warps + kWarps - 1) / kWarps);
  if (head_dim == 64) launch_after(qk_norm_rope_kernel<64, PAGES>, grid, kWarps * 32, 0, s, a);
  else if (head_dim == 128) launch_after(qk_norm_rope_kernel<128, PAGES>, grid, kWarps * 32, 0, s, a);
  else launch_after(qk_norm_rope_kernel<256, PAGES>, grid, kWarps * 32, 0, s, a);
  B200_LAUNCH_CHECK();
  return B200_OK;
}

}  // namespace

extern "C" b200_status b200_qk_norm_rope(const b200_norm_rope* shape, const void* d_q, const void* d_k, int32_t q_stride, int32_t k_stride,
                                         const void* d_q_weight, const void* d_k_weight, const int32_t* d_positions, int32_t rows, void* d_q_out,
                                         void* d_k_out, int32_t q_out_stride, int32_t k_out_stride, void* stream) {
  NormRopeArgs a{};
  b200_status st = fill(a, "qk_norm_rope", shape, d_q, d_k, q_stride, k_stride, d_q_weight, d_k_weight, d_positions, rows, d_q_out, q_out_stride);
  if (st != B200_OK) return st;
  if (rows > 0 && shape->n_kv_heads > 0 && (!d_k_out || ((uintptr_t)d_k_out & 15) != 0 || k_out_stride % 8 != 0 || k_out_stride < shape->n_kv_heads * shape->head_dim)) {
    b200_set_error("qk_norm_rope: rows start on 16 bytes, strides are multiples of 8 elements and hold all heads");
    return B200_ERR_INVALID_ARGUMENT;
  }
  st = b200_require_device();
  if (st != B200_OK) return st;
  if (rows == 0 || a.hq + a.hkv == 0) return B200_OK;
  a.k_out = (__nv_bfloat16*)d_k_out; a.k_out_stride = k_out_stride;
  return launch<false>(a, shape->head_dim, (cudaStream_t)stream);
}

extern "C" b200_status b200_kv_norm_rope_append(b200_kv* kv, int32_t layer, const b200_norm_rope* shape, const void* d_q, void* d_k, const void* d_v,
                                                int32_t q_stride, int32_t k_stride, int32_t v_stride, const void* d_q_weight, const void* d_k_weight,
                                                const int32_t* d_positions, const int32_t* d_row_seq, int32_t rows, void* d_q_out, int32_t q_out_stride,
                                                void* stream) {
  if (!kv) { b200_set_error("norm_rope_append: no pool"); return B200_ERR_INVALID_ARGUMENT; }
  const b200_kv_config& c = kv->cfg;
  if (kv->layered) { b200_set_error("norm_rope_append: layered pools are written by the decoder step"); return B200_ERR_UNSUPPORTED; }
  if (layer < 0 || layer >= c.n_layers) { b200_set_error("norm_rope_append: layer %d out of range", layer); return B200_ERR_INVALID_ARGUMENT; }
  NormRopeArgs a{};
  b200_status st = fill(a, "norm_rope_append", shape, d_q, d_k, q_stride, k_stride, d_q_weight, d_k_weight, d_positions, rows, d_q_out, q_out_stride);
  if (st != B200_OK) return st;
  if (shape->head_dim != c.head_dim || shape->n_kv_heads != c.n_kv_heads) {
    b200_set_error("norm_rope_append: %d heads of %d, the pool has %d of %d", shape->n_kv_heads, shape->head_dim, c.n_kv_heads, c.head_dim);
    return B200_ERR_INVALID_ARGUMENT;
  }
  if (rows > 0 && (!d_row_seq || !d_v || ((uintptr_t)d_v & 15) != 0 || v_stride % 8 != 0 || v_stride < c.n_kv_heads * c.head_dim)) {
    b200_set_error("norm_rope_append: rows start on 16 bytes, strides are multiples of 8 elements and hold all heads");
    return B200_ERR_INVALID_ARGUMENT;
  }
  st = b200_require_device();
  if (st != B200_OK) return st;
  if (rows == 0) return B200_OK;
  if (c.kv_dtype != B200_KV_BF16) {  // a page's scale depends on all its new rows: they pass through d_k
    a.k_out = (__nv_bfloat16*)d_k; a.k_out_stride = k_stride;
    st = launch<false>(a, shape->head_dim, (cudaStream_t)stream);
    return st != B200_OK ? st : b200_kv_append_strided(kv, layer, d_k, d_v, k_stride, v_stride, rows, stream);
  }
  a.v = (const __nv_bfloat16*)d_v; a.v_stride = v_stride; a.row_seq = d_row_seq; a.d = kv->dev; a.layer = layer;
  return launch<true>(a, shape->head_dim, (cudaStream_t)stream);
}
