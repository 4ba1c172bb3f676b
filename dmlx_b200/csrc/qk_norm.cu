// Norm of every query and key head and the rotation behind it, in one pass over the rows; into pages as well.
//
// n = x / sqrt(mean(x^2) + eps) * w over a head's D numbers, then the first rot_dim of them rotate in pairs by position * theta^(-2 i / rot_dim).
// Everything between the load and the store is f32, and there is one rounding at the end.  The angle of a far position does not fit f32 (position
// 2^20 has 4 bits left behind the point of a turn), so it is kept in turns: position * (frequency / 2 pi) in f64, its whole turns dropped, and
// what is left goes to sincospif, which is exact about the 2 pi.
//
// A head is D / 8 lanes of eight neighbouring elements, so a warp takes 512 bytes (32 / (D / 8) heads) at once.  A pair (i, i + rot_dim / 2) lies
// in two lanes at the same place, and one shuffle of a word brings two partners; a pair (2 i, 2 i + 1) lies in a word.  Either way
//   y = (x cos w - x' sin w') r,  r = 1 / sqrt(mean + eps),  x' the partner, sin with its sign,
// so a head costs two packed operations per two elements beside the norm, with the products of angles and weights in registers for all heads that
// a warp takes of its row.  The block's rows have their angles computed once, by all its threads.  Few rows: more warps for each.
//
// Bound by what it reads and writes: 8192 rows of 32 + 8 heads of 128 take 34.6 us, 4.8 TB/s (kAhead loads in flight a warp, 32 warps per SM, the first of
// them ahead of the angles, else 36.0; 64 warps 41, 128 warps 49, every round's loads ahead 52, requested into L2 ahead 39); 257 rows of 16 + 4 heads of 64
// take 2.9 us, one row 3.5, a launch's latency.
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
  int rows, hq, hkv, rot, interleaved, block_rows;
  float eps;
  KvDev d;
  int layer;
  double turns[kMostPairs];  // frequency / (2 pi) of each pair
};

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 widen(uint32_t w) { return make_float2(ptx::bf16_lo(w), ptx::bf16_hi(w)); }

// PAGES: k goes into the row's page, and so does v.  ROWS rows of a block, kWarps / ROWS warps for each, and gridDim.y blocks for the same rows.
template <int D, bool PAGES, bool NEXT>
__global__ void __launch_bounds__(kWarps * 32, 4) qk_norm_rope_kernel(const __grid_constant__ NormRopeArgs a) {
  after_previous();
  constexpr int LANES = D / 8, HEADS = 32 / LANES;  // lanes of a head; heads of a load
  __shared__ float2 turn[kWarps * (D / 2)];         // [row of the block][pair] cosine, sine
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rows = a.block_rows, per_row = kWarps / rows;
  const int row = blockIdx.x * rows + warp / per_row, parts = per_row * gridDim.y, part = blockIdx.y * per_row + warp % per_row;
  const int at = (lane % LANES) * 8, sub = lane / LANES;  // this lane's elements of a head; its head of a load
  const int half = a.rot / 2;
  const int head0 = part * HEADS + sub, step = parts * HEADS;
  // The first loads of q are on their way while the angles are computed.
  uint4 in[kAhead];
  auto load = [&](const __nv_bfloat16* src, int head, int heads) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) in[u] = head + u * step < heads ? *reinterpret_cast<const uint4*>(src + (size_t)(u * step) * D) : make_uint4(0, 0, 0, 0);
  };
  const int first = head0 * D + at;
  load(a.q + (size_t)min(row, a.rows - 1) * a.q_stride + first, head0, a.hq);
  for (int i = threadIdx.x; i < rows * half; i += kWarps * 32) {
    const int r = i / half, pair = i - r * half;
    const double t = (double)(blockIdx.x * rows + r < a.rows ? a.positions[blockIdx.x * rows + r] : 0) * a.turns[pair];
    float sn, cs;
    sincospif((float)(2.0 * (t - rint(t))), &sn, &cs);
    turn[r * half + pair] = make_float2(cs, sn);
  }
  __syncthreads();
  if (row >= a.rows) return;
  const bool turns_here = at < a.rot, second = !NEXT && at >= half;
  const int partner = (lane & ~(LANES - 1)) | ((turns_here ? (second ? at - half : at + half) : at) / 8);
  const uint32_t neighbours = turns_here ? 0x1032 : 0x3210;  // (what does not turn is its own partner: 0 times another infinite number is not 0)
  // The row's heads, loads part, part + parts, ...: `src` and `dst` head 0 of the row, dst_head elements between heads there.
  auto heads_of = [&](const __nv_bfloat16* src, int heads, const __nv_bfloat16* weight, __nv_bfloat16* dst, int dst_head, bool writes, bool loaded) {
    float2 cw[4], sw[4];  // cosine times the weight of each of the lane's elements; sine, with its sign, times the partner's
    {
      const uint4 one = make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u);
      const uint4 own = weight ? *reinterpret_cast<const uint4*>(weight + at) : one;
      const uint4 other = NEXT || !weight ? own : *reinterpret_cast<const uint4*>(weight + (partner & (LANES - 1)) * 8);
      const uint32_t wo[4] = {own.x, own.y, own.z, own.w}, wp[4] = {other.x, other.y, other.z, other.w};
      const float2* tr = turn + (warp / per_row) * half;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        cw[e] = widen(wo[e]);
        sw[e] = make_float2(0.f, 0.f);
        if (!turns_here) continue;
        if constexpr (NEXT) {
          const float2 cs = tr[at / 2 + e];
          sw[e] = make_float2(-cs.y * cw[e].y, cs.y * cw[e].x);
          cw[e] = make_float2(cs.x * cw[e].x, cs.x * cw[e].y);
        } else {
          const float2 c0 = tr[(second ? at - half : at) + 2 * e], c1 = tr[(second ? at - half : at) + 2 * e + 1], p = widen(wp[e]);
          const float sign = second ? 1.f : -1.f;
          sw[e] = make_float2(sign * c0.y * p.x, sign * c1.y * p.y);
          cw[e] = make_float2(c0.x * cw[e].x, c1.x * cw[e].y);
        }
      }
    }
    int head = head0;
    src += first;
    dst += (size_t)head * dst_head + at;
    for (int h0 = part * HEADS; h0 < heads; h0 += kAhead * step) {  // (h0: the same in the whole warp)
      if (!loaded || h0 != part * HEADS) load(src, head, heads);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        if (h0 + u * step >= heads) break;
        const uint32_t w[4] = {in[u].x, in[u].y, in[u].z, in[u].w};
        float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int e = 0; e < 4; ++e) s2 = fma2(widen(w[e]), widen(w[e]), s2);
        float ss = s2.x + s2.y;
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float r = rsqrtf(ss * (1.0f / D) + a.eps);
        uint4 out;
        uint32_t* o = reinterpret_cast<uint32_t*>(&out);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t other = NEXT ? __byte_perm(w[e], 0u, neighbours) : __shfl_sync(0xffffffffu, w[e], partner);
          const float2 y = mul2(fma2(widen(other), sw[e], mul2(widen(w[e]), cw[e])), make_float2(r, r));
          const __nv_bfloat162 p = __floats2bfloat162_rn(y.x, y.y);
          o[e] = *reinterpret_cast<const uint32_t*>(&p);
        }
        if (writes && head + u * step < heads) *reinterpret_cast<uint4*>(dst + (size_t)(u * step) * dst_head) = out;
      }
      head += kAhead * step;
      src += (size_t)(kAhead * step) * D;
      dst += (size_t)(kAhead * step) * dst_head;
    }
  };
  heads_of(a.q + (size_t)row * a.q_stride, a.hq, a.q_weight, a.q_out + (size_t)row * a.q_out_stride, D, true, true);
  if constexpr (!PAGES) {
    heads_of(a.k + (size_t)row * a.k_stride, a.hkv, a.k_weight, a.k_out + (size_t)row * a.k_out_stride, D, true, false);
  } else {
    // a step whose reservation failed has no page for this row: nothing of it is written there (the error word is set)
    const int pos = a.positions[row], seq = a.row_seq[row], page_idx = pos / a.d.page_size;
    const bool have_page = pos >= 0 && seq >= 0 && seq < a.d.max_seqs && page_idx < a.d.seq_pages[seq];
    const int page = have_page ? a.d.block_table[(size_t)seq * a.d.max_pages_per_seq + page_idx] : 0, head_step = a.d.page_size * D;
    const size_t tile = (((size_t)a.layer * a.d.n_pages + page) * a.hkv * a.d.page_size + (have_page ? pos - page_idx * a.d.page_size : 0)) * (size_t)D;
    heads_of(a.k + (size_t)row * a.k_stride, a.hkv, a.k_weight, (__nv_bfloat16*)a.d.k_pool + tile, head_step, have_page, false);
    if (have_page)
      for (int h = part * HEADS + sub; h < a.hkv; h += parts * HEADS)
        *reinterpret_cast<uint4*>((__nv_bfloat16*)a.d.v_pool + tile + (size_t)h * head_step + at) =
            *reinterpret_cast<const uint4*>(a.v + (size_t)row * a.v_stride + (size_t)h * D + at);
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
  // The frequencies of the last call's rotation: a model has one or two.
  static thread_local struct { int rot = 0; double theta = 0.0, turns[kMostPairs]; } last;
  if (last.rot != s->rot_dim || last.theta != s->theta) {
    for (int i = 0; i < s->rot_dim / 2; ++i) last.turns[i] = pow(s->theta, -2.0 * i / s->rot_dim) / (2.0 * M_PI);
    last.rot = s->rot_dim;
    last.theta = s->theta;
  }
  std::copy(last.turns, last.turns + s->rot_dim / 2, a.turns);
  return B200_OK;
}

template <int D, bool PAGES>
void launch_as(const NormRopeArgs& a, dim3 grid, cudaStream_t s) {
  if (a.interleaved) launch_after(qk_norm_rope_kernel<D, PAGES, true>, grid, kWarps * 32, 0, s, a);
  else launch_after(qk_norm_rope_kernel<D, PAGES, false>, grid, kWarps * 32, 0, s, a);
}

template <bool PAGES>
b200_status launch(NormRopeArgs& a, int head_dim, cudaStream_t s) {
  const int heads = 256 / head_dim, loads = std::max(1, std::max((a.hq + heads - 1) / heads, (a.hkv + heads - 1) / heads));
  // warps for a row: enough that there are 32 on every SM, no more than the row has loads
  const int want = std::min(loads, std::max(1, (32 * b200_sm_count() + a.rows - 1) / a.rows));
  a.block_rows = want >= kWarps ? 1 : want > kWarps / 2 ? 1 : want > kWarps / 4 ? 2 : want > 1 ? 4 : 8;
  const dim3 grid((a.rows + a.block_rows - 1) / a.block_rows, (want + kWarps - 1) / kWarps);
  if (head_dim == 64) launch_as<64, PAGES>(a, grid, s);
  else if (head_dim == 128) launch_as<128, PAGES>(a, grid, s);
  else launch_as<256, PAGES>(a, grid, s);
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
