// Products of rows and weights in 8-bit integers, and the gated feed-forward block made of them:
//   y[t][n] = (sum_k q[t][k] w[n][k]) scale[n] step[t] + bias[n],   q[t][k] = round(127 x[t][k] / max_k |x[t][k]|),  step[t] = max_k |x[t][k]| / 127.
//
// The sums are exact (int32 on tcgen05.mma kind::i8), so neither the order of K nor what shares a tile changes a bit of a row.
//
// Few rows are bound by the weights: one row of 4096 to 6144 7.0 us in a graph, one through a block of 14336 32 (176 MB, 5.5 TB/s), 96 through it 42.  Many are bound by
// the tensor cores under the power cap.  In a run of a second and more (1.49 GHz in the middle, the cap its only reason) 8192 rows of 4096 to 6144 take 185 us; with an event
// between its kernels, which ends their overlap, 33 for the rows and 157 for the product (2.6 PFLOP/s).  Through a block of 14336 they take 1204 to 1220; apart in the same run
// 36 the rows, 720 gate and up (2.7 PFLOP/s), 124 the inner rows, 329 down (2.9): 1208.  The first milliseconds are faster, as the clock falls only then: 155 and 1067 in a graph.
#include <cuda_bf16.h>
#include <math.h>

#include <algorithm>
#include <new>
#include <type_traits>

#include "common.h"
#include "i8.cuh"
#include "launch.cuh"
#include "ptx.cuh"
#include "qmm.cuh"
#include "rows.cuh"

namespace {

// ---- rows into 8 bits ----------------------------------------------------------------------------------------------------
// A row waits in registers while its largest is looked for: a block for each, or a warp where a row is short.  Bound by what it reads and writes, and by its
// arithmetic in turn: 8192 rows of 4096 22.6 us (4.4 TB/s), 96 1.9.  (A warp for each of eight neighbouring rows, whose bytes lie together: 38.)
struct QuantizeArgs {
  const __nv_bfloat16* x;
  long long x_stride;
  signed char* q;
  float* scale;
  int rows, k, chunks, aligned;
};

// NV: vectors of eight columns of a thread; 0: any number, the row is read twice.  WARP: a warp for a row.  FIT: rows start on 16 bytes and are whole vectors.
template <int NV, bool WARP, bool FIT>
__global__ void __launch_bounds__(WARP ? 256 : 1024) i8_quantize_kernel(QuantizeArgs a) {
  after_previous();
  __shared__ uint32_t part[32];
  const int threads = WARP ? 32 : blockDim.x, t = WARP ? threadIdx.x & 31 : threadIdx.x;
  const int row = WARP ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= a.rows) return;
  const __nv_bfloat16* x = a.x + (size_t)row * a.x_stride;
  const int vectors = a.chunks * (kI8Chunk / 8);
  auto load = [&](int v) { return load_eight(x, v * 8, a.k, FIT || a.aligned); };
  Eight<__nv_bfloat16> keep[NV > 0 ? NV : 1];
  uint32_t most = 0u;
  if constexpr (NV > 0) {
    load_eights(keep, x, a.k, FIT || a.aligned, [&](int u) { return (t + u * threads) * 8; });
#pragma unroll
    for (int u = 0; u < NV; ++u) most = most_of(most, keep[u]);
  } else {
    for (int v = t; v < vectors; v += threads) most = most_of(most, load(v));
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if constexpr (!WARP) {
    if ((t & 31) == 0) part[t >> 5] = most;
    __syncthreads();
    most = __reduce_max_sync(0xffffffffu, (t & 31) < (threads >> 5) ? part[t & 31] : 0u);
  }
  const I8Scale s = I8Scale::of(__uint_as_float(most));
  if (t == 0) a.scale[row] = s.step();
  // (a round further on is threads / 16 blocks further on, at the same place)
  signed char* to = a.q + i8_at(row, t * 8, a.chunks);
  auto put = [&](const Eight<__nv_bfloat16>& raw, int round) {
    float f[8];
    widen(raw, f);
    *reinterpret_cast<uint2*>(to + (size_t)round * (threads / 16) * kI8Block) = s.quantize(f);
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int u = 0; u < NV; ++u)
      if (t + u * threads < vectors) put(keep[u], u);
  } else {
    for (int v = t, u = 0; v < vectors; v += threads, ++u) put(load(v), u);
  }
}

template <bool FIT>
void launch_quantize(const QuantizeArgs& a, cudaStream_t s) {
  const int vectors = a.chunks * (kI8Chunk / 8), rows = a.rows;
  if (vectors <= 32 * 2) {
    const int warps = rows >= 8 * b200_sm_count() ? 8 : 1;
    const unsigned grid = (unsigned)((rows + warps - 1) / warps);
    if (vectors <= 32) launch_after(i8_quantize_kernel<1, true, FIT>, grid, warps * 32, 0, s, a);
    else launch_after(i8_quantize_kernel<2, true, FIT>, grid, warps * 32, 0, s, a);
  } else if (vectors <= 4 * 1024) {
    // few rows: more threads, each with fewer loads to wait for (96 rows of 4096 1.9 us with one, 2.8 with four; 8192 46 and 22.6)
    const int nv = rows > 4 * b200_sm_count() || vectors > 2048 ? 4 : vectors > 1024 ? 2 : 1, threads = (vectors + 32 * nv - 1) / (32 * nv) * 32;
    if (nv == 1) launch_after(i8_quantize_kernel<1, false, FIT>, rows, threads, 0, s, a);
    else if (nv == 2) launch_after(i8_quantize_kernel<2, false, FIT>, rows, threads, 0, s, a);
    else launch_after(i8_quantize_kernel<4, false, FIT>, rows, threads, 0, s, a);
  } else {
    launch_after(i8_quantize_kernel<0, false, FIT>, rows, 1024, 0, s, a);
  }
}

b200_status quantize(const __nv_bfloat16* x, long long x_stride, int rows, int k, const I8RowsDev& to, cudaStream_t s) {
  QuantizeArgs a;
  a.x = x; a.x_stride = x_stride; a.q = to.q; a.scale = to.scale; a.rows = rows; a.k = k; a.chunks = i8_chunks(k);
  a.aligned = ((uintptr_t)x & 15) == 0 && x_stride % 8 == 0;
  if (a.aligned && k % 8 == 0) launch_quantize<true>(a, s);
  else launch_quantize<false>(a, s);
  B200_LAUNCH_CHECK();
  return B200_OK;
}

// The feed-forward block's inner rows, of which the product that made them has left the largest of every 32 channels, so that nothing waits for a row to be
// read and a row may be many blocks'.  A block's warps take eight neighbouring rows, whose bytes lie together.  Bound by what it reads and writes: 8192 rows of 14336
// 118 us, 5 TB/s (141 as a block for each row); behind a short product, whose results are still on their way to memory, 130.
constexpr int kInnerThreads = 256, kInnerAhead = 4;  // (loads of 256 columns that a warp has in flight)

__global__ void __launch_bounds__(kInnerThreads, 3) i8_quantize_inner_kernel(const float* h, long long h_stride, const float* most, int groups, signed char* __restrict__ q,
                                                                             float* __restrict__ steps, int rows, int k, int chunks, int per_block) {
  after_previous();
  const int lane = threadIdx.x & 31, row = blockIdx.x * (kInnerThreads / 32) + (threadIdx.x >> 5);
  if (row >= rows) return;
  const int first = blockIdx.y * per_block, last = min(first + per_block, chunks * kI8Chunk);
  const float* from = h + (size_t)row * h_stride + lane * 8;
  float4 keep[kInnerAhead][2];
  auto load = [&](int c0) {  // (rows are whole vectors, what lies behind the last column of the last one is not looked at)
#pragma unroll
    for (int u = 0; u < kInnerAhead; ++u) {
      keep[u][0] = keep[u][1] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (c0 + u * 256 + lane * 8 < k) {
        keep[u][0] = *reinterpret_cast<const float4*>(from + c0 + u * 256);
        keep[u][1] = *reinterpret_cast<const float4*>(from + c0 + u * 256 + 4);
      }
    }
  };
  load(first);
  uint32_t m = 0u;
  for (int g = lane; g < groups; g += 32) m = max(m, __float_as_uint(most[(size_t)row * groups + g]));
  const I8Scale s = I8Scale::of(__uint_as_float(__reduce_max_sync(0xffffffffu, m)));
  if (blockIdx.y == 0 && lane == 0) steps[row] = s.step();
  signed char* to = q + i8_at(row, first + lane * 8, chunks);
  for (int c0 = first; c0 < last; c0 += kInnerAhead * 256, to += kInnerAhead * 2 * kI8Block) {
    if (c0 > first) load(c0);
#pragma unroll
    for (int u = 0; u < kInnerAhead; ++u) {
      float f[8] = {keep[u][0].x, keep[u][0].y, keep[u][0].z, keep[u][0].w, keep[u][1].x, keep[u][1].y, keep[u][1].z, keep[u][1].w};
      const int left = k - (c0 + u * 256 + lane * 8);
      if (left < 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e >= left) f[e] = 0.f;
      }
      if (c0 + u * 256 + lane * 8 < last) *reinterpret_cast<uint2*>(to + u * 2 * kI8Block) = s.quantize(f);
    }
  }
}

b200_status quantize_inner(const b200_i8_rows* r, int rows, int k, cudaStream_t s) {
  const int chunks = i8_chunks(k), eights = (rows + 7) / 8;
  // Columns: fewer blocks where there are enough of them (8192 rows through a block of 14336 1018 us, 1044 with 1024 columns a block; no more than 4096: 1015).
  int per_block = kInnerAhead * 256;
  while (per_block < 4096 && (long long)eights * ((chunks * kI8Chunk + per_block - 1) / per_block) >= 8 * b200_sm_count()) per_block *= 2;
  launch_after(i8_quantize_inner_kernel, dim3(eights, (chunks * kI8Chunk + per_block - 1) / per_block), kInnerThreads, 0, s, r->h, (long long)r->h_stride, r->most, chunks * 4,
               r->hidden.q, r->hidden.scale, rows, k, chunks, per_block);
  B200_LAUNCH_CHECK();
  return B200_OK;
}

// ---- what the handles hold, into and out of its order -----------------------------------------------------------------------
// A thread for sixteen columns of a row of the laid-out weight.
__global__ void i8_lay_out_kernel(const signed char* src, const float* scales, int n, int k, int chunks, int tile0, int tile_step, int tiles, signed char* __restrict__ q,
                                  float* __restrict__ scale) {
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  const int per_row = chunks * 8;
  const long long row = i / per_row;
  const int piece = (int)(i - row * per_row);
  if (row >= (long long)tiles * kI8Tile) return;
  uint32_t w[4] = {0u, 0u, 0u, 0u};
  if (row < n)
    for (int e = 0; e < 16; ++e)
      if (piece * 16 + e < k) w[e / 4] |= (uint32_t)(unsigned char)src[(size_t)row * k + piece * 16 + e] << (8 * (e % 4));
  const int to = (int)(tile0 + row / kI8Tile * tile_step), r = (int)(row % kI8Tile);
  *reinterpret_cast<uint4*>(q + ((size_t)to * chunks + piece / 8) * kI8Block + r * kI8Chunk + (((piece % 8) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
  if (piece == 0) scale[(size_t)to * kI8Tile + r] = row < n ? scales[row] : 0.f;
}

__global__ void i8_rows_get_kernel(I8RowsDev from, int rows, int k, int chunks, signed char* __restrict__ q, float* __restrict__ steps) {
  after_previous();
  const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= (long long)rows * k) return;
  const int row = (int)(i / k), c = (int)(i - (long long)row * k);
  if (q) q[i] = from.q[i8_at(row, c, chunks)];
  if (steps && c == 0) steps[row] = from.scale[row];
}

// ---- products ----------------------------------------------------------------------------------------------------------------
struct MmArgs {
  const signed char* w;
  const float* w_scale;
  const signed char* q;
  const float* step;
  const float* bias;
  void* y;
  long long y_stride;
  float* most;  // a feed-forward block's inner rows: [row][tiles * 2] the largest magnitude of 32 channels
  int* err;
  int rows, n, chunks, tiles, tn, stages, shares;
  int over_stages, pushed_at, raw_at, bars_at;  // places in shared memory (i8_stream_kernel)
  // Rows that the kernel brings into 8 bits itself
  const void* raw;
  long long raw_stride;
  int raw_inner, raw_fit, k;  // f32, with the largest of every 32 channels in raw_most; or bf16, which go into q_out and step_out as well
  const float* raw_most;
  signed char* q_out;
  float* step_out;
  int y_vec;       // rows of y start on 16 bytes
  int y_f32, act;  // (a feed-forward block's inner rows are f32)
};

// D[tmem] (+)= A B of signed 8-bit integers, 32-bit sums.
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor: signed 8-bit A and B (both K-major), 32-bit sums, tile m x n.
__device__ __forceinline__ uint32_t idesc_i8(uint32_t m, uint32_t n) { return 2u << 4 | 1u << 7 | 1u << 10 | (n >> 3) << 17 | (m >> 4) << 24; }

// What follows is the same for every kernel, so the compiler is told which products and sums to fuse: a row's bits must not depend on the kernel that has it.
// A sum as a number of the product.
__device__ __forceinline__ float scaled(uint32_t sum, float w, float step, float bias) { return __fmaf_rn(__fmul_rn((float)(int)sum, w), step, bias); }
__device__ __forceinline__ float scaled(uint32_t sum, float w, float step) { return __fmul_rn(__fmul_rn((float)(int)sum, w), step); }
// The exponentials are the hardware's, off by 2 + 1.16 |z| of their last place: 2^-20 of a number at |z| of 9, whose own size is 1e-3 then, beside a step of 1/127 of the row's
// largest in which the result is held.
template <int ACT>
__device__ __forceinline__ float activated(float g) {
  if constexpr (ACT == B200_ACT_SILU) return __fdividef(g, __fadd_rn(1.0f, __expf(-g)));  // (a divisor past 2^126 makes 0, as it should)
  if constexpr (ACT == B200_ACT_GELU) return __fmul_rn(__fmul_rn(0.5f, g), __fadd_rn(1.0f, erff(__fmul_rn(g, 0.70710678118654752f))));
  // 0.5 g (1 + tanh z) = g / (1 + e^-2z)
  return __fdividef(g, __fadd_rn(1.0f, __expf(__fmul_rn(-1.5957691216057308f, __fmaf_rn(__fmul_rn(__fmul_rn(0.044715f, g), g), g, g)))));
}
// y[j] = act(y[j]) * up[j]; the activation is chosen once.
template <int N>
__device__ __forceinline__ void gate_with(int act, float (&y)[N], const float (&up)[N]) {
  auto each = [&](auto which) {
#pragma unroll
    for (int j = 0; j < N; ++j) y[j] = __fmul_rn(activated<decltype(which)::value>(y[j]), up[j]);
  };
  if (act == B200_ACT_SILU) each(std::integral_constant<int, B200_ACT_SILU>{});
  else if (act == B200_ACT_GELU) each(std::integral_constant<int, B200_ACT_GELU>{});
  else each(std::integral_constant<int, B200_ACT_GELU_TANH>{});
}

// ---- up to a few hundred rows: streams of weights ----
// A weight tile (gated: the gate's and up's tile of the same channels) by up to tn rows and a share of K per CTA.  The weights are the MMA's M, the rows
// its N, so that few rows waste nothing; a lane of tensor memory is a channel.  Warp 0 loads, warp 1 multiplies, eight bring the sums to the output, each every
// other sixteen rows of 32 channels.
// Bound by the weights, which come at the rate of memory only if every SM asks for them (an SM gets 16 KB of them in 0.27 us, however many are on their way): a
// cluster of up to eight CTAs shares K, an SM for each.  A CTA brings a share of the rows to the output and gets the others' sums of these
// pushed into its shared memory, where the stages were unless there is room beside them, with a barrier that counts their bytes.
constexpr int kStreamThreads = 320, kStreamShared = 112 * 1024, kStreamAlone = 226 * 1024, kMostShares = 8;  // (shared memory of two CTAs on an SM, of one)

// Weights that go through L2 once, where all rows are one tile's, leave it ahead of what else is there.  (Among it are the instructions, which a kernel fetches anew: behind
// 117 MB of weights the last ones came from memory, 4 to 8 us for the output of one row.)  With more tiles of rows they are read again, and stay as anything else does.
__device__ __forceinline__ uint64_t weights_in_l2(bool once) {
  uint64_t p;
  if (once) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  else asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(p));
  return p;
}
__device__ __forceinline__ void bulk_g2s_with(void* dst_smem, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(ptx::smem_u32(dst_smem)), "l"(src), "r"(bytes),
               "r"(ptx::smem_u32(bar)), "l"(policy) : "memory");
}
// Four words to another CTA of the cluster, counted by a barrier there.
__device__ __forceinline__ void push4(uint32_t mapped, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t mapped_bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(mapped), "r"(a), "r"(b), "r"(c), "r"(d),
               "r"(mapped_bar) : "memory");
}
// Waits for what the other CTAs push.  It comes from outside this CTA, so the wait acquires in the cluster's scope: by an ordinary one, of this CTA's, the sums would not be
// ordered ahead of the loads behind it.
__device__ __forceinline__ bool wait_pushed(uint32_t bar) {
  for (uint32_t i = 0; i < ptx::kSpinLimit; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar)
        : "memory");
    if (ok) return true;
    if (i > 64) __nanosleep(64);
  }
  return false;
}
// The rows that a CTA of the cluster brings to the output: CTA q the q-th so many, a multiple of four.
__host__ __device__ constexpr int rows_per_rank(int rows_here, int shares) { return ((rows_here + shares - 1) / shares + 3) / 4 * 4; }
// What it gets pushed: [other CTA][gate, up][four rows][channel][row].
__host__ __device__ constexpr int pushed_bytes(int rows_here, int shares, int parts) { return (shares - 1) * parts * rows_per_rank(rows_here, shares) * kI8Tile * 4; }

// Tensor memory of a CTA.  Those of a cluster wait for one another while they hold theirs, so a CTA on the same SM may never have to wait for its own: a
// launch asks for at least kSharedPerCol bytes of shared memory a column, of which an SM's 228 KB (a KB of them for itself in every CTA) are 512 columns' at most.
__host__ __device__ constexpr uint32_t stream_cols(int tn, int parts) { return tn * parts < 32 ? 32u : (uint32_t)(tn * parts); }
constexpr int kSharedPerCol = 440;

// Sums of four rows from `col` on, of this warp's 32 channels.
__device__ __forceinline__ void tmem_ld4(uint32_t taddr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(taddr) : "memory");
}

// RAW's rows; their numbers at most; blocks of K in a share at most, and times the rows (four rows through a block of 14336: 35.1 us with kernels of their own for
// the rows, 37.6 without; two 34.8 and 33.8; four through one of 8192 17.8 and 16.7).
constexpr int kRawRows = 4, kRawNumbers = 16384, kRawChunks = 32, kRawWork = 64;

// Warps 2 to 9: rows into 8 bits, as i8_quantize_kernel and i8_quantize_inner_kernel do, blocks chunk0 and on as an operand of 16 rows each at `to` (the rows that
// are not there hold anything), steps into `steps`; `out` and `first`: into the handle too, and the steps.
template <typename T>
__device__ __forceinline__ void raw_rows(const MmArgs& a, const T* x, bool fit, unsigned char* to, int chunk0, int chunks, bool out, bool first, uint64_t* ready, float* steps,
                                         uint32_t* part) {
  constexpr bool kInner = sizeof(T) == 4;
  constexpr int kAhead = 4, kWarps = kStreamThreads / 32 - 2;
  // The rows at the same time, each by as many warps.
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) - 2, warps = a.rows == 1 ? kWarps : a.rows == 2 ? kWarps / 2 : kWarps / 4, threads = warps * 32;
  const int r = warp / warps, t = (warp - r * warps) * 32 + lane;
  const bool there = r < a.rows;
  const T* row = x + (size_t)(there ? r : 0) * a.raw_stride;
  uint32_t m = 0u;
  if constexpr (kInner) {
    for (int g = t; g < a.chunks * 4; g += threads) m = max(m, __float_as_uint(a.raw_most[(size_t)(there ? r : 0) * (a.chunks * 4) + g]));
  } else {
#pragma unroll 1
    for (int v = t; v * 8 < a.k; v += kAhead * threads) {
      Eight<T> e[kAhead];
      load_eights(e, row, a.k, fit, [&](int u) { return (v + u * threads) * 8; });
#pragma unroll
      for (int u = 0; u < kAhead; ++u) m = most_of(m, e[u]);
    }
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) part[warp] = m;
  asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");
  if (there) {
    const I8Scale s = I8Scale::of(__uint_as_float(__reduce_max_sync(0xffffffffu, part[r * warps + lane % warps])));
    if (t == 0) {
      steps[r] = s.step();
      if (out && first && !kInner) a.step_out[r] = s.step();
    }
#pragma unroll 1
    for (int v = t; v < chunks * 16; v += kAhead * threads) {
      Eight<T> e[kAhead];
      load_eights(e, row, a.k, fit, [&](int u) { return chunk0 * kI8Chunk + (v + u * threads) * 8; });
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int at = v + u * threads, piece = at & 15;
        if (at >= chunks * 16) break;
        float f[8];
        widen(e[u], f);
        const uint2 q = s.quantize(f);
        *reinterpret_cast<uint2*>(to + (at >> 4) * 16 * kI8Chunk + r * kI8Chunk + (((piece >> 1) ^ r) << 4) + (piece & 1) * 8) = q;
        if (out && !kInner) *reinterpret_cast<uint2*>(a.q_out + i8_at(r, chunk0 * kI8Chunk + at * 8, a.chunks)) = q;
      }
    }
  }
  ptx::fence_proxy_async_smem();
  asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory");  // the steps are there
  if (lane == 0) ptx::mbar_arrive(ready);
}

// RAW: up to kRawRows rows that are not 8 bits yet: every CTA looks for their largest numbers itself and keeps its share of K in shared memory, while the first
// weights come.  (A kernel of its own for one row costs 2.5 us, and as much of the host's time.)
template <bool GATED, bool RAW>
__global__ void __launch_bounds__(kStreamThreads, 2) i8_stream_kernel(MmArgs a) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  constexpr int W = GATED ? 2 : 1;
  const int S = a.stages, stage_bytes = W * kI8Block + (RAW ? 0 : a.tn * kI8Chunk);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + a.bars_at);
  uint64_t* done = full + S;
  uint64_t* sums = done + S;
  uint64_t* pushed = sums + 1;
  uint64_t* rows_ready = pushed + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(rows_ready + 1);
  float* raw_steps = reinterpret_cast<float*>(tmem_slot + 1);                    // [kRawRows]
  uint32_t* raw_part = reinterpret_cast<uint32_t*>(raw_steps + kRawRows);        // [warp]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int shares = a.shares, rank = shares > 1 ? (int)ptx::cluster_rank() : 0;
  const int tile = blockIdx.x / shares, t0 = blockIdx.y * a.tn, rows_here = min(a.tn, a.rows - t0), n_here = (rows_here + 15) / 16 * 16;
  const int per_share = (a.chunks + shares - 1) / shares, chunk0 = rank * per_share, chunks = min(per_share, a.chunks - chunk0);  // (never none)
  const int per_rank = rows_per_rank(rows_here, shares), mine0 = min(rows_here, rank * per_rank), mine1 = min(rows_here, mine0 + per_rank);
  const uint32_t cols = stream_cols(a.tn, W);
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&done[s], 1);
    }
    ptx::mbar_init(sums, 1);
    ptx::mbar_init(pushed, 1);
    ptx::mbar_init(rows_ready, 8);
    ptx::mbar_fence_init();
    ptx::mbar_expect_tx(pushed, (shares - 1) * W * ((mine1 - mine0 + 3) / 4) * kI8Tile * 16);
  }
  __syncthreads();
  if (shares > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // this CTA's barriers are there
  const uint64_t policy = weights_in_l2(gridDim.y == 1);
  auto load_weights = [&](int i, int s) {
    ptx::mbar_expect_tx(&full[s], W * kI8Block + (RAW ? 0 : n_here * kI8Chunk));
    for (int h = 0; h < W; ++h)
      bulk_g2s_with(smem + (size_t)s * stage_bytes + h * kI8Block, a.w + ((size_t)(tile * W + h) * a.chunks + chunk0 + i) * kI8Block, kI8Block, &full[s], policy);
  };
  auto load_rows = [&](int i, int s) {  // (a tile of 256 rows is two of the layout's)
    for (int r = 0; r < n_here && !RAW; r += kI8Tile) {
      const int row = t0 + r;
      ptx::bulk_g2s(smem + (size_t)s * stage_bytes + W * kI8Block + r * kI8Chunk,
                    a.q + ((size_t)(row / kI8Tile) * a.chunks + chunk0 + i) * kI8Block + row % kI8Tile * kI8Chunk, min(kI8Tile, n_here - r) * kI8Chunk, &full[s]);
    }
  };
  const int ahead = min(S, chunks);  // weights asked for before the kernels ahead have ended
  if (threadIdx.x == 0)
    for (int i = 0; i < ahead; ++i) load_weights(i, i);
  wait_previous();
  if (threadIdx.x == 0)
    for (int i = 0; i < ahead; ++i) load_rows(i, i);
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, cols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;
  if (warp == 0) {
    if (lane == 0) {
      int s = ahead == S ? 0 : ahead, issued = ahead;
      uint32_t ph = 0;
      for (int i = ahead; i < chunks; ++i) {
        ok = ptx::mbar_wait(&done[s], ph);
        if (!ok) break;
        load_weights(i, s);
        load_rows(i, s);
        ++issued;
        if (++s == S) { s = 0; ph ^= 1u; }
      }
      let_next_start();
      if (!ok)  // copies are on their way into this memory
        for (int i = max(0, issued - S); i < issued; ++i) ptx::mbar_wait(&full[i % S], (i / S) & 1);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (ptx::elect_one()) {
      const uint32_t idesc = idesc_i8(kI8Tile, n_here);
      int s = 0;
      uint32_t ph = 0;
      if constexpr (RAW) ok = ptx::mbar_wait(rows_ready, 0);
      const int todo = ok ? chunks : 0;
      for (int i = 0; i < todo; ++i) {
        ok = ptx::mbar_wait(&full[s], ph);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        const uint32_t at = ptx::smem_u32(smem + (size_t)s * stage_bytes);
        const uint64_t db = ptx::umma_desc_k_sw128(RAW ? ptx::smem_u32(smem + a.raw_at) + i * 16 * kI8Chunk : at + W * kI8Block);
#pragma unroll
        for (int h = 0; h < W; ++h) {
          const uint64_t da = ptx::umma_desc_k_sw128(at + h * kI8Block);
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) umma_i8(tmem + h * a.tn, da + 2 * k4, db + 2 * k4, idesc, (i > 0 || k4 > 0) ? 1u : 0u);
        }
        ptx::umma_commit(&done[s]);
        if (++s == S) { s = 0; ph ^= 1u; }
      }
      ptx::umma_commit(sums);
      if (!ok) ptx::mbar_wait(sums, 0);
    }
    __syncwarp();
  }
  const int quarter = warp & 3, half = (warp - 2) >> 2, channel = tile * kI8Tile + quarter * 32 + lane;
  const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16);
  float ws = 0.f, us = 0.f, bias = 0.f;
  auto steps_of = [&](int c0) { return c0 + (lane & 15) < mine1 ? (RAW ? raw_steps[(c0 + lane) % kRawRows] : a.step[t0 + c0 + (lane & 15)]) : 0.f; };  // sixteen rows' in the lanes
  if constexpr (RAW) {
    if (warp >= 2) {
      const bool out = blockIdx.x < shares;
      unsigned char* to = smem + a.raw_at;
      if (!GATED && a.raw_inner) raw_rows(a, (const float*)a.raw, true, to, chunk0, chunks, false, false, rows_ready, raw_steps, raw_part);
      else if (a.raw_fit) raw_rows(a, (const __nv_bfloat16*)a.raw, true, to, chunk0, chunks, out, rank == 0, rows_ready, raw_steps, raw_part);
      else raw_rows(a, (const __nv_bfloat16*)a.raw, false, to, chunk0, chunks, out, rank == 0, rows_ready, raw_steps, raw_part);
    }
  }
  // Sixteen rows' sums, as far as they go.
  auto load_sums = [&](int c0, int end, uint32_t (&v)[16], uint32_t (&u)[16]) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = u[j] = 0u;
#pragma unroll
    for (int g = 0; g < 16; g += 4)
      if (c0 + g < end) {
        tmem_ld4(acc + c0 + g, v[g], v[g + 1], v[g + 2], v[g + 3]);
        if constexpr (GATED) tmem_ld4(acc + a.tn + c0 + g, u[g], u[g + 1], u[g + 2], u[g + 3]);
      }
    ptx::tmem_ld_wait();
  };
  if (warp >= 2) {
    const size_t scale_at = (size_t)tile * W * kI8Tile + quarter * 32 + lane;
    ws = a.w_scale[scale_at];
    if (GATED) us = a.w_scale[scale_at + kI8Tile];
    if (!GATED && a.bias && channel < a.n) bias = a.bias[channel];
    // Once without sums, while these are made: the instructions are then there when they are needed.
#pragma unroll 1
    for (int live = 0; live < 2; ++live) {
      int end = live ? mine1 : mine0 + half * 16 + 1;  // (one round)
      if (live) {
        ok = ptx::mbar_wait(sums, 0);
        ok = __all_sync(0xffffffffu, ok);
        ptx::tc_fence_after_sync();
        if (shares > 1) {
          asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // the others' barriers are there
          if (a.over_stages) ptx::cluster_sync();                              // nobody's stages are in use
          if (ok) {
#pragma unroll 1
            for (int i = 1; i < shares; ++i) {
              const int q = rank + i < shares ? rank + i : rank + i - shares, q0 = min(rows_here, q * per_rank), q1 = min(rows_here, q0 + per_rank);
              const uint32_t bar = ptx::map_to_rank(ptx::smem_u32(pushed), q), part = per_rank / 4 * kI8Tile * 16;
              uint32_t to = ptx::map_to_rank(ptx::smem_u32(smem + a.pushed_at), q) + (rank - (rank > q)) * W * part + (half * 4 * kI8Tile + quarter * 32 + lane) * 16;
#pragma unroll 1
              for (int c0 = q0 + half * 16; c0 < q1; c0 += 32, to += 8 * kI8Tile * 16) {
                uint32_t v[16], u[16];
                load_sums(c0, q1, v, u);
#pragma unroll
                for (int g = 0; g < 16; g += 4)
                  if (c0 + g < q1) {
                    push4(to + g / 4 * kI8Tile * 16, v[g], v[g + 1], v[g + 2], v[g + 3], bar);
                    if constexpr (GATED) push4(to + part + g / 4 * kI8Tile * 16, u[g], u[g + 1], u[g + 2], u[g + 3], bar);
                  }
              }
            }
          }
          __syncwarp();
          asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
          if (mine0 < mine1) ok &= (bool)__all_sync(0xffffffffu, wait_pushed(ptx::smem_u32(pushed)));  // (where a wait here ran out, too: the others push all the same)
        }
        if (!ok) end = 0;
      }
#pragma unroll 1
      for (int c0 = mine0 + half * 16; c0 < end; c0 += 32) {
        uint32_t v[16], u[16];
        const float steps = steps_of(c0);  // (ahead of the stores, which loads do not pass)
        load_sums(c0, live ? mine1 : 0, v, u);
        const uint4* from = reinterpret_cast<const uint4*>(smem + a.pushed_at) + (c0 - mine0) / 4 * kI8Tile + quarter * 32 + lane;
#pragma unroll 1
        for (int q = 0; q < shares - 1; ++q, from += W * (per_rank / 4) * kI8Tile) {
#pragma unroll
          for (int g = 0; g < 16; g += 4)
            if (live && c0 + g < mine1) {
              const uint4 p = from[g / 4 * kI8Tile];
              v[g] += p.x; v[g + 1] += p.y; v[g + 2] += p.z; v[g + 3] += p.w;
              if constexpr (GATED) {
                const uint4 p2 = from[(per_rank / 4 + g / 4) * kI8Tile];
                u[g] += p2.x; u[g + 1] += p2.y; u[g + 2] += p2.z; u[g + 3] += p2.w;
              }
            }
        }
        // All sixteen are worked out before the first is stored: one after the other each took 100 cycles of latencies.
        float y[16], up[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float step = __shfl_sync(0xffffffffu, steps, j);
          y[j] = scaled(v[j], ws, step, bias);
          if constexpr (GATED) up[j] = scaled(u[j], us, step);
        }
        if constexpr (GATED) {
          gate_with(a.act, y, up);
          uint32_t most = 0u;  // lane j keeps row j's
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(y[j]) & 0x7fffffffu);
            if (lane == j) most = m;
          }
          if (live && c0 + lane < mine1 && lane < 16) a.most[(size_t)(t0 + c0 + lane) * (a.tiles * 2) + tile * 4 + quarter] = __uint_as_float(most);
        }
        const size_t at = (size_t)(t0 + c0) * a.y_stride + channel;
        const int rows_left = live && channel < a.n ? mine1 - c0 : 0;
        if (GATED || a.y_f32) {
          float* to = reinterpret_cast<float*>(a.y) + at;
#pragma unroll
          for (int j = 0; j < 16; ++j, to += a.y_stride)
            if (j < rows_left) *to = y[j];
        } else {
          __nv_bfloat16* to = reinterpret_cast<__nv_bfloat16*>(a.y) + at;
#pragma unroll
          for (int j = 0; j < 16; ++j, to += a.y_stride)
            if (j < rows_left) *to = __float2bfloat16(y[j]);
        }
      }
    }
  } else if (shares > 1) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (a.over_stages) ptx::cluster_sync();
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  if (!ok) atomicExch(a.err, B200_ERR_DEVICE_FLAGGED);
  __syncwarp();
  ptx::tc_fence_before_sync();
  if (shares > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // nobody leaves while something may be pushed to it
  __syncthreads();
  if (warp == 1) ptx::tmem_dealloc(tmem, cols);
}

// ---- many rows: pairs of CTAs ----
// Two CTAs share an MMA of 256 rows by 256 weight rows: each brings 128 of both and holds the sums of its 128 rows, so that an MMA reads 8 KiB of each CTA's
// shared memory in the 128 cycles that it takes.  Persistent: a pair walks the items, a tile of rows by a pair of weight tiles (gated: the gate's and
// up's of the same 128 channels), rows fastest within bands of kPairBand tiles, so that both
// operands come from L2 (8192 rows through a block of 14336 1017 us in a graph, bands of 4, 8 and 32 tiles 1057, 1031 and 1023).  An item's sums are half of tensor memory: eight
// warps drain one half while the MMAs fill the other.
// Where there are fewer items than pairs, a cluster of up to four pairs shares an item's K, an item to a cluster: groups of 32 columns go to the pairs in
// turn, and a CTA gets the others' sums of its groups pushed into its shared memory, where the stages were.
// Warps: 0 loads both operands of this CTA, 1 multiplies (in a pair's first CTA), 2 tells the first CTA that this one's stage is complete, 4-11 bring the
// sums to the output.
constexpr int kPairThreads = 384, kPairStage = 2 * kI8Block, kPairStages = 6, kPairRows = 256, kPairBand = 16, kMostPairs = 4;
constexpr int kPairPitch = 20;  // epilogue: words between rows in a warp's staging tile of 32 rows by 16 words
constexpr int kPairShared = 1024 + kPairStages * kPairStage + 8 * 32 * kPairPitch * 4 + 8 * 2 * kI8Tile * 4 + 8 * (3 * kPairStages + 6) + 16;
// (A pair's CTAs hold all tensor memory of their SMs while they wait for one another, so none may lie beside another kernel's that holds some: what is left has no room
// for a CTA of i8_stream_kernel, whose one block of weights and rows is 18 KB.)
static_assert(kPairShared > (228 - 20) * 1024, "a pair's CTA has its SM for itself");

__device__ __forceinline__ void umma2_i8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// ptx::umma2_commit in a cluster of several pairs.
__device__ __forceinline__ void commit_pair(uint32_t bar, uint16_t ctas) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(ctas) : "memory");
}

// A warp's 32 rows by 32 columns from the item's column c0 on, whose sums are v (gated: with up's in u), to the output, through shared memory, so that a
// store is 64 contiguous bytes of a row.  scales: these columns' factors, and 128 floats behind them up's, or the bias.
template <bool GATED>
__device__ __forceinline__ void store_sums(const MmArgs& a, uint32_t (&v)[32], const uint32_t (&u)[GATED ? 32 : 1], float* mine, const float* scales, int first_tile, int c0, int row0, float row_step) {
  const int lane = threadIdx.x & 31, rows_here = min(32, a.rows - row0), n0 = (GATED ? first_tile / 2 : first_tile) * kI8Tile + c0, cols = min(32, a.n - n0);
  if (rows_here <= 0) return;
  if (cols <= 0) {  // (nothing is the largest there)
    if (GATED && lane < rows_here) a.most[(size_t)(row0 + lane) * (a.tiles * 2) + n0 / 32] = 0.f;
    return;
  }
  float y[32], up[GATED ? 32 : 1];
#pragma unroll
  for (int j4 = 0; j4 < 8; ++j4) {
    const float4 w4 = *reinterpret_cast<const float4*>(scales + 4 * j4), o4 = *reinterpret_cast<const float4*>(scales + kI8Tile + 4 * j4);
    const float w[4] = {w4.x, w4.y, w4.z, w4.w}, o[4] = {o4.x, o4.y, o4.z, o4.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = 4 * j4 + e;
      y[j] = scaled(v[j], w[e], row_step, GATED ? 0.f : o[e]);
      if constexpr (GATED) up[j] = scaled(u[j], o[e], row_step);
    }
  }
  if constexpr (GATED) gate_with(a.act, y, up);
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(y[j]);
  if constexpr (GATED) {
    uint32_t most = 0u;
#pragma unroll
    for (int j = 0; j < 32; ++j) most = max(most, v[j] & 0x7fffffffu);
    if (lane < rows_here) a.most[(size_t)(row0 + lane) * (a.tiles * 2) + n0 / 32] = __uint_as_float(most);
  }
  if (GATED || a.y_f32) {
#pragma unroll
    for (int x = 0; x < 32; x += 16) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<uint4*>(mine + lane * kPairPitch + 4 * q) = make_uint4(v[x + 4 * q], v[x + 4 * q + 1], v[x + 4 * q + 2], v[x + 4 * q + 3]);
      __syncwarp();
      float* out = reinterpret_cast<float*>(a.y) + (size_t)row0 * a.y_stride + n0 + x;
      if (a.y_vec && cols == 32) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = q * 8 + (lane >> 2), c = (lane & 3) * 4;
          if (r < rows_here) *reinterpret_cast<float4*>(out + (size_t)r * a.y_stride + c) = *reinterpret_cast<const float4*>(mine + r * kPairPitch + c);
        }
      } else if (x + (lane & 15) < cols) {
        for (int r = lane >> 4; r < rows_here; r += 2) out[(size_t)r * a.y_stride + (lane & 15)] = mine[r * kPairPitch + (lane & 15)];
      }
      __syncwarp();
    }
  } else {
    uint32_t* words = reinterpret_cast<uint32_t*>(mine);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t h[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(v[8 * q + 2 * e]), __uint_as_float(v[8 * q + 2 * e + 1]));
        h[e] = *reinterpret_cast<const uint32_t*>(&b);
      }
      *reinterpret_cast<uint4*>(words + lane * kPairPitch + 4 * q) = make_uint4(h[0], h[1], h[2], h[3]);
    }
    __syncwarp();
    __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.y) + (size_t)row0 * a.y_stride + n0;
    if (a.y_vec && cols == 32) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = q * 8 + (lane >> 2), c = (lane & 3) * 4;
        if (r < rows_here) *reinterpret_cast<uint4*>(out + (size_t)r * a.y_stride + 2 * c) = *reinterpret_cast<const uint4*>(words + r * kPairPitch + c);
      }
    } else if (lane < cols) {
      for (int r = 0; r < rows_here; ++r) out[(size_t)r * a.y_stride + lane] = reinterpret_cast<const __nv_bfloat16*>(words + r * kPairPitch)[lane];
    }
    __syncwarp();
  }
}

template <bool GATED>
__global__ void __launch_bounds__(kPairThreads, 1) i8_pair_kernel(MmArgs a) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  constexpr int S = kPairStages, W = GATED ? 2 : 1, G = GATED ? 4 : 8;  // G: groups of 32 columns of an item
  float* staging = reinterpret_cast<float*>(smem + (size_t)S * kPairStage);
  float* scale_rows = staging + 8 * 32 * kPairPitch;  // [epilogue warp][factors of 128 columns, up's or the bias]
  uint64_t* bars = reinterpret_cast<uint64_t*>(scale_rows + 8 * 2 * kI8Tile);
  const uint32_t smem_u = ptx::smem_u32(smem), full = ptx::smem_u32(bars);  // [S] this CTA's half of the stage has landed
  const uint32_t done = full + 8u * S;        // [S] the MMAs that read the stage are done
  const uint32_t ready = done + 8u * S;       // [S] first CTA: both CTAs' halves have landed
  const uint32_t acc_full = ready + 8u * S;   // [2] an item's sums are complete
  const uint32_t acc_free = acc_full + 16u;   // [2] first CTA: both CTAs have read them
  const uint32_t drain = acc_free + 16u;
  const uint32_t pushed = drain + 8u;         // the other pairs' sums are here
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 3 * S + 6);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t in_cluster = ptx::cluster_rank(), rank = in_cluster & 1u, leader = in_cluster & ~1u;
  const uint16_t both = (uint16_t)(3u << leader);
  const int shares = a.shares, share = (int)in_cluster / 2;
  const int per_share = (a.chunks + shares - 1) / shares, chunk0 = share * per_share, chunks = min(per_share, a.chunks - chunk0);  // (never none)
  const int row_tiles = (a.rows + kPairRows - 1) / kPairRows, pairs = (a.tiles + 1) / 2;
  const int items = row_tiles * pairs, first_item = blockIdx.x / (2 * shares), step = gridDim.x / (2 * shares);
  struct Item { int tile, row; };  // this CTA's weight tile and first row
  auto item_of = [&](int i) {
    const int band = kPairBand * pairs, b = i / band, rest = i - b * band, high = min(kPairBand, row_tiles - b * kPairBand);
    return Item{2 * (rest / high) + (int)rank, (b * kPairBand + rest % high) * kPairRows + (int)rank * kI8Tile};
  };
  const int own_groups = (G - share + shares - 1) / shares, most_groups = (G + shares - 1) / shares;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      ptx::mbar_init(&bars[s], 1);
      ptx::mbar_init(&bars[S + s], 1);
      ptx::mbar_init(&bars[2 * S + s], 2);
    }
    for (int q = 0; q < 2; ++q) {
      ptx::mbar_init(&bars[3 * S + q], 1);
      ptx::mbar_init(&bars[3 * S + 2 + q], 16);
    }
    ptx::mbar_init(&bars[3 * S + 4], 1);
    ptx::mbar_init(&bars[3 * S + 5], 1);
    ptx::mbar_fence_init();
    ptx::mbar_expect_tx_addr(pushed, (uint32_t)((shares - 1) * own_groups * W) * kI8Block);
  }
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // this CTA's barriers are there
  // (what does not exist is not loaded: its products go nowhere)
  auto load_weights = [&](const Item& it, int c, uint32_t s) {
    const bool rows_there = it.row < a.rows, tile_there = it.tile < a.tiles;
    ptx::mbar_expect_tx_addr(full + 8u * s, (rows_there ? kI8Block : 0) + (tile_there ? kI8Block : 0));
    if (tile_there) ptx::bulk_g2s_addr(smem_u + s * kPairStage + kI8Block, a.w + ((size_t)it.tile * a.chunks + chunk0 + c) * kI8Block, kI8Block, full + 8u * s);
  };
  auto load_rows = [&](const Item& it, int c, uint32_t s) {
    if (it.row < a.rows) ptx::bulk_g2s_addr(smem_u + s * kPairStage, a.q + ((size_t)(it.row / kI8Tile) * a.chunks + chunk0 + c) * kI8Block, kI8Block, full + 8u * s);
  };
  const int ahead = min(S, chunks);  // weights asked for before the kernels ahead have ended
  const Item first = item_of(first_item);
  if (threadIdx.x == 0)
    for (int c = 0; c < ahead; ++c) load_weights(first, c, (uint32_t)c);
  wait_previous();
  if (threadIdx.x == 0)
    for (int c = 0; c < ahead; ++c) load_rows(first, c, (uint32_t)c);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // the others' are
  if (warp == 1) {
    ptx::tmem_alloc2(tmem_slot, 512);
    ptx::tmem_relinquish2();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;
  const int quarter = warp & 3, half = (warp - 4) >> 2;  // of the epilogue's warps
  float *mine = staging + (warp - 4) * 32 * kPairPitch, *scales = scale_rows + (warp - 4) * 2 * kI8Tile;
  // The factors of the four groups of columns that this warp brings to the output, asked for before their sums are there.
  const int my_group = shares > 1 ? share + (half + 2 * (lane / 8)) * shares : GATED ? lane / 8 : half * 4 + lane / 8;
  auto fetch_scales = [&](int first_tile) {
    const int c = my_group * 32 + lane % 8 * 4, n = first_tile * kI8Tile + c;
    const float4 none = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool there = my_group < G && first_tile + c / kI8Tile < a.tiles;
    float4 w = there ? *reinterpret_cast<const float4*>(a.w_scale + n) : none, o = none;
    if (GATED) {
      if (there) o = *reinterpret_cast<const float4*>(a.w_scale + n + kI8Tile);
    } else if (a.bias && there) {
      o = make_float4(n < a.n ? a.bias[n] : 0.f, n + 1 < a.n ? a.bias[n + 1] : 0.f, n + 2 < a.n ? a.bias[n + 2] : 0.f, n + 3 < a.n ? a.bias[n + 3] : 0.f);
    }
    __syncwarp();
    *reinterpret_cast<float4*>(scales + lane * 4) = w;
    *reinterpret_cast<float4*>(scales + kI8Tile + lane * 4) = o;
    __syncwarp();
  };
  const uint32_t acc0 = tmem + ((uint32_t)(quarter * 32) << 16);
  float row_step = 0.f;
  if (warp == 0) {
    if (lane == 0) {
      uint32_t s = 0, ph = 1;
      long long issued = 0;
      for (int i = first_item; i < items && ok; i += step) {
        const Item it = item_of(i);
        for (int c = 0; c < chunks; ++c) {
          if (issued >= ahead) {
            ok = ptx::mbar_wait_addr(done + 8u * s, ph);
            if (!ok) break;
            load_weights(it, c, s);
            load_rows(it, c, s);
          }
          ++issued;
          if (++s == (uint32_t)S) { s = 0; ph ^= 1u; }
        }
      }
      let_next_start();
      if (!ok)  // copies are on their way into this memory
        for (long long i = issued > S ? issued - S : 0; i < issued; ++i) ptx::mbar_wait_addr(full + 8u * (uint32_t)(i % S), (uint32_t)(i / S) & 1u);
    }
  } else if (warp == 2) {
    if (lane == 0) {
      const uint32_t to = ptx::map_to_rank(ready, leader);
      uint32_t s = 0, ph = 0;
      for (int i = first_item; i < items && ok; i += step)
        for (int c = 0; c < chunks; ++c) {
          ok = ptx::mbar_wait_addr(full + 8u * s, ph);
          if (!ok) break;
          ptx::mbar_arrive_cluster(to + 8u * s);
          if (++s == (uint32_t)S) { s = 0; ph ^= 1u; }
        }
    }
  } else if (warp == 1) {
    if (rank == 0 && ptx::elect_one()) {
      const uint32_t idesc = idesc_i8(2 * kI8Tile, 2 * kI8Tile);
      uint32_t s = 0, ph = 0, n_item = 0;
      for (int i = first_item; i < items && ok; i += step, ++n_item) {
        const uint32_t set = n_item & 1u, acc = tmem + set * 256u;
        if (n_item >= 2) ok = ptx::mbar_wait_cluster(acc_free + 8u * set, ((n_item >> 1) - 1u) & 1u);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        for (int c = 0; c < chunks; ++c) {
          ok = ptx::mbar_wait_cluster(ready + 8u * s, ph);
          if (!ok) break;
          ptx::tc_fence_after_sync();
          const uint64_t da = ptx::umma_desc_k_sw128(smem_u + s * kPairStage), db = ptx::umma_desc_k_sw128(smem_u + s * kPairStage + kI8Block);
#pragma unroll
          for (int k4 = 0; k4 < 4; ++k4) umma2_i8(acc, da + 2 * k4, db + 2 * k4, idesc, (c > 0 || k4 > 0) ? 1u : 0u);
          commit_pair(done + 8u * s, both);
          if (++s == (uint32_t)S) { s = 0; ph ^= 1u; }
        }
        if (ok) commit_pair(acc_full + 8u * set, both);
      }
      if (!ok) {  // the MMAs on the way read both CTAs' shared memory
        commit_pair(drain, both);
        ptx::mbar_wait_addr(drain, 0);
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    // A lane is a row.
    const uint32_t to = ptx::map_to_rank(acc_free, leader);
    uint32_t n_item = 0;
    for (int i = first_item; i < items; i += step, ++n_item) {
      const Item it = item_of(i);
      const uint32_t set = n_item & 1u;
      const int row0 = it.row + quarter * 32;
      row_step = row0 + lane < a.rows ? a.step[row0 + lane] : 0.f;
      fetch_scales(it.tile - (int)rank);
      ok = ptx::mbar_wait_addr(acc_full + 8u * set, (n_item >> 1) & 1u);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      ptx::tc_fence_after_sync();
      if (shares > 1) break;
#pragma unroll 1  // (an epilogue that runs once per CTA waits for its instructions)
      for (int g = half * (G / 2); g < half * (G / 2) + G / 2; ++g) {
        uint32_t v[32], u[GATED ? 32 : 1];
        ptx::tmem_ld32(acc0 + set * 256u + (uint32_t)(g * 32), v);
        if constexpr (GATED) ptx::tmem_ld32(acc0 + set * 256u + (uint32_t)(kI8Tile + g * 32), u);
        ptx::tmem_ld_wait();
        store_sums<GATED>(a, v, u, mine, scales + (GATED ? g : g % 4) * 32, it.tile - (int)rank, g * 32, row0, row_step);
      }
      // all that this warp reads of the item's sums has been read
      ptx::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive_cluster_relaxed(to + 8u * set);
    }
  }
  if (shares > 1) {
    __syncwarp();
    ptx::cluster_sync();  // nobody's stages are in use
    if (warp >= 4) {
      const Item it = item_of(first_item);
      // [other pair][group][gate, up][four columns][row]
      auto place = [&](int from, int group, int part, int j4) { return (((((from * most_groups + group) * W + part) * 8 + j4) * kI8Tile) + quarter * 32 + lane) * 16; };
#pragma unroll 1
      for (int g = half; g < G && ok; g += 2) {
        const int owner = g % shares;
        if (owner == share) continue;
        const uint32_t cta = (uint32_t)owner * 2 + rank, to = ptx::map_to_rank(smem_u, cta), bar = ptx::map_to_rank(pushed, cta);
        const int from = share - (share > owner);
#pragma unroll
        for (int part = 0; part < W; ++part) {
          uint32_t v[32];
          ptx::tmem_ld32(acc0 + (uint32_t)(part * kI8Tile + g * 32), v);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int j4 = 0; j4 < 8; ++j4) push4(to + place(from, g / shares, part, j4), v[4 * j4], v[4 * j4 + 1], v[4 * j4 + 2], v[4 * j4 + 3], bar);
        }
      }
      ok &= (bool)__all_sync(0xffffffffu, wait_pushed(pushed));  // (where a wait here ran out, too: the others push all the same)
#pragma unroll 1
      for (int i = half; i < own_groups && ok; i += 2) {
        const int g = share + i * shares;
        uint32_t v[32], u[GATED ? 32 : 1];
        ptx::tmem_ld32(acc0 + (uint32_t)(g * 32), v);
        if constexpr (GATED) ptx::tmem_ld32(acc0 + (uint32_t)(kI8Tile + g * 32), u);
        ptx::tmem_ld_wait();
#pragma unroll 1
        for (int from = 0; from < shares - 1; ++from) {
#pragma unroll
          for (int j4 = 0; j4 < 8; ++j4) {
            const uint4 p = *reinterpret_cast<const uint4*>(smem + place(from, i, 0, j4));
            v[4 * j4] += p.x; v[4 * j4 + 1] += p.y; v[4 * j4 + 2] += p.z; v[4 * j4 + 3] += p.w;
            if constexpr (GATED) {
              const uint4 q = *reinterpret_cast<const uint4*>(smem + place(from, i, 1, j4));
              u[4 * j4] += q.x; u[4 * j4 + 1] += q.y; u[4 * j4 + 2] += q.z; u[4 * j4 + 3] += q.w;
            }
          }
        }
        store_sums<GATED>(a, v, u, mine, scales + (i >> 1) * 32, it.tile - (int)rank, g * 32, it.row + quarter * 32, row_step);
      }
    }
  }
  if (!ok) atomicExch(a.err, B200_ERR_DEVICE_FLAGGED);
  __syncwarp();
  ptx::tc_fence_before_sync();
  ptx::cluster_sync();  // nobody leaves while its memory may be read, written or arrived on
  if (warp == 1) ptx::tmem_dealloc2(tmem, 512);
}

// A launch in clusters of `size` (1: none) whose start-up overlaps the end of the kernel ahead.
template <class... P>
void launch_clusters(void (*kernel)(P...), int size, dim3 grid, int threads, size_t smem, cudaStream_t s, P... args) {
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // (as launch_after)
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = size;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = size > 1 ? 2 : 1;
  (void)cudaLaunchKernelEx(&cfg, kernel, args...);
}

// What a product is expected to take with one kernel or the other.  Microseconds of launches one behind the other in a graph, fitted to 2048 x 2048 to 4096 x 14336
// and 28672 x 4096 at 1 to 1024 rows: a block of weights reaches an SM in 0.27 us however few rows go with it, a row that a CTA brings to the output costs
// 0.02 us, one whose sums it pushes as much, and a cluster 0.55 for each of its CTAs.  4096 x 4096: 256 rows as 64 tiles of 128 in two shares 9.0 us (model 8.6), as
// 32 of 256 in four 10.7 (10.8), as pairs in two shares 11.6 (12.1); 512 rows as 128 tiles of 128 12.2 (11.8), as pairs 13.0 (12.1); 1024 rows as pairs 15.8 (15.8),
// as tiles 18.6 (16.1 at least).
struct Plan {
  float us = 1e30f;
  bool pair = false;
  int tn = 0, shares = 1;
};

template <bool GATED>
Plan plan_of(const MmArgs& a, const int* stream_at_once, const int* pairs_at_once) {
  constexpr int W = GATED ? 2 : 1;
  Plan best;
  const auto split = [&](int n, int least) { return n == 1 || (a.chunks >= least * n && (n - 1) * ((a.chunks + n - 1) / n) < a.chunks); };  // into n shares, none of them empty
  const int tiles = a.tiles / W, sms = b200_sm_count();
  for (int tn = 16; W * tn <= 256; tn *= 2) {
    const long long row_tiles = (a.rows + tn - 1) / tn;
    const int rows_here = std::min(a.rows, tn);
    if (row_tiles > 4096) continue;
    for (int n = 1; n <= kMostShares; ++n) {
      const long long ctas = tiles * row_tiles * n;
      if (!split(n, 2) || pushed_bytes(rows_here, n, W) > kStreamAlone - 2048 || (n > 1 && ctas > stream_at_once[n])) continue;
      const int own = std::min(rows_here, rows_per_rank(rows_here, n));
      float us = 0.6f + 0.02f * W * own + (float)((a.chunks + n - 1) / n) * W * std::max(0.27f, 0.0014f * tn);
      if (n > 1) us += 0.55f * n + 0.02f * W * (rows_here - own);
      if (ctas > sms) us *= 1.18f * ctas / sms;
      if (us < best.us) best = {us, false, tn, n};
    }
    if (tn >= a.rows) break;
  }
  const long long items = (long long)((a.rows + kPairRows - 1) / kPairRows) * ((a.tiles + 1) / 2);
  for (int n = 1; n <= kMostPairs; ++n) {
    if (!split(n, 4) || pairs_at_once[n] < 1 || (n > 1 && items > pairs_at_once[n])) continue;
    const float waves = (float)((items + pairs_at_once[n] - 1) / pairs_at_once[n]);
    const float us = (n == 1 ? 6.4f : 7.0f) + waves * ((GATED ? 2.5f : 0.8f) + 0.27f * ((a.chunks + n - 1) / n));
    if (us < best.us) best = {us, true, 0, n};
  }
  return best;
}

// Rows that are not 8 bits yet: bf16, or the inner rows of a feed-forward block.
struct RawRows {
  const void* x = nullptr;
  long long stride = 0;
  const b200_i8_rows* inner = nullptr;
};

template <bool GATED>
b200_status launch_product(MmArgs& a, const I8RowsDev& to, const RawRows& raw, cudaStream_t s) {
  constexpr int W = GATED ? 2 : 1;
  // What runs at the same time with an SM for each CTA, by the cluster's size: CTAs of the one kernel, clusters of the other.  (The occupancy calculation counts
  // one CTA of a kernel that allocates tensor memory to an SM; of i8_stream_kernel's two share that memory.)
  static int at_once[kMostShares + 1] = {}, pairs_at_once[kMostPairs + 1] = {};
  if (at_once[1] == 0) {
    B200_CUDA_TRY(cudaFuncSetAttribute(i8_stream_kernel<GATED, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kStreamAlone));
    B200_CUDA_TRY(cudaFuncSetAttribute(i8_stream_kernel<GATED, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kStreamAlone));
    B200_CUDA_TRY(cudaFuncSetAttribute(i8_pair_kernel<GATED>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairShared));
    for (int n = kMostPairs; n > 0; --n) pairs_at_once[n] = ctas_in_clusters(i8_pair_kernel<GATED>, 2 * n, 1, b200_sm_count(), kPairThreads, kPairShared) / (2 * n);
    for (int n = kMostShares; n > 0; --n) at_once[n] = ctas_in_clusters(i8_stream_kernel<GATED, false>, n, 1, b200_sm_count(), kStreamThreads, kStreamAlone);
    if (at_once[1] < 1 || pairs_at_once[1] < 1) {
      at_once[1] = 0;
      b200_set_error("i8: the kernels do not fit the device");
      return B200_ERR_CAPACITY;
    }
  }
  const Plan plan = plan_of<GATED>(a, at_once, pairs_at_once);
  a.shares = plan.shares;
  const int per_share = (a.chunks + a.shares - 1) / a.shares;
  const bool in_kernel = raw.x && !plan.pair && a.rows <= kRawRows && per_share <= kRawChunks && a.rows * per_share <= kRawWork && (raw.inner || a.rows * a.k <= kRawNumbers);
  if (raw.x && !in_kernel) {
    const b200_status st = raw.inner ? quantize_inner(raw.inner, a.rows, a.k, s) : quantize((const __nv_bfloat16*)raw.x, raw.stride, a.rows, a.k, to, s);
    if (st != B200_OK) return st;
  }
  if (plan.pair) {
    const long long items = (long long)((a.rows + kPairRows - 1) / kPairRows) * ((a.tiles + 1) / 2);
    if (items > 0x3fffffff) { b200_set_error("i8: %d rows of %d channels in one call", a.rows, a.n); return B200_ERR_CAPACITY; }
    launch_clusters(i8_pair_kernel<GATED>, 2 * a.shares, dim3((unsigned)(2 * a.shares * std::min<long long>(items, pairs_at_once[a.shares]))), kPairThreads, kPairShared, s, a);
  } else {
    a.tn = plan.tn;
    const int tiles = a.tiles / W, row_tiles = (a.rows + a.tn - 1) / a.tn, stage = W * kI8Block + (in_kernel ? 0 : a.tn * kI8Chunk);
    const int room = ((long long)tiles * row_tiles * a.shares <= at_once[a.shares] ? kStreamAlone : kStreamShared) - 2048;
    const int pushed = pushed_bytes(std::min(a.rows, a.tn), a.shares, W), raw_bytes = in_kernel ? per_share * 16 * kI8Chunk : 0;
    // What is pushed has a place beside the stages where that is a quarter of the room at most (an eighth: 200 rows of 4096 to 4096 9.1 us in place of 8.8; half: 256 through a
    // block of 14336 66 in place of 61).
    a.over_stages = pushed > room / 4;
    a.stages = std::min(per_share, (room - raw_bytes - (a.over_stages ? 0 : pushed)) / stage);
    a.raw_at = a.stages * stage;
    a.pushed_at = a.over_stages ? 0 : a.stages * stage + raw_bytes;
    a.bars_at = std::max(a.stages * stage + raw_bytes, a.pushed_at + pushed);
    const size_t shared = std::max<size_t>(a.bars_at + 2048, kSharedPerCol * stream_cols(a.tn, W));
    if (in_kernel) {
      a.raw = raw.x; a.raw_stride = raw.stride; a.raw_inner = raw.inner != nullptr; a.q_out = to.q; a.step_out = to.scale;
      a.raw_fit = ((uintptr_t)raw.x & 15) == 0 && raw.stride % 8 == 0;
      if (raw.inner) a.raw_most = raw.inner->most;
      launch_clusters(i8_stream_kernel<GATED, true>, a.shares, dim3(tiles * a.shares, row_tiles), kStreamThreads, shared, s, a);
    } else {
      launch_clusters(i8_stream_kernel<GATED, false>, a.shares, dim3(tiles * a.shares, row_tiles), kStreamThreads, shared, s, a);
    }
  }
  B200_LAUNCH_CHECK();
  return B200_OK;
}

b200_status product(const b200_i8_weight* w, const I8RowsDev& x, const RawRows& raw, int rows, const float* bias, int act, void* y, long long y_stride, int y_f32, float* most, cudaStream_t s) {
  MmArgs a{};
  b200_status st = b200_qmm_ensure_err_word(&a.err);
  if (st != B200_OK) return st;
  a.w = w->q; a.w_scale = w->scale; a.q = x.q; a.step = x.scale; a.bias = bias; a.y = y; a.y_stride = y_stride; a.y_f32 = y_f32; a.act = act; a.most = most;
  a.rows = rows; a.n = w->n; a.chunks = w->chunks; a.tiles = w->tiles; a.k = w->k;
  a.y_vec = ((uintptr_t)y & 15) == 0 && y_stride * (w->gated || y_f32 ? 4 : 2) % 16 == 0;
  return w->gated ? launch_product<true>(a, x, raw, s) : launch_product<false>(a, x, raw, s);
}

// ---- handles -------------------------------------------------------------------------------------------------------------------
b200_status create_weight(int n, int k, bool gated, const int8_t* const* q, const float* const* scales, b200_i8_weight** out) {
  if (!out) { b200_set_error("i8 weight: no place for the handle"); return B200_ERR_INVALID_ARGUMENT; }
  *out = nullptr;
  const int parts = gated ? 2 : 1;
  for (int p = 0; p < parts; ++p)
    if (!q[p] || !scales[p] || ((uintptr_t)scales[p] & 3) != 0) { b200_set_error("i8 weight: no numbers, or no scales"); return B200_ERR_INVALID_ARGUMENT; }
  if (n <= 0 || k <= 0 || n > 1 << 24 || k > kI8MaxK) { b200_set_error("i8 weight: %d x %d (at most %d x %d)", n, k, 1 << 24, kI8MaxK); return B200_ERR_INVALID_ARGUMENT; }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  int* err = nullptr;
  st = b200_qmm_ensure_err_word(&err);  // (not in the first product, which may be captured)
  if (st != B200_OK) return st;
  auto* w = new (std::nothrow) b200_i8_weight();
  if (!w) { b200_set_error("i8 weight: out of host memory"); return B200_ERR_CAPACITY; }
  const int tiles = (n + kI8Tile - 1) / kI8Tile;
  w->n = n; w->k = k; w->gated = gated; w->tiles = tiles * parts; w->chunks = i8_chunks(k);
  cudaError_t e = cudaDeviceSynchronize();  // (the numbers may be another stream's work)
  if (e == cudaSuccess) e = cudaMalloc((void**)&w->q, (size_t)w->tiles * w->chunks * kI8Block);
  if (e == cudaSuccess) e = cudaMalloc((void**)&w->scale, sizeof(float) * (size_t)w->tiles * kI8Tile);
  int device = 0;
  if (e == cudaSuccess) e = cudaGetDevice(&device);
  void *q_copy = nullptr, *scale_copy = nullptr;
  for (int p = 0; p < parts && e == cudaSuccess; ++p) {
    auto here = [&](const void* from, size_t bytes, void*& copy) -> const void* {  // in this device's memory
      cudaPointerAttributes at{};
      if (cudaPointerGetAttributes(&at, from) == cudaSuccess && at.type == cudaMemoryTypeDevice && at.device == device) return from;
      cudaGetLastError();
      if (!copy) e = cudaMalloc(&copy, bytes);
      if (e == cudaSuccess) e = cudaMemcpy(copy, from, bytes, cudaMemcpyDefault);
      return copy;
    };
    const void* q_here = here(q[p], (size_t)n * k, q_copy);
    const void* scale_here = e == cudaSuccess ? here(scales[p], sizeof(float) * (size_t)n, scale_copy) : nullptr;
    if (e != cudaSuccess) break;
    const long long pieces = (long long)tiles * kI8Tile * w->chunks * 8;
    i8_lay_out_kernel<<<(unsigned)((pieces + 255) / 256), 256>>>((const signed char*)q_here, (const float*)scale_here, n, k, w->chunks, p, parts, tiles, w->q, w->scale);
    ++g_b200_launch_counter;
    e = cudaGetLastError();
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
  }
  if (q_copy) cudaFree(q_copy);
  if (scale_copy) cudaFree(scale_copy);
  if (e != cudaSuccess) {
    b200_set_error("i8 weight: %d x %d: %s", n, k, cudaGetErrorString(e));
    cudaGetLastError();
    b200_i8_weight_destroy(w);
    return B200_ERR_CUDA;
  }
  *out = w;
  return B200_OK;
}

// The checks of x and the rows that a product reads.
b200_status take_rows(const char* who, b200_i8_rows* r, const void* d_x, int64_t x_stride, int32_t rows, int32_t k) {
  if (rows < 0 || rows > r->max_rows) { b200_set_error("%s: %d rows, the handle is for %d", who, rows, r->max_rows); return rows < 0 ? B200_ERR_INVALID_ARGUMENT : B200_ERR_CAPACITY; }
  if (k > r->max_k) { b200_set_error("%s: rows of %d columns, the handle is for %d", who, k, r->max_k); return B200_ERR_CAPACITY; }
  if (rows == 0) {  // (whether x is there or not)
    r->rows = 0;
    r->k = k;
    return B200_OK;
  }
  if (!d_x) {
    if (r->rows != rows || r->k != k) {
      b200_set_error("%s: %d rows of %d columns, the handle holds %d of %d", who, rows, k, std::max(0, r->rows), r->k);
      return B200_ERR_INVALID_ARGUMENT;
    }
    return B200_OK;
  }
  if (rows > 1 && x_stride < k) { b200_set_error("%s: rows of %d columns %lld apart", who, k, (long long)x_stride); return B200_ERR_INVALID_ARGUMENT; }
  if (((uintptr_t)d_x & 1) != 0) { b200_set_error("%s: x is not on a number's boundary", who); return B200_ERR_INVALID_ARGUMENT; }
  r->rows = -1;  // (until the rows are on their way)
  return B200_OK;
}

b200_status taken(b200_i8_rows* r, int32_t rows, int32_t k, b200_status st) {
  if (st == B200_OK) { r->rows = rows; r->k = k; }
  return st;
}

b200_status check_out(const char* who, const void* d_y, int64_t y_stride, int32_t rows, int32_t n, int size) {
  if (rows > 0 && (!d_y || ((uintptr_t)d_y & (size - 1)) != 0 || (rows > 1 && y_stride < n))) {
    b200_set_error("%s: no place for %d rows of %d columns", who, rows, n);
    return B200_ERR_INVALID_ARGUMENT;
  }
  return B200_OK;
}

b200_status feed_forward(const b200_i8_weight* gate_up, const b200_i8_weight* down, b200_i8_rows* r, const void* d_x, int64_t x_stride, int32_t rows, int32_t activation,
                         void* d_y, int64_t y_stride, bool y_f32, void* stream) {
  if (!gate_up || !down || !r) { b200_set_error("i8 ffn: no weights, or no rows"); return B200_ERR_INVALID_ARGUMENT; }
  if (!gate_up->gated || down->gated || down->k != gate_up->n) {
    b200_set_error("i8 ffn: %s weight of %d channels in front of %s of %d columns", gate_up->gated ? "a gated" : "a plain", gate_up->n, down->gated ? "a gated one" : "one", down->k);
    return B200_ERR_INVALID_ARGUMENT;
  }
  if (activation < B200_ACT_SILU || activation > B200_ACT_GELU_TANH) { b200_set_error("i8 ffn: activation %d", activation); return B200_ERR_INVALID_ARGUMENT; }
  if (down->k > r->max_hidden) { b200_set_error("i8 ffn: %d channels inside the block, the handle is for %d", down->k, r->max_hidden); return B200_ERR_CAPACITY; }
  b200_status st = check_out("i8 ffn", d_y, y_stride, rows, down->n, y_f32 ? 4 : 2);
  if (st == B200_OK) st = b200_require_device();
  if (st == B200_OK) st = take_rows("i8 ffn", r, d_x, x_stride, rows, gate_up->k);
  if (st != B200_OK || rows == 0) return st;
  cudaStream_t s = (cudaStream_t)stream;
  st = taken(r, rows, gate_up->k, product(gate_up, r->x, RawRows{d_x, x_stride, nullptr}, rows, nullptr, activation, r->h, r->h_stride, 0, r->most, s));
  if (st == B200_OK) st = product(down, r->hidden, RawRows{r->h, r->h_stride, r}, rows, nullptr, 0, d_y, y_stride, y_f32, nullptr, s);
  return st;
}

}  // namespace

extern "C" b200_status b200_i8_weight_create(int32_t n, int32_t k, const int8_t* q, const float* scales, b200_i8_weight** out) {
  return create_weight(n, k, false, &q, &scales, out);
}

extern "C" b200_status b200_i8_weight_create_gated(int32_t n, int32_t k, const int8_t* gate_q, const float* gate_scales, const int8_t* up_q, const float* up_scales,
                                                   b200_i8_weight** out) {
  const int8_t* q[2] = {gate_q, up_q};
  const float* scales[2] = {gate_scales, up_scales};
  return create_weight(n, k, true, q, scales, out);
}

extern "C" void b200_i8_weight_destroy(b200_i8_weight* w) {
  if (!w) return;
  for (void* p : {(void*)w->q, (void*)w->scale}) if (p) cudaFree(p);
  delete w;
}

extern "C" b200_status b200_i8_rows_create(int32_t max_rows, int32_t max_k, int32_t max_hidden, b200_i8_rows** out) {
  if (!out) { b200_set_error("i8 rows: no place for the handle"); return B200_ERR_INVALID_ARGUMENT; }
  *out = nullptr;
  if (max_rows <= 0 || max_rows > 1 << 24 || max_k <= 0 || max_k > kI8MaxK || max_hidden < 0 || max_hidden > kI8MaxK) {
    b200_set_error("i8 rows: %d rows of %d columns, %d inside a block (at most %d, %d and %d)", max_rows, max_k, max_hidden, 1 << 24, kI8MaxK, kI8MaxK);
    return B200_ERR_INVALID_ARGUMENT;
  }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  auto* r = new (std::nothrow) b200_i8_rows();
  if (!r) { b200_set_error("i8 rows: out of host memory"); return B200_ERR_CAPACITY; }
  r->max_rows = max_rows; r->max_k = max_k; r->max_hidden = max_hidden; r->h_stride = (max_hidden + 7) / 8 * 8;
  const size_t tiles = (max_rows + kI8Tile - 1) / kI8Tile;
  cudaError_t e = cudaSuccess;
  auto make = [&](I8RowsDev& d, int k) {
    const size_t bytes = tiles * i8_chunks(k) * kI8Block;
    if (e == cudaSuccess) e = cudaMalloc((void**)&d.q, bytes);
    if (e == cudaSuccess) e = cudaMalloc((void**)&d.scale, sizeof(float) * tiles * kI8Tile);
    if (e == cudaSuccess) e = cudaMemset(d.q, 0, bytes);
    if (e == cudaSuccess) e = cudaMemset(d.scale, 0, sizeof(float) * tiles * kI8Tile);
  };
  make(r->x, max_k);
  if (max_hidden > 0) {
    make(r->hidden, max_hidden);
    if (e == cudaSuccess) e = cudaMalloc((void**)&r->h, sizeof(float) * (size_t)max_rows * r->h_stride);
    if (e == cudaSuccess) e = cudaMalloc((void**)&r->most, sizeof(float) * (size_t)max_rows * i8_chunks(max_hidden) * 4);
  }
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  if (e != cudaSuccess) {
    b200_set_error("i8 rows: %d rows of %d columns, %d inside a block: %s", max_rows, max_k, max_hidden, cudaGetErrorString(e));
    cudaGetLastError();
    b200_i8_rows_destroy(r);
    return B200_ERR_CUDA;
  }
  *out = r;
  return B200_OK;
}

extern "C" void b200_i8_rows_destroy(b200_i8_rows* r) {
  if (!r) return;
  for (void* p : {(void*)r->x.q, (void*)r->x.scale, (void*)r->hidden.q, (void*)r->hidden.scale, (void*)r->h, (void*)r->most}) if (p) cudaFree(p);
  delete r;
}

extern "C" b200_status b200_i8_quantize(b200_i8_rows* r, const void* d_x, int64_t x_stride, int32_t rows, int32_t k, void* stream) {
  if (!r || k <= 0 || (rows > 0 && !d_x)) { b200_set_error("i8 quantize: no handle, or no rows"); return B200_ERR_INVALID_ARGUMENT; }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  st = take_rows("i8 quantize", r, d_x, x_stride, rows, k);
  if (st != B200_OK || rows == 0) return st;
  return taken(r, rows, k, quantize((const __nv_bfloat16*)d_x, x_stride, rows, k, r->x, (cudaStream_t)stream));
}

extern "C" b200_status b200_i8_rows_get(const b200_i8_rows* r, void* d_q, float* d_steps, void* stream) {
  if (!r || r->rows < 0 || ((uintptr_t)d_steps & 3) != 0) { b200_set_error("i8 rows: nothing there, or no place for it"); return B200_ERR_INVALID_ARGUMENT; }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  if (r->rows == 0 || (!d_q && !d_steps)) return B200_OK;
  const long long numbers = (long long)r->rows * r->k;
  launch_after(i8_rows_get_kernel, (unsigned)((numbers + 255) / 256), 256, 0, (cudaStream_t)stream, r->x, r->rows, r->k, i8_chunks(r->k), (signed char*)d_q, d_steps);
  B200_LAUNCH_CHECK();
  return B200_OK;
}

extern "C" b200_status b200_i8_mm(const b200_i8_weight* w, b200_i8_rows* r, const void* d_x, int64_t x_stride, int32_t rows, const float* d_bias, void* d_y,
                                  int64_t y_stride, int32_t y_f32, void* stream) {
  if (!w || !r) { b200_set_error("i8 mm: no weight, or no rows"); return B200_ERR_INVALID_ARGUMENT; }
  if (w->gated) { b200_set_error("i8 mm: the weight is a feed-forward block's gate and up"); return B200_ERR_INVALID_ARGUMENT; }
  if (((uintptr_t)d_bias & 3) != 0) { b200_set_error("i8 mm: the bias is not on a number's boundary"); return B200_ERR_INVALID_ARGUMENT; }
  b200_status st = check_out("i8 mm", d_y, y_stride, rows, w->n, y_f32 ? 4 : 2);
  // (rows become 8 bits in the same kernel where they are few, while others' columns are stored already)
  const int size = y_f32 ? 4 : 2;
  const RowsAt y{d_y, rows, y_stride * size, (long long)w->n * size};
  if (st == B200_OK && (rows_overlap(y, {d_x, rows, x_stride * 2, (long long)w->k * 2}) || rows_overlap(y, {d_bias, 1, 0, (long long)w->n * 4}))) {
    b200_set_error("i8 mm: y lies over x or the bias");
    return B200_ERR_INVALID_ARGUMENT;
  }
  if (st == B200_OK) st = b200_require_device();
  if (st == B200_OK) st = take_rows("i8 mm", r, d_x, x_stride, rows, w->k);
  if (st != B200_OK || rows == 0) return st;
  return taken(r, rows, w->k, product(w, r->x, RawRows{d_x, x_stride, nullptr}, rows, d_bias, 0, d_y, y_stride, y_f32 != 0, nullptr, (cudaStream_t)stream));
}

extern "C" b200_status b200_i8_ffn(const b200_i8_weight* gate_up, const b200_i8_weight* down, b200_i8_rows* r, const void* d_x, int64_t x_stride, int32_t rows,
                                   int32_t activation, void* d_y, int64_t y_stride, void* stream) {
  return feed_forward(gate_up, down, r, d_x, x_stride, rows, activation, d_y, y_stride, false, stream);
}

extern "C" b200_status b200_i8_ffn_f32(const b200_i8_weight* gate_up, const b200_i8_weight* down, b200_i8_rows* r, const void* d_x, int64_t x_stride, int32_t rows,
                                       int32_t activation, float* d_y, int64_t y_stride, void* stream) {
  return feed_forward(gate_up, down, r, d_x, x_stride, rows, activation, d_y, y_stride, true, stream);
}
