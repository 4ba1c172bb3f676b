// Low-rank adapters of many requests beside a projection that they share: out[r] = y[r] + s_a B_a (A_a x[r]) with a = the row's adapter.
//
// The plan sorts a batch's rows by adapter and cuts each adapter's rows into tiles.  A cluster of eight CTAs takes a tile through both products
// in one launch: its 64 warps share K between them for u = A x (f32), the parts are summed through distributed shared memory, and each CTA then
// has all of u for its share of the N columns of y.  So u never goes to memory, a tile's x, y, A and B cross the chip once, and there is no second
// launch to wait for.  A tile of a step that has few of them is given to several clusters, which all form u and share the columns.
//
// The products run on mma.sync m16n8k16 with fragments straight from global memory: a lane loads 16 (or 8) neighbouring bytes of a row, which are
// its places of the MMA's K in one or two steps (both operands agree on the order), and in the second product its places of N as well, so that it
// holds eight neighbouring columns of y.  At ranks up to 64 a byte of x or y has fewer than 64 multiplications, an order below what would ask for
// more than mma.sync.
//
// A row's u is summed in the same order whatever shares its tile: within a warp's 1/64 of K by the MMAs, then over the eight warps, then over the
// eight CTAs.  It goes into the second product as two bf16 numbers (u - hi, exactly, and that rounded), which leaves 2^-17 of it, and the sum with
// y is rounded once.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <vector>

#include "common.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace cg = cooperative_groups;

// Adapters of one projection.  Rank rows are padded to rs (16, 32, 64 or 128).
struct b200_lora {
  int n_adapters = 0, n = 0, k = 0, max_rank = 0, rs = 0;
  __nv_bfloat16 *a = nullptr, *b = nullptr;  // [adapter][rs][k], [adapter][n][rs]
  int* rank = nullptr;                       // [adapter], 0: none
  float* scale = nullptr;
};

// The rows of a step by adapter: order[max_rows], tiles of {adapter or -1, first place in order, rows, -}, header {tiles}.
struct b200_lora_batch {
  int max_rows = 0, max_adapters = 0, max_rank = 0, max_tiles = 0, rows = -1;
  int* order = nullptr;
  int4* tiles = nullptr;
  int* hdr = nullptr;
};

namespace {

constexpr int kCluster = 8, kWarps = 8, kThreads = kWarps * 32;
constexpr int kMaxAdapters = 4096, kMaxRank = 128;
constexpr int kEnoughTiles = 72;  // about twice the clusters that run at a time: beyond that, larger tiles rather than more of them

__host__ __device__ constexpr int most_tile_rows(int rs) { return rs > 64 ? 64 : 128; }

// ---- the plan ------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(1024) lora_plan_kernel(const int* row_adapter, int rows, int n_adapters, int most_rows, int* __restrict__ order,
                                                         int4* __restrict__ tiles, int* __restrict__ hdr) {
  after_previous();
  __shared__ int count[kMaxAdapters + 1], warp_sums[32], total[4], carry[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bins = n_adapters + 1;
  for (int i = tid; i < bins; i += blockDim.x) count[i] = 0;
  if (tid < 4) total[tid] = 0;
  if (tid < 2) carry[tid] = 0;
  __syncthreads();
  auto bin = [&](int r) {
    const int a = row_adapter[r];
    return a >= 0 && a < n_adapters ? a : n_adapters;
  };
  for (int r = tid; r < rows; r += blockDim.x) atomicAdd(&count[bin(r)], 1);
  __syncthreads();
  int mine[4] = {0, 0, 0, 0};  // tiles of 16, 32, 64, 128 rows
  for (int i = tid; i < bins; i += blockDim.x) {
#pragma unroll
    for (int s = 0; s < 4; ++s) mine[s] += (count[i] + (16 << s) - 1) >> (4 + s);
  }
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const int t = __reduce_add_sync(0xffffffffu, mine[s]);
    if (lane == 0 && t) atomicAdd(&total[s], t);
  }
  __syncthreads();
  int shift = 4;
  while ((1 << shift) < most_rows && total[shift - 4] > kEnoughTiles) ++shift;
  // places of each adapter's rows and tiles: a scan over the bins
  for (int base = 0; base < bins; base += blockDim.x) {
    const int i = base + tid, c = i < bins ? count[i] : 0, t = (c + (1 << shift) - 1) >> shift;
    int ic = c, it = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int uc = __shfl_up_sync(0xffffffffu, ic, o), ut = __shfl_up_sync(0xffffffffu, it, o);
      if (lane >= o) { ic += uc; it += ut; }
    }
    if (lane == 31) warp_sums[warp] = ic;
    __syncthreads();
    int before_c = carry[0], before_t = carry[1];
    for (int w = 0; w < warp; ++w) before_c += warp_sums[w];
    __syncthreads();
    if (lane == 31) warp_sums[warp] = it;
    __syncthreads();
    for (int w = 0; w < warp; ++w) before_t += warp_sums[w];
    const int first = before_c + ic - c;
    if (i < bins) {
      for (int j = 0; j < t; ++j) tiles[before_t + it - t + j] = make_int4(i < n_adapters ? i : -1, first + (j << shift), min(1 << shift, c - (j << shift)), 0);
      count[i] = first;
    }
    __syncthreads();
    if (tid == (int)blockDim.x - 1) { carry[0] = before_c + ic; carry[1] = before_t + it; }
    __syncthreads();
  }
  // (rows of an adapter in any order: no row's result depends on its place)
  for (int r = tid; r < rows; r += blockDim.x) order[atomicAdd(&count[bin(r)], 1)] = r;
  if (tid == 0) hdr[0] = carry[1];
}

// ---- the products ---------------------------------------------------------------------------------------------------
struct LoraArgs {
  const __nv_bfloat16 *a, *b, *x, *y;
  __nv_bfloat16* out;
  const int* rank;
  const float* scale;
  const int* order;
  const int4* tiles;
  const int* hdr;
  int n_adapters, n, k, rows;
  int x_stride, y_stride, out_stride;
  int most_parts;  // clusters that may share a tile's columns
};

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// What bf16 leaves of u; nothing where u is no finite number.
__device__ __forceinline__ float rest(float u) {
  const float hi = __bfloat162float(__float2bfloat16(u));
  return isfinite(hi) ? u - hi : 0.f;
}

template <int RS>
struct Shape {
  static constexpr int TM = most_tile_rows(RS), RC = RS > 64 ? 64 : RS, NT = RC / 8, KS = RS / 16;
  static constexpr int MG = RS > 32 ? 1 : 2;          // groups of 16 rows at a time: registers
  static constexpr int PAD = RC + 8, UPAD = RS + 8;   // strides without bank conflicts
  static constexpr int kPart = kWarps * MG * 16 * PAD * 4, kHalves = 2 * TM * UPAD * 2;
  static constexpr int kShared = (kPart > kHalves ? kPart : kHalves) + TM * RS * 4 + TM * 4;
};

template <int RS>
__global__ void __launch_bounds__(kThreads, 2) lora_kernel(const __grid_constant__ LoraArgs a) {
  after_previous();
  using Z = Shape<RS>;
  extern __shared__ __align__(16) unsigned char smem[];
  float* part = reinterpret_cast<float*>(smem);                       // [warp][row of the round][PAD]
  __nv_bfloat16* halves = reinterpret_cast<__nv_bfloat16*>(smem);     // [hi, lo][row][UPAD], when the parts have been summed
  float* u = reinterpret_cast<float*>(smem + (Z::kPart > Z::kHalves ? Z::kPart : Z::kHalves));  // [row][RS]: this CTA's share of K
  int* row_of = reinterpret_cast<int*>(u + Z::TM * RS);
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = cluster.block_rank(), clusters = gridDim.x / kCluster, me = blockIdx.x / kCluster;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int n_tiles = a.hdr[0];
  const int parts = max(1, min(a.most_parts, clusters / max(n_tiles, 1)));
  const int each = (a.k + 64 * 32 - 1) / (64 * 32) * 32;  // a warp's share of K
  const int k0 = (cta * kWarps + warp) * each, k1 = min(a.k, k0 + each);

  for (int item = me; item < n_tiles * parts; item += clusters) {
    const int4 tile = a.tiles[item / parts];
    const int share = item % parts, count = tile.z, groups = (count + 15) / 16;
    const int rank = tile.x >= 0 ? min(a.rank[tile.x], RS) : 0, rk = (rank + 15) / 16 * 16;
    if (rank == 0 && a.out == a.y) continue;  // (the whole cluster)
    for (int i = tid; i < Z::TM; i += kThreads) row_of[i] = i < count ? a.order[tile.y + i] : -1;
    __syncthreads();
    // ---- u: this warp's part of K, round by round of MG * 16 rows ----
    if (rank > 0) {
      const float scale = a.scale[tile.x];
      for (int c0 = 0; c0 < rk; c0 += Z::RC) {
        const __nv_bfloat16* aw = a.a + ((size_t)tile.x * RS + c0) * a.k;
        const int nts = min(Z::NT, (rk - c0) / 8);
        for (int m0 = 0; m0 < groups; m0 += Z::MG) {
          float acc[Z::MG][Z::NT][4];
#pragma unroll
          for (int m = 0; m < Z::MG; ++m)
#pragma unroll
            for (int j = 0; j < Z::NT; ++j) acc[m][j][0] = acc[m][j][1] = acc[m][j][2] = acc[m][j][3] = 0.f;
          const __nv_bfloat16* xr[Z::MG][2];
#pragma unroll
          for (int m = 0; m < Z::MG; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int at = (m0 + m) * 16 + h * 8 + g, r = at < Z::TM ? row_of[at] : -1;
              xr[m][h] = r >= 0 ? a.x + (size_t)r * a.x_stride : nullptr;
            }
#pragma unroll 2
          for (int kk = k0 + 8 * t; kk - 8 * t < k1; kk += 32) {
            const bool in = kk < k1;
            const uint4 zero = make_uint4(0, 0, 0, 0);
            uint4 xv[Z::MG][2], av[Z::NT];
#pragma unroll
            for (int m = 0; m < Z::MG; ++m)
#pragma unroll
              for (int h = 0; h < 2; ++h) xv[m][h] = in && xr[m][h] ? *reinterpret_cast<const uint4*>(xr[m][h] + kk) : zero;
#pragma unroll
            for (int j = 0; j < Z::NT; ++j) av[j] = in && j < nts ? *reinterpret_cast<const uint4*>(aw + (size_t)(j * 8 + g) * a.k + kk) : zero;
#pragma unroll
            for (int j = 0; j < Z::NT; ++j) {
              if (j >= nts) continue;
#pragma unroll
              for (int m = 0; m < Z::MG; ++m) {
                mma(acc[m][j], xv[m][0].x, xv[m][1].x, xv[m][0].y, xv[m][1].y, av[j].x, av[j].y);
                mma(acc[m][j], xv[m][0].z, xv[m][1].z, xv[m][0].w, xv[m][1].w, av[j].z, av[j].w);
              }
            }
          }
          float* mine = part + warp * Z::MG * 16 * Z::PAD;
#pragma unroll
          for (int m = 0; m < Z::MG; ++m)
#pragma unroll
            for (int j = 0; j < Z::NT; ++j) {
              *reinterpret_cast<float2*>(mine + (m * 16 + g) * Z::PAD + j * 8 + 2 * t) = make_float2(acc[m][j][0], acc[m][j][1]);
              *reinterpret_cast<float2*>(mine + (m * 16 + 8 + g) * Z::PAD + j * 8 + 2 * t) = make_float2(acc[m][j][2], acc[m][j][3]);
            }
          __syncthreads();
          for (int i = tid; i < Z::MG * 16 * (Z::RC / 4); i += kThreads) {
            const int row = i / (Z::RC / 4), c = i % (Z::RC / 4) * 4;
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
              const float4 v = *reinterpret_cast<const float4*>(part + (w * Z::MG * 16 + row) * Z::PAD + c);
              s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
            if (m0 * 16 + row < Z::TM) *reinterpret_cast<float4*>(u + (m0 * 16 + row) * RS + c0 + c) = s;
          }
          __syncthreads();
        }
      }
      // ---- the cluster's sum, as two bf16 numbers ----
      const int per_row = rk / 4, quads = groups * 16 * per_row;
      auto sum_of = [&](int i, uint2& hi, uint2& lo) {
        const int row = i / per_row, c = (i - row * per_row) * 4;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < kCluster; ++r) {
          const float4 v = *reinterpret_cast<const float4*>(cluster.map_shared_rank(u, r) + row * RS + c);
          s[0] += v.x; s[1] += v.y; s[2] += v.z; s[3] += v.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = c + e < rank ? s[e] * scale : 0.f;  // (a padded rank has no part in it, whatever x holds)
        hi = make_uint2(pack(s[0], s[1]), pack(s[2], s[3]));
        lo = make_uint2(pack(rest(s[0]), rest(s[1])), pack(rest(s[2]), rest(s[3])));
        return row * Z::UPAD + c;
      };
      cluster.sync();
      const bool few = quads <= 512;
      if (few) {  // every CTA sums all of it; nobody writes his share of K again before all have read it (below)
        for (int i = tid; i < quads; i += kThreads) {
          uint2 hi, lo;
          const int at = sum_of(i, hi, lo);
          *reinterpret_cast<uint2*>(halves + at) = hi;
          *reinterpret_cast<uint2*>(halves + Z::TM * Z::UPAD + at) = lo;
        }
        __syncthreads();
      } else {    // every CTA sums an eighth and hands it to all
        const int from = (int)((long long)quads * cta / kCluster), to = (int)((long long)quads * (cta + 1) / kCluster);
        for (int i = from + tid; i < to; i += kThreads) {
          uint2 hi, lo;
          const int at = sum_of(i, hi, lo);
#pragma unroll
          for (int r = 0; r < kCluster; ++r) {
            __nv_bfloat16* there = cluster.map_shared_rank(halves, r);
            *reinterpret_cast<uint2*>(there + at) = hi;
            *reinterpret_cast<uint2*>(there + Z::TM * Z::UPAD + at) = lo;
          }
        }
        cluster.sync();
      }
    }
    // ---- out = y + u B^T: 32 columns a warp at a time; lane (g, t) has columns 8 t .. 8 t + 7 of rows g and g + 8 ----
    const int chunks = (a.n + 31) / 32, ks = rk / 16;
    for (int c = (share * kCluster + cta) * kWarps + warp; c < chunks; c += parts * kCluster * kWarps) {
      uint2 bv[4][Z::KS];  // MMA column g of n-tile j is column 8 (g / 2) + 2 j + g % 2
      const int n_lane = c * 32 + 8 * (g >> 1) + (g & 1);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int s = 0; s < Z::KS; ++s)
          bv[j][s] = s < ks && n_lane + 2 * j < a.n ? *reinterpret_cast<const uint2*>(a.b + ((size_t)tile.x * a.n + n_lane + 2 * j) * RS + s * 16 + 4 * t) : make_uint2(0, 0);
      const int col = c * 32 + 8 * t;
      auto load_y = [&](int m, uint4 (&v)[2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = m < groups ? row_of[m * 16 + h * 8 + g] : -1;
          v[h] = r >= 0 && col < a.n ? *reinterpret_cast<const uint4*>(a.y + (size_t)r * a.y_stride + col) : make_uint4(0, 0, 0, 0);
        }
      };
      uint4 next[2];
      load_y(0, next);
      for (int m = 0; m < groups; ++m) {
        uint4 yv[2] = {next[0], next[1]};
        load_y(m + 1, next);
        float acc[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
        const __nv_bfloat16* ur = halves + (m * 16 + g) * Z::UPAD + 4 * t;
#pragma unroll
        for (int s = 0; s < Z::KS; ++s) {
          if (s >= ks) continue;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint2 up = *reinterpret_cast<const uint2*>(ur + half * Z::TM * Z::UPAD + s * 16);
            const uint2 down = *reinterpret_cast<const uint2*>(ur + half * Z::TM * Z::UPAD + 8 * Z::UPAD + s * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) mma(acc[j], up.x, down.x, up.y, down.y, bv[j][s].x, bv[j][s].y);
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = row_of[m * 16 + h * 8 + g];
          if (r < 0 || col >= a.n) continue;
          uint4 o = yv[h];
          if (rank > 0) {
            uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = pack(ptx::bf16_lo(w[j]) + acc[j][2 * h], ptx::bf16_hi(w[j]) + acc[j][2 * h + 1]);
          }
          *reinterpret_cast<uint4*>(a.out + (size_t)r * a.out_stride + col) = o;
        }
      }
    }
    if (rank > 0) cluster.sync();  // (another CTA may still be reading this one's u)
    else __syncthreads();
  }
}

template <int RS>
b200_status launch(LoraArgs& a, int max_tiles, cudaStream_t s) {
  using Z = Shape<RS>;
  static int resident = 0;  // clusters that run at a time
  if (resident == 0) {
    B200_CUDA_TRY(cudaFuncSetAttribute(lora_kernel<RS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Z::kShared));
    resident = std::max(1, ctas_in_clusters(lora_kernel<RS>, kCluster, 8, b200_sm_count(), kThreads, Z::kShared) / kCluster);
  }
  a.most_parts = std::max(1, (a.n + 31) / 32 / (kCluster * kWarps));
  const int clusters = (int)std::min<long long>(resident, (long long)max_tiles * a.most_parts);
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kCluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(clusters * kCluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Z::kShared;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  (void)cudaLaunchKernelEx(&cfg, lora_kernel<RS>, a);
  B200_LAUNCH_CHECK();
  return B200_OK;
}

int max_tiles_of(int rows, int adapters) { return std::min(rows, adapters + 1) + rows / 16; }

bool fits(const void* p, int stride, int width) { return p && ((uintptr_t)p & 15) == 0 && stride % 8 == 0 && stride >= width; }

}  // namespace

extern "C" b200_status b200_lora_create(int32_t n_adapters, int32_t n, int32_t k, int32_t max_rank, b200_lora** out) {
  if (!out) { b200_set_error("lora: no place for the handle"); return B200_ERR_INVALID_ARGUMENT; }
  *out = nullptr;
  if (n_adapters <= 0 || n_adapters > kMaxAdapters || max_rank <= 0 || max_rank > kMaxRank) {
    b200_set_error("lora: %d adapters of rank %d (at most %d, and %d)", n_adapters, max_rank, kMaxAdapters, kMaxRank);
    return B200_ERR_INVALID_ARGUMENT;
  }
  if (n <= 0 || k <= 0 || n % 8 != 0 || k % 8 != 0) { b200_set_error("lora: a projection of %d x %d (multiples of 8)", n, k); return B200_ERR_INVALID_ARGUMENT; }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  auto* l = new b200_lora();
  l->n_adapters = n_adapters; l->n = n; l->k = k; l->max_rank = max_rank;
  l->rs = max_rank <= 16 ? 16 : max_rank <= 32 ? 32 : max_rank <= 64 ? 64 : 128;
  const size_t a_bytes = (size_t)n_adapters * l->rs * k * 2, b_bytes = (size_t)n_adapters * l->rs * n * 2;
  cudaError_t e = cudaMalloc((void**)&l->a, a_bytes);
  if (e == cudaSuccess) e = cudaMalloc((void**)&l->b, b_bytes);
  if (e == cudaSuccess) e = cudaMalloc((void**)&l->rank, sizeof(int) * n_adapters);
  if (e == cudaSuccess) e = cudaMalloc((void**)&l->scale, sizeof(float) * n_adapters);
  if (e == cudaSuccess) e = cudaMemset(l->a, 0, a_bytes);
  if (e == cudaSuccess) e = cudaMemset(l->b, 0, b_bytes);
  if (e == cudaSuccess) e = cudaMemset(l->rank, 0, sizeof(int) * n_adapters);
  if (e == cudaSuccess) e = cudaMemset(l->scale, 0, sizeof(float) * n_adapters);
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  if (e != cudaSuccess) {
    b200_set_error("lora: %d adapters of rank %d for %d x %d: %s", n_adapters, max_rank, n, k, cudaGetErrorString(e));
    cudaGetLastError();
    b200_lora_destroy(l);
    return B200_ERR_CUDA;
  }
  *out = l;
  return B200_OK;
}

extern "C" void b200_lora_destroy(b200_lora* l) {
  if (!l) return;
  for (void* p : {(void*)l->a, (void*)l->b, (void*)l->rank, (void*)l->scale}) if (p) cudaFree(p);
  delete l;
}

extern "C" b200_status b200_lora_set(b200_lora* l, int32_t adapter, int32_t rank, float scale, const void* h_a, const void* h_b) {
  if (!l || adapter < 0 || adapter >= l->n_adapters) { b200_set_error("lora: adapter %d out of range", adapter); return B200_ERR_INVALID_ARGUMENT; }
  if (rank < 0 || rank > l->max_rank) { b200_set_error("lora: rank %d, the handle holds up to %d", rank, l->max_rank); return B200_ERR_INVALID_ARGUMENT; }
  if (rank > 0 && (!h_a || !h_b)) { b200_set_error("lora: an adapter of rank %d without matrices", rank); return B200_ERR_INVALID_ARGUMENT; }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  __nv_bfloat16 *a = l->a + (size_t)adapter * l->rs * l->k, *b = l->b + (size_t)adapter * l->rs * l->n;
  B200_CUDA_TRY(cudaMemset(b, 0, (size_t)l->rs * l->n * 2));
  if (rank > 0) {
    B200_CUDA_TRY(cudaMemcpy(a, h_a, (size_t)rank * l->k * 2, cudaMemcpyHostToDevice));
    B200_CUDA_TRY(cudaMemcpy2D(b, (size_t)l->rs * 2, h_b, (size_t)rank * 2, (size_t)rank * 2, l->n, cudaMemcpyHostToDevice));
  }
  B200_CUDA_TRY(cudaMemcpy(l->scale + adapter, &scale, sizeof(float), cudaMemcpyHostToDevice));
  B200_CUDA_TRY(cudaMemcpy(l->rank + adapter, &rank, sizeof(int), cudaMemcpyHostToDevice));
  B200_CUDA_TRY(cudaDeviceSynchronize());
  return B200_OK;
}

extern "C" b200_status b200_lora_batch_create(int32_t max_rows, int32_t max_adapters, int32_t max_rank, b200_lora_batch** out) {
  if (!out) { b200_set_error("lora batch: no place for the handle"); return B200_ERR_INVALID_ARGUMENT; }
  *out = nullptr;
  if (max_rows <= 0 || max_rows > 1 << 24 || max_adapters <= 0 || max_adapters > kMaxAdapters || max_rank <= 0 || max_rank > kMaxRank) {
    b200_set_error("lora batch: %d rows, %d adapters of rank %d (at most %d, %d and %d)", max_rows, max_adapters, max_rank, 1 << 24, kMaxAdapters, kMaxRank);
    return B200_ERR_INVALID_ARGUMENT;
  }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  auto* b = new b200_lora_batch();
  b->max_rows = max_rows; b->max_adapters = max_adapters; b->max_rank = max_rank; b->max_tiles = max_tiles_of(max_rows, max_adapters);
  cudaError_t e = cudaMalloc((void**)&b->order, sizeof(int) * max_rows);
  if (e == cudaSuccess) e = cudaMalloc((void**)&b->tiles, sizeof(int4) * b->max_tiles);
  if (e == cudaSuccess) e = cudaMalloc((void**)&b->hdr, sizeof(int) * 4);
  if (e == cudaSuccess) e = cudaMemset(b->hdr, 0, sizeof(int) * 4);
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  if (e != cudaSuccess) {
    b200_set_error("lora batch: %d rows: %s", max_rows, cudaGetErrorString(e));
    cudaGetLastError();
    b200_lora_batch_destroy(b);
    return B200_ERR_CUDA;
  }
  *out = b;
  return B200_OK;
}

extern "C" void b200_lora_batch_destroy(b200_lora_batch* b) {
  if (!b) return;
  for (void* p : {(void*)b->order, (void*)b->tiles, (void*)b->hdr}) if (p) cudaFree(p);
  delete b;
}

extern "C" b200_status b200_lora_plan(b200_lora_batch* b, const int32_t* d_row_adapter, int32_t rows, void* stream) {
  if (!b || rows < 0 || (rows > 0 && !d_row_adapter)) { b200_set_error("lora plan: no batch, or no rows"); return B200_ERR_INVALID_ARGUMENT; }
  if (rows > b->max_rows) { b200_set_error("lora plan: %d rows, the batch holds %d", rows, b->max_rows); return B200_ERR_CAPACITY; }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  b->rows = rows;
  if (rows == 0) return B200_OK;
  launch_after(lora_plan_kernel, 1, rows <= 256 ? 256 : 1024, 0, (cudaStream_t)stream, d_row_adapter, rows, b->max_adapters,
               most_tile_rows(b->max_rank), b->order, b->tiles, b->hdr);
  B200_LAUNCH_CHECK();
  return B200_OK;
}

extern "C" b200_status b200_lora_apply(const b200_lora* l, const b200_lora_batch* b, const void* d_x, int32_t x_stride, const void* d_y, int32_t y_stride,
                                       void* d_out, int32_t out_stride, void* stream) {
  if (!l || !b) { b200_set_error("lora: no adapters, or no batch"); return B200_ERR_INVALID_ARGUMENT; }
  if (b->rows < 0) { b200_set_error("lora: the batch has no plan"); return B200_ERR_INVALID_ARGUMENT; }
  if (l->n_adapters != b->max_adapters || l->max_rank > b->max_rank) {
    b200_set_error("lora: %d adapters of rank %d, the batch is for %d of %d", l->n_adapters, l->max_rank, b->max_adapters, b->max_rank);
    return B200_ERR_INVALID_ARGUMENT;
  }
  if (b->rows > 0 && (!fits(d_x, x_stride, l->k) || !fits(d_y, y_stride, l->n) || !fits(d_out, out_stride, l->n) || (d_out == d_y && out_stride != y_stride))) {
    b200_set_error("lora: rows start on 16 bytes, strides are multiples of 8 elements and hold a row; out is y itself or apart from it");
    return B200_ERR_INVALID_ARGUMENT;
  }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  if (b->rows == 0) return B200_OK;
  LoraArgs a;
  a.a = l->a; a.b = l->b; a.x = (const __nv_bfloat16*)d_x; a.y = (const __nv_bfloat16*)d_y; a.out = (__nv_bfloat16*)d_out;
  a.rank = l->rank; a.scale = l->scale; a.order = b->order; a.tiles = b->tiles; a.hdr = b->hdr;
  a.n_adapters = l->n_adapters; a.n = l->n; a.k = l->k; a.rows = b->rows;
  a.x_stride = x_stride; a.y_stride = y_stride; a.out_stride = out_stride;
  const int tiles = max_tiles_of(b->rows, b->max_adapters);
  cudaStream_t s = (cudaStream_t)stream;
  return l->rs == 16 ? launch<16>(a, tiles, s) : l->rs == 32 ? launch<32>(a, tiles, s) : l->rs == 64 ? launch<64>(a, tiles, s) : launch<128>(a, tiles, s);
}
