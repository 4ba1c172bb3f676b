// Low-rank adapters of many requests beside a projection that they share: out[r] = y[r] + s_a B_a (A_a x[r]) with a = the row's adapter.
//
// The plan sorts a batch's rows by adapter and cuts each adapter's rows into tiles.  Then two kernels per projection:
//   * down: an item is a tile and a quarter of K, u = A x in f32, a warp for 16 rows; the block that is the last of its tile adds the quarters up;
//   * up: out = y + u B^T by steps of 32 rows of an adapter and 256 columns, of which every block has an equal share.
// Both are bound by what they read and write once (x and A; y, B and out).  The first kernel's operands come through a ring in shared memory, loads of
// later items under way while the present one is multiplied (cp.async; the rows of a tile may lie anywhere), or straight into registers where a tile
// has few rows; the second kernel's go straight into registers.  Its blocks are on their SMs, with y and B on the way, when the first one ends.
//
// Measured: 256 rows of 64 adapters of rank 16 at 4096 -> 6144, 16.5 us from HBM and 12.7 from L2 (and 3.3 for the plan); 1583 rows of 33 adapters of rank up
// to 64 at 4096 -> 28672, 92 to 95 us, 2.7 TB/s of what it cannot do without; 8192 rows of 5 of rank 32 at 14336 -> 4096, 93 to 95 us, 4.0 TB/s: 60 us of them
// are the first product's, which reads x at 3.9 TB/s.
//
// The products run on mma.sync m16n8k16.  A lane takes 16 neighbouring bytes of a row of x as its places of K in two MMAs, four neighbouring ranks
// as its places in one of the second product, and eight neighbouring columns of y as its places of N.  A, B and u lie in memory as the lanes take
// them, so that a warp's share of an MMA is 512 contiguous bytes.  At ranks up to 64 a byte of x or y has fewer than 64 multiplications, an order
// below what would ask for more than mma.sync.
//
// A row's u is summed in the same order whatever shares its tile: 1/64 of K by the MMAs, sixteen of those, then the quarters.  It goes into the
// second product as two bf16 numbers (u - hi, exactly, and that rounded), which leaves 2^-17 of it, and the sum with y is rounded once.
#include <cuda_bf16.h>

#include <algorithm>
#include <memory>
#include <new>

#include "common.h"
#include "launch.cuh"
#include "ptx.cuh"

// Adapters of one projection.  Rank rows are padded to rs (16, 32, 64 or 128), k and n to 32, with zeros.
//   a: [adapter][step of 32 of K][8 ranks][lane (g, t)] 16 bytes: rank g of the eight, K 8 t .. 8 t + 7 of the step
//   b: [adapter][32 columns][16 ranks][2][lane (g, t)] 16 bytes, two halves of 8: half h of the i-th: column 8 (g / 2) + 2 (2 i + h) + g % 2, ranks 4 t .. 4 t + 3
struct b200_lora {
  int n_adapters = 0, n = 0, k = 0, max_rank = 0, rs = 0;
  uint4 *a = nullptr, *b = nullptr;
  int* rank = nullptr;  // [adapter], 0: none
  float* scale = nullptr;
  size_t a_units() const { return (size_t)(k + 31) / 32 * rs * 4; }  // of 16 bytes, of an adapter
  size_t b_units() const { return (size_t)(n + 31) / 32 * rs * 4; }
};

// The rows of a step by adapter: order[max_rows]; tiles of {adapter or -1, first place in order, rows, first slot} (those of many rows from the front
// on, those of few from the back); groups of 32 rows of an adapter {adapter, first place, rows, -}, each two slots of 16; header {tiles of many rows,
// groups, tiles of few}.  And what goes from the first product to the second.
struct b200_lora_batch {
  int max_rows = 0, max_adapters = 0, max_rank = 0, max_tiles = 0, rows = -1;
  int* order = nullptr;
  int4* tiles = nullptr;
  int* hdr = nullptr;
  int4* groups = nullptr;   // [max_tiles]
  int* done = nullptr;      // [max_tiles] quarters of a tile that are there
  float* parts = nullptr;   // [quarter][max_rows][rank rows]
  uint32_t* u = nullptr;    // [slot][16 ranks][hi, lo][lane (g, t)] rows g and g + 8, ranks 4 t and 4 t + 1, then the same of 4 t + 2 and 4 t + 3
};

namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kSlices = 4;        // of K
constexpr int kFewRows = 16;      // of a tile whose slice of K the warps of a block share
constexpr int kMaxAdapters = 4096, kMaxRank = 128, kMaxWidth = 1 << 24, kTileRows = 128, kGroupRows = 32;

int rank_rows(int rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

// ---- the plan ------------------------------------------------------------------------------------------------------
// Places, tiles and groups are handed out as the atomics come: no row's result depends on its place, its tile or its block.
__global__ void __launch_bounds__(1024) lora_plan_kernel(const int* row_adapter, int rows, int n_adapters, int max_tiles, int enough_tiles, int* __restrict__ order,
                                                         int4* __restrict__ tiles, int4* __restrict__ groups, int* __restrict__ hdr) {
  after_previous();
  __shared__ int count[kMaxAdapters + 1], total[4], next[4];  // next: place, group, tile of many rows, tile of few
  const int tid = threadIdx.x, lane = tid & 31, bins = n_adapters + 1;
  for (int i = tid; i < bins; i += blockDim.x) count[i] = 0;
  if (tid < 4) total[tid] = next[tid] = 0;
  __syncthreads();
  // Adds one to the count of each lane's adapter (prompts are runs of one, so lanes with the same one add together); the count before, for this lane.
  auto count_rows = [&](int r) {
    int b = -1;
    if (r < rows) {
      const int a = row_adapter[r];
      b = a >= 0 && a < n_adapters ? a : n_adapters;
    }
    const unsigned same = __match_any_sync(0xffffffffu, b);
    const int first = __ffs(same) - 1;
    int before = 0;
    if (lane == first && b >= 0) before = atomicAdd(&count[b], __popc(same));
    return __shfl_sync(0xffffffffu, before, first) + __popc(same & ((1u << lane) - 1));
  };
  for (int base = 0; base < rows; base += blockDim.x) count_rows(base + tid);
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
  while ((1 << shift) < kTileRows && total[shift - 4] > enough_tiles) ++shift;
  for (int i = tid; i < bins; i += blockDim.x) {
    const int c = count[i];
    if (c == 0) continue;
    const int adapter = i < n_adapters ? i : -1, first = atomicAdd(&next[0], c), group = atomicAdd(&next[1], (c + kGroupRows - 1) / kGroupRows);
    for (int j = 0; j < c; j += kGroupRows) groups[group + j / kGroupRows] = make_int4(adapter, first + j, min(kGroupRows, c - j), 0);
    for (int j = 0; j < c; j += 1 << shift) {
      const int n = min(1 << shift, c - j);
      const int at = n > kFewRows ? atomicAdd(&next[2], 1) : max_tiles - 1 - atomicAdd(&next[3], 1);
      tiles[at] = make_int4(adapter, first + j, n, group * (kGroupRows / 16) + j / 16);
    }
    count[i] = first;
  }
  __syncthreads();
  for (int base = 0; base < rows; base += blockDim.x) {
    const int at = count_rows(base + tid);
    if (base + tid < rows) order[at] = base + tid;
  }
  if (tid == 0) { hdr[0] = next[2]; hdr[1] = next[1]; hdr[2] = next[3]; }
}

// ---- the products ---------------------------------------------------------------------------------------------------
struct LoraArgs {
  const uint4 *a, *b;
  const __nv_bfloat16 *x, *y;
  __nv_bfloat16* out;
  const int* rank;
  const float* scale;
  const int* order;
  const int4 *tiles, *groups;
  const int* hdr;
  int* done;
  float* parts;
  uint32_t* u;
  int max_rows, max_tiles, rows, n, k;  // rows: of x, y and out; the plan of a graph's launches may come to have others
  int x_stride, y_stride, out_stride;
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
// 16 bytes to shared memory, zeros where there is nothing to copy.
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_groups() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}

// ---- down: rings of chunks of 64 of K, a chunk [128 rows of x][128 bytes], 16-byte pieces of odd rows exchanged in halves, then A's -----------------
template <int RS>
struct Down {
  static constexpr int NT = RS / 8, CHUNK = (kTileRows + RS) * 128;
  static constexpr int STAGES = RS == 64 ? 4 : RS > 64 ? 6 : 5, PER_SM = RS > 64 ? 1 : 2;
  static constexpr int kShared = STAGES * CHUNK;
};

template <int RS>
__global__ void __launch_bounds__(kThreads, Down<RS>::PER_SM) lora_down_kernel(const __grid_constant__ LoraArgs a) {
  after_previous();
  using Z = Down<RS>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int s_last;
  const uint32_t ring = ptx::smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int n_items = a.hdr[0] * kSlices, n_few = a.hdr[2] * kSlices;
  const int each = (a.k + 64 * 32 - 1) / (64 * 32) * 32, per_slice = 64 / kSlices * each, k_steps = (a.k + 31) / 32;  // 1/64 of K; a slice of it

  // The last block of a tile to come here adds its quarters up, times the scale.  Ranks that are padding have no part in it, whatever x holds.
  auto finish = [&](int tile_at, const int4& tile) {
    __threadfence();
    __syncthreads();
    if (tid == 0) s_last = atomicAdd(&a.done[tile_at], 1) == kSlices - 1;
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    const int rank = min(a.rank[tile.x], RS), per_row = (rank + 15) / 16 * 4;
    const float scale = a.scale[tile.x];
    for (int i = tid; i < tile.z * per_row; i += kThreads) {
      const int row = i / per_row, c = (i - row * per_row) * 4;
      float s[4] = {0.f, 0.f, 0.f, 0.f};
      float4 v[kSlices];
#pragma unroll
      for (int q = 0; q < kSlices; ++q) v[q] = __ldcg(reinterpret_cast<const float4*>(a.parts + ((size_t)q * a.max_rows + tile.y + row) * RS + c));
#pragma unroll
      for (int q = 0; q < kSlices; ++q) { s[0] += v[q].x; s[1] += v[q].y; s[2] += v[q].z; s[3] += v[q].w; }
#pragma unroll
      for (int e = 0; e < 4; ++e) s[e] = c + e < rank ? s[e] * scale : 0.f;
      uint32_t* to = a.u + ((((size_t)(tile.w + row / 16) * (RS / 16) + c / 16) * 2) * 32 + row % 8 * 4 + c % 16 / 4) * 4 + row % 16 / 8;
      to[0] = pack(s[0], s[1]);
      to[2] = pack(s[2], s[3]);
      to[128] = pack(rest(s[0]), rest(s[1]));
      to[130] = pack(rest(s[2]), rest(s[3]));
    }
    if (tid == 0) a.done[tile_at] = 0;
  };

  // ---- loads, ahead of the products and across items: this thread copies piece `piece` of rows row0, row0 + 32, ... ----
  const int piece = tid & 7, row0 = tid >> 3;
  const uint32_t x_to = ring + row0 * 128 + ((piece ^ ((row0 & 1) << 2)) << 4);
  struct Cursor { int item, chunk, chunks, k0, rk; int4 tile; };
  Cursor lc{};
  const __nv_bfloat16* xp[kTileRows / 32];  // null: no such row
  const uint4* ap = nullptr;
  auto enter = [&](Cursor& c, int item) {  // the next item from `item` on that has something to do
    for (;; item += gridDim.x) {
      c.item = item;
      if (item >= n_items) return;
      c.tile = a.tiles[item / kSlices];
      c.chunk = 0;
      c.rk = c.tile.x >= 0 ? (min(a.rank[c.tile.x], RS) + 15) / 16 * 16 : 0;
      c.k0 = item % kSlices * per_slice;
      c.chunks = max(1, (min(a.k - c.k0, per_slice) + 63) / 64);
      if (c.rk > 0) return;
    }
  };
  auto enter_loads = [&](int item) {
    enter(lc, item);
    if (lc.item >= n_items) return;
#pragma unroll
    for (int i = 0; i < kTileRows / 32; ++i) {
      const int row = row0 + 32 * i < lc.tile.z ? a.order[lc.tile.y + row0 + 32 * i] : a.rows;
      xp[i] = row < a.rows ? a.x + (size_t)row * a.x_stride + lc.k0 + piece * 8 : nullptr;
    }
    ap = a.a + ((size_t)lc.tile.x * k_steps + lc.k0 / 32) * (RS * 4);
  };
  uint32_t load_slot = 0, use_slot = 0;
  auto issue = [&]() {
    if (lc.item < n_items) {
      const int k = lc.chunk * 64;
      const bool in = lc.k0 + k + piece * 8 < a.k;
      const uint32_t to = load_slot * Z::CHUNK;
#pragma unroll
      for (int i = 0; i < kTileRows / 32; ++i)
        if (xp[i]) copy16(x_to + to + i * 32 * 128, in ? xp[i] + k : a.x, in);
#pragma unroll
      for (int i = tid; i < RS * 8; i += kThreads)  // two steps of [8 ranks][lane]
        if (i % (RS * 4) < lc.rk * 4) copy16(ring + to + kTileRows * 128 + i * 16, lc.k0 / 32 + lc.chunk * 2 + i / (RS * 4) < k_steps ? ap + lc.chunk * (RS * 8) + i : a.a, lc.k0 / 32 + lc.chunk * 2 + i / (RS * 4) < k_steps);
      if (++lc.chunk == lc.chunks) enter_loads(lc.item + gridDim.x);
    }
    commit();
    if (++load_slot == Z::STAGES) load_slot = 0;
  };
  enter_loads(blockIdx.x);
  if (lc.item < n_items)
    for (int i = 0; i < Z::STAGES - 1; ++i) issue();

  Cursor c{};
  for (enter(c, blockIdx.x); c.item < n_items; enter(c, c.item + gridDim.x)) {
    float acc[Z::NT][4], sum[Z::NT][4];
#pragma unroll
    for (int j = 0; j < Z::NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = sum[j][e] = 0.f;
    const bool works = warp * 16 < c.tile.z;
    const int nts = c.rk / 8, steps = each / 32;
    int within = 0;
    for (int chunk = 0; chunk < c.chunks; ++chunk) {
      wait_groups<Z::STAGES - 2>();
      __syncthreads();  // (the chunk is there, and the one before it has been used)
      issue();
      const uint32_t stage = ring + use_slot * Z::CHUNK, xa = stage + (warp * 16 + g) * 128, aw = stage + kTileRows * 128 + lane * 16;
      if (++use_slot == Z::STAGES) use_slot = 0;
      if (!works) continue;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const uint32_t at = (uint32_t)((s * 4 + t) ^ ((g & 1) << 2)) << 4;
        const uint4 va = lds16(xa + at), vb = lds16(xa + 8 * 128 + at);
#pragma unroll
        for (int j = 0; j < Z::NT; ++j) {
          if (j >= nts) continue;
          const uint4 w = lds16(aw + (s * Z::NT + j) * 512);
          mma(acc[j], va.x, vb.x, va.y, vb.y, w.x, w.y);
          mma(acc[j], va.z, vb.z, va.w, vb.w, w.z, w.w);
        }
        if (++within == steps) {  // 1/64 of K is complete
          within = 0;
#pragma unroll
          for (int j = 0; j < Z::NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) { sum[j][e] += acc[j][e]; acc[j][e] = 0.f; }
        }
      }
    }
    if (works) {
      float* parts = a.parts + ((size_t)(c.item % kSlices) * a.max_rows + c.tile.y) * RS;
      const int ra = warp * 16 + g, rb = ra + 8;
#pragma unroll
      for (int j = 0; j < Z::NT; ++j) {
        if (j >= nts) continue;
        // (the last 1/64 of K may be cut short by the end of it)
        if (ra < c.tile.z) *reinterpret_cast<float2*>(parts + (size_t)ra * RS + j * 8 + 2 * t) = make_float2(sum[j][0] + acc[j][0], sum[j][1] + acc[j][1]);
        if (rb < c.tile.z) *reinterpret_cast<float2*>(parts + (size_t)rb * RS + j * 8 + 2 * t) = make_float2(sum[j][2] + acc[j][2], sum[j][3] + acc[j][3]);
      }
    }
    finish(c.item / kSlices, c.tile);
  }
  wait_groups<0>();
  __syncthreads();
  // ---- tiles of few rows: the warps share the slice, straight from memory; the sums of its 1/64s of K go to shared memory ----
  constexpr int SHARE = 64 / kSlices / kWarps, PAD = RS + 8;  // 1/64s of a warp; floats between rows of their sums, [1/64][row][PAD] in place of the ring
  float* sums = reinterpret_cast<float*>(smem);
  for (int item = blockIdx.x + (n_items + gridDim.x - 1 - blockIdx.x) / gridDim.x * gridDim.x; item < n_items + n_few; item += gridDim.x) {
    const int tile_at = a.max_tiles - 1 - (item - n_items) / kSlices, slice = (item - n_items) % kSlices;
    const int4 tile = a.tiles[tile_at];
    const int rank = tile.x >= 0 ? min(a.rank[tile.x], RS) : 0, nts = (rank + 15) / 16 * 2;
    if (rank == 0) continue;
    const int row_a = g < tile.z ? a.order[tile.y + g] : a.rows, row_b = g + 8 < tile.z ? a.order[tile.y + 8 + g] : a.rows;
    const bool on_a = row_a < a.rows, on_b = row_b < a.rows;
    const __nv_bfloat16 *xa = a.x + (size_t)(on_a ? row_a : 0) * a.x_stride, *xb = a.x + (size_t)(on_b ? row_b : 0) * a.x_stride;
    const uint4* aw = a.a + (size_t)tile.x * k_steps * (RS * 4) + lane;
    auto load16 = [](const __nv_bfloat16* p, bool there) { return there ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0); };
#pragma unroll(RS > 32 ? 1 : SHARE)
    for (int i = 0; i < SHARE; ++i) {
      const int part = warp * SHARE + i, k0 = slice * per_slice + part * each, k1 = min(a.k, k0 + each);
      float acc[Z::NT][4];
#pragma unroll
      for (int j = 0; j < Z::NT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
#pragma unroll(RS > 32 ? 1 : 2)
      for (int kk = k0; kk < k1; kk += 32) {
        const bool in = kk + 8 * t < k1;
        const uint4 va = load16(xa + kk + 8 * t, in && on_a), vb = load16(xb + kk + 8 * t, in && on_b);
        uint4 w[Z::NT];
#pragma unroll
        for (int j = 0; j < Z::NT; ++j) w[j] = j < nts ? aw[(size_t)(kk / 32) * (RS * 4) + j * 32] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int j = 0; j < Z::NT; ++j) {
          if (j >= nts) continue;
          mma(acc[j], va.x, vb.x, va.y, vb.y, w[j].x, w[j].y);
          mma(acc[j], va.z, vb.z, va.w, vb.w, w[j].z, w[j].w);
        }
      }
      float* mine = sums + part * 16 * PAD;
#pragma unroll
      for (int j = 0; j < Z::NT; ++j) {
        *reinterpret_cast<float2*>(mine + g * PAD + j * 8 + 2 * t) = make_float2(acc[j][0], acc[j][1]);
        *reinterpret_cast<float2*>(mine + (8 + g) * PAD + j * 8 + 2 * t) = make_float2(acc[j][2], acc[j][3]);
      }
    }
    __syncthreads();
    // added in the order in which a warp by itself comes to them
    for (int i = tid; i < tile.z * (RS / 4); i += kThreads) {
      const int row = i / (RS / 4), e = i % (RS / 4) * 4;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int part = 0; part < 64 / kSlices; ++part) {
        const float4 w = *reinterpret_cast<const float4*>(sums + (part * 16 + row) * PAD + e);
        v.x += w.x; v.y += w.y; v.z += w.z; v.w += w.w;
      }
      *reinterpret_cast<float4*>(a.parts + ((size_t)slice * a.max_rows + tile.y + row) * RS + e) = v;
    }
    finish(tile_at, tile);
  }
}

// ---- up: 32 columns for a warp, steps of 32 rows ------------------------------------------------------------------------------------------------------
// Its part of B stays in registers; lane (g, t) has columns 8 t .. 8 t + 7 of rows g, g + 8, g + 16 and g + 24.  The warps of a block take neighbouring
// columns, so what they read of y is contiguous and u comes from their L1.  Nothing passes through shared memory: with y by cp.async, u and B in bulk
// and warps for that alone, those warps' issue was what everything waited for (1850 cycles for 32 rows of 256 columns, 1140 for their products).
// What bounds it is how many bytes are on their way: 2 KB of y a warp, a step of 32 rows ahead (1583 rows of rank 64 to 28672 columns 70 us; 16 rows
// ahead, and B loaded before the next y instead of behind it, 88), and blocks per SM as the registers for that allow.
template <int RS>
struct Up {
  static constexpr int KS = RS / 16, COLS = kWarps * 32, PER_SM = RS == 16 ? 3 : RS <= 64 ? 2 : 1;
};

// (Everything but u was there when the kernel ahead began, and that one lets this one start behind its own wait: only u is waited for.)
template <int RS>
__global__ void __launch_bounds__(kThreads, Up<RS>::PER_SM) lora_up_kernel(const __grid_constant__ LoraArgs a) {
  using Z = Up<RS>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int groups = a.hdr[1], col_blocks = (a.n + Z::COLS - 1) / Z::COLS, n_blocks = (a.n + 31) / 32;
  const long long all = (long long)groups * col_blocks;
  const int begin = (int)(all * blockIdx.x / gridDim.x), end = (int)(all * (blockIdx.x + 1) / gridDim.x);
  if (begin < end) {
    // Ahead of the step at hand: y of the next one, the rows' numbers of the one behind it, and the group behind that.
    struct Place { int block, at; };  // range of columns, group
    auto behind = [&](Place p) { return ++p.at == groups ? Place{p.block + 1, 0} : p; };
    auto group_of = [&](int s, const Place& p) { return s < end ? a.groups[p.at] : make_int4(-1, 0, 0, 0); };  // {adapter, first place, rows, -}
    auto rows_of = [&](const int4& gr, int (&r)[4]) {  // g, g + 8, g + 16, g + 24 of the group; -1: none
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = g + 8 * i < gr.z ? a.order[gr.y + g + 8 * i] : -1;
    };
    // (Whether the call has a row is asked where it is used, its number being under way until then.  Another load in place of one that is left out: with the
    // condition widened, 1583 rows of rank 128 to 28672 columns took 217 us for 207.)
    auto there = [&](int r) { return (unsigned)r < (unsigned)a.rows; };
    auto load_y = [&](const int (&r)[4], int block, uint4 (&y)[4]) {
      const int col = (block * kWarps + warp) * 32 + 8 * t;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = r[i] >= 0 && col < a.n ? *reinterpret_cast<const uint4*>(a.y + (size_t)min(r[i], a.rows - 1) * a.y_stride + col) : make_uint4(0, 0, 0, 0);
    };
    Place p0{begin / groups, 0}, p1, p2;
    p0.at = begin - p0.block * groups;
    p1 = behind(p0);
    p2 = behind(p1);
    int4 g0 = group_of(begin, p0), g1 = group_of(begin + 1, p1), g2 = group_of(begin + 2, p2);
    int r0[4], r1[4];
    uint4 y0[4];
    rows_of(g0, r0);
    rows_of(g1, r1);
    load_y(r0, p0.block, y0);
    auto ranks_of = [&](int adapter) { return adapter >= 0 ? (min(a.rank[adapter], RS) + 15) / 16 : 0; };  // in sixteens
    auto load_b = [&](int adapter, int block, int ks, uint4 (&v)[Z::KS][2]) {
      const uint4* bp = a.b + ((size_t)max(adapter, 0) * n_blocks + min(block * kWarps + warp, n_blocks - 1)) * Z::KS * 64 + lane;
#pragma unroll
      for (int k = 0; k < Z::KS; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) v[k][i] = k < ks ? bp[(k * 2 + i) * 32] : make_uint4(0, 0, 0, 0);
    };
    uint4 bv[Z::KS][2];
    int ks = ranks_of(g0.x);
    load_b(g0.x, p0.block, ks, bv);
    for (int s = begin; s < end; ++s) {
      const int col = (p0.block * kWarps + warp) * 32 + 8 * t, slot = p0.at * (kGroupRows / 16);
      const bool other = s + 1 < end && (g1.x != g0.x || p1.block != p0.block);  // another part of B is next
      if (other && g1.x >= 0 && p1.block * kWarps + warp < n_blocks && lane < RS / 2)  // on its way to L2, as it is laid out: all RS ranks, of 128 the first 64
        asm volatile("prefetch.global.L2 [%0];" ::"l"(a.b + ((size_t)g1.x * n_blocks + p1.block * kWarps + warp) * Z::KS * 64 + lane * 8));
      uint4 y1[4];
      load_y(r1, p1.block, y1);
      int r2[4];
      rows_of(g2, r2);
      const Place p3 = behind(p2);
      const int4 g3 = group_of(s + 3, p3);
      if (s == begin) after_previous();
#pragma unroll
      for (int m = 0; m < kGroupRows / 16; ++m) {
        if (m * 16 >= g0.z || (ks == 0 && a.out == a.y)) continue;
        float acc[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
        const uint4* up = reinterpret_cast<const uint4*>(a.u) + (size_t)(slot + m) * Z::KS * 64 + lane;
#pragma unroll
        for (int k = 0; k < Z::KS; ++k) {
          if (k >= ks) continue;
          const uint4 u[2] = {__ldca(up + (k * 2) * 32), __ldca(up + (k * 2 + 1) * 32)};
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              mma(acc[2 * i], u[half].x, u[half].y, u[half].z, u[half].w, bv[k][i].x, bv[k][i].y);
              mma(acc[2 * i + 1], u[half].x, u[half].y, u[half].z, u[half].w, bv[k][i].z, bv[k][i].w);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!there(r0[2 * m + h]) || col >= a.n) continue;
          uint4 o = y0[2 * m + h];
          if (ks > 0) {
            uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = pack(ptx::bf16_lo(w[j]) + acc[j][2 * h], ptx::bf16_hi(w[j]) + acc[j][2 * h + 1]);
          }
          *reinterpret_cast<uint4*>(a.out + (size_t)r0[2 * m + h] * a.out_stride + col) = o;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) { r0[i] = r1[i]; r1[i] = r2[i]; y0[i] = y1[i]; }
      if (other) {
        ks = ranks_of(g1.x);
        load_b(g1.x, p1.block, ks, bv);
      }
      p0 = p1; p1 = p2; p2 = p3;
      g0 = g1; g1 = g2; g2 = g3;
    }
  } else {
    after_previous();
  }
}

template <int RS>
b200_status launch(LoraArgs& a, int max_tiles, cudaStream_t s) {
  static bool configured = false;
  if (!configured) {
    B200_CUDA_TRY(cudaFuncSetAttribute(lora_down_kernel<RS>, cudaFuncAttributeMaxDynamicSharedMemorySize, Down<RS>::kShared));
    configured = true;
  }
  const long long sms = b200_sm_count(), items = (long long)max_tiles * ((a.n + Up<RS>::COLS - 1) / Up<RS>::COLS);
  launch_after(lora_down_kernel<RS>, (unsigned)std::min<long long>((long long)max_tiles * kSlices, sms * Down<RS>::PER_SM), kThreads, Down<RS>::kShared, s, a);
  B200_LAUNCH_CHECK();
  launch_after(lora_up_kernel<RS>, (unsigned)std::min<long long>(items, sms * Up<RS>::PER_SM), kThreads, 0, s, a);
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
  if (n <= 0 || k <= 0 || n % 8 != 0 || k % 8 != 0 || n > kMaxWidth || k > kMaxWidth) {
    b200_set_error("lora: a projection of %d x %d (multiples of 8, at most %d)", n, k, kMaxWidth);
    return B200_ERR_INVALID_ARGUMENT;
  }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  auto* l = new (std::nothrow) b200_lora();
  if (!l) { b200_set_error("lora: out of host memory"); return B200_ERR_CAPACITY; }
  l->n_adapters = n_adapters; l->n = n; l->k = k; l->max_rank = max_rank;
  l->rs = rank_rows(max_rank);
  const size_t a_bytes = n_adapters * l->a_units() * 16, b_bytes = n_adapters * l->b_units() * 16;
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
  if (rank > 0) {  // into the lanes' order
    const uint16_t *ha = (const uint16_t*)h_a, *hb = (const uint16_t*)h_b;
    const int rs = l->rs, ks = rs / 16;
    const size_t a_size = l->a_units() * 8, b_size = l->b_units() * 8;
    std::unique_ptr<uint16_t[]> a(new (std::nothrow) uint16_t[a_size]()), b(new (std::nothrow) uint16_t[b_size]());
    if (!a || !b) { b200_set_error("lora: out of host memory for an adapter of %d x %d", l->n, l->k); return B200_ERR_CAPACITY; }
    for (int r = 0; r < rank; ++r)
      for (int k = 0; k < l->k; ++k) a[((((size_t)(k / 32) * (rs / 8) + r / 8) * 32 + r % 8 * 4 + k % 32 / 8) * 8) + k % 8] = ha[(size_t)r * l->k + k];
    for (int n = 0; n < l->n; ++n) {
      const int c = n % 32, g = c / 8 * 2 + c % 2, j = c / 2 % 4;
      for (int r = 0; r < rank; ++r)
        b[(((((size_t)(n / 32) * ks + r / 16) * 2 + j / 2) * 32 + g * 4 + r % 16 / 4) * 2 + j % 2) * 4 + r % 4] = hb[(size_t)n * rank + r];
    }
    B200_CUDA_TRY(cudaMemcpy(l->a + adapter * l->a_units(), a.get(), a_size * 2, cudaMemcpyHostToDevice));
    B200_CUDA_TRY(cudaMemcpy(l->b + adapter * l->b_units(), b.get(), b_size * 2, cudaMemcpyHostToDevice));
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
  auto* b = new (std::nothrow) b200_lora_batch();
  if (!b) { b200_set_error("lora batch: out of host memory"); return B200_ERR_CAPACITY; }
  b->max_rows = max_rows; b->max_adapters = max_adapters; b->max_rank = max_rank; b->max_tiles = max_tiles_of(max_rows, max_adapters);
  cudaError_t e = cudaMalloc((void**)&b->order, sizeof(int) * max_rows);
  if (e == cudaSuccess) e = cudaMalloc((void**)&b->tiles, sizeof(int4) * b->max_tiles);
  if (e == cudaSuccess) e = cudaMalloc((void**)&b->hdr, sizeof(int) * 4);
  if (e == cudaSuccess) e = cudaMalloc((void**)&b->groups, sizeof(int4) * b->max_tiles);
  if (e == cudaSuccess) e = cudaMalloc((void**)&b->done, sizeof(int) * b->max_tiles);
  if (e == cudaSuccess) e = cudaMalloc((void**)&b->parts, sizeof(float) * kSlices * (size_t)max_rows * rank_rows(max_rank));
  if (e == cudaSuccess) e = cudaMalloc((void**)&b->u, (size_t)b->max_tiles * kGroupRows * rank_rows(max_rank) * 4);
  if (e == cudaSuccess) e = cudaMemset(b->hdr, 0, sizeof(int) * 4);
  if (e == cudaSuccess) e = cudaMemset(b->done, 0, sizeof(int) * b->max_tiles);
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
  for (void* p : {(void*)b->order, (void*)b->tiles, (void*)b->hdr, (void*)b->groups, (void*)b->done, (void*)b->parts, (void*)b->u}) if (p) cudaFree(p);
  delete b;
}

extern "C" b200_status b200_lora_plan(b200_lora_batch* b, const int32_t* d_row_adapter, int32_t rows, void* stream) {
  if (!b || rows < 0 || (rows > 0 && !d_row_adapter)) { b200_set_error("lora plan: no batch, or no rows"); return B200_ERR_INVALID_ARGUMENT; }
  if (rows > b->max_rows) { b200_set_error("lora plan: %d rows, the batch holds %d", rows, b->max_rows); return B200_ERR_CAPACITY; }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  b->rows = rows;
  if (rows == 0) {  // (for layers in a graph: none of their rows are there)
    B200_CUDA_TRY(cudaMemsetAsync(b->hdr, 0, sizeof(int) * 4, (cudaStream_t)stream));
    return B200_OK;
  }
  // A tile is kSlices items of the first product: beyond one for each of its blocks, larger tiles rather than more of them (2097 rows of two adapters of
  // rank 128, one block per SM, at 14336 -> 4096: 99 us; with room for two blocks per SM, so smaller tiles, 166).
  const int enough = b200_sm_count() * (b->max_rank > 64 ? Down<128>::PER_SM : Down<64>::PER_SM) / kSlices;
  launch_after(lora_plan_kernel, 1, rows <= 256 ? 256 : 1024, 0, (cudaStream_t)stream, d_row_adapter, rows, b->max_adapters,
               b->max_tiles, enough, b->order, b->tiles, b->groups, b->hdr);
  B200_LAUNCH_CHECK();
  return B200_OK;
}

extern "C" b200_status b200_lora_apply(const b200_lora* l, b200_lora_batch* b, const void* d_x, int32_t x_stride, const void* d_y, int32_t y_stride,
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
  const int tiles = max_tiles_of(b->rows, b->max_adapters);
  if ((long long)tiles * ((l->n + kWarps * 32 - 1) / (kWarps * 32)) > 0x7fffffff) { b200_set_error("lora: %d rows of %d columns in one call", b->rows, l->n); return B200_ERR_CAPACITY; }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  if (b->rows == 0) return B200_OK;
  LoraArgs a;
  a.a = l->a; a.b = l->b; a.x = (const __nv_bfloat16*)d_x; a.y = (const __nv_bfloat16*)d_y; a.out = (__nv_bfloat16*)d_out;
  a.rank = l->rank; a.scale = l->scale; a.order = b->order; a.tiles = b->tiles; a.groups = b->groups; a.hdr = b->hdr;
  a.done = b->done; a.parts = b->parts; a.u = b->u;
  a.max_rows = b->max_rows; a.max_tiles = b->max_tiles; a.rows = b->rows; a.n = l->n; a.k = l->k;
  a.x_stride = x_stride; a.y_stride = y_stride; a.out_stride = out_stride;
  cudaStream_t s = (cudaStream_t)stream;
  return l->rs == 16 ? launch<16>(a, tiles, s) : l->rs == 32 ? launch<32>(a, tiles, s) : l->rs == 64 ? launch<64>(a, tiles, s) : launch<128>(a, tiles, s);
}
