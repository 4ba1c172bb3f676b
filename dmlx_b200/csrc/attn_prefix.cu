// Attention of a batch whose sequences share pages: what several rows see of a page is computed for all of them at once.
//
// Sequences come to share pages by fork and by prefix sharing, which hand on pages from the front, and a page that is written by one of them is
// copied first.  So two sequences that have the same page at one place have the same pages before it, and the rows of a step form a tree: a node is
// a range of pages and the rows that see all of them.  A row's context is its nodes from the root on, and the pages behind them that it has alone.
// Softmax over the parts: each gives m = max s, l = sum 2^(s - m) and o = sum 2^(s - m) v, and the parts are joined as 2^(m_i - m) l_i and
// 2^(m_i - m) o_i (f32).
//
// Four kernels.  The plan (one block, once per step) finds the tree by the first page that rows of a group have not compared yet: equal pages make
// a group, its smallest common length a node.  Then, per layer:
//   * nodes with more than 16 query rows per kv head: tcgen05.  An item is up to 256 query rows (row, head of the GQA group), a range of the
//     node's pages, and a kv head; S = Q K^T into tensor memory, P = 2^(S - m) in 16 bits in its place, O += P V with P read from there.  Every key is
//     seen by every row, so there are no masks;
//   * everything else, smaller nodes and the rows' own pages: a warp per item on mma.sync, 16 query rows, pages by TMA into rings of its own;
//   * the join.
// The first two run at the same time: the plan gives the nodes as many SMs as lets both end together.
//
// Of 128 keys and 256 query rows the tensor-core kernel's exponentials and its products take 2048 cycles each; a block of both takes 3750, since a tile's
// next scores wait for its last product (P lies where they go) and the two tiles overlap only in part; an item has 22000 more around its blocks, for q,
// the first pages and 128 KB of parts.  The warps' kernel is bound by the stream of pages.  Measured per layer, 32 query heads on 8, 128 dims, pages in
// HBM: 256 rows behind 8192 shared tokens with up to 512 of their own 88 us (one after the other 110: 52 the nodes' on all SMs, 51 the warps', 10 the
// join), 64 rows behind 2048 28 us, 128 rows behind 4096 on FP8 pages 39.5 us; plans 11 to 16 us.
#include <cuda_bf16.h>
#include <cuda_fp8.h>

#include <algorithm>
#include <new>

#include "common.h"
#include "kv_pool.cuh"
#include "launch.cuh"
#include "ptx.cuh"
#include "tma.cuh"

namespace {

constexpr int kMaxRows = 4096;
constexpr int kLevels = 3;        // nodes that a row may go through
constexpr int kItemUnits = 44, kBlockUnits = 10, kTileUnits = 6;  // of time, of the tensor-core kernel
constexpr int kMinPages = 2;      // of a node: below that a part of its own costs more than it saves
constexpr int kWarpRows = 16;     // query rows of an item of the warps' kernel
constexpr int kBlockKeys = 128, kBlockPages = 4, kTileRows = 128;
constexpr float kHidden = -1e30f;   // score of a key that a row does not see
constexpr float kNoScale = -1e28f;  // scale of a row that has seen no key
constexpr uint32_t kPolls = 1u << 21;

struct Node {
  int seq;            // a slot whose table holds the node's pages
  int first, count;   // its rows: places of `members`
  int p0, p1;         // pages
};
struct Member { int row, slot; };  // a row of a node; the place of its first part
struct alignas(16) ItemA { int seq, first, count, p0, p1, part, tiles, pad; };  // pages of slot seq's table for `count` members from `first` on; their part behind `slot`
struct alignas(16) ItemB { int seq, first, count, p0, p1, ctx, part, pad; };  // count 0: own pages of the row `first`, its part `part`, and ctx tokens that it sees; else members, as above

enum { H_ITEMS_A = 0, H_ITEMS_B, H_NEXT_A, H_NEXT_B, H_WORKERS_A, H_ROWS, H_COUNT = 16 };  // H_WORKERS_A: blocks that work on the large nodes; H_ROWS: of the plan

struct PlanDev {
  int *hdr, *row_seq, *row_ctx, *row_base, *member_node;
  Node* nodes;
  Member* members;
  ItemA* items_a;
  ItemB* items_b;
  float *part_o, *part_ml;  // [slot][q head][D], [slot][q head]{max in log2, sum}
  int max_rows, max_slots;
};

// Rows of a tile of 128: whole GQA groups.
__host__ __device__ constexpr int tile_members(int group) { return kTileRows / group; }

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// ---- the plan ------------------------------------------------------------------------------------------------------------
// A large node's rows in items of equal size, of one tile if all of them fit, else of two each: how many parts a row has depends on the node alone, not on
// its place among the members, which atomics hand out.  A chunk gives a row one part, or two where the item's one tile of rows has its blocks of keys go to
// the two softmax groups in turn.
__host__ __device__ __forceinline__ bool is_large(int count, int group) { return count * group > kWarpRows; }
__device__ __forceinline__ bool one_tile(const Node& n, int group) { return n.count <= tile_members(group); }
__device__ __forceinline__ int items_of(const Node& n, int group) { return ceil_div(n.count, 2 * tile_members(group)); }  // of a chunk
__device__ __forceinline__ int even_length(int pages, int len) { return ceil_div(ceil_div(pages, ceil_div(pages, len)), kBlockPages) * kBlockPages; }  // of as many chunks
__device__ __forceinline__ int large_parts(int pages, int len, bool one) {  // len: pages of a chunk, a multiple of kBlockPages
  const int chunks = ceil_div(pages, len), last = pages - (chunks - 1) * len;
  return one ? 2 * chunks - (last <= kBlockPages ? 1 : 0) : chunks;
}

constexpr int kLengthsA = 12;  // pages of a chunk: all, 256, 192, 128, 96, ..., 12, 8
__device__ __forceinline__ int length_a(int k) { return k == 0 ? 1 << 28 : k & 1 ? 512 >> (k + 1) / 2 : 384 >> k / 2; }
constexpr int kLengthsB = 6;  // all, 32, 16, 8, 4, 2
__device__ __forceinline__ int length_b(int k) { return k == 0 ? 1 << 28 : 64 >> k; }

struct PlanShared {
  int n_nodes, n_members, more, warp_sums[32], carry;
  int max_a[kLengthsA], items_a[kLengthsA], units_a[kLengthsA], slots_a[kLengthsA];
  int items_b[kLengthsB], slots_b[kLengthsB];
  int units_b, longest_b, workers_a, pick_a, pick_b, next_a, next_b;
};

// Common pages of two sequences that agree up to `lo` (at least one page behind it too): a search in steps of 16 probes.
__device__ __forceinline__ int common_pages(const int* a, const int* b, int lo, int hi) {
  while (lo < hi) {  // agree on [0, lo), may on [0, hi)
    const int step = max(1, (hi - lo + 15) / 16);
    int agree = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int p = lo + (i + 1) * step;
      const bool same = p <= hi && a[min(p, hi) - 1] == b[min(p, hi) - 1];
      agree += same ? 1 : 0;  // (pages agree from the front on, so the probes that do come first)
    }
    const int next = lo + agree * step;
    hi = min(hi, next + step - 1);
    lo = next;
  }
  return lo;
}

__global__ void __launch_bounds__(1024) prefix_plan_kernel(KvDev d, PlanDev p, const int* row_seq, const int* row_ctx, int rows, int hash_size, int group,
                                                           int workers, int warps, float per_page) {
  after_previous();
  extern __shared__ __align__(16) unsigned char dyn[];
  unsigned long long* keys = reinterpret_cast<unsigned long long*>(dyn);  // [hash_size]
  int* leader = reinterpret_cast<int*>(keys + hash_size);                 // [hash_size] smallest row of the entry
  int* count = leader + hash_size;
  int* common = count + hash_size;   // pages that all rows of the entry have in common
  int* place = common + hash_size;   // of the entry's next row among the members, -1: no node
  int* depth = place + hash_size;    // [rows] pages compared
  int* from = depth + rows;          // pages covered by nodes
  int* grp = from + rows;            // the row's group: its smallest row
  int* entry = grp + rows;
  int* full = entry + rows;          // pages that the row sees whole
  int* parts = full + rows;          // parts so far
  __shared__ PlanShared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr unsigned long long kEmpty = ~0ull;
  if (tid == 0) { s.n_nodes = 0; s.n_members = 0; }
  for (int i = tid; i < rows; i += blockDim.x) {
    const int seq = row_seq[i];
    const bool there = seq >= 0 && seq < d.max_seqs;
    // (behind its pages a slot's table names what it had before: rows that ask for it would agree there with rows that they share nothing with before)
    const int ctx = there ? min(max(row_ctx[i], 0), d.seq_pages[seq] * d.page_size) : 0;
    p.row_seq[i] = there ? seq : 0;
    p.row_ctx[i] = ctx;
    full[i] = ctx / d.page_size;
    depth[i] = 0; from[i] = 0; grp[i] = 0; parts[i] = 0;
  }
  __syncthreads();
  // ---- the tree, a level at a time ----
  int level_first[kLevels + 1];
  int levels = 0;
  for (int round = 0; round < 4 * kLevels && levels < kLevels; ++round) {
    for (int i = tid; i < hash_size; i += blockDim.x) { keys[i] = kEmpty; leader[i] = 0x7fffffff; count[i] = 0; common[i] = 0x7fffffff; place[i] = -1; }
    if (tid == 0) s.more = 0;
    __syncthreads();
    level_first[levels] = s.n_members;
    for (int base = 0; base < rows; base += blockDim.x) {
      const int i = base + tid;
      const bool on = i < rows && depth[i] < full[i];
      if (i < rows) entry[i] = -1;
      unsigned long long key = kEmpty;
      if (on) key = (unsigned long long)(unsigned)grp[i] << 32 | (unsigned)d.block_table[(size_t)p.row_seq[i] * d.max_pages_per_seq + depth[i]];
      // the lanes that agree with the first of them go in as one
      const unsigned active = __ballot_sync(0xffffffffu, on);
      if (active == 0) continue;
      const int lead = __ffs(active) - 1;
      const unsigned long long first = __shfl_sync(0xffffffffu, key, lead);
      const unsigned alike = __ballot_sync(0xffffffffu, on && key == first);
      const bool mine = alike >> lane & 1u;
      unsigned at = 0;
      if (on && (!mine || lane == lead)) {
        at = ((unsigned)key * 2654435761u ^ (unsigned)(key >> 32) * 40503u) & (hash_size - 1);
        for (int probe = 0; probe < hash_size; ++probe) {
          const unsigned long long had = atomicCAS(&keys[at], kEmpty, key);
          if (had == kEmpty || had == key) break;
          at = (at + 1) & (hash_size - 1);
        }
        atomicMin(&leader[at], i);  // (the first lane has the smallest row of its group)
        atomicAdd(&count[at], mine ? __popc(alike) : 1);
      }
      const unsigned of_lead = __shfl_sync(0xffffffffu, at, lead);
      if (on) entry[i] = (int)(mine ? of_lead : at);
    }
    __syncthreads();
    for (int base = 0; base < rows; base += blockDim.x) {
      const int i = base + tid, e = i < rows ? entry[i] : -1;
      const bool on = e >= 0 && count[max(e, 0)] >= 2;
      int have = 0x7fffffff;
      if (on) {
        const int l = leader[e];
        have = l == i ? full[i]
                      : common_pages(d.block_table + (size_t)p.row_seq[i] * d.max_pages_per_seq, d.block_table + (size_t)p.row_seq[l] * d.max_pages_per_seq,
                                     depth[i] + 1, min(full[i], full[l]));
      }
      const unsigned active = __ballot_sync(0xffffffffu, on);
      if (active == 0) continue;
      const int lead = __ffs(active) - 1, first = __shfl_sync(0xffffffffu, e, lead);
      const bool mine = on && e == first;
      const int least = __reduce_min_sync(0xffffffffu, mine ? have : 0x7fffffff);
      if (on && (!mine || lane == lead)) atomicMin(&common[e], mine ? least : have);
    }
    __syncthreads();
    for (int i = tid; i < rows; i += blockDim.x) {
      const int e = entry[i];
      if (e < 0 || leader[e] != i || count[e] < 2 || common[e] - from[i] < kMinPages) continue;
      const int node = atomicAdd(&s.n_nodes, 1), first = atomicAdd(&s.n_members, count[e]);
      p.nodes[node] = Node{p.row_seq[i], first, count[e], from[i], common[e]};
      place[e] = first;
      keys[e] = (unsigned long long)(unsigned)node;  // (the key has done its work)
    }
    __syncthreads();
    for (int i = tid; i < rows; i += blockDim.x) {
      const int e = entry[i];
      if (e < 0) continue;
      if (count[e] < 2) { depth[i] = full[i]; continue; }
      if (place[e] >= 0) {
        const int at = atomicAdd(&place[e], 1);
        p.members[at].row = i;
        p.member_node[at] = (int)keys[e];
        from[i] = common[e];
      }
      depth[i] = common[e];
      grp[i] = leader[e];
      s.more = 1;
    }
    __syncthreads();
    const bool more = s.more != 0;
    if (s.n_members > level_first[levels]) ++levels;
    __syncthreads();
    if (!more) break;
  }
  level_first[levels] = s.n_members;
  for (int l = levels + 1; l <= kLevels; ++l) level_first[l] = s.n_members;
  // ---- lengths of chunks ----
  if (tid < kLengthsA) { s.max_a[tid] = 0; s.items_a[tid] = 0; s.units_a[tid] = 0; s.slots_a[tid] = 0; }
  if (tid < kLengthsB) { s.items_b[tid] = 0; s.slots_b[tid] = 0; }
  if (tid == 0) { s.next_a = 0; s.next_b = 0; s.carry = 0; s.units_b = 0; s.longest_b = 0; }
  __syncthreads();
  const int n_nodes = s.n_nodes, warp_members = kWarpRows / group;
  for (int u = tid; u < n_nodes * kLengthsA; u += blockDim.x) {  // a thread per node and length
    const Node n = p.nodes[u / kLengthsA];
    const int k = u % kLengthsA, pages = n.p1 - n.p0;
    if (is_large(n.count, group)) {
      // in units of 500 cycles: a block of two tiles of rows kBlockUnits, of one kTileUnits, with the memory busy beside; an item's fill, drain and way out kItemUnits
      const bool one = one_tile(n, group);
      const int len = even_length(pages, length_a(k)), chunks = ceil_div(pages, len), blocks = ceil_div(pages, kBlockPages), of_block = one ? kTileUnits : kBlockUnits;
      const int tiles = items_of(n, group);
      atomicMax(&s.max_a[k], of_block * min(blocks, len / kBlockPages) + kItemUnits);
      atomicAdd(&s.items_a[k], tiles * chunks);
      atomicAdd(&s.units_a[k], tiles * (of_block * blocks + kItemUnits * chunks));
      atomicAdd(&s.slots_a[k], n.count * large_parts(pages, len, one));
    } else if (k < kLengthsB) {
      const int chunks = ceil_div(pages, length_b(k)), tiles = ceil_div(n.count, warp_members);
      atomicAdd(&s.items_b[k], tiles * chunks);
      atomicAdd(&s.slots_b[k], n.count * chunks);
      if (k == 0) { atomicAdd(&s.units_b, tiles * pages); atomicMax(&s.longest_b, pages); }
    }
  }
  int own_chunks[kLengthsB] = {}, own_pages = 0, longest = 0;
  for (int i = tid; i < rows; i += blockDim.x) {
    const int pages = ceil_div(p.row_ctx[i], d.page_size) - from[i];
#pragma unroll
    for (int k = 0; k < kLengthsB; ++k) own_chunks[k] += ceil_div(pages, length_b(k));
    own_pages += pages;
    longest = max(longest, pages);
  }
#pragma unroll
  for (int k = 0; k < kLengthsB; ++k) {
    const int c = __reduce_add_sync(0xffffffffu, own_chunks[k]);
    if (lane == 0) { atomicAdd(&s.items_b[k], c); atomicAdd(&s.slots_b[k], c); }
  }
  own_pages = __reduce_add_sync(0xffffffffu, own_pages);
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (lane == 0) { atomicAdd(&s.units_b, own_pages); atomicMax(&s.longest_b, longest); }
  __syncthreads();
  if (warp == 0) {
    // Lengths of both kinds of chunks, and how many blocks work on the nodes, by the shortest estimated time of those whose parts fit; a lane per choice.
    // The rest runs beside the nodes, on the SMs that they leave and on theirs when they are done.  Of an SM it takes 2.3 units an item and `per_page` a
    // page (0.6 us and, of 128 dims in 16 bits, 0.2), up to two thirds of the SMs, whose loads are all that the memory gives; the last items end one by one.
    const float of_item = per_page * __fdividef(warps, workers) * 0.6f, most = 0.68f * workers, heads = d.n_kv_heads;
    const float of_slot = 6e-6f * d.n_kv_heads * group * d.head_dim;  // written and read again
    auto share_up = [](float a, float b) { return __float2int_ru(__fdividef(a, b)); };  // (a little too much or too little does no harm)
    float best = 3e38f;
    int choice = 0;
    for (int c = lane; c < kLengthsA * 2 * kLengthsB; c += 32) {
      const int k = c / (2 * kLengthsB), b = c % kLengthsB, slots = s.slots_a[k] + s.slots_b[b];
      const float items = s.items_a[k] * heads, rounds = max(share_up(items, workers), 1) + c / kLengthsB % 2;
      const int mine = min(max(share_up(items, rounds), 1), workers);
      const float nodes = fmaxf(__fdividef(s.units_a[k] * heads, mine), 0.875f * rounds * s.max_a[k]);
      const float rest = (s.units_b * per_page + 2.3f * s.items_b[b]) * heads, rate = fmaxf(fminf(workers - mine, most), 0.01f), beside = __fdividef(rest, rate);
      const float pages = fminf(beside, nodes + __fdividef(fmaxf(rest - nodes * rate, 0.f), most)) + of_item * min(length_b(b), s.longest_b);
      const float cost = fmaxf(nodes, pages) + of_slot * slots;
      if ((slots <= p.max_slots || (k == 0 && b == 0)) && cost < best) { best = cost; choice = (k * kLengthsB + b) << 16 | mine; }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, best, o);
      const int theirs = __shfl_xor_sync(0xffffffffu, choice, o);
      if (other < best || (other == best && theirs < choice)) { best = other; choice = theirs; }
    }
    if (lane == 0) { s.pick_a = (choice >> 16) / kLengthsB; s.pick_b = (choice >> 16) % kLengthsB; s.workers_a = choice & 0xffff; }
  }
  __syncthreads();
  const int len_a = length_a(s.pick_a), len_b = length_b(s.pick_b);
  // ---- places of the parts: a row's nodes from the root on, then its own pages ----
  for (int l = 0; l < levels; ++l) {
    for (int at = level_first[l] + tid; at < level_first[l + 1]; at += blockDim.x) {
      const Node n = p.nodes[p.member_node[at]];
      const int row = p.members[at].row, pages = n.p1 - n.p0;
      p.members[at].slot = parts[row];
      parts[row] += is_large(n.count, group) ? large_parts(pages, even_length(pages, len_a), one_tile(n, group)) : ceil_div(pages, len_b);
    }
    __syncthreads();
  }
  for (int base = 0; base < rows; base += blockDim.x) {
    const int i = base + tid;
    const int own = i < rows ? ceil_div(ceil_div(p.row_ctx[i], d.page_size) - from[i], len_b) : 0, all = i < rows ? parts[i] + own : 0;
    int incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    if (lane == 31) s.warp_sums[warp] = incl;
    __syncthreads();
    int start = s.carry + incl - all;
    for (int w = 0; w < warp; ++w) start += s.warp_sums[w];
    if (i < rows) {
      p.row_base[i] = start;
      depth[i] = start;
      if (own > 0) {
        const int at = atomicAdd(&s.next_b, own);
        const int pages = ceil_div(p.row_ctx[i], d.page_size);
        for (int c = 0; c < own; ++c) {
          const int p0 = from[i] + c * min(len_b, pages);
          p.items_b[at + c] = ItemB{p.row_seq[i], i, 0, p0, min(pages, p0 + min(len_b, pages)), p.row_ctx[i], start + parts[i] + c, 0};
        }
      }
    }
    __syncthreads();
    if (tid == (int)blockDim.x - 1) s.carry = start + all;
    __syncthreads();
  }
  for (int at = tid; at < s.n_members; at += blockDim.x) p.members[at].slot += depth[p.members[at].row];
  // items of the nodes, a warp per node
  for (int i = warp; i < n_nodes; i += blockDim.x / 32) {
    const Node n = p.nodes[i];
    const int pages = n.p1 - n.p0, large = is_large(n.count, group) ? 1 : 0, len = large ? even_length(pages, len_a) : min(len_b, pages), chunks = ceil_div(pages, len);
    const int tiles = large ? items_of(n, group) : 1, each = ceil_div(n.count, tiles), one = one_tile(n, group) ? 1 : 0;
    int at = 0;
    if (lane == 0) at = atomicAdd(large ? &s.next_a : &s.next_b, tiles * chunks);
    at = __shfl_sync(0xffffffffu, at, 0);
    for (int c = lane; c < tiles * chunks; c += 32) {
      const int tile = c % tiles, chunk = c / tiles, p0 = n.p0 + chunk * len, p1 = min(n.p1, p0 + len);
      if (large) {
        p.items_a[at + c] = ItemA{n.seq, n.first + tile * each, min(each, n.count - tile * each), p0, p1, one ? 2 * chunk : chunk, one ? 1 : 2, 0};
      } else {
        p.items_b[at + c] = ItemB{n.seq, n.first, n.count, p0, p1, 0x7fffffff, chunk, 0};
      }
    }
  }
  __syncthreads();
  if (tid == 0) {
    p.row_base[rows] = s.carry;
    p.hdr[H_ITEMS_A] = s.next_a;
    p.hdr[H_ITEMS_B] = s.next_b;
    p.hdr[H_NEXT_A] = 0;
    p.hdr[H_NEXT_B] = 0;
    p.hdr[H_WORKERS_A] = s.workers_a;
    p.hdr[H_ROWS] = rows;
  }
}

// ---- arguments and small things that the kernels share ------------------------------------------------------------------
struct Args {
  KvDev d;
  PlanDev p;
  int layer, rows, n_q_heads, group;  // rows of q and out; the plan of a graph's launches may come to have others (row numbers that q lacks are not read)
  bool nodes;  // whether the kernel of the large nodes is ahead of the warps'
  const __nv_bfloat16* q;
  int q_stride;
  __nv_bfloat16* out;
  int out_stride;
  float scale_log2;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Bounded; once a wait has run out nothing is waited for any more, so that every role comes to its end.
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, bool& ok) {
  if (!ok) return;
  for (uint32_t i = 0; i < kPolls; ++i)
    if (ptx::mbar_try_wait(bar, parity)) return;
  ok = false;
}
__device__ __forceinline__ const int* table_of(const Args& a, int seq) { return a.d.block_table + (size_t)seq * a.d.max_pages_per_seq; }

// ---- everything but the large nodes: a warp per item ------------------------------------------------------------------------
// 16 query rows are all that mma.sync needs for one tile, and the pages of few rows come as fast as the memory gives them: about 2180 pages of 8 heads, 285 MB
// in K and V, 51 us on all SMs, 5.6 TB/s; 59 us on 92 of them, 68 on 74.  K and V are loads of their own, so that a warp's next page is on its way before
// this one's values have been used.  (Of 128 dims: a layer of 256, 64 and 4 rows takes 89.2, 27.9 and 10.7 us; with twelve warps of two stages 87.6, 29.3 and
// 11.1, with seven of four 94.5, 27.8 and 9.8.)
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <bool F16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t lo16) {
  uint32_t d;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(d) : "h"((unsigned short)lo16));
  return d;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <int D, bool FP8>
struct ShapeB {
  static constexpr int TILE = 32 * D * (FP8 ? 1 : 2);  // bytes of a page's K or V of one head
  static constexpr int WARPS = D == 64 ? 12 : 8, STAGES = FP8 || D == 64 ? 4 : 3;  // registers, then shared memory (a stage holds K or V of a page)
  static constexpr int QUEUE = 8;                      // items that a warp's loads may be ahead of its products
  static constexpr size_t kShared = (size_t)WARPS * STAGES * TILE + 1024 + sizeof(uint64_t) * WARPS * STAGES + sizeof(int) * WARPS * QUEUE;
};

// bf16: K and V as they are; FP8: the codes widened to f16 in registers (exact), K's dims and V's output columns in the order in which ldmatrix gives
// the bytes, the page's K scale on the scores, its V scale (over the item's largest) on P, which f16 takes with three bits more than bf16 down to 2^-14 of
// the row's largest weight and within 2^-25 of it below.
template <int D, bool FP8>
__device__ __forceinline__ void warp_items(const CUtensorMap& kmap, const CUtensorMap& vmap, const Args& a) {
  using Z = ShapeB<D, FP8>;
  constexpr int TILE = Z::TILE, STAGES = Z::STAGES, KS = D / 16, NO = D / 8;
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~(uintptr_t)1023);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  unsigned char* tiles = smem + (size_t)warp * STAGES * TILE;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + (size_t)Z::WARPS * STAGES * TILE) + warp * STAGES;
  int* queue = reinterpret_cast<int*>(reinterpret_cast<uint64_t*>(smem + (size_t)Z::WARPS * STAGES * TILE) + Z::WARPS * STAGES) + warp * Z::QUEUE;
  const int H = a.d.n_kv_heads, G = a.group, n_items = a.p.hdr[H_ITEMS_B] * H;
  if (lane == 0) {
    for (int s = 0; s < STAGES; ++s) ptx::mbar_init(&full[s], 1);
    ptx::mbar_fence_init();
  }
  __syncwarp();

  // ---- loads: the items come off a counter; K and V of page after page, ahead of the products ----
  int p_head = 0, p_begin = 0, p_page = 0, p_end = 0, p_ids = 0, p_id = 0;
  const int* p_table = nullptr;
  uint32_t taken = 0, loaded = 0, load_slot = 0;
  bool p_more = true, p_value = false;
  auto enter = [&]() {  // the next item's number into the queue (-1: no more)
    int id = 0;
    if (lane == 0) id = atomicAdd(&a.p.hdr[H_NEXT_B], 1);
    id = __shfl_sync(0xffffffffu, id, 0);
    p_more = id < n_items;
    if (lane == 0) queue[taken % Z::QUEUE] = p_more ? id : -1;
    __syncwarp();
    ++taken;
    if (!p_more) return;
    const ItemB it = a.p.items_b[id / H];
    p_head = id % H;
    p_table = table_of(a, it.seq);
    p_begin = p_page = it.p0;
    p_end = it.p1;
  };
  auto load_tile = [&]() {
    if (!p_more) return;
    if (!p_value) {
      const int rel = p_page - p_begin;
      if ((rel & 31) == 0) p_ids = p_page + lane < p_end ? p_table[p_page + lane] : 0;
      p_id = __shfl_sync(0xffffffffu, p_ids, rel & 31);
    }
    if (lane == 0) {
      ptx::fence_proxy_async_smem();
      const CUtensorMap* map = p_value ? &vmap : &kmap;
      ptx::mbar_expect_tx(&full[load_slot], TILE);
#pragma unroll
      for (int b = 0; b < (FP8 ? 1 : D / 64); ++b) ptx::tma_load_3d(tiles + load_slot * TILE + b * 4096, map, b * 64, (p_id * H + p_head) * 32, a.layer, &full[load_slot]);
    }
    ++loaded;
    if (++load_slot == STAGES) load_slot = 0;
    if (p_value && ++p_page >= p_end) enter();
    p_value = !p_value;
  };
  enter();
  for (int i = 0; i < STAGES; ++i) load_tile();

  bool alive = true;
  uint32_t used = 0, use_slot = 0, use_lap = 0;
  auto next_tile = [&]() {  // the address of the next tile in turn, when it is there
    // (each lane polls for itself: what follows wants the whole warp, whether the tile came or not)
    alive = __all_sync(0xffffffffu, ptx::mbar_wait(&full[use_slot], use_lap & 1u));
    return ptx::smem_u32(tiles + use_slot * TILE);
  };
  auto done_tile = [&]() {
    __syncwarp();
    ++used;
    if (++use_slot == STAGES) { use_slot = 0; ++use_lap; }
    load_tile();
  };
  const int ld_r = lane & 7, ld_m = lane >> 3;
  for (uint32_t n = 0; alive; ++n) {
    const int id = queue[n % Z::QUEUE];
    if (id < 0) break;
    const ItemB it = a.p.items_b[id / H];
    const int item_head = id % H;
    // a node of more than 16 query rows does not come here: its members are all in this item
    const int members = max(it.count, 1);
    const bool low = members * G > 8;  // whether rows 8 to 15 of the tile are used
    int row[2], slot[2], qh[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = g + 8 * h, m = r / G;
      row[h] = slot[h] = -1;
      qh[h] = item_head * G + r - m * G;
      if (m < members) {
        if (it.count == 0) { row[h] = it.first; slot[h] = it.part; }
        else { const Member mb = a.p.members[it.first + m]; row[h] = mb.row; slot[h] = mb.slot + it.part; }
      }
      if (row[h] >= a.rows) row[h] = -1;
    }
    uint32_t qa[KS][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __nv_bfloat16* qr = a.q + (size_t)max(row[h], 0) * a.q_stride + (size_t)qh[h] * D;
#pragma unroll
      for (int c = 0; c < KS; ++c) {
        if constexpr (FP8) {  // K slots (2t, 2t + 1) are dims 16 c + 4 t + {0, 1}, slots (2t + 8, 2t + 9) dims 16 c + 4 t + {2, 3}
          const uint2 w = row[h] >= 0 ? *reinterpret_cast<const uint2*>(qr + 16 * c + 4 * t) : make_uint2(0, 0);
          qa[c][h] = pack_f16(ptx::bf16_lo(w.x), ptx::bf16_hi(w.x));
          qa[c][2 + h] = pack_f16(ptx::bf16_lo(w.y), ptx::bf16_hi(w.y));
        } else {
          qa[c][h] = row[h] >= 0 ? *reinterpret_cast<const uint32_t*>(qr + 16 * c + 2 * t) : 0u;
          qa[c][2 + h] = row[h] >= 0 ? *reinterpret_cast<const uint32_t*>(qr + 16 * c + 8 + 2 * t) : 0u;
        }
      }
    }
    float my_ks = 1.f, my_vr = 1.f, v_ref = 1.f;
    auto page_scales = [&](int page0) {  // lane i: the scales of page page0 + i
      my_ks = 0.f; my_vr = 0.f;
      if (page0 + lane < it.p1) {
        const size_t at = ((size_t)a.layer * a.d.n_pages + table_of(a, it.seq)[page0 + lane]) * H + item_head;
        my_ks = a.d.k_scale[at];
        my_vr = a.d.v_scale[at];
      }
    };
    if constexpr (FP8) {
      v_ref = 0.f;
      for (int base = it.p0; base < it.p1; base += 32) { page_scales(base); v_ref = fmaxf(v_ref, my_vr); }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v_ref = fmaxf(v_ref, __shfl_xor_sync(0xffffffffu, v_ref, o));
    }
    const float v_inv = v_ref > 0.f ? 1.0f / v_ref : 0.f;

    float o[NO][4];
#pragma unroll
    for (int j = 0; j < NO; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m_run[2] = {kNoScale, kNoScale}, l_run[2] = {0.f, 0.f};
    for (int pg = it.p0; pg < it.p1; ++pg) {
      const uint32_t kbase = next_tile();
      if (!alive) break;
      float ks = a.scale_log2, vr = 1.f;
      if constexpr (FP8) {
        const int rel = pg - it.p0;
        if ((rel & 31) == 0) page_scales(pg);
        ks = __shfl_sync(0xffffffffu, my_ks, rel & 31) * a.scale_log2;
        vr = __shfl_sync(0xffffffffu, my_vr, rel & 31) * v_inv;
      }
      float sc[4][4];
#pragma unroll
      for (int nt = 0; nt < 4; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
      if constexpr (FP8) {
#pragma unroll
        for (int kk = 0; kk < KS / 4; ++kk)
#pragma unroll
          for (int nt = 0; nt < 4; ++nt) {
            const int r = nt * 8 + ld_r, cc = 4 * kk + ld_m;
            uint32_t b[4];
            ldsm_x4(kbase + r * 128 + ((cc ^ (r & 7)) << 4), b);
#pragma unroll
            for (int m = 0; m < 4; ++m) mma<true>(sc[nt], qa[4 * kk + m], e4m3x2_to_f16x2(b[m]), e4m3x2_to_f16x2(b[m] >> 16));
          }
      } else {
#pragma unroll
        for (int kk = 0; kk < KS / 2; ++kk)
#pragma unroll
          for (int nt = 0; nt < 4; ++nt) {
            const int r = nt * 8 + ld_r, cc = 4 * kk + ld_m;
            uint32_t b[4];
            ldsm_x4(kbase + (cc >> 3) * 4096 + r * 128 + (((cc & 7) ^ (r & 7)) << 4), b);
            mma<false>(sc[nt], qa[2 * kk], b[0], b[1]);
            mma<false>(sc[nt], qa[2 * kk + 1], b[2], b[3]);
          }
      }
      done_tile();  // (the scores are in registers)
      const int left = it.ctx - pg * 32;  // keys of this page that are seen
      uint32_t pa[2][4];
      float corr[2] = {1.f, 1.f};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h == 1 && !low) {
          pa[0][1] = pa[0][3] = pa[1][1] = pa[1][3] = 0u;
          continue;
        }
        float mx = kHidden;
#pragma unroll
        for (int nt = 0; nt < 4; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // (a score that is no number weighs nothing, as a hidden one)
            sc[nt][2 * h + e] = nt * 8 + 2 * t + e < left ? fmaxf(sc[nt][2 * h + e] * ks, kHidden) : kHidden;
            mx = fmaxf(mx, sc[nt][2 * h + e]);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m_run[h], mx);
        corr[h] = ex2(m_run[h] - m_new);
        float sum = 0.f;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
          float pv[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            pv[e] = ex2(sc[2 * kt + (e >> 1)][2 * h + (e & 1)] - m_new);
            sum += pv[e];
          }
          pa[kt][h] = FP8 ? pack_f16(pv[0] * vr, pv[1] * vr) : pack_bf16(pv[0], pv[1]);
          pa[kt][2 + h] = FP8 ? pack_f16(pv[2] * vr, pv[3] * vr) : pack_bf16(pv[2], pv[3]);
        }
        l_run[h] = l_run[h] * corr[h] + sum;
        m_run[h] = m_new;
      }
      if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
        for (int j = 0; j < NO; ++j) { o[j][0] *= corr[0]; o[j][1] *= corr[0]; o[j][2] *= corr[1]; o[j][3] *= corr[1]; }
      }
      const uint32_t vbase = next_tile();
      if (!alive) break;
      const bool whole = left >= 32;  // else what lies behind the context may be anything, and 0 times it no number
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        const int k0 = kt * 16 + 2 * t;  // this lane's keys: k0, k0 + 1, k0 + 8, k0 + 9
        if constexpr (FP8) {
#pragma unroll
          for (int jj = 0; jj < KS / 2; ++jj) {
            const int r = kt * 16 + (ld_m & 1) * 8 + ld_r, cc = 2 * jj + (ld_m >> 1);
            uint32_t b[4];
            ldsm_x4_trans(vbase + r * 128 + ((cc ^ (r & 7)) << 4), b);
            if (!whole) {  // (of a word: key, dim: two bytes of the first key, two of the second)
              const uint32_t low_keys = (k0 < left ? 0xFFFFu : 0u) | (k0 + 1 < left ? 0xFFFF0000u : 0u), high_keys = (k0 + 8 < left ? 0xFFFFu : 0u) | (k0 + 9 < left ? 0xFFFF0000u : 0u);
              b[0] &= low_keys; b[2] &= low_keys; b[1] &= high_keys; b[3] &= high_keys;
            }
            // bytes (key 2t, dim 2g), (2t, 2g+1), (2t+1, 2g), (2t+1, 2g+1) -> (even dims | odd dims)
            const uint32_t p0 = __byte_perm(b[0], 0u, 0x3120), p1 = __byte_perm(b[1], 0u, 0x3120), p2 = __byte_perm(b[2], 0u, 0x3120), p3 = __byte_perm(b[3], 0u, 0x3120);
            mma<true>(o[4 * jj], pa[kt], e4m3x2_to_f16x2(p0), e4m3x2_to_f16x2(p1));
            mma<true>(o[4 * jj + 1], pa[kt], e4m3x2_to_f16x2(p0 >> 16), e4m3x2_to_f16x2(p1 >> 16));
            mma<true>(o[4 * jj + 2], pa[kt], e4m3x2_to_f16x2(p2), e4m3x2_to_f16x2(p3));
            mma<true>(o[4 * jj + 3], pa[kt], e4m3x2_to_f16x2(p2 >> 16), e4m3x2_to_f16x2(p3 >> 16));
          }
        } else {
#pragma unroll
          for (int jj = 0; jj < NO / 2; ++jj) {
            const int r = kt * 16 + (ld_m & 1) * 8 + ld_r, cc = 2 * jj + (ld_m >> 1);
            uint32_t b[4];
            ldsm_x4_trans(vbase + (cc >> 3) * 4096 + r * 128 + (((cc & 7) ^ (r & 7)) << 4), b);
            if (!whole) {
              const uint32_t low_keys = (k0 < left ? 0xFFFFu : 0u) | (k0 + 1 < left ? 0xFFFF0000u : 0u), high_keys = (k0 + 8 < left ? 0xFFFFu : 0u) | (k0 + 9 < left ? 0xFFFF0000u : 0u);
              b[0] &= low_keys; b[2] &= low_keys; b[1] &= high_keys; b[3] &= high_keys;
            }
            mma<false>(o[2 * jj], pa[kt], b[0], b[1]);
            mma<false>(o[2 * jj + 1], pa[kt], b[2], b[3]);
          }
        }
      }
      done_tile();
    }
    if (!alive) break;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
      l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
      if (slot[h] < 0) continue;
      const size_t at = (size_t)slot[h] * a.n_q_heads + qh[h];
      float* po = a.p.part_o + at * D;
      if constexpr (FP8) {
#pragma unroll
        for (int c = 0; c < KS; ++c)  // dims 16 c + 4 t + {0, 1, 2, 3} = column 2t of tiles 2c and 2c + 1, then column 2t + 1
          *reinterpret_cast<float4*>(po + 16 * c + 4 * t) =
              make_float4(o[2 * c][2 * h] * v_ref, o[2 * c + 1][2 * h] * v_ref, o[2 * c][2 * h + 1] * v_ref, o[2 * c + 1][2 * h + 1] * v_ref);
      } else {
#pragma unroll
        for (int j = 0; j < NO; ++j) *reinterpret_cast<float2*>(po + j * 8 + 2 * t) = make_float2(o[j][2 * h], o[j][2 * h + 1]);
      }
      if (t == 0) *reinterpret_cast<float2*>(a.p.part_ml + at * 2) = make_float2(m_run[h], l_run[h]);
    }
  }
  if (!alive) {  // leave no copy in flight behind
    const uint32_t first = loaded > STAGES ? loaded - STAGES : 0;
    for (uint32_t i = first > used ? first : used; i < loaded; ++i) ptx::mbar_wait(&full[i % STAGES], (i / STAGES) & 1u);
    if (lane == 0) atomicExch(a.d.state + ST_ATTN_ERR, B200_ERR_DEVICE_FLAGGED);
  }
}
// The kernel ahead, the nodes', waits for all that is before it and then lets this one start, on the SMs that it leaves and later on its own.  Neither
// reads what the other writes, and the waits here are for copies of its own, so this one waits for the nodes' only at its end: what follows waits for this one alone.
template <int D, bool FP8>
__global__ void __launch_bounds__(ShapeB<D, FP8>::WARPS * 32, 1) prefix_warp_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ Args a) {
  if (!a.nodes) wait_previous();
  warp_items<D, FP8>(kmap, vmap, a);
  let_next_start();
  wait_previous();
}

// ---- large nodes: tcgen05 ---------------------------------------------------------------------------------------------------
// Warps 0-7 and 8-15: softmax of a tile each, two threads a row (64 of a block's 128 keys); warp 16: loads of pages; warp 17: products; on FP8 pools warps
// 18 and 19 widen the pages' codes to f16, which is exact, q and P being f16 there too.  An item of two tiles has both use every block of keys; one of one
// tile has its blocks in turn to the two softmax groups, with sums and parts of their own.
// A row keeps its scale until a score is 2^kLate above it, so that a block is one vote of the two warps of a row and no exchange of maxima: all that a
// late scale costs is that the largest weight is no longer 1, and so is rounded like the others.
// (256 rows behind 8192 tokens, on all SMs: 52 us.  With one thread a row, two warps on each of the SM's quarters, 61: 3560 cycles of softmax had nothing
// to hide their latency behind.  64 keys at a time into two places of tensor memory, the next scores ahead of the softmax, 63, since products of 64
// columns take longer per key; a row in four lanes of one warp, with nothing to agree on, 56; a warp of products for each tile slows both, 82 for 66.)
constexpr int kSoftWarps = 16, kLoadWarp = 16, kMmaWarp = 17, kWidenWarps = 2, kWiden = kWidenWarps * 32;
__host__ __device__ constexpr int threads_a(bool fp8) { return (kMmaWarp + 1 + (fp8 ? kWidenWarps : 0)) * 32; }
constexpr float kLate = 4.f;

template <int D, bool FP8>
struct ShapeA {
  static constexpr int BOXES = D / 64, SLOT = BOXES * kBlockKeys * 128, QBYTES = BOXES * kTileRows * 128;
  static constexpr int SLOTS = FP8 ? 3 : D == 128 ? 5 : 8;
  static constexpr int RAW = kBlockKeys * D, RAWS = FP8 ? 4 : 0;  // FP8: slots of codes in front of the slots of operands
};
template <int D, bool FP8>
struct SharedA {
  using Z = ShapeA<D, FP8>;
  uint64_t full[Z::SLOTS], free[Z::SLOTS], raw_full[4], raw_free[4], q_full, q_free, s_full[2], p_ready[2], o_full[2], item_full[2], item_free[2], drain;
  float exchange[2][2][kTileRows];  // [tile][half of the keys]: a row's maximum, its sum
  int item[2][8];  // {kind, head, seq, first member, members, first page, last page + 1, chunk}; kind: tiles of rows, 0 = no more
  uint32_t tmem;
};

template <int D, bool FP8>
constexpr size_t shared_a() { return 2 * ShapeA<D, FP8>::QBYTES + ShapeA<D, FP8>::SLOTS * ShapeA<D, FP8>::SLOT + ShapeA<D, FP8>::RAWS * ShapeA<D, FP8>::RAW + sizeof(SharedA<D, FP8>); }

// Waits for `count` threads, of whole warps, at barrier `id`; whether any of them says so.  (The barrier is `.aligned` and has no limit: a warp's lanes
// come to it together, also out of a wait that each of them polls for itself.)
__device__ __forceinline__ bool any_of(int id, int count, bool mine) {
  __syncwarp();
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred.aligned q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"(mine ? 1u : 0u), "r"(id), "r"(count) : "memory");
  return r != 0;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <int D, bool FP8>
__global__ void __launch_bounds__(threads_a(FP8), 1) prefix_node_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ Args a) {
  after_previous();  // (the warps' kernel takes the SMs that this one leaves)
  using Z = ShapeA<D, FP8>;
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned char* qbuf = smem;                    // [tile][box][128 rows][128 B]
  unsigned char* ring = smem + 2 * Z::QBYTES;    // [slot][box][128 keys][128 B], K and V in turn
  unsigned char* raw = ring + Z::SLOTS * Z::SLOT;  // [slot][128 keys][D]
  SharedA<D, FP8>& sh = *reinterpret_cast<SharedA<D, FP8>*>(raw + Z::RAWS * Z::RAW);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_items = a.p.hdr[H_ITEMS_A] * a.d.n_kv_heads;
  const int workers = a.p.hdr[H_WORKERS_A];
  if (n_items == 0 || (int)blockIdx.x >= workers) return;  // (whole blocks)
  if (threadIdx.x == 0) {
    for (int s = 0; s < Z::SLOTS; ++s) { ptx::mbar_init(&sh.full[s], FP8 ? kWiden : 1); ptx::mbar_init(&sh.free[s], 1); }
    for (int s = 0; s < 4; ++s) { ptx::mbar_init(&sh.raw_full[s], 1); ptx::mbar_init(&sh.raw_free[s], kWiden); }
    ptx::mbar_init(&sh.q_full, kSoftWarps * 32);
    ptx::mbar_init(&sh.q_free, 1);
    for (int t = 0; t < 2; ++t) {
      ptx::mbar_init(&sh.s_full[t], 1);
      ptx::mbar_init(&sh.p_ready[t], kSoftWarps * 16);
      ptx::mbar_init(&sh.o_full[t], 1);
      ptx::mbar_init(&sh.item_full[t], 1);
      ptx::mbar_init(&sh.item_free[t], 1 + kSoftWarps + (FP8 ? kWidenWarps : 0));
    }
    ptx::mbar_init(&sh.drain, 1);
    ptx::mbar_fence_init();
  }
  if (warp == kMmaWarp) {
    ptx::tmem_alloc(&sh.tmem, 512);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = sh.tmem;
  auto tmem_s = [&](int t) { return tmem + (uint32_t)(t * 128); };
  auto tmem_o = [&](int t) { return tmem + (uint32_t)(256 + t * D); };
  bool ok = (ptx::smem_u32(smem) & 1023) == 0;
  const int G = a.group, members = tile_members(G);
  // The next item of the list into `it`.  Everybody but the loads takes items from there in the same order.
  auto take_item = [&](uint32_t n, int (&it)[8]) {
    wait(&sh.item_full[n & 1u], (n >> 1) & 1u, ok);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 8; ++i) it[i] = sh.item[n & 1u][i];
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive(&sh.item_free[n & 1u]);
  };

  if (warp == kLoadWarp) {
    // ---- pages; the warp stays together, lane 0 issues ----
    uint32_t loads = 0;
    constexpr int RING = FP8 ? 4 : Z::SLOTS;
    uint64_t *full = FP8 ? sh.raw_full : sh.full, *free = FP8 ? sh.raw_free : sh.free;
    auto wait_all = [&](uint64_t* bar, uint32_t parity) {
      wait(bar, parity, ok);
      ok = __all_sync(0xffffffffu, ok);
    };
    for (uint32_t n = 0;; ++n) {
      int id = blockIdx.x;  // (the counter hands out what is behind the first round)
      if (n > 0) {
        if (lane == 0) id = workers + atomicAdd(&a.p.hdr[H_NEXT_A], 1);
        id = __shfl_sync(0xffffffffu, id, 0);
      }
      const bool there = id < n_items;
      ItemA it{};
      if (there) it = a.p.items_a[id / a.d.n_kv_heads];
      const int head = id % a.d.n_kv_heads, seq = it.seq, p0 = it.p0, p1 = it.p1;
      wait_all(&sh.item_free[n & 1u], ((n >> 1) & 1u) ^ 1u);
      const int kind = ok && there ? it.tiles : 0;
      if (lane == 0) {
        int* to = sh.item[n & 1u];
        to[0] = kind; to[1] = head; to[2] = seq; to[3] = it.first; to[4] = it.count; to[5] = p0; to[6] = p1; to[7] = it.part;
        ptx::mbar_arrive(&sh.item_full[n & 1u]);
      }
      __syncwarp();
      if (kind == 0) break;
      // lanes hold the ids of 32 pages, and of the 32 behind them
      const int* table = table_of(a, seq);
      int ids = p0 + lane < p1 ? table[p0 + lane] : 0, more = 0;
      for (int pg = p0; pg < p1 && ok; pg += kBlockPages) {
        const int rel = pg - p0;
        if (n == 0 && rel == kBlockPages) wait_all(&sh.q_full, 0);  // (at the start all blocks load at once; q comes before what can wait)
        if (!ok) break;
        if ((rel & 31) == 0) {
          if (rel > 0) ids = more;
          more = pg + 32 + lane < p1 ? table[pg + 32 + lane] : 0;
        }
        const int pages = min(kBlockPages, p1 - pg);
        int row0[kBlockPages];
#pragma unroll
        for (int p = 0; p < kBlockPages; ++p) row0[p] = (__shfl_sync(0xffffffffu, ids, (rel & 31) + p) * a.d.n_kv_heads + head) * 32;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const uint32_t s = loads % RING;
          wait_all(&free[s], ((loads / RING) & 1u) ^ 1u);
          if (!ok) break;
          if (lane == 0) {
            const CUtensorMap* map = kv ? &vmap : &kmap;
            if constexpr (FP8) {
              ptx::mbar_expect_tx(&full[s], pages * 32 * D);
              for (int p = 0; p < pages; ++p) ptx::tma_load_3d(raw + s * Z::RAW + p * 4096, map, 0, row0[p], a.layer, &full[s]);
            } else {
              ptx::mbar_expect_tx(&full[s], pages * Z::BOXES * 4096);
              for (int x = 0; x < Z::BOXES; ++x)
                for (int p = 0; p < pages; ++p)
                  ptx::tma_load_3d(ring + s * Z::SLOT + x * kBlockKeys * 128 + p * 4096, map, x * 64, row0[p], a.layer, &full[s]);
            }
          }
          __syncwarp();
          ++loads;
        }
      }
    }
    if (!ok) {  // leave no copy in flight behind
      bool drained = true;
      for (uint32_t i = loads > (uint32_t)RING ? loads - RING : 0; i < loads; ++i) wait(&full[i % RING], (i / RING) & 1u, drained);
    }
  } else if (warp == kMmaWarp) {
    // ---- products ----
    if (ptx::elect_one()) {
      constexpr uint32_t kF16 = ~((1u << 7) | (1u << 10));  // both operands
      const uint32_t id_s = ptx::umma_idesc_bf16(kTileRows, kBlockKeys) & (FP8 ? kF16 : ~0u), id_o = (ptx::umma_idesc_bf16(kTileRows, D) | ptx::kUmmaBMn) & (FP8 ? kF16 : ~0u);
      const uint64_t q_desc = ptx::umma_desc_k_sw128(ptx::smem_u32(qbuf)), k_desc = ptx::umma_desc_k_sw128(ptx::smem_u32(ring));
      const uint64_t v_desc = ptx::umma_desc_mn_sw128(ptx::smem_u32(ring), kBlockKeys * 128);
      uint32_t n_p[2] = {0, 0}, n_q = 0, load0 = 0;  // softmaxes waited for; items; loads of the items before
      auto slot_of = [&](int k) { return (load0 + k) % Z::SLOTS; };  // K of the item's block j is its load 2 j, V 2 j + 1
      auto arrived = [&](int k) {
        wait(&sh.full[slot_of(k)], ((load0 + k) / Z::SLOTS) & 1u, ok);
        ptx::tc_fence_after_sync();
      };
      for (uint32_t n = 0;; ++n) {
        wait(&sh.item_full[n & 1u], (n >> 1) & 1u, ok);
        if (!ok) break;
        const int kind = sh.item[n & 1u][0], n_pages = sh.item[n & 1u][6] - sh.item[n & 1u][5];
        ptx::mbar_arrive(&sh.item_free[n & 1u]);
        if (kind == 0) break;
        const int nb = (n_pages + kBlockPages - 1) / kBlockPages;
        wait(&sh.q_full, n_q & 1u, ok);
        ++n_q;
        ptx::tc_fence_after_sync();
        auto qk = [&](int t, int j, int q_tile) {  // S of softmax group t from block j
          const uint64_t k0 = k_desc + (uint64_t)(slot_of(2 * j) * (Z::SLOT >> 4)), q0 = q_desc + (uint64_t)(q_tile * (Z::QBYTES >> 4));
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t at = (uint32_t)((k >> 2) * (kBlockKeys * 128 >> 4) + (k & 3) * 2);
            ptx::umma_bf16(tmem_s(t), q0 + at, k0 + at, id_s, k > 0 ? 1u : 0u);
          }
          ptx::umma_commit(&sh.s_full[t]);
        };
        auto pv = [&](int t, int j, bool first) {
          const uint64_t v0 = v_desc + (uint64_t)(slot_of(2 * j + 1) * (Z::SLOT >> 4));
          const int steps = min(kBlockPages, n_pages - j * kBlockPages) * 2;  // (what lies behind the last page is not read)
          wait(&sh.p_ready[t], n_p[t] & 1u, ok);
          ++n_p[t];
          ptx::tc_fence_after_sync();
          for (int k = 0; k < steps; ++k) ptx::umma_bf16_tmem_a(tmem_o(t), tmem_s(t) + (k >> 2) * 64 + (k & 3) * 8, v0 + k * (2048 >> 4), id_o, first && k == 0 ? 0u : 1u);
        };
        if (kind == 2) {
          arrived(0);
          qk(0, 0, 0);
          qk(1, 0, 1);
          ptx::umma_commit(&sh.free[slot_of(0)]);
          if (nb == 1) ptx::umma_commit(&sh.q_free);
          for (int j = 0; j < nb && ok; ++j) {
            const bool last = j + 1 == nb;
            arrived(2 * j + 1);
            pv(0, j, j == 0);
            if (last) {
              ptx::umma_commit(&sh.o_full[0]);
            } else {
              arrived(2 * j + 2);
              qk(0, j + 1, 0);
            }
            pv(1, j, j == 0);
            ptx::umma_commit(&sh.free[slot_of(2 * j + 1)]);
            if (last) {
              ptx::umma_commit(&sh.o_full[1]);
            } else {
              qk(1, j + 1, 1);
              ptx::umma_commit(&sh.free[slot_of(2 * j + 2)]);
              if (j + 2 == nb) ptx::umma_commit(&sh.q_free);
            }
          }
        } else {
          for (int j = 0; j < min(nb, 2); ++j) {
            arrived(2 * j);
            qk(j, j, 0);
            ptx::umma_commit(&sh.free[slot_of(2 * j)]);
            // (K of block 1 comes behind V of block 0 in the ring, and more slots than three follow before V's is used again)
          }
          if (nb <= 2) ptx::umma_commit(&sh.q_free);
          for (int j = 0; j < nb && ok; ++j) {
            const int t = j & 1;
            arrived(2 * j + 1);
            pv(t, j, j < 2);
            ptx::umma_commit(&sh.free[slot_of(2 * j + 1)]);
            if (j + 2 < nb) {
              arrived(2 * j + 4);
              qk(t, j + 2, 0);
              ptx::umma_commit(&sh.free[slot_of(2 * j + 4)]);
              if (j + 3 == nb) ptx::umma_commit(&sh.q_free);
            } else {
              ptx::umma_commit(&sh.o_full[t]);
            }
          }
        }
        load0 += 2 * nb;
      }
      const bool fine = ok;
      ok = true;
      ptx::umma_commit(&sh.drain);
      wait(&sh.drain, 0, ok);
      ok = ok && fine;
    }
    __syncwarp();
  } else if (warp < kSoftWarps) {
    // ---- the item's rows of q, then softmax: two threads per row ----
    const int g = warp >> 3, half = (warp >> 2) & 1, r = (warp & 3) * 32 + lane, m = r / G, head = r - m * G, pair = 1 + (warp >> 3) * 4 + (warp & 3);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    uint32_t n_s = 0, n_o = 0;
    for (uint32_t n = 0;; ++n) {
      int it[8];
      take_item(n, it);
      if (any_of(9 + g, 256, !ok)) { ok = false; break; }  // (a tile's threads meet at barriers that wait without limit, so they leave together)
      if (it[0] == 0) break;
      wait(&sh.q_free, (n & 1u) ^ 1u, ok);
      {
        constexpr int PIECES = D / 8;  // 16-byte pieces of a row
        constexpr int EACH = kTileRows * PIECES / 256;  // of a thread, all under way at once
        if (g < it[0]) {
          const int by_group = 65536 / a.group + 1;  // x * by_group >> 16 is x / G up to 127
          uint4 w[EACH];
          int row[EACH];
#pragma unroll
          for (int e = 0; e < EACH; ++e) {
            const int qr = ((threadIdx.x & 255) + e * 256) / PIECES, qm = qr * by_group >> 16, member = g * members + qm;
            row[e] = qm < members && member < it[4] ? a.p.members[it[3] + member].row : -1;
            if (row[e] >= a.rows) row[e] = -1;
          }
#pragma unroll
          for (int e = 0; e < EACH; ++e) {
            const int qr = ((threadIdx.x & 255) + e * 256) / PIECES, qh = qr - (qr * by_group >> 16) * G;
            const __nv_bfloat16* src = a.q + (size_t)max(row[e], 0) * a.q_stride + (size_t)(it[1] * G + qh) * D + (threadIdx.x % PIECES) * 8;
            w[e] = row[e] >= 0 ? *reinterpret_cast<const uint4*>(src) : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int e = 0; e < EACH; ++e) {
            const int c = threadIdx.x % PIECES, qr = ((threadIdx.x & 255) + e * 256) / PIECES;
            const uint32_t dst = ptx::smem_u32(qbuf + g * Z::QBYTES + (c >> 3) * (kTileRows * 128) + qr * 128 + (((c & 7) ^ (qr & 7)) << 4));
            uint32_t x[4] = {w[e].x, w[e].y, w[e].z, w[e].w};
            if constexpr (FP8) {
#pragma unroll
              for (int i = 0; i < 4; ++i) x[i] = pack_f16(ptx::bf16_lo(x[i]), ptx::bf16_hi(x[i]));
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]) : "memory");
          }
        }
      }
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(&sh.q_full);
      const bool alone = it[0] == 1;  // one tile of rows: the groups take the blocks in turn
      const int n_pages = it[6] - it[5], nb = (n_pages + kBlockPages - 1) / kBlockPages, member = (alone ? 0 : g * members) + m;
      const bool on = m < members && member < it[4];
      const int slot = on ? a.p.members[it[3] + member].slot + it[7] + (alone ? g : 0) : 0;
      const int j0 = alone ? g : 0, step = alone ? 2 : 1;
      float scale = kNoScale, l = 0.f;  // log2 units; the sum of this thread's keys
      float my_ks = 0.f, my_vs = 0.f, v_ref = 1.f;
      auto page_scales = [&](int page0) {  // lane i: the scales of page page0 + i of the item
        my_ks = my_vs = 0.f;
        if (page0 + lane < n_pages) {
          const size_t at = ((size_t)a.layer * a.d.n_pages + table_of(a, it[2])[it[5] + page0 + lane]) * a.d.n_kv_heads + it[1];
          my_ks = a.d.k_scale[at];
          my_vs = a.d.v_scale[at];
        }
      };
      if constexpr (FP8) {  // P is multiplied by a page's V scale over the item's largest
        v_ref = 0.f;
        for (int base = 0; base < n_pages; base += 32) { page_scales(base); v_ref = fmaxf(v_ref, my_vs); }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v_ref = fmaxf(v_ref, __shfl_xor_sync(0xffffffffu, v_ref, o));
      }
      const float v_inv = v_ref > 0.f ? 1.0f / v_ref : 0.f;
      const uint32_t t_s = tmem_s(g) + lanes, t_o = tmem_o(g) + lanes + half * (D / 2);
      for (int j = j0; j < nb; j += step) {
        const int pages = min(kBlockPages, n_pages - j * kBlockPages) - 2 * half;  // of this thread's two that there are
        float ks[2] = {a.scale_log2, a.scale_log2}, vs[2] = {1.f, 1.f};
        if constexpr (FP8) {
          const int rel = j * kBlockPages;
          if (j < j0 + step || (rel & 31) < kBlockPages * step) page_scales(rel & ~31);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            ks[c] = __shfl_sync(0xffffffffu, my_ks, (rel & 31) + 2 * half + c) * a.scale_log2;
            vs[c] = __shfl_sync(0xffffffffu, my_vs, (rel & 31) + 2 * half + c) * v_inv;
          }
        }
        wait(&sh.s_full[g], n_s & 1u, ok);
        ++n_s;
        ptx::tc_fence_after_sync();
        __syncwarp();
        uint32_t u[2][32];
#pragma unroll
        for (int c = 0; c < 2; ++c) ptx::tmem_ld32(t_s + half * 64 + c * 32, u[c]);
        ptx::tmem_ld_wait();
        if (pages < 2) {  // (columns behind the last page hold anything)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            if (c >= pages) {
              ks[c] = a.scale_log2;
#pragma unroll
              for (int i = 0; i < 32; ++i) u[c][i] = __float_as_uint(kHidden);
            }
        }
        float top = kHidden;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx[4] = {kHidden, kHidden, kHidden, kHidden};
#pragma unroll
          for (int i = 0; i < 32; ++i) mx[i & 3] = max_nan(mx[i & 3], __uint_as_float(u[c][i]));
          top = max_nan(top, max_nan(max_nan(mx[0], mx[1]), max_nan(mx[2], mx[3])) * ks[c]);
        }
        if (__any_sync(0xffffffffu, top != top)) {  // a score that is no number weighs nothing, as a hidden one does
          const bool none = top != top;
          top = none ? kHidden : top;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (none) {
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                // (on 8-bit pages behind the page's scale, which would make so little of kHidden that it is above kNoScale)
                const float x = fmaxf(FP8 ? __uint_as_float(u[c][i]) * ks[c] : __uint_as_float(u[c][i]), kHidden);
                u[c][i] = __float_as_uint(x);
                top = fmaxf(top, FP8 ? x : x * ks[c]);
              }
              if (FP8) ks[c] = 1.f;
            }
          }
          __syncwarp();
        }
        ptx::tc_fence_before_sync();
        if (any_of(pair, 64, top > scale + kLate)) {
          sh.exchange[g][half][r] = top;
          any_of(pair, 64, false);
          top = fmaxf(top, sh.exchange[g][half ^ 1][r]);
          const bool late = top > scale + kLate;
          const float corr = late ? ex2(scale - top) : 1.f;
          if (late) scale = top;
          l *= corr;
          ptx::tc_fence_after_sync();
          if (j != j0 && __any_sync(0xffffffffu, late)) {  // (the scores' arrival says that the product before them is done)
#pragma unroll 1
            for (int c = 0; c < D / 2; c += 16) {
              uint32_t w[16];
              ptx::tmem_ld16(t_o + c, w);
              ptx::tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(__uint_as_float(w[i]) * corr);
              ptx::tmem_st16(t_o + c, w);
            }
          }
        }
        ptx::tc_fence_after_sync();
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        const float2 m2 = make_float2(-scale, -scale);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t p[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float2 x = fma2(make_float2(__uint_as_float(u[c][2 * i]), __uint_as_float(u[c][2 * i + 1])), make_float2(ks[c], ks[c]), m2);
            const float2 e = make_float2(ex2(x.x), ex2(x.y));
            sum[i & 1] = add2(sum[i & 1], e);
            p[i] = FP8 ? pack_f16(e.x * vs[c], e.y * vs[c]) : pack_bf16(e.x, e.y);
          }
          ptx::tmem_st16(t_s + half * 64 + c * 16, p);  // (over scores of its own that are in registers)
        }
        const float2 both = add2(sum[0], sum[1]);
        l += both.x + both.y;
        ptx::tmem_st_wait();
        ptx::tc_fence_before_sync();
        ptx::mbar_arrive(&sh.p_ready[g]);
      }
      // ---- the row's part leaves, half of its columns from each thread ----
      if (j0 < nb) {
        wait(&sh.o_full[g], n_o & 1u, ok);
        sh.exchange[g][half][r] = l;  // (the sums are there, so all threads have read the last maxima)
        any_of(pair, 64, false);
        l += sh.exchange[g][half ^ 1][r];
        wait(&sh.q_free, n & 1u, ok);  // (all the item's scores have been computed: both groups' may come from the first tile)
        ++n_o;
        ptx::tc_fence_after_sync();
        __syncwarp();
        const int q_head = it[1] * G + head;
        if (on && half == 0) *reinterpret_cast<float2*>(a.p.part_ml + ((size_t)slot * a.n_q_heads + q_head) * 2) = make_float2(scale, l);
        // 16 columns of 32 rows at a time through the tile's place for q (its products are done), so that four lanes write 64 bytes of a row
        unsigned char* pass = qbuf + g * Z::QBYTES + (warp & 7) * 2048;
        const int row4 = lane >> 2, piece4 = lane & 3;
        int to_slot[4], to_head[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // of rows row4 + 8 i of this warp
          to_slot[i] = __shfl_sync(0xffffffffu, on ? slot : -1, row4 + 8 * i);
          to_head[i] = __shfl_sync(0xffffffffu, q_head, row4 + 8 * i);
        }
#pragma unroll
        for (int c = 0; c < D / 2; c += 16) {
          uint32_t w[16];
          ptx::tmem_ld16(t_o + c, w);
          ptx::tmem_ld_wait();
          if constexpr (FP8) {
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(__uint_as_float(w[i]) * v_ref);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(pass + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int from = row4 + 8 * i;
            const uint4 v = *reinterpret_cast<const uint4*>(pass + from * 64 + ((piece4 ^ ((from >> 1) & 3)) << 4));
            if (to_slot[i] >= 0) *reinterpret_cast<uint4*>(a.p.part_o + ((size_t)to_slot[i] * a.n_q_heads + to_head[i]) * D + half * (D / 2) + c + piece4 * 4) = v;
          }
          __syncwarp();
        }
        ptx::fence_proxy_async_smem();
        ptx::tc_fence_before_sync();
        any_of(9 + g, 256, false);  // (all of it has left before the next q takes its place)
      }
    }
  } else if constexpr (FP8) {
    // ---- operands from codes: two keys per thread ----
    const int me = threadIdx.x - (kMmaWarp + 1) * 32;
    uint32_t loads = 0;
    for (uint32_t n = 0;; ++n) {
      int it[8];
      take_item(n, it);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok || it[0] == 0) break;
      const int nb = (it[6] - it[5] + kBlockPages - 1) / kBlockPages;
      for (int k = 0; k < 2 * nb; ++k, ++loads) {
        const uint32_t from = loads % 4, to = loads % Z::SLOTS;
        wait(&sh.raw_full[from], (loads / 4) & 1u, ok);
        wait(&sh.free[to], ((loads / Z::SLOTS) & 1u) ^ 1u, ok);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
#pragma unroll
        for (int key = me; key < kBlockKeys; key += kWiden) {
          const unsigned char* src = raw + from * Z::RAW + key * 128;
          unsigned char* dst = ring + to * Z::SLOT + key * 128;
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            const uint4 w = *reinterpret_cast<const uint4*>(src + ((c ^ (key & 7)) << 4));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t lo = h ? w.z : w.x, hi = h ? w.w : w.y;
              const int cc = 2 * c + h;
              *reinterpret_cast<uint4*>(dst + (cc >> 3) * kBlockKeys * 128 + (((cc & 7) ^ (key & 7)) << 4)) =
                  make_uint4(e4m3x2_to_f16x2(lo), e4m3x2_to_f16x2(lo >> 16), e4m3x2_to_f16x2(hi), e4m3x2_to_f16x2(hi >> 16));
            }
          }
        }
        ptx::fence_proxy_async_smem();
        ptx::mbar_arrive(&sh.raw_free[from]);
        ptx::mbar_arrive(&sh.full[to]);
      }
    }
  }
  if (!ok) atomicExch(a.d.state + ST_ATTN_ERR, B200_ERR_DEVICE_FLAGGED);
  ptx::tc_fence_before_sync();
  __syncthreads();
  ptx::tc_fence_after_sync();
  if (warp == kMmaWarp) ptx::tmem_dealloc(tmem, 512);
}

// ---- the join: a warp per (row, query head) -----------------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(256) prefix_join_kernel(const __grid_constant__ Args a) {
  after_previous();
  const int u = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (blockIdx.x == 0 && threadIdx.x == 0) { a.p.hdr[H_NEXT_A] = 0; a.p.hdr[H_NEXT_B] = 0; }  // for the next layer
  const int row = u / a.n_q_heads, qh = u - row * a.n_q_heads;
  // (all on their way together; there is room for the places of a.rows rows whatever the plan)
  const int planned = a.p.hdr[H_ROWS], large = a.p.hdr[H_ITEMS_A], error = a.d.state[ST_ATTN_ERR], s0 = a.p.row_base[min(row, a.rows)], s1 = a.p.row_base[min(row + 1, a.rows)];
  if (!a.nodes && large > 0) {  // a plan of more rows than the launches are for
    if (blockIdx.x == 0 && threadIdx.x == 0) atomicExch(a.d.state + ST_ATTN_ERR, B200_ERR_INVALID_ARGUMENT);
    return;
  }
  if (row >= min(a.rows, planned) || error != 0) return;
  constexpr int V = D / 32;
  const float2* ml = reinterpret_cast<const float2*>(a.p.part_ml) + qh;
  const float* po = a.p.part_o + (size_t)qh * D + lane * V;
  float mm = kNoScale, ll = 0.f, acc[V] = {};
  for (int base = s0; base < s1; base += 32) {
    const int n = min(32, s1 - base);
    const float2 mine = lane < n ? ml[(size_t)(base + lane) * a.n_q_heads] : make_float2(kNoScale, 0.f);
    float top = mine.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float m_new = fmaxf(mm, top), corr = ex2(mm - m_new), w = lane < n ? ex2(mine.x - m_new) : 0.f;
    float l = lane < n ? mine.y * w : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    ll = ll * corr + l;
    mm = m_new;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] *= corr;
    for (int c = 0; c < n; c += 8) {
      float v[8][V];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float* src = po + (size_t)(base + min(c + i, n - 1)) * a.n_q_heads * D;
        if constexpr (V == 4) { const float4 f = *reinterpret_cast<const float4*>(src); v[i][0] = f.x; v[i][1] = f.y; v[i][2] = f.z; v[i][3] = f.w; }
        else { const float2 f = *reinterpret_cast<const float2*>(src); v[i][0] = f.x; v[i][1] = f.y; }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float wi = __shfl_sync(0xffffffffu, w, (c + i) & 31);
        if (c + i >= n) continue;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = fmaf(v[i][e], wi, acc[e]);
      }
    }
  }
  const float inv = 1.0f / ll;  // (a row without a key has ll = 0 and is written as zeros)
  uint32_t* dst = reinterpret_cast<uint32_t*>(a.out + (size_t)row * a.out_stride + (size_t)qh * D + lane * V);
#pragma unroll
  for (int e = 0; e < V; e += 2) dst[e / 2] = ll != 0.f ? pack_bf16(acc[e] * inv, acc[e + 1] * inv) : 0u;
}

}  // namespace

struct b200_prefix_attn {
  b200_kv* kv = nullptr;
  int max_rows = 0, rows = -1;
  void* buf = nullptr;  // everything below, one allocation
  PlanDev p;
};

namespace {

template <int D, bool FP8>
b200_status launch_layer(const b200_kv* kv, const Args& a, cudaStream_t s) {
  static bool configured = false;
  constexpr size_t shared_nodes = shared_a<D, FP8>();
  if (!configured) {
    B200_CUDA_TRY((cudaFuncSetAttribute(prefix_node_kernel<D, FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)shared_nodes)));
    B200_CUDA_TRY((cudaFuncSetAttribute(prefix_warp_kernel<D, FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ShapeB<D, FP8>::kShared)));
    configured = true;
  }
  if (a.nodes) {
    launch_after(prefix_node_kernel<D, FP8>, b200_sm_count(), threads_a(FP8), shared_nodes, s, kv->kmap, kv->vmap, a);
    B200_LAUNCH_CHECK();
  }
  launch_after(prefix_warp_kernel<D, FP8>, b200_sm_count(), ShapeB<D, FP8>::WARPS * 32, ShapeB<D, FP8>::kShared, s, kv->kmap, kv->vmap, a);
  B200_LAUNCH_CHECK();
  launch_after(prefix_join_kernel<D>, (a.rows * a.n_q_heads + 7) / 8, 256, 0, s, a);
  B200_LAUNCH_CHECK();
  return B200_OK;
}

}  // namespace

extern "C" b200_status b200_prefix_attn_create(b200_kv* kv, int32_t max_rows, b200_prefix_attn** out) {
  if (!out) { b200_set_error("prefix attention: no place for the handle"); return B200_ERR_INVALID_ARGUMENT; }
  *out = nullptr;
  if (!kv) { b200_set_error("prefix attention: no pool"); return B200_ERR_INVALID_ARGUMENT; }
  if (max_rows <= 0 || max_rows > kMaxRows) { b200_set_error("prefix attention: %d rows (at most %d)", max_rows, kMaxRows); return B200_ERR_INVALID_ARGUMENT; }
  const b200_kv_config& c = kv->cfg;
  if (kv->layered) { b200_set_error("prefix attention: layered pools are read by the decoder step's attention"); return B200_ERR_UNSUPPORTED; }
  const int group = c.n_q_heads / c.n_kv_heads;
  if (group > kWarpRows || (c.kv_dtype != B200_KV_BF16 && c.head_dim != 128)) {
    b200_set_error("prefix attention: %d query heads per kv head (at most %d); FP8 pages have head_dim 128", group, kWarpRows);
    return B200_ERR_UNSUPPORTED;
  }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  auto* h = new (std::nothrow) b200_prefix_attn();
  if (!h) { b200_set_error("prefix attention: out of host memory"); return B200_ERR_CAPACITY; }
  h->kv = kv; h->max_rows = max_rows;
  // A row has at most kLevels nodes of one or two parts, and its own pages; beyond that, room for the chunks of few rows.
  PlanDev& p = h->p;
  p.max_rows = max_rows;
  p.max_slots = (2 * kLevels + 1) * max_rows + 1024;
  size_t bytes = 0;
  auto place = [&](size_t n) { const size_t at = bytes; bytes += (n + 255) / 256 * 256; return at; };
  const size_t r = max_rows, slots = p.max_slots;
  const size_t hdr = place(sizeof(int) * H_COUNT), seq = place(4 * r), ctx = place(4 * r), base = place(4 * (r + 1));
  const size_t nodes = place(sizeof(Node) * (kLevels * r / 2 + 1)), members = place(sizeof(Member) * kLevels * r), of_node = place(4 * kLevels * r);
  const size_t items_a = place(sizeof(ItemA) * slots), items_b = place(sizeof(ItemB) * slots);
  const size_t part_o = place(sizeof(float) * slots * c.n_q_heads * c.head_dim), part_ml = place(sizeof(float) * 2 * slots * c.n_q_heads);
  cudaError_t e = cudaMalloc(&h->buf, bytes);
  if (e == cudaSuccess) e = cudaMemset(h->buf, 0, sizeof(int) * H_COUNT);
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  if (e != cudaSuccess) {
    b200_set_error("prefix attention: %zu bytes: %s", bytes, cudaGetErrorString(e));
    cudaGetLastError();
    b200_prefix_attn_destroy(h);
    return B200_ERR_CUDA;
  }
  char* b = (char*)h->buf;
  p.hdr = (int*)(b + hdr); p.row_seq = (int*)(b + seq); p.row_ctx = (int*)(b + ctx); p.row_base = (int*)(b + base);
  p.nodes = (Node*)(b + nodes); p.members = (Member*)(b + members); p.member_node = (int*)(b + of_node);
  p.items_a = (ItemA*)(b + items_a); p.items_b = (ItemB*)(b + items_b); p.part_o = (float*)(b + part_o); p.part_ml = (float*)(b + part_ml);
  *out = h;
  return B200_OK;
}

extern "C" void b200_prefix_attn_destroy(b200_prefix_attn* h) {
  if (!h) return;
  if (h->buf) cudaFree(h->buf);
  delete h;
}

extern "C" b200_status b200_prefix_attn_plan(b200_prefix_attn* h, const int32_t* d_row_seq, const int32_t* d_row_ctx, int32_t rows, void* stream) {
  if (!h || rows < 0 || (rows > 0 && (!d_row_seq || !d_row_ctx))) { b200_set_error("prefix attention: no handle, or no rows"); return B200_ERR_INVALID_ARGUMENT; }
  if (rows > h->max_rows) { b200_set_error("prefix attention: %d rows, the handle holds %d", rows, h->max_rows); return B200_ERR_CAPACITY; }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  h->rows = rows;
  if (rows == 0) {  // (for layers in a graph: none of their rows are there)
    B200_CUDA_TRY(cudaMemsetAsync(h->p.hdr, 0, sizeof(int) * H_COUNT, (cudaStream_t)stream));
    return B200_OK;
  }
  int hash = 64;
  while (hash < rows || (hash < 2 * rows && hash < 4096)) hash *= 2;
  const size_t shared = (size_t)hash * (8 + 4 * 4) + (size_t)rows * 4 * 6;
  static bool configured = false;
  if (!configured) {
    B200_CUDA_TRY(cudaFuncSetAttribute(prefix_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 4096 * 24 + kMaxRows * 24));
    configured = true;
  }
  const b200_kv_config& c = h->kv->cfg;
  const bool fp8 = c.kv_dtype != B200_KV_BF16;
  const int warps = fp8 ? ShapeB<128, true>::WARPS : c.head_dim == 128 ? ShapeB<128, false>::WARPS : ShapeB<64, false>::WARPS;
  launch_after(prefix_plan_kernel, 1, rows <= 256 ? 256 : 1024, shared, (cudaStream_t)stream, h->kv->dev, h->p, d_row_seq, d_row_ctx, rows, hash,
               c.n_q_heads / c.n_kv_heads, b200_sm_count(), b200_sm_count() * warps, fp8 ? 1.15f : c.head_dim == 128 ? 0.75f : 0.4f);
  B200_LAUNCH_CHECK();
  return B200_OK;
}

extern "C" b200_status b200_prefix_attn_run(b200_prefix_attn* h, int32_t layer, const void* d_q, int32_t q_stride, void* d_out, int32_t out_stride, void* stream) {
  if (!h) { b200_set_error("prefix attention: no handle"); return B200_ERR_INVALID_ARGUMENT; }
  const b200_kv* kv = h->kv;
  const b200_kv_config& c = kv->cfg;
  if (h->rows < 0) { b200_set_error("prefix attention: the handle has no plan"); return B200_ERR_INVALID_ARGUMENT; }
  if (layer < 0 || layer >= c.n_layers) { b200_set_error("prefix attention: layer %d out of range", layer); return B200_ERR_INVALID_ARGUMENT; }
  const int width = c.n_q_heads * c.head_dim;
  auto fits = [&](const void* p, int stride) { return p && ((uintptr_t)p & 15) == 0 && stride % 8 == 0 && stride >= width; };
  if (h->rows > 0 && (!fits(d_q, q_stride) || !fits(d_out, out_stride))) {
    b200_set_error("prefix attention: rows start on 16 bytes, strides are multiples of 8 elements and hold all heads");
    return B200_ERR_INVALID_ARGUMENT;
  }
  b200_status st = b200_require_device();
  if (st != B200_OK) return st;
  if (h->rows == 0) return B200_OK;
  Args a;
  a.d = kv->dev; a.p = h->p; a.layer = layer; a.rows = h->rows; a.n_q_heads = c.n_q_heads; a.group = c.n_q_heads / c.n_kv_heads;
  a.nodes = is_large(h->rows, a.group);  // (else no node is: the least rows take one launch less)
  a.q = (const __nv_bfloat16*)d_q; a.q_stride = q_stride; a.out = (__nv_bfloat16*)d_out; a.out_stride = out_stride;
  a.scale_log2 = 1.4426950408889634f / sqrtf((float)c.head_dim);
  cudaStream_t s = (cudaStream_t)stream;
  if (c.kv_dtype != B200_KV_BF16) return launch_layer<128, true>(kv, a, s);
  return c.head_dim == 128 ? launch_layer<128, false>(kv, a, s) : launch_layer<64, false>(kv, a, s);
}
