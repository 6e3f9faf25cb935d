// Pages of the paged KV cache on gfx950: copied, forked, grown, freed and compacted. The state is
// on the device -- block tables, sequence lengths and one reference count per block (0: free) --
// so a captured decode loop can share and move pages without asking the host. It has the roles
// of the reference's BlockManager (src/engine/block_manager.py:75-246: ref counts of shared
// blocks, allocation for new tokens, release when the last holder goes), whose host lists the
// C++ host core keeps for callers that schedule there.
//
// Blocks are given out lowest number first, in the order of the call's list, so results do not
// depend on the order in which work-groups run; counts change by integer atomics, whose order
// does not show.
#include <algorithm>

#include "common.h"

namespace pk {
namespace {

// ---------------------------------------------------------------- copying ---------------

constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;
constexpr int kCopyVecs = kCopyThreads * kCopyUnroll;  // 16-byte vectors of one piece (16 KiB)
constexpr int kCopyGroups = 2048;                      // work-groups of a copy launch at most (8 per CU)

// Which pages to copy: a pair's source, target and tokens, from the caller's lists or a plan.
struct CopyList {
  const int32_t* src;
  const int32_t* dst;
  const int32_t* tokens;     // nullptr: whole pages
  const int4* heads;         // forks: (src, tokens, first target in dst, -) of every run of targets; the entry
                             // after the last one has their end
  const int32_t* num_pairs;  // on the device (forks, compaction), or nullptr: max_pairs
  int32_t max_pairs;
};

// Pieces of 16 KiB of one page of one layer's K or V, dealt to the work-groups round robin, all
// loads of a piece before its stores; a fork's piece is read once for all targets in a row that
// want it. A copy is bound by HBM: each byte is read once and written once, past the caches. Measured,
// us with non-temporal loads and stores, stores alone, neither: 16 pages of 512 KiB in 28 layers 180,
// 185, 189 (0.94 GB moved); 128 forks of 16 parents, whose pages are the next read, 168, 149, 172.
template <bool kHeads>
__device__ __forceinline__ void copy_pages(const PageCaches& c, const CopyList& list, int32_t group,
                                           int32_t groups) {
  const int32_t pairs = list.num_pairs ? min(*list.num_pairs, list.max_pairs) : list.max_pairs;
  const int32_t pieces = (c.block_size * c.row_vec + kCopyVecs - 1) / kCopyVecs;
  const int32_t per_pair = c.layers * 2 * pieces;
  const int32_t total = pairs * per_pair;  // below kCopyMaxPieces (checked on the host)
  for (int32_t u = group; u < total; u += groups) {
    const int32_t i = u / per_pair;
    int32_t rem = u - i * per_pair;
    const int32_t layer = rem / (2 * pieces);
    rem -= layer * 2 * pieces;
    const bool is_v = rem >= pieces;
    const int32_t piece = is_v ? rem - pieces : rem;
    int32_t src, tokens = c.block_size, first = i, last = i + 1;
    if constexpr (kHeads) {
      const int4 head = list.heads[i];
      src = head.x;
      tokens = head.y;
      first = head.z;
      last = list.heads[i + 1].z;
    } else {
      src = list.src[i];
      if (list.tokens) tokens = min(list.tokens[i], c.block_size);
    }
    const int32_t n = tokens * c.row_vec;
    const int32_t base = piece * kCopyVecs + (int32_t)threadIdx.x;
    if (src < 0 || src >= c.num_blocks || piece * kCopyVecs >= n) continue;
    u32x4* cache = reinterpret_cast<u32x4*>(is_v ? c.v : c.k) + layer * (is_v ? c.v_layer_vec : c.k_layer_vec);
    const int64_t block_vec = is_v ? c.v_block_vec : c.k_block_vec;
    const u32x4* from = cache + src * block_vec;
    u32x4 v[kCopyUnroll];
#pragma unroll
    for (int j = 0; j < kCopyUnroll; ++j)
      if (base + j * kCopyThreads < n)
        v[j] = kHeads ? from[base + j * kCopyThreads] : __builtin_nontemporal_load(from + base + j * kCopyThreads);
    for (int32_t t = first; t < last; ++t) {
      const int32_t dst = list.dst[t];
      if (dst < 0 || dst >= c.num_blocks || src == dst) continue;
      u32x4* to = cache + dst * block_vec;
#pragma unroll
      for (int j = 0; j < kCopyUnroll; ++j)
        if (base + j * kCopyThreads < n) __builtin_nontemporal_store(v[j], to + base + j * kCopyThreads);
    }
  }
}

__global__ __launch_bounds__(kCopyThreads) void copy_pages_kernel(const PageCaches c, const CopyList list) {
  copy_pages<false>(c, list, blockIdx.x, gridDim.x);
}

int32_t copy_groups(const PageCaches& c, int64_t pairs) {
  return (int32_t)std::min<int64_t>(copy_pieces(c, pairs), kCopyGroups);
}

// ---------------------------------------------------------------- allocation ------------

constexpr int kPoolThreads = 1024;  // one work-group decides who gets which block
constexpr int kPoolWaves = kPoolThreads / kWave;

// Exclusive prefix sum over the work-group's threads, and the total; `part` has kPoolWaves
// entries. Every thread of the work-group has to call it.
__device__ __forceinline__ int32_t pool_scan(int32_t v, int32_t* part, int32_t* total) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  int32_t incl = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int32_t o = __shfl_up(incl, d, kWave);
    if (lane >= d) incl += o;
  }
  __syncthreads();  // the previous call's sums have been read
  if (lane == kWave - 1) part[wave] = incl;
  __syncthreads();
  int32_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPoolWaves; ++w) {
    const int32_t p = part[w];
    if (w < wave) before += p;
    all += p;
  }
  *total = all;
  return before + incl - v;
}

// The block of the nth (0-based) free entry of ref_counts for every thread that needs one, -1 if
// the pool has fewer: free blocks are listed in LDS, lowest first, until `want` are found.
__device__ __forceinline__ int32_t pool_take(const int32_t* ref_counts, int32_t num_blocks, bool need, int32_t nth,
                                             int32_t want, int32_t* part, int32_t* found) {
  int32_t have = 0;
  for (int32_t base = 0; base < num_blocks && have < want; base += 4 * kPoolThreads) {
    const int32_t b = base + 4 * (int32_t)threadIdx.x;
    bool is_free[4];
    int32_t n = 0, sum;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      is_free[j] = b + j < num_blocks && ref_counts[min(b + j, num_blocks - 1)] == 0;
      n += is_free[j];
    }
    int32_t at = have + pool_scan(n, part, &sum);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (is_free[j] && at < kPoolThreads) found[at++] = b + j;
    have += sum;
  }
  __syncthreads();
  return need && nth < min(have, kPoolThreads) ? found[nth] : -1;
}

// Whether entry i of the list (n entries in LDS, 16-byte aligned) names a row that an earlier entry
// names too: every thread reads the same four entries at a time, none waits for a comparison.
__device__ __forceinline__ bool listed_before(const int32_t* rows, int32_t n, int32_t i, int32_t row) {
  bool found = false;
  if (i / kWave * kWave >= n) return found;  // no entry in this wavefront
#pragma unroll 4
  for (int32_t j = 0; j < n; j += 4) {
    const int4 r = *reinterpret_cast<const int4*>(rows + j);
    found |= (r.x == row && j < i) | (r.y == row && j + 1 < i) | (r.z == row && j + 2 < i) | (r.w == row && j + 3 < i);
  }
  return found;
}

// What a fork leaves for the launch that applies it.
struct ForkPlan {
  int4* heads;       // runs of children in a row that copy the same tokens (CopyList::heads), and the end
  int32_t* targets;  // their new blocks
  int32_t* blocks;   // of every child: its new block, or -1
  int32_t* lens;     // of every child: its length, -1: it stays as it was
  int32_t* runs;     // number of runs
};

ForkPlan fork_plan(void* ws, int32_t n) {
  ForkPlan f;
  f.heads = static_cast<int4*>(ws);
  f.targets = reinterpret_cast<int32_t*>(f.heads + n + 1);
  f.blocks = f.targets + n;
  f.lens = f.blocks + n;
  f.runs = f.lens + n;
  return f;
}

// Who gets which block in a fork: a chain of dependent loads and prefix sums, 5.2 us for 4 forks and 7.0
// for 128. The children's lengths and the new blocks' counts are written
// here, tables and shared counts by the launch that copies.
__global__ __launch_bounds__(kPoolThreads) void fork_plan_kernel(const PageTables t, const int32_t* parents,
                                                                 const int32_t* children, int32_t n,
                                                                 int32_t* new_blocks, const ForkPlan f) {
  __shared__ __attribute__((aligned(16))) int32_t rows[kPoolThreads];
  __shared__ int32_t found[kPoolThreads], part[kPoolWaves];
  const int32_t i = threadIdx.x;
  int32_t parent = -1, child = -1, length = 0;
  if (i < n) {
    parent = parents[i];
    child = children[i];
    if (parent >= 0 && parent < t.rows) length = max(min(t.lens[parent], t.max_len), 0);
  }
  rows[i] = child;
  __syncthreads();
  const bool listed = listed_before(rows, n, i, child);
  const bool ok = i < n && child >= 0 && child < t.rows && t.lens[child] == 0 && !listed;
  const int32_t full = length / t.block_size, tail = length - full * t.block_size;
  const bool need = ok && tail > 0;
  const int32_t src = need ? t.tables[parent * t.stride + full] : -1;
  int32_t want;
  const int32_t nth = pool_scan(need, part, &want);
  // (pool_take's barriers order every read of the lengths before the writes below)
  const int32_t block = pool_take(t.ref_counts, t.num_blocks, need, nth, want, part, found);
  const bool done = ok && (!need || block >= 0), copies = need && done;
  // The copies, in order (blocks run out for the last ones, so nth counts those that got one),
  // and the runs of one source and length among them.
  __syncthreads();  // `found` has been read
  rows[i] = copies ? src : -2;
  found[i] = tail;
  __syncthreads();
  const bool head = copies && (i == 0 || rows[i - 1] != src || found[i - 1] != tail);
  int32_t runs, copied;
  const int32_t run = pool_scan(head, part, &runs);
  pool_scan(copies, part, &copied);
  if (i == 0) {
    *f.runs = runs;
    f.heads[runs] = make_int4(-1, 0, copied, 0);
  }
  if (i >= n) return;
  new_blocks[i] = !ok ? -3 : !need ? -1 : block >= 0 ? block : -2;
  f.blocks[i] = copies ? block : -1;
  f.lens[i] = done ? length : -1;
  if (head) f.heads[run] = make_int4(src, tail, nth, 0);
  if (copies) {
    f.targets[nth] = block;
    t.ref_counts[block] = 1;
  }
  if (done) t.lens[child] = length;
}

// Work-groups [0, n): child i's table row, and one more holder for the pages it shares. The
// others copy the new pages' tokens.
__global__ __launch_bounds__(kCopyThreads) void fork_apply_kernel(const PageTables t, const PageCaches c,
                                                                  const int32_t* parents, const int32_t* children,
                                                                  int32_t n, const ForkPlan f) {
  if ((int32_t)blockIdx.x >= n) {
    copy_pages<true>(c, CopyList{nullptr, f.targets, nullptr, f.heads, f.runs, n}, blockIdx.x - n, gridDim.x - n);
    return;
  }
  const int32_t i = blockIdx.x;
  const int32_t length = f.lens[i];
  if (length < 0) return;
  const int32_t full = length / t.block_size;
  const int32_t* from = t.tables + parents[i] * t.stride;  // read only where full > 0: the parent is a row then
  int32_t* to = t.tables + children[i] * t.stride;
  for (int32_t j = threadIdx.x; j < t.width; j += kCopyThreads) {
    int32_t b = -1;
    if (j < full) {
      b = from[j];
      if (b >= 0 && b < t.num_blocks) atomicAdd(t.ref_counts + b, 1);
    } else if (j == full) {
      b = f.blocks[i];
    }
    to[j] = b;
  }
}

// One more token for every listed sequence: its slot, a new block where it starts one. -1 and
// nothing changed where the row is no row, is listed before, its table is full or the pool empty.
__global__ __launch_bounds__(kPoolThreads) void extend_kernel(const PageTables t, const int32_t* list, int32_t n,
                                                              int32_t* slots) {
  __shared__ __attribute__((aligned(16))) int32_t rows[kPoolThreads];
  __shared__ int32_t found[kPoolThreads], part[kPoolWaves];
  const int32_t i = threadIdx.x;
  int32_t row = -1;
  if (i < n) row = list[i];
  rows[i] = row;
  __syncthreads();
  int32_t length = -1;
  const bool listed = listed_before(rows, n, i, row);
  if (row >= 0 && row < t.rows && !listed) length = t.lens[row];
  const bool ok = length >= 0 && length < t.max_len;
  const int32_t page = ok ? length / t.block_size : 0, off = ok ? length - page * t.block_size : 0;
  const bool need = ok && off == 0;
  int32_t block = ok && !need ? t.tables[row * t.stride + page] : -1;
  int32_t want;
  const int32_t nth = pool_scan(need, part, &want);
  const int32_t got = pool_take(t.ref_counts, t.num_blocks, need, nth, want, part, found);
  if (need) block = got;
  if (i >= n) return;
  const bool done = ok && block >= 0 && block < t.num_blocks;
  slots[i] = done ? block * t.block_size + off : -1;
  if (!done) return;
  t.lens[row] = length + 1;
  if (need) {
    t.tables[row * t.stride + page] = block;
    t.ref_counts[block] = 1;
  }
}

// One wavefront per listed row. The exchange makes a row that is listed twice free its pages once.
__global__ __launch_bounds__(kWave) void free_kernel(const PageTables t, const int32_t* list) {
  const int32_t row = list[blockIdx.x];
  if (row < 0 || row >= t.rows) return;
  int32_t length = 0;
  if (threadIdx.x == 0) length = atomicExch(t.lens + row, 0);
  length = min(__builtin_amdgcn_readfirstlane(length), t.max_len);
  const int32_t pages = length <= 0 ? 0 : (length - 1) / t.block_size + 1;
  int32_t* table = t.tables + row * t.stride;
  for (int32_t j = threadIdx.x; j < pages; j += kWave) {
    const int32_t b = table[j];
    table[j] = -1;
    if (b >= 0 && b < t.num_blocks) atomicSub(t.ref_counts + b, 1);
  }
}

// ---------------------------------------------------------------- compaction ------------

// The kth live block at or past num_live moves to the kth free block before it: the fewest moves
// that make the live blocks the first ones, and no block is both read and written. One
// work-group: count the live blocks, list both sides in order, move the counts. 160 blocks 4.7 us.
__global__ __launch_bounds__(kPoolThreads) void compact_plan_kernel(int32_t* ref_counts, int32_t num_blocks,
                                                                    int32_t* block_map, int32_t* num_live,
                                                                    int32_t* src, int32_t* dst, int32_t* moves) {
  __shared__ int32_t part[kPoolWaves];
  int32_t n = 0, live;
  for (int32_t b = threadIdx.x; b < num_blocks; b += kPoolThreads) n += ref_counts[b] > 0;
  pool_scan(n, part, &live);
  int32_t holes = 0, movers = 0;
  for (int32_t base = 0; base < num_blocks; base += 4 * kPoolThreads) {
    const int32_t b = base + 4 * (int32_t)threadIdx.x;
    bool is_live[4];
    int32_t nh = 0, nm = 0, sh, sm;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      is_live[j] = b + j < num_blocks && ref_counts[min(b + j, num_blocks - 1)] > 0;
      if (b + j < num_blocks) {
        nh += !is_live[j] && b + j < live;
        nm += is_live[j] && b + j >= live;
        block_map[b + j] = is_live[j] ? b + j : -1;
      }
    }
    int32_t h = holes + pool_scan(nh, part, &sh);
    int32_t m = movers + pool_scan(nm, part, &sm);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (b + j < num_blocks) {
        if (!is_live[j] && b + j < live) dst[h++] = b + j;
        if (is_live[j] && b + j >= live) src[m++] = b + j;
      }
    }
    holes += sh;
    movers += sm;
  }
  __syncthreads();  // the lists, and the map's identity, before the moves
  for (int32_t k = threadIdx.x; k < movers; k += kPoolThreads) {
    const int32_t s = src[k], d = dst[k];
    block_map[s] = d;
    ref_counts[d] = ref_counts[s];
    ref_counts[s] = 0;
  }
  if (threadIdx.x == 0) {
    *num_live = live;
    *moves = movers;
  }
}

// Work-groups [0, table_groups): the tables' entries of the pages in use, renamed. The others copy.
__global__ __launch_bounds__(kCopyThreads) void compact_apply_kernel(const PageTables t, const PageCaches c,
                                                                     const int32_t* block_map, const CopyList list,
                                                                     int32_t table_groups) {
  if ((int32_t)blockIdx.x >= table_groups) {
    copy_pages<false>(c, list, blockIdx.x - table_groups, gridDim.x - table_groups);
    return;
  }
  const int64_t total = (int64_t)t.rows * t.width;
  for (int64_t e = blockIdx.x * (int64_t)kCopyThreads + threadIdx.x; e < total;
       e += (int64_t)table_groups * kCopyThreads) {
    const int64_t row = e / t.width;
    const int32_t j = (int32_t)(e - row * t.width);
    const int32_t length = min(t.lens[row], t.max_len);
    if (length <= 0 || j > (length - 1) / t.block_size) continue;
    const int32_t b = t.tables[row * t.stride + j];
    if (b < 0 || b >= t.num_blocks) continue;
    const int32_t to = block_map[b];
    if (to >= 0 && to != b) t.tables[row * t.stride + j] = to;
  }
}

}  // namespace

int64_t copy_pieces(const PageCaches& c, int64_t pairs) {
  return pairs * c.layers * 2 * (((int64_t)c.block_size * c.row_vec + kCopyVecs - 1) / kCopyVecs);
}

hipError_t launch_copy_blocks(const PageCaches& c, const int32_t* src, const int32_t* dst, const int32_t* tokens,
                              int32_t num_pairs, hipStream_t stream) {
  const int32_t groups = copy_groups(c, num_pairs);
  if (groups <= 0) return hipSuccess;
  hipLaunchKernelGGL(copy_pages_kernel, dim3(groups), dim3(kCopyThreads), 0, stream, c,
                     CopyList{src, dst, tokens, nullptr, nullptr, num_pairs});
  return hipGetLastError();
}

size_t fork_workspace_bytes(int32_t n) {
  return n <= 0 ? 0 : (size_t)(n + 1) * sizeof(int4) + (size_t)(3 * n + 1) * sizeof(int32_t);
}

hipError_t launch_fork_sequences(const PageTables& t, const PageCaches& c, const int32_t* parents,
                                 const int32_t* children, int32_t n, int32_t* new_blocks, void* workspace,
                                 hipStream_t stream) {
  const ForkPlan f = fork_plan(workspace, n);
  hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kPoolThreads), 0, stream, t, parents, children, n, new_blocks,
                     f);
  if (hipError_t err = hipGetLastError(); err != hipSuccess) return err;
  hipLaunchKernelGGL(fork_apply_kernel, dim3(n + copy_groups(c, n)), dim3(kCopyThreads), 0, stream, t, c, parents,
                     children, n, f);
  return hipGetLastError();
}

hipError_t launch_extend_sequences(const PageTables& t, const int32_t* rows, int32_t n, int32_t* slots,
                                   hipStream_t stream) {
  hipLaunchKernelGGL(extend_kernel, dim3(1), dim3(kPoolThreads), 0, stream, t, rows, n, slots);
  return hipGetLastError();
}

hipError_t launch_free_sequences(const PageTables& t, const int32_t* rows, int32_t n, hipStream_t stream) {
  hipLaunchKernelGGL(free_kernel, dim3(n), dim3(kWave), 0, stream, t, rows);
  return hipGetLastError();
}

size_t compact_workspace_bytes(int32_t num_blocks) {  // both sides of the moves, and their number
  return num_blocks <= 0 ? 0 : ((size_t)2 * num_blocks + 4) * sizeof(int32_t);
}

hipError_t launch_compact_blocks(const PageTables& t, const PageCaches& c, int32_t* block_map, int32_t* num_live,
                                 void* workspace, hipStream_t stream) {
  int32_t* moves = static_cast<int32_t*>(workspace);
  int32_t *src = moves + 4, *dst = src + t.num_blocks;
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPoolThreads), 0, stream, t.ref_counts, t.num_blocks,
                     block_map, num_live, src, dst, moves);
  if (hipError_t err = hipGetLastError(); err != hipSuccess) return err;
  const int64_t entries = (int64_t)t.rows * t.width;
  const int32_t table_groups = (int32_t)std::min<int64_t>((entries + kCopyThreads - 1) / kCopyThreads, 1024);
  const int32_t groups = copy_groups(c, t.num_blocks / 2);  // every other block may move, not more
  if (table_groups + groups == 0) return hipSuccess;
  hipLaunchKernelGGL(compact_apply_kernel, dim3(table_groups + groups), dim3(kCopyThreads), 0, stream, t, c,
                     block_map, CopyList{src, dst, nullptr, nullptr, moves, t.num_blocks}, table_groups);
  return hipGetLastError();
}

}  // namespace pk
