// Low-rank adapters of many requests beside a shared projection, on gfx950: every token row m has
// an adapter a = adapter_ids[m] of its own (outside [0, num_adapters): none),
//   t[m, i]   = scale[a] * sum_k x[m, k] A[a, i, k]                          (shrink)
//   out[m, c] = bf16(base[m, c] + sum_j t[m, q rank + j] B[a, c, j])         (expand)
// where q is the slice (merged projection) of output column c and base is x W^T, whose sums are
// computed next to the shrink (lora_linear, at most 128 rows), or given (lora_add). The reference
// has no adapters; the projections are those of linear.hip.
//
// The work is reading: W or base once, out once, and the adapters in use once each; the products
// are 16-64 wide and free next to that. So rows are brought together by adapter, and a group of
// up to 16 or 64 rows of ONE adapter is an MFMA tile that reads A and B once for all of them:
//   * up to kLoraSmallRows rows: the groups are the equal ids within 16 consecutive rows. Nothing is
//     sorted: the work-group of a row that is not the first of its group has nothing to do.
//   * more: one work-group sorts the rows by adapter (counts, offsets, positions) and lists the
//     tiles of 64.
// Every row's sums are taken in the same order whatever shares its tile, so a row's result does
// not depend on the other rows of the batch beyond the choice between the two forms.
//
// t is kept in fp32. For the expand it is split into two bf16, t = hi + lo with a remainder
// below 2^-16 |t|, and both halves are multiplied (the products with bf16 B are exact in the
// fp32 sum), so t costs no rounding of the output's size. The output is rounded once.
//
// MFMA: v_mfma_f32_16x16x32_bf16, D[i][j] = sum_k A[i][k] B[k][j]; lane (r = lane & 15, h = lane
// >> 4) supplies row r of both operands at k = 8 h .. 8 h + 7 and holds D[4 h .. 4 h + 3][r]. The
// token rows are the second operand, so a lane's four values are neighbours in one row of t
// or out.
#include "linear_core.h"

namespace pk {
namespace {

constexpr int kLoraThreads = 256;
constexpr int kLoraWaves = kLoraThreads / kWave;
constexpr int kLoraTile = 64;        // rows of a sorted tile
constexpr int kLoraSmallTile = 16;   // rows of a tile that is not sorted
constexpr int kPlanThreads = 1024;

__device__ __forceinline__ f32x4 mfma16(const u32x4 a, const u32x4 b, const f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}

// The adapter of a row, -1 for none.
__device__ __forceinline__ int32_t adapter_of(const LoraArgs& p, int32_t row) {
  const int32_t id = p.ids[row];
  return id >= 0 && id < p.num_adapters ? id : -1;
}

// A tile: its adapter, and each of its R rows' index in x (-1: not a row of the tile), in LDS.
// Not sorted: the rows of [16 tile, 16 tile + 16) with the adapter of row `slot`; false if an
// earlier row has that adapter. Every thread of the work-group calls it.
__device__ __forceinline__ bool small_tile(const LoraArgs& p, int32_t slot, int32_t* rows, int32_t* id) {
  const int lane = threadIdx.x & (kWave - 1);
  const int32_t row = (slot & ~(kLoraSmallTile - 1)) + lane;
  const bool is_row = lane < kLoraSmallTile && row < p.rows;
  const int32_t mine = is_row ? adapter_of(p, row) : -2;
  const int j = slot & (kLoraSmallTile - 1);
  *id = __builtin_amdgcn_readlane(mine, j);
  const uint64_t group = __ballot(mine == *id);
  if (__builtin_ctzll(group) != j) return false;
  if (threadIdx.x < kLoraSmallTile) rows[threadIdx.x] = mine == *id ? row : -1;
  __syncthreads();
  return true;
}

__device__ __forceinline__ bool sorted_tile(const LoraArgs& p, int32_t tile, int32_t* rows, int32_t* id) {
  if (tile >= *p.num_tiles) return false;
  const int4 t = p.tiles[tile];  // adapter, first position, rows
  *id = t.x;
  if (threadIdx.x < kLoraTile) rows[threadIdx.x] = (int)threadIdx.x < t.z ? p.perm[t.y + threadIdx.x] : -1;
  __syncthreads();
  return true;
}

// ---------------------------------------------------------------- shrink ----------------

constexpr int shrink_smem_bytes(int r, int cb) { return kLoraWaves * r * (cb * 16 + 4) * 4; }

// t of R rows of one adapter at its columns [c0, c0 + 16 CB). The four wavefronts take the k range
// in turns of 64 (128 contiguous bytes of every row), U turns' loads before their products,
// and add up in LDS.
template <int R, int CB, int U>
__device__ __forceinline__ void shrink_tile(const LoraArgs& p, const int32_t id, const int32_t c0, const int32_t* rows,
                                            char* smem) {
  constexpr int kSubs = R / 16, kStride = CB * 16 + 4;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int r = lane & 15, h = lane >> 4;
  const int32_t width = p.num_slices * p.rank;
  const uint16_t *xr[kSubs], *ar[CB];
#pragma unroll
  for (int s = 0; s < kSubs; ++s) {
    const int32_t row = rows[16 * s + r];
    xr[s] = p.x + (int64_t)max(row, 0) * p.x_stride;  // (what the missing rows give is not stored)
  }
#pragma unroll
  for (int c = 0; c < CB; ++c)
    ar[c] = p.a + id * p.a_adapter + (int64_t)min(c0 + 16 * c + r, width - 1) * p.a_row;
  f32x4 acc[kSubs][CB];
#pragma unroll
  for (int s = 0; s < kSubs; ++s)
#pragma unroll
    for (int c = 0; c < CB; ++c) acc[s][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int kTurn = kLoraWaves * 64;
  for (int32_t k0 = wave * 64; k0 < p.k; k0 += U * kTurn) {
    u32x4 xv[2 * U][kSubs], av[2 * U][CB];
#pragma unroll
    for (int u = 0; u < 2 * U; ++u) {
      const int32_t kp = k0 + (u >> 1) * kTurn + (u & 1) * 32 + 8 * h;
      const bool in = kp < p.k;  // k is a multiple of 8
      const int32_t at = in ? kp : 0;
      const u32x4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int s = 0; s < kSubs; ++s) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(xr[s] + at);
        xv[u][s] = in ? v : zero;
      }
#pragma unroll
      for (int c = 0; c < CB; ++c) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(ar[c] + at);
        av[u][c] = in ? v : zero;
      }
    }
#pragma unroll
    for (int u = 0; u < 2 * U; ++u)
#pragma unroll
      for (int s = 0; s < kSubs; ++s)
#pragma unroll
        for (int c = 0; c < CB; ++c) acc[s][c] = mfma16(av[u][c], xv[u][s], acc[s][c]);
  }
  float* red = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int s = 0; s < kSubs; ++s)
#pragma unroll
    for (int c = 0; c < CB; ++c)
      *reinterpret_cast<f32x4*>(red + (wave * R + 16 * s + r) * kStride + 16 * c + 4 * h) = acc[s][c];
  __syncthreads();
  const float scale = p.scales ? p.scales[id] : 1.0f;
  for (int e = threadIdx.x; e < R * CB * 4; e += kLoraThreads) {
    const int i = e / (CB * 4), c = (e - i * (CB * 4)) * 4;
    const int32_t row = rows[i];
    if (row < 0 || c0 + c >= width) continue;
    f32x4 v[kLoraWaves];
#pragma unroll
    for (int w = 0; w < kLoraWaves; ++w) v[w] = *reinterpret_cast<const f32x4*>(red + (w * R + i) * kStride + c);
    f32x4 sum;
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] = ((v[0][j] + v[1][j]) + (v[2][j] + v[3][j])) * scale;
    *reinterpret_cast<f32x4*>(p.t + (int64_t)row * width + c0 + c) = sum;
  }
}

// Work-group = (row, 16 columns of t).
__device__ __forceinline__ void shrink_small(const LoraArgs& p, int32_t group, int32_t* rows, char* smem) {
  const int32_t blocks = (p.num_slices * p.rank + 15) / 16;
  const int32_t slot = group / blocks;
  int32_t id;
  if (!small_tile(p, slot, rows, &id) || id < 0) return;
  shrink_tile<kLoraSmallTile, 1, 4>(p, id, (group - slot * blocks) * 16, rows, smem);
}

__global__ __launch_bounds__(kLoraThreads) void lora_shrink_small_kernel(const LoraArgs p) {
  __shared__ __attribute__((aligned(16))) char smem[shrink_smem_bytes(kLoraSmallTile, 1)];
  __shared__ int32_t rows[kLoraSmallTile];
  shrink_small(p, blockIdx.x, rows, smem);
}

// Work-group = (sorted tile, 64 columns of t).
__global__ __launch_bounds__(kLoraThreads) void lora_shrink_kernel(const LoraArgs p) {
  __shared__ __attribute__((aligned(16))) char smem[shrink_smem_bytes(kLoraTile, 4)];
  __shared__ int32_t rows[kLoraTile];
  const int32_t blocks = (p.num_slices * p.rank + 63) / 64;
  const int32_t tile = blockIdx.x / blocks;
  int32_t id;
  if (!sorted_tile(p, tile, rows, &id) || id < 0) return;
  shrink_tile<kLoraTile, 4, 2>(p, id, (blockIdx.x - tile * blocks) * 64, rows, smem);
}

// The sums of a decode step's projection (work-groups [0, lin_groups)) and the shrink of its
// adapters, which need nothing of each other, in one launch.
template <int NB>
__global__ __launch_bounds__(kLinThreads) void lora_linear_kernel(const LinArgs a, const LoraArgs p,
                                                                  const int32_t lin_groups) {
  __shared__ __attribute__((aligned(16))) char smem[lin_smem_bytes(1, 1)];
  __shared__ int32_t rows[kLoraSmallTile];
  if ((int32_t)blockIdx.x < lin_groups)
    linear_tile<1, 1, NB, kEpiPartial>(a, blockIdx.x, smem);
  else
    shrink_small(p, blockIdx.x - lin_groups, rows, smem);
}

// ---------------------------------------------------------------- expand ----------------

constexpr int lora_rank32(int rank) { return (rank + 31) / 32 * 32; }
constexpr int expand_row_bytes(int rank) { return lora_rank32(rank) * 4 + 16; }  // hi, lo, and 16 against bank conflicts

__device__ __forceinline__ void split_bf16(float v, uint32_t* hi, uint32_t* lo) {
  const uint32_t b = f32_to_bf16(v);
  const float head = __uint_as_float(b << 16);
  *hi = b;
  // an infinite head (t infinite, or beyond bf16) has no remainder
  *lo = (b & 0x7f80u) == 0x7f80u ? 0u : f32_to_bf16(v - head);
}

// out of R rows of one adapter at columns [begin, end) of slice q: 64 columns a wavefront and turn.
// MFMA row i of tile u is column 32 (u >> 1) + 8 (i >> 2) + 4 (u & 1) + (i & 3) of the turn, so a lane
// holds 8 neighbouring columns of a row in two tiles: 16-byte loads and stores, 64 contiguous
// bytes of every row in one instruction. NCH: 32-wide pieces of the rank.
// kPartial: base is the sum of p.ks fp32 partial products, else bf16 rows of y.
template <int R, int NCH, bool kPartial>
__device__ __forceinline__ void expand_tile(const LoraArgs& p, const int32_t id, const int32_t q, const int32_t begin,
                                            const int32_t end, const int32_t* rows, char* smem) {
  constexpr int kSubs = R / 16;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int r = lane & 15, h = lane >> 4;
  const int row_bytes = expand_row_bytes(p.rank), lo_at = lora_rank32(p.rank) * 2;
  if (id >= 0) {
    const int quads = lora_rank32(p.rank) / 4;
    const int64_t width = p.num_slices * p.rank;
    for (int e = threadIdx.x; e < R * quads; e += kLoraThreads) {
      const int i = e / quads, j = (e - i * quads) * 4;
      const int32_t row = rows[i];
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
      if (row >= 0 && j < p.rank) v = *reinterpret_cast<const f32x4*>(p.t + row * width + q * p.rank + j);
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int n = 0; n < 4; ++n) split_bf16(v[n], &hi[n], &lo[n]);
      char* to = smem + i * row_bytes + j * 2;
      *reinterpret_cast<u32x2*>(to) = u32x2{hi[0] | hi[1] << 16, hi[2] | hi[3] << 16};
      *reinterpret_cast<u32x2*>(to + lo_at) = u32x2{lo[0] | lo[1] << 16, lo[2] | lo[3] << 16};
    }
    __syncthreads();
  }
  const uint16_t* bp = p.b + max(id, 0) * p.b_adapter;
  for (int32_t c0 = begin + 64 * wave; c0 < end; c0 += 64 * kLoraWaves) {
    const bool both = c0 + 32 < end;  // ranges are multiples of 32 columns
    u32x4 bv[NCH][4];
    if (id >= 0) {
#pragma unroll
      for (int ch = 0; ch < NCH; ++ch)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int32_t col = c0 + (both ? 32 * (u >> 1) : 0) + 8 * (r >> 2) + 4 * (u & 1) + (r & 3);
          const int32_t j = 32 * ch + 8 * h;
          bv[ch][u] = u32x4{0u, 0u, 0u, 0u};
          if (j < p.rank) bv[ch][u] = *reinterpret_cast<const u32x4*>(bp + col * p.b_row + j);
        }
    }
#pragma unroll
    for (int s = 0; s < kSubs; ++s) {
      const int32_t row = rows[16 * s + r];
      // the base's 2 x 8 columns
      f32x4 acc[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      u32x4 yv[2];
      if constexpr (!kPartial) {
#pragma unroll
        for (int v = 0; v < 2; ++v)
          if (row >= 0 && (v == 0 || both))
            yv[v] = *reinterpret_cast<const u32x4*>(p.y + row * p.y_stride + c0 + 32 * v + 8 * h);
      }
      if (id >= 0) {
#pragma unroll
        for (int ch = 0; ch < NCH; ++ch) {
          const char* at = smem + (16 * s + r) * row_bytes + 64 * ch + 16 * h;
          const bool in = 32 * ch < lo_at / 2;
          u32x4 hi = {0u, 0u, 0u, 0u}, lo = hi;
          if (in) {
            hi = *reinterpret_cast<const u32x4*>(at);
            lo = *reinterpret_cast<const u32x4*>(at + lo_at);
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            acc[u] = mfma16(bv[ch][u], lo, acc[u]);
            acc[u] = mfma16(bv[ch][u], hi, acc[u]);
          }
        }
      }
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        if (row < 0 || (v == 1 && !both)) continue;
        const int32_t col = c0 + 32 * v + 8 * h;
        float base[8];
        if constexpr (kPartial) {
#pragma unroll
          for (int e = 0; e < 8; ++e) base[e] = 0.f;
          for (int k = 0; k < p.ks; ++k) {
            const float* pp = p.part + ((int64_t)k * p.rows + row) * p.n_out + col;
            const f32x4 a = *reinterpret_cast<const f32x4*>(pp), b = *reinterpret_cast<const f32x4*>(pp + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              base[e] += a[e];
              base[4 + e] += b[e];
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            base[2 * e] = bf16_lo(yv[v][e]);
            base[2 * e + 1] = bf16_hi(yv[v][e]);
          }
        }
        if (id >= 0) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            base[e] += acc[2 * v][e];
            base[4 + e] += acc[2 * v + 1][e];
          }
        }
        u32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = pack_bf16x2(base[2 * e], base[2 * e + 1]);
        *reinterpret_cast<u32x4*>(p.out + row * p.out_stride + col) = o;
      }
    }
  }
}

// Work-group = (row or sorted tile, p.group_cols columns of one slice).
template <bool kSorted, int NCH, bool kPartial>
__global__ __launch_bounds__(kLoraThreads) void lora_expand_kernel(const LoraArgs p) {
  constexpr int R = kSorted ? kLoraTile : kLoraSmallTile;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ int32_t rows[R];
  const int32_t tile = blockIdx.x / p.col_groups;
  int32_t g = blockIdx.x - tile * p.col_groups, q = 0;
  for (; q < p.num_slices - 1; ++q) {
    const int32_t n = (p.slice_begin[q + 1] - p.slice_begin[q] + p.group_cols - 1) / p.group_cols;
    if (g < n) break;
    g -= n;
  }
  int32_t id;
  if constexpr (kSorted) {
    if (!sorted_tile(p, tile, rows, &id)) return;
  } else {
    if (!small_tile(p, tile, rows, &id)) return;
  }
  if (!kPartial && id < 0 && p.out == p.y) return;  // rows without an adapter stay as they are
  const int32_t begin = p.slice_begin[q] + g * p.group_cols;
  expand_tile<R, NCH, kPartial>(p, id, q, begin, min(begin + p.group_cols, p.slice_begin[q + 1]), rows, smem);
}

// ---------------------------------------------------------------- sorting ---------------

// One work-group: rows per adapter (bucket num_adapters: none), the buckets' first positions and
// tiles, then every row's position. A wavefront whose rows have one adapter, the common case
// of a prefill step, counts them in one LDS atomic. Rows of one adapter come in any order.
__global__ __launch_bounds__(kPlanThreads) void lora_plan_kernel(const LoraArgs p) {
  extern __shared__ int32_t count[];  // num_adapters + 1
  __shared__ int32_t part[2][kPlanThreads / kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int32_t buckets = p.num_adapters + 1;
  for (int32_t b = threadIdx.x; b < buckets; b += kPlanThreads) count[b] = 0;
  __syncthreads();
  const auto take = [&](int32_t row) -> int32_t {  // the row's place in its bucket's counter
    const bool is_row = row < p.rows;
    int32_t b = is_row ? adapter_of(p, row) : -1;
    if (b < 0) b = p.num_adapters;
    const uint64_t live = __ballot(is_row);
    if (live == 0) return 0;
    const int32_t first = __builtin_amdgcn_readfirstlane(b);  // (rows ascend with the lane: lane 0 is one)
    if (__ballot(is_row && b != first) == 0) {
      int32_t at = 0;
      if (lane == 0) at = atomicAdd(count + first, __popcll(live));
      return __builtin_amdgcn_readfirstlane(at) + lane;
    }
    return is_row ? atomicAdd(count + b, 1) : 0;
  };
  for (int32_t row0 = 0; row0 < p.rows; row0 += kPlanThreads) take(row0 + threadIdx.x);
  __syncthreads();
  // first positions and first tiles of the buckets: exclusive sums over them, a stretch of
  // neighbouring buckets a thread
  const int32_t per = (buckets + kPlanThreads - 1) / kPlanThreads;
  const int32_t b0 = min((int32_t)threadIdx.x * per, buckets), b1 = min(b0 + per, buckets);
  int32_t n = 0, t = 0;
  for (int32_t b = b0; b < b1; ++b) {
    n += count[b];
    t += (count[b] + kLoraTile - 1) / kLoraTile;
  }
  int32_t in = n, it = t;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int32_t on = __shfl_up(in, d, kWave), ot = __shfl_up(it, d, kWave);
    if (lane >= d) {
      in += on;
      it += ot;
    }
  }
  if (lane == kWave - 1) {
    part[0][wave] = in;
    part[1][wave] = it;
  }
  __syncthreads();
  in -= n;
  it -= t;
  int32_t tiles = 0;
  for (int w = 0; w < kPlanThreads / kWave; ++w) {
    if (w < wave) {
      in += part[0][w];
      it += part[1][w];
    }
    tiles += part[1][w];
  }
  for (int32_t b = b0; b < b1; ++b) {
    const int32_t c = count[b];
    for (int32_t i = 0; i < c; i += kLoraTile)
      p.tiles[it++] = make_int4(b < p.num_adapters ? b : -1, in + i, min(c - i, kLoraTile), 0);
    count[b] = in;  // from here on the bucket's next free position
    in += c;
  }
  if (threadIdx.x == 0) *p.num_tiles = tiles;
  __syncthreads();
  for (int32_t row0 = 0; row0 < p.rows; row0 += kPlanThreads) {
    const int32_t row = row0 + threadIdx.x;
    const int32_t at = take(row);
    if (row < p.rows) p.perm[at] = row;
  }
}

// ---------------------------------------------------------------- launches --------------

int64_t lora_max_tiles(int32_t rows, int32_t num_adapters) {
  return rows / kLoraTile + std::min<int64_t>((int64_t)num_adapters + 1, rows);
}

int32_t lora_col_groups(LoraArgs& p, int32_t group_cols) {
  p.group_cols = group_cols;
  p.col_groups = 0;
  for (int q = 0; q < p.num_slices; ++q)
    p.col_groups += (p.slice_begin[q + 1] - p.slice_begin[q] + group_cols - 1) / group_cols;
  return p.col_groups;
}

template <bool kSorted, bool kPartial>
hipError_t launch_expand(const LoraArgs& p, int64_t tiles, hipStream_t stream) {
  const dim3 grid((unsigned)(tiles * p.col_groups)), block(kLoraThreads);
  const unsigned lds = (kSorted ? kLoraTile : kLoraSmallTile) * expand_row_bytes(p.rank);
  if (p.rank <= 32)
    hipLaunchKernelGGL((lora_expand_kernel<kSorted, 1, kPartial>), grid, block, lds, stream, p);
  else if (p.rank <= 64)
    hipLaunchKernelGGL((lora_expand_kernel<kSorted, 2, kPartial>), grid, block, lds, stream, p);
  else
    hipLaunchKernelGGL((lora_expand_kernel<kSorted, 4, kPartial>), grid, block, lds, stream, p);
  return hipGetLastError();
}

size_t round16(size_t n) { return (n + 15) & ~(size_t)15; }

size_t t_bytes(const LoraArgs& p) { return (size_t)p.rows * p.num_slices * p.rank * sizeof(float); }

}  // namespace

size_t lora_linear_workspace_bytes(const LoraArgs& p) {
  const LinCfg c = choose_config(p.rows, p.n_out / kLinTile, p.k, 1);
  return t_bytes(p) + (size_t)c.ks * p.rows * p.n_out * sizeof(float);
}

size_t lora_add_workspace_bytes(const LoraArgs& p) {
  if (p.rows <= kLoraSmallRows) return t_bytes(p);
  return t_bytes(p) + 16 + (size_t)lora_max_tiles(p.rows, p.num_adapters) * sizeof(int4) +
         round16((size_t)p.rows * sizeof(int32_t));
}

hipError_t launch_lora_linear(const LoraArgs& args, const void* w, int64_t w_stride, void* ws, hipStream_t stream) {
  LoraArgs p = args;
  const LinCfg c = choose_config(p.rows, p.n_out / kLinTile, p.k, 1);
  p.t = static_cast<float*>(ws);
  p.part = p.t + (size_t)p.rows * p.num_slices * p.rank;
  p.ks = c.ks;
  LinArgs a{};
  a.x = p.x;
  a.x_stride = p.x_stride;
  a.w = static_cast<const uint16_t*>(w);
  a.w_stride = w_stride;
  a.rows = p.rows;
  a.n_out = p.n_out;
  a.k = p.k;
  a.ks = c.ks;
  a.part = p.part;
  const int32_t lin_groups = (p.n_out / kLinTile) * c.ks * c.mgroups;
  const int32_t shrink = p.num_adapters > 0 ? p.rows * ((p.num_slices * p.rank + 15) / 16) : 0;
  const dim3 grid(lin_groups + shrink), block(kLinThreads);
  switch (c.nb) {
    case 1: hipLaunchKernelGGL(lora_linear_kernel<1>, grid, block, 0, stream, a, p, lin_groups); break;
    case 2: hipLaunchKernelGGL(lora_linear_kernel<2>, grid, block, 0, stream, a, p, lin_groups); break;
    default: hipLaunchKernelGGL(lora_linear_kernel<4>, grid, block, 0, stream, a, p, lin_groups); break;
  }
  if (hipError_t err = hipGetLastError(); err != hipSuccess) return err;
  lora_col_groups(p, 64 * kLoraWaves);
  return launch_expand<false, true>(p, p.rows, stream);
}

hipError_t launch_lora_add(const LoraArgs& args, void* ws, hipStream_t stream) {
  LoraArgs p = args;
  p.t = static_cast<float*>(ws);
  const int32_t width = p.num_slices * p.rank;
  if (p.rows <= kLoraSmallRows) {
    if (p.num_adapters > 0) {
      hipLaunchKernelGGL(lora_shrink_small_kernel, dim3(p.rows * ((width + 15) / 16)), dim3(kLoraThreads), 0, stream,
                         p);
      if (hipError_t err = hipGetLastError(); err != hipSuccess) return err;
    }
    lora_col_groups(p, 64 * kLoraWaves);
    return launch_expand<false, false>(p, p.rows, stream);
  }
  const int64_t tiles = lora_max_tiles(p.rows, p.num_adapters);
  char* at = static_cast<char*>(ws) + t_bytes(p);
  p.num_tiles = reinterpret_cast<int32_t*>(at);
  p.tiles = reinterpret_cast<int4*>(at + 16);
  p.perm = reinterpret_cast<int32_t*>(at + 16 + tiles * sizeof(int4));
  hipLaunchKernelGGL(lora_plan_kernel, dim3(1), dim3(kPlanThreads), (p.num_adapters + 1) * sizeof(int32_t), stream, p);
  if (hipError_t err = hipGetLastError(); err != hipSuccess) return err;
  if (p.num_adapters > 0) {
    hipLaunchKernelGGL(lora_shrink_kernel, dim3((unsigned)(tiles * ((width + 63) / 64))), dim3(kLoraThreads), 0, stream,
                       p);
    if (hipError_t err = hipGetLastError(); err != hipSuccess) return err;
  }
  lora_col_groups(p, 64 * kLoraWaves);
  return launch_expand<true, false>(p, tiles, stream);
}

}  // namespace pk
