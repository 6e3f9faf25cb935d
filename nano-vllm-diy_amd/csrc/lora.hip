// Low-rank adapters of many requests beside a shared projection, on gfx950: every token row m has
// an adapter a = adapter_ids[m] of its own (outside [0, num_adapters): none),
//   t[m, i]   = scale[a] * sum_k x[m, k] A[a, i, k]                          (shrink)
//   out[m, c] = bf16(base[m, c] + sum_j t[m, q rank + j] B[a, c, j])         (expand)
// where q is the slice (merged projection) of output column c and base is x W^T, whose sums are
// computed next to the shrink (lora_linear, at most 128 rows), or given (lora_add). The reference
// has no adapters; the projections are those of linear.hip.
//
// The work is reading: W or base, out, and the adapters in use; the products are 16-64 wide and free
// next to that. So rows are brought together by adapter, and a group of up to 16 or 64 rows of ONE
// adapter is an MFMA tile that reads A and B once for all of them. An adapter whose rows are in several
// groups is read by each, mostly from the caches:
//   * few rows (small_add): the groups are the equal ids within 16 consecutive rows. Nothing is sorted:
//     there is a work-group for every group that 16 rows can have, 16 or one for each adapter and one
//     for none, and those without a group end.
//   * more: one work-group sorts the rows by adapter (counts, offsets, positions) and lists the
//     tiles of 64.
// Every row's sums are taken in the same order whatever shares its tile. A row of lora_add has the same
// bits alone and in any batch, sorted or not. For lora_linear the number of rows picks the projection's K
// split and the form that adds the adapters, and with them the order of the sums; the other rows' values
// and adapters change nothing.
//
// t is kept in fp32. For the expand it is split into two bf16, t = hi + lo with a remainder
// below 2^-16 |t|, and both halves are multiplied (the products with bf16 B are exact in the
// fp32 sum), so t costs no rounding of the output's size. The output is rounded once. An infinite B
// gives NaN where lo is 0 or of the other sign, and the formula's infinity elsewhere and in the
// epilogue that multiplies in fp32 (LoraAddend).
//
// MFMA: v_mfma_f32_16x16x32_bf16, D[i][j] = sum_k A[i][k] B[k][j]; lane (r = lane & 15, h = lane
// >> 4) supplies row r of both operands at k = 8 h .. 8 h + 7 and holds D[4 h .. 4 h + 3][r]. The
// token rows are the second operand, so a lane's four values are neighbours in one row of t
// or out.
#include <type_traits>

#include "linear_core.h"

namespace pk {
namespace {

constexpr int kLoraThreads = 256;
constexpr int kLoraWaves = kLoraThreads / kWave;
constexpr int kLoraTile = 64;        // rows of a sorted tile
constexpr int kLoraSmallTile = 16;   // rows of a tile that is not sorted
constexpr int kPlanThreads = 1024;
constexpr int kPlanTurns = 4;        // turns of 4096 rows whose ids are loaded together

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
// Not sorted: of the rows of [16 t, 16 t + 16) those with the jth group's adapter, t = slot /
// tile_slots and j = slot % tile_slots; false if there is none. Every thread calls it.
__device__ __forceinline__ bool small_tile(const LoraArgs& p, int32_t slot, int32_t* rows, int32_t* id) {
  const int lane = threadIdx.x & (kWave - 1);
  const int32_t tile = slot / p.tile_slots, row = tile * kLoraSmallTile + lane;
  const bool is_row = lane < kLoraSmallTile && row < p.rows;
  const int32_t mine = is_row ? adapter_of(p, row) : -2;
  const int32_t j = slot - tile * p.tile_slots;
  if (p.tile_slots == kLoraSmallTile) {  // the group of row j, if that is its first row
    if (tile * kLoraSmallTile + j >= p.rows) return false;
    *id = __builtin_amdgcn_readlane(mine, j);
    if (__builtin_ctzll(__ballot(mine == *id)) != j) return false;
  } else {
    uint64_t left = __ballot(is_row);
    for (int i = 0;; ++i) {
      if (left == 0) return false;
      *id = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
      if (i == j) break;
      left &= ~__ballot(mine == *id);
    }
  }
  if (threadIdx.x < kLoraSmallTile) rows[threadIdx.x] = mine == *id ? row : -1;
  __syncthreads();
  return true;
}

// Sorted: R rows of the tile from its row `first` on (its record and its rows are loaded together;
// an unused tile has no rows).
template <int R>
__device__ __forceinline__ bool sorted_tile(const LoraArgs& p, int32_t tile, int32_t first, int32_t* rows,
                                            int32_t* id) {
  if (tile >= p.max_tiles) return false;
  const int32_t i = first + threadIdx.x;
  const int2 t = p.tiles[tile];  // adapter, rows
  const int32_t row = threadIdx.x < R ? p.perm[(int64_t)tile * kLoraTile + i] : -1;
  *id = t.x;
  if (first >= t.y) return false;
  if (threadIdx.x < R) rows[threadIdx.x] = i < t.y ? row : -1;
  __syncthreads();
  return true;
}

// ---------------------------------------------------------------- shrink ----------------

// A chunk is 64 elements of k: 128 contiguous bytes of every row, in LDS with 16 bytes between rows.
constexpr int kChunk = 64;
constexpr int kChunkStride = kChunk * 2 + 16;
constexpr int shrink_smem_bytes(int r, int cb) {
  const int chunks = kLoraWaves * (r + cb * 16) * kChunkStride, sums = kLoraWaves * r * (cb * 16 + 4) * 4;
  return chunks > sums ? chunks : sums;
}

// This wavefront's LDS writes before its reads and its reads before its next writes: a
// wavefront's LDS operations run in order, so only the compiler has to be told.
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// t of R rows of one adapter at its columns [c0, c0 + 16 CB). The four wavefronts take the chunks of
// k in turn (each its own: no barrier) and add up in LDS at the end. A chunk's x and A rows are
// loaded 8 rows an instruction and put into the MFMA's order through LDS: loaded in that
// order, four neighbouring lanes would hold four rows, four cache lines instead of one, and
// the L1 would be the bound. The loads are U chunks ahead.
// store(i, c, v): t of the tile's row i at columns c0 + c .. + 3, scaled.
template <int R, int CB, int U, class Store>
__device__ __forceinline__ void shrink_tile(const LoraArgs& p, const int32_t id, const int32_t c0, const int32_t* rows,
                                            char* smem, const Store& store) {
  constexpr int kSubs = R / 16, kLoads = (R + 16 * CB) / 8, kStride = CB * 16 + 4;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int r = lane & 15, h = lane >> 4;
  const int32_t width = p.num_slices * p.rank;
  const uint16_t* src[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int m = 8 * i + (lane >> 3);
    if (8 * i < R)
      src[i] = p.x + (int64_t)max(rows[m], 0) * p.x_stride;  // (what the missing rows give is not stored)
    else
      src[i] = p.a + id * p.a_adapter + (int64_t)min(c0 + m - R, width - 1) * p.a_row;
    src[i] += 8 * (lane & 7);
  }
  char* mine = smem + wave * (R + 16 * CB) * kChunkStride;
  char* put = mine + (lane >> 3) * kChunkStride + 16 * (lane & 7);
  const char* get = mine + r * kChunkStride + 16 * h;
  f32x4 acc[kSubs][CB];
#pragma unroll
  for (int s = 0; s < kSubs; ++s)
#pragma unroll
    for (int c = 0; c < CB; ++c) acc[s][c] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int32_t kTurn = kLoraWaves * kChunk;
  u32x4 st[U][kLoads];
  const auto load = [&](int u, int32_t at) {
    const bool in = at + 8 * (lane & 7) < p.k;  // k is a multiple of 8
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      st[u][i] = u32x4{0u, 0u, 0u, 0u};
      if (in) st[u][i] = *reinterpret_cast<const u32x4*>(src[i] + at);
    }
  };
#pragma unroll
  for (int u = 0; u < U; ++u) load(u, wave * kChunk + u * kTurn);
  for (int32_t k0 = wave * kChunk; k0 < p.k; k0 += U * kTurn) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) *reinterpret_cast<u32x4*>(put + i * 8 * kChunkStride) = st[u][i];
      if (k0 + U * kTurn < p.k) load(u, k0 + (U + u) * kTurn);
      wave_lds_fence();
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        u32x4 xv[kSubs];
#pragma unroll
        for (int s = 0; s < kSubs; ++s)
          xv[s] = *reinterpret_cast<const u32x4*>(get + 16 * s * kChunkStride + 64 * q);
#pragma unroll
        for (int c = 0; c < CB; ++c) {
          const u32x4 av = *reinterpret_cast<const u32x4*>(get + (R + 16 * c) * kChunkStride + 64 * q);
#pragma unroll
          for (int s = 0; s < kSubs; ++s) acc[s][c] = mfma16(av, xv[s], acc[s][c]);
        }
      }
      wave_lds_fence();
    }
  }
  __syncthreads();  // every wavefront is done with its chunks before they hold the sums
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
    f32x4 v[kLoraWaves];
#pragma unroll
    for (int w = 0; w < kLoraWaves; ++w) v[w] = *reinterpret_cast<const f32x4*>(red + (w * R + i) * kStride + c);
    f32x4 sum;
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[j] = ((v[0][j] + v[1][j]) + (v[2][j] + v[3][j])) * scale;
    store(i, c, sum);
  }
}

// shrink_tile's sums to p.t, for the expand's launch.
template <int R, int CB, int U>
__device__ __forceinline__ void shrink_to_memory(const LoraArgs& p, const int32_t id, const int32_t c0,
                                                 const int32_t* rows, char* smem) {
  const int32_t width = p.num_slices * p.rank;
  shrink_tile<R, CB, U>(p, id, c0, rows, smem, [&](int i, int c, const f32x4 v) {
    const int32_t row = rows[i];
    if (row >= 0 && c0 + c < width) *reinterpret_cast<f32x4*>(p.t + (int64_t)row * width + c0 + c) = v;
  });
}

// Work-group = (group of rows, 16 CB columns of t).
template <int CB>
__device__ __forceinline__ void shrink_small(const LoraArgs& p, int32_t group, int32_t* rows, char* smem) {
  const int32_t blocks = (p.num_slices * p.rank + 16 * CB - 1) / (16 * CB);
  const int32_t slot = group / blocks;
  int32_t id;
  if (!small_tile(p, slot, rows, &id) || id < 0) return;
  shrink_to_memory<kLoraSmallTile, CB, 4>(p, id, (group - slot * blocks) * 16 * CB, rows, smem);
}

__global__ __launch_bounds__(kLoraThreads) void lora_shrink_small_kernel(const LoraArgs p) {
  __shared__ __attribute__((aligned(16))) char smem[shrink_smem_bytes(kLoraSmallTile, 1)];
  __shared__ int32_t rows[kLoraSmallTile];
  shrink_small<1>(p, blockIdx.x, rows, smem);
}

// Work-group = (R rows of a sorted tile, 16 CB columns of t). 16384 rows of k = 1024, 48 columns 10.0 us (x
// alone 6.6 at a copy's rate): the rest is the chain from the tile's rows to their first loads.
template <int R, int CB>
__global__ __launch_bounds__(kLoraThreads) void lora_shrink_kernel(const LoraArgs p) {
  __shared__ __attribute__((aligned(16))) char smem[shrink_smem_bytes(R, CB)];
  __shared__ int32_t rows[R];
  const int32_t blocks = (p.num_slices * p.rank + 16 * CB - 1) / (16 * CB);
  // the blocks of one tile's rows are 8 work-groups apart: one XCD, whose L2 gives the rows to all
  const int32_t part = blockIdx.x / (8 * blocks) * 8 + blockIdx.x % 8, block = blockIdx.x % (8 * blocks) / 8;
  constexpr int kParts = kLoraTile / R;
  int32_t id;
  if (!sorted_tile<R>(p, part / kParts, part % kParts * R, rows, &id) || id < 0) return;
  shrink_to_memory<R, CB, 1>(p, id, block * 16 * CB, rows, smem);
}

// The partial sums of a decode step's projection (work-groups [0, lin_groups)) and the shrink of its
// adapters, which need nothing of each other, in one launch; the expand adds the partial sums. 128 rows,
// 64 adapters of rank 64 in use on 3072 x 1024: 12.0 us. W, x and A read once are 32 MB; it reads 49,
// since the 16-row groups hold 108 times one of the 64 adapters.
template <int NB, int CB>
__global__ __launch_bounds__(kLinThreads) void lora_linear_kernel(const LinArgs a, const LoraArgs p,
                                                                  const int32_t lin_groups) {
  __shared__ __attribute__((aligned(16))) char smem[lin_smem_bytes(1, 1)];
  __shared__ int32_t rows[kLoraSmallTile];
  if ((int32_t)blockIdx.x < lin_groups)
    linear_tile<1, 1, NB, kEpiPartial>(a, blockIdx.x, smem, NoAddend{});
  else
    shrink_small<CB>(p, blockIdx.x - lin_groups, rows, smem);
}

// A projection whose K is not split, after the shrink's launch: the work-group adds its rows' adapters
// to its sums, products in fp32, for ranks up to 16. A row's B is 64 pieces of 16 bytes (two a
// column), one after the other in memory; the row's eight threads take them in turn, whole cache
// lines, before the K walk, which hides them. Their products with t go through LDS to the threads
// that have the columns.
//
// kShrink: t is computed here too, after the K walk, by every work-group for its slice, which saves the
// shrink's launch and reads the rows' A in every work-group. Rank 16, every row an adapter of its own, one
// launch and two, us in a graph over eight sets of weights in turn: 1024 x 4096 1 row 7.7 and 9.2, 2 rows 9.8
// and 9.9, 3 rows 10.7 and 9.8, 4 rows 12.0 and 9.9; 1024 x 6144 1 row 8.6 and 10.3, 2 rows 10.1 and 10.4, 4
// rows 12.3 and 10.3. Outside a graph the second launch also costs 3.3 us of host time.
constexpr int kOneLaunchRows = 2;

template <bool kShrink>
struct LoraAddend {
  const LoraArgs& p;
  int32_t* rows;   // LDS, 16 (kShrink)
  float* t_here;   // LDS, [16][16] (kShrink)
  int32_t id, slice;
  u32x4 b[8];
  f32x4 t[2];
  __device__ __forceinline__ int half() const { return threadIdx.x & 1; }
  __device__ __forceinline__ void load(int row0, int n0) {
    const int32_t m = row0 + (threadIdx.x >> 3), piece = threadIdx.x & 7;
    id = m < p.rows ? adapter_of(p, m) : -1;
    slice = 0;
    while (slice < p.num_slices - 1 && n0 >= p.slice_begin[slice + 1]) ++slice;  // (multiples of 32 columns)
    if (id < 0) return;
    const uint16_t* bp = p.b + id * p.b_adapter + (n0 + (piece >> 1)) * p.b_row + 8 * half();
    const bool in = 8 * half() < p.rank;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      b[i] = u32x4{0u, 0u, 0u, 0u};
      if (in) b[i] = *reinterpret_cast<const u32x4*>(bp + 4 * i * p.b_row);
    }
    if constexpr (!kShrink) load_t(p.t + (int64_t)m * (p.num_slices * p.rank) + slice * p.rank);
  }
  __device__ __forceinline__ void load_t(const float* row) {
    t[0] = t[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (8 * half() < p.rank) {
      t[0] = *reinterpret_cast<const f32x4*>(row + 8 * half());
      t[1] = *reinterpret_cast<const f32x4*>(row + 8 * half() + 4);
    }
  }
  __device__ __forceinline__ void prepare(char* lds) {
    if constexpr (kShrink) {
      for (int j = 0; j < p.rows; ++j) {  // the rows' adapters, each once
        int32_t a;
        if (!small_tile(p, j, rows, &a) || a < 0) continue;
        shrink_tile<kLoraSmallTile, 1, 4>(p, a, slice * p.rank, rows, lds, [&](int i, int c, const f32x4 v) {
          if (rows[i] >= 0) *reinterpret_cast<f32x4*>(t_here + 16 * i + c) = v;
        });
        __syncthreads();
      }
      if (id >= 0) load_t(t_here + 16 * (threadIdx.x >> 3));
    }
  }
  // [row][64] products of the pieces, 4 floats between rows
  __device__ __forceinline__ void put(char* lds) const {
    float* at = reinterpret_cast<float*>(lds) + (threadIdx.x >> 3) * 68 + (threadIdx.x & 7);
    if (id < 0) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float d = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        d = fmaf(bf16_lo(b[i][e]), t[e >> 1][2 * (e & 1)], d);
        d = fmaf(bf16_hi(b[i][e]), t[e >> 1][2 * (e & 1) + 1], d);
      }
      at[8 * i] = d;
    }
  }
  __device__ __forceinline__ void add(const char* lds, float4& v) const {
    if (id < 0) return;
    const float* at = reinterpret_cast<const float*>(lds) + (threadIdx.x >> 3) * 68 + 8 * (threadIdx.x & 7);
    const f32x4 d0 = *reinterpret_cast<const f32x4*>(at), d1 = *reinterpret_cast<const f32x4*>(at + 4);
    v = make_float4(v.x + (d0[0] + d0[1]), v.y + (d0[2] + d0[3]), v.z + (d1[0] + d1[1]), v.w + (d1[2] + d1[3]));
  }
};

template <int NB, bool kShrink>
__global__ __launch_bounds__(kLinThreads) void lora_linear_expand_kernel(const LinArgs a, const LoraArgs p) {
  __shared__ __attribute__((aligned(16))) char smem[lin_smem_bytes(1, 1)];
  __shared__ __attribute__((aligned(16))) float t_here[kShrink ? kLoraSmallTile * 16 : 4];
  __shared__ int32_t rows[kLoraSmallTile];
  linear_tile<1, 1, NB, kEpiStore>(a, blockIdx.x, smem, LoraAddend<kShrink>{p, rows, t_here});
}

// ---------------------------------------------------------------- expand ----------------

// t = hi + lo. The head is within bf16's range, so that a finite t stays finite; an infinite or NaN t is
// in lo.
__device__ __forceinline__ void split_bf16(float v, uint32_t* hi, uint32_t* lo) {
  constexpr float kLargest = 0x1.fep127f;
  const uint32_t b = f32_to_bf16(__builtin_amdgcn_fmed3f(v, -kLargest, kLargest));
  *hi = b;
  *lo = f32_to_bf16(v - __uint_as_float(b << 16));
}

// How both expand kernels multiply. A wavefront has 16 rows and 128 columns: t's rows are the
// MFMA's first operand, B's the second, and row j of MFMA tile u is column 8 j + u, so that a lane's
// eight tiles give 8 neighbouring columns of a row and 16 lanes 256 contiguous bytes of it: whole
// cache lines of base and out. B is loaded along its rows and ordered through LDS, KP elements of
// the rank at a time with 16 bytes between rows. Of t both halves are multiplied; with KP = 16
// they fit one MFMA (k 0-15 hi, 16-31 lo).
template <int KP>
struct ExpandShape {
  static constexpr int kRowBytes = KP * 2 + 16;
  static constexpr int kChunks = KP / 8;                   // 16-byte pieces of a B row
  static constexpr int kSteps = KP > 32 ? KP / 32 : 1;     // MFMA steps
  // LDS row of a column: column 8 j + u of 128 at 16 u + j, so a tile's rows are neighbours
  __device__ static __forceinline__ int at(int c) { return (c & ~127) | (c & 7) << 4 | (c & 127) >> 3; }
};

// A lane's part of t, both halves: row t_row (of one slice), elements j0 + 32 n + 8 h of KP.
template <int KP>
__device__ __forceinline__ void load_t(const float* t_row, int32_t rank, int32_t j0, int h,
                                       u32x4 (&hi)[ExpandShape<KP>::kSteps], u32x4 (&lo)[ExpandShape<KP>::kSteps]) {
#pragma unroll
  for (int n = 0; n < ExpandShape<KP>::kSteps; ++n) {
    const int32_t j = j0 + 32 * n + 8 * (KP == 16 ? h & 1 : h);
    f32x4 v[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    if (j < rank) {
      v[0] = *reinterpret_cast<const f32x4*>(t_row + j);
      v[1] = *reinterpret_cast<const f32x4*>(t_row + j + 4);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint32_t ha, la, hb, lb;
      split_bf16(v[e >> 1][2 * (e & 1)], &ha, &la);
      split_bf16(v[e >> 1][2 * (e & 1) + 1], &hb, &lb);
      hi[n][e] = ha | hb << 16;
      lo[n][e] = la | lb << 16;
      if (KP == 16 && h >= 2) hi[n][e] = lo[n][e];
    }
  }
}

// acc[u] += t B^T over KP elements; b: LDS row of the wavefront's first column.
template <int KP>
__device__ __forceinline__ void expand_mfma(const char* b, int r, int h, const u32x4 (&hi)[ExpandShape<KP>::kSteps],
                                            const u32x4 (&lo)[ExpandShape<KP>::kSteps], f32x4 (&acc)[8]) {
  constexpr int kRowBytes = ExpandShape<KP>::kRowBytes;
#pragma unroll
  for (int n = 0; n < ExpandShape<KP>::kSteps; ++n) {
    const char* get = b + r * kRowBytes + 64 * n + 16 * (KP == 16 ? h & 1 : h);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const u32x4 bv = *reinterpret_cast<const u32x4*>(get + 16 * u * kRowBytes);
      if constexpr (KP != 16) acc[u] = mfma16(lo[n], bv, acc[u]);
      acc[u] = mfma16(hi[n], bv, acc[u]);
    }
  }
}

// The slice of column group g (of `cols` columns each) and its first column.
__device__ __forceinline__ int32_t group_slice(const LoraArgs& p, int32_t g, int32_t cols, int32_t* begin) {
  int32_t q = 0;
  for (; q < p.num_slices - 1; ++q) {
    const int32_t n = (p.slice_begin[q + 1] - p.slice_begin[q] + cols - 1) / cols;
    if (g < n) break;
    g -= n;
  }
  *begin = p.slice_begin[q] + g * cols;
  return q;
}

// Work-group = (group of rows of one adapter, up to 128 WAVES columns of a slice): 128 columns a
// wavefront. Everything is asked for before the first wait.
// kBase: where base is from -- kBasePartial: the sum of p.ks fp32 partial products, kBaseRows: bf16
// rows of y, kBaseRowsShrink: those, and t is computed here, by every work-group of the row again, instead of
// by a launch before (the rank is KP at most then).
enum Base { kBasePartial = 0, kBaseRows = 1, kBaseRowsShrink = 2 };

template <int KP, int WAVES, int kBase>
__global__ __launch_bounds__(WAVES* kWave, kBase == kBaseRowsShrink && KP == 16 ? 3 : 1) void
lora_expand_small_kernel(const LoraArgs p) {
  using S = ExpandShape<KP>;
  constexpr bool kPartial = kBase == kBasePartial, kShrink = kBase == kBaseRowsShrink;
  static_assert(!kShrink || WAVES == kLoraWaves, "shrink_tile's work-group");
  constexpr int kThreads = WAVES * kWave, kCols = 128 * WAVES;
  constexpr int kLoads = kCols * S::kChunks / kThreads, CB = (KP + 15) / 16;
  constexpr int kBBytes = kCols * S::kRowBytes, kShrinkBytes = kShrink ? shrink_smem_bytes(kLoraSmallTile, CB) : 0;
  __shared__ __attribute__((aligned(16))) char smem[kBBytes > kShrinkBytes ? kBBytes : kShrinkBytes];
  __shared__ __attribute__((aligned(16))) float t_here[kShrink ? kLoraSmallTile * KP : 4];
  __shared__ int32_t rows[kLoraSmallTile];
  const int32_t slot = blockIdx.x / p.col_groups;
  int32_t id, begin;
  if (!small_tile(p, slot, rows, &id)) return;
  if (!kPartial && id < 0 && p.out == p.y) return;  // rows without an adapter stay as they are
  const int32_t q = group_slice(p, blockIdx.x - slot * p.col_groups, kCols, &begin);
  const int32_t end = min(begin + kCols, p.slice_begin[q + 1]);
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int r = lane & 15, h = lane >> 4;
  const int32_t col = begin + 128 * wave + 8 * r;  // this lane's columns
  const bool in = col < end;                       // ranges are multiples of 32 columns
  int32_t row[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) row[i] = rows[4 * h + i];
  u32x4 yv[4];
  if constexpr (!kPartial) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (in && row[i] >= 0) yv[i] = *reinterpret_cast<const u32x4*>(p.y + row[i] * p.y_stride + col);
  }
  f32x4 acc[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (id >= 0) {
    const uint16_t* bp = p.b + id * p.b_adapter;
    const float* tp = kShrink ? t_here + r * KP
                              : p.t + (int64_t)max(rows[r], 0) * (p.num_slices * p.rank) + q * p.rank;
#pragma unroll 1
    for (int32_t j0 = 0; j0 < p.rank; j0 += KP) {
      u32x4 st[kLoads], hi[S::kSteps], lo[S::kSteps];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int e = i * kThreads + threadIdx.x, c = e / S::kChunks, j = j0 + e % S::kChunks * 8;
        st[i] = u32x4{0u, 0u, 0u, 0u};
        if (begin + c < end && j < p.rank) st[i] = *reinterpret_cast<const u32x4*>(bp + (begin + c) * p.b_row + j);
      }
      if constexpr (kShrink) {
        shrink_tile<kLoraSmallTile, CB, 2 / CB>(p, id, q * p.rank, rows, smem, [&](int i, int c, const f32x4 v) {
          *reinterpret_cast<f32x4*>(t_here + i * KP + c) = v;
        });
        __syncthreads();  // t is there, and the sums it was added from are free for B
      }
      load_t<KP>(tp, p.rank, j0, h, hi, lo);
      if (j0) __syncthreads();  // the previous piece has been read
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int e = i * kThreads + threadIdx.x;
        *reinterpret_cast<u32x4*>(smem + S::at(e / S::kChunks) * S::kRowBytes + e % S::kChunks * 16) = st[i];
      }
      __syncthreads();
      expand_mfma<KP>(smem + 128 * wave * S::kRowBytes, r, h, hi, lo, acc);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (!in || row[i] < 0) continue;
    float f[8];
    if constexpr (kPartial) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = 0.f;
      const float* pp = p.part + (int64_t)row[i] * p.n_out + col;
      for (int k0 = 0; k0 < p.ks; k0 += 4) {  // four splits' loads together, added in order
        f32x4 a[4], b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float* at = pp + (int64_t)min(k0 + k, p.ks - 1) * p.rows * p.n_out;
          a[k] = *reinterpret_cast<const f32x4*>(at);
          b[k] = *reinterpret_cast<const f32x4*>(at + 4);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (k0 + k < p.ks)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              f[e] += a[k][e];
              f[4 + e] += b[k][e];
            }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[2 * e] = bf16_lo(yv[i][e]);
        f[2 * e + 1] = bf16_hi(yv[i][e]);
      }
    }
    if (id >= 0) {
#pragma unroll
      for (int u = 0; u < 8; ++u) f[u] += acc[u][i];
    }
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = pack_bf16x2(f[2 * e], f[2 * e + 1]);
    if constexpr (!kPartial)
      if (id < 0) o = yv[i];
    *reinterpret_cast<u32x4*>(p.out + row[i] * p.out_stride + col) = o;
  }
}

// Work-group = (sorted tile, up to kSortedCols columns of a slice): 16 rows a wavefront, all four the
// same columns, which they walk 128 at a time. The walk's loads are one turn ahead of its
// products: B's next rows and the base's next columns are in flight while this turn multiplies
// and stores. t stays in registers: NP pieces of KP elements of the rank. Bound by HBM: 16384 x 4096,
// rank 16 56.8 us, 4.7 TB/s of base and out (a copy's rate); 13001 x 6144, rank 64 76 us, 4.2 TB/s.
// 1024 columns a work-group 61 and 80, 256 and 384 within 2 %.
constexpr int kSortedCols = 512;

template <int KP, int NP>
__global__ __launch_bounds__(kLoraThreads) void lora_expand_kernel(const LoraArgs p) {
  using S = ExpandShape<KP>;
  constexpr int kLoads = 128 * S::kChunks / kLoraThreads;
  constexpr int kBuf = 128 * S::kRowBytes;
  __shared__ __attribute__((aligned(16))) char smem[2 * kBuf];
  __shared__ int32_t rows[kLoraTile];
  const int32_t tile = blockIdx.x / p.col_groups;
  int32_t id, begin;
  if (!sorted_tile<kLoraTile>(p, tile, 0, rows, &id)) return;
  if (id < 0 && p.out == p.y) return;  // rows without an adapter stay as they are
  const int32_t q = group_slice(p, blockIdx.x - tile * p.col_groups, kSortedCols, &begin);
  const int32_t end = min(begin + kSortedCols, p.slice_begin[q + 1]);
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int r = lane & 15, h = lane >> 4;
  int32_t row[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) row[i] = rows[16 * wave + 4 * h + i];
  const uint16_t* bp = p.b + max(id, 0) * p.b_adapter;
  u32x4 st[kLoads], yv[4], hi[NP][S::kSteps], lo[NP][S::kSteps];
  const auto load_b = [&](int32_t c0, int32_t j0) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int e = i * kLoraThreads + threadIdx.x, c = e / S::kChunks, j = j0 + e % S::kChunks * 8;
      st[i] = u32x4{0u, 0u, 0u, 0u};
      if (c0 + c < end && j < p.rank) st[i] = *reinterpret_cast<const u32x4*>(bp + (c0 + c) * p.b_row + j);
    }
  };
  const auto load_y = [&](int32_t c0, u32x4 (&y)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c0 + 8 * r < end && row[i] >= 0)
        y[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p.y + row[i] * p.y_stride + c0 + 8 * r));
  };
  if (id >= 0) load_b(begin, 0);
  load_y(begin, yv);
  if (id >= 0) {
    const float* tp = p.t + (int64_t)max(rows[16 * wave + r], 0) * (p.num_slices * p.rank) + q * p.rank;
#pragma unroll
    for (int n = 0; n < NP; ++n) load_t<KP>(tp, p.rank, n * KP, h, hi[n], lo[n]);
  }
  int buf = 0;
  for (int32_t c0 = begin; c0 < end; c0 += 128) {
    u32x4 next[4];
    f32x4 acc[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) acc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (c0 + 128 < end) load_y(c0 + 128, next);
    if (id >= 0) {
#pragma unroll
      for (int n = 0; n < NP; ++n) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
          const int e = i * kLoraThreads + threadIdx.x;
          *reinterpret_cast<u32x4*>(smem + buf * kBuf + S::at(e / S::kChunks) * S::kRowBytes + e % S::kChunks * 16) =
              st[i];
        }
        if (n + 1 < NP) load_b(c0, (n + 1) * KP);
        else if (c0 + 128 < end) load_b(c0 + 128, 0);
        // one barrier a turn: the buffer written next was last read before it
        lin_lds_barrier();
        expand_mfma<KP>(smem + buf * kBuf, r, h, hi[n], lo[n], acc);
        buf ^= 1;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (c0 + 8 * r >= end || row[i] < 0) continue;
      float f[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f[2 * e] = bf16_lo(yv[i][e]) + acc[2 * e][i];
        f[2 * e + 1] = bf16_hi(yv[i][e]) + acc[2 * e + 1][i];
      }
      u32x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = pack_bf16x2(f[2 * e], f[2 * e + 1]);
      if (id < 0) o = yv[i];
      // base and out non-temporal: whole lines, used once (16384 rows on qkv, caches cold: 74.0 us for
      // the three launches, 77.7 with ordinary loads, 81.7 with ordinary stores as well)
      __builtin_nontemporal_store(o, reinterpret_cast<u32x4*>(p.out + row[i] * p.out_stride + c0 + 8 * r));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) yv[i] = next[i];
  }
}

// ---------------------------------------------------------------- sorting ---------------

// One work-group: every row's place among the rows of its adapter (bucket num_adapters: none), the
// buckets' first tiles, then every row's position. A lane has 4 neighbouring rows, a wavefront 256
// at a time; 256 rows of one adapter, the common case of a prefill step, count as one entry, and the
// entries of all kPlanTurns turns ask the counters in one LDS atomic, lane i for turn i. The work is
// instructions on one CU, so what is done per row is what counts: 16384 rows of 8 adapters 11.8 us
// with one row a lane, 7.0 so.
// Rows of one adapter come in any order, which no result shows: a row's sums are its own.
typedef int32_t i32x4_u __attribute__((ext_vector_type(4), aligned(4)));

__global__ __launch_bounds__(kPlanThreads) void lora_plan_kernel(const LoraArgs p) {
  extern __shared__ int32_t count[];  // rows of every bucket, and behind them its first tile
  __shared__ int32_t part[kPlanThreads / kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int32_t buckets = p.num_adapters + 1;
  int32_t* first_tile = count + buckets;
  for (int32_t b = threadIdx.x; b < buckets; b += kPlanThreads) count[b] = 0;
  __syncthreads();
  constexpr int kTurn = 4 * kPlanThreads, kStep = kPlanTurns * kTurn;
  const bool one_step = p.rows <= kStep;  // then adapters and places stay in registers
  int32_t b[kPlanTurns][4], place[kPlanTurns][4];
  const int32_t my_row = 4 * (int32_t)threadIdx.x;
  const auto load_ids = [&](int32_t row0) {
#pragma unroll
    for (int i = 0; i < kPlanTurns; ++i) {
      const int32_t row = row0 + i * kTurn + my_row;
      if (row + 3 < p.rows) {
        const i32x4_u v = *reinterpret_cast<const i32x4_u*>(p.ids + row);
#pragma unroll
        for (int e = 0; e < 4; ++e) b[i][e] = v[e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) b[i][e] = p.ids[min(row + e, p.rows - 1)];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) b[i][e] = b[i][e] >= 0 && b[i][e] < p.num_adapters ? b[i][e] : p.num_adapters;
    }
  };
  for (int32_t row0 = 0; row0 < p.rows; row0 += kStep) {
    load_ids(row0);
    uint32_t mixed = 0;
    int32_t bucket = 0, n = 0;  // of turn `lane`
#pragma unroll
    for (int i = 0; i < kPlanTurns; ++i) {
      const int32_t left = p.rows - (row0 + i * kTurn + 4 * kWave * wave);  // rows from the wavefront's first on
      if (left <= 0) continue;
      // (rows past the end repeat the last one's id: the same bucket as a row that counts)
      const int32_t first = __builtin_amdgcn_readfirstlane(b[i][0]);
      const bool other = b[i][0] != first || b[i][1] != first || b[i][2] != first || b[i][3] != first;
      if (__ballot(other) != 0) mixed |= 1u << i;
      else if (lane == i) {
        bucket = first;
        n = min(left, 4 * kWave);
      }
    }
    int32_t at = 0;
    if (n > 0) at = atomicAdd(count + bucket, n);
#pragma unroll
    for (int i = 0; i < kPlanTurns; ++i) {
      const int32_t row = row0 + i * kTurn + my_row, mine = min(p.rows - row, 4);
      int32_t first = __builtin_amdgcn_readlane(at, i) + 4 * lane;
      const bool same = b[i][0] == b[i][1] && b[i][0] == b[i][2] && b[i][0] == b[i][3];
      if ((mixed >> i & 1) && same && mine > 0) first = atomicAdd(count + b[i][0], mine);
#pragma unroll
      for (int e = 0; e < 4; ++e) place[i][e] = first + e;
      if ((mixed >> i & 1) && !same) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < mine) place[i][e] = atomicAdd(count + b[i][e], 1);
      }
      if (!one_step) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e < mine) p.place[row + e] = place[i][e];
      }
    }
  }
  __syncthreads();
  // the buckets' first tiles: an exclusive sum over them, a stretch of neighbours a thread
  const int32_t per = (buckets + kPlanThreads - 1) / kPlanThreads;
  const int32_t b0 = min((int32_t)threadIdx.x * per, buckets), b1 = min(b0 + per, buckets);
  int32_t t = 0;
  for (int32_t i = b0; i < b1; ++i) t += (count[i] + kLoraTile - 1) / kLoraTile;
  int32_t it = t;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int32_t o = __shfl_up(it, d, kWave);
    if (lane >= d) it += o;
  }
  if (lane == kWave - 1) part[wave] = it;
  __syncthreads();
  it -= t;
  int32_t tiles = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / kWave; ++w) {
    if (w < wave) it += part[w];
    tiles += part[w];
  }
  for (int32_t i = b0; i < b1; ++i) {
    first_tile[i] = it;
    it += (count[i] + kLoraTile - 1) / kLoraTile;
  }
  for (int32_t i = tiles + threadIdx.x; i < p.max_tiles; i += kPlanThreads) p.tiles[i] = make_int2(-1, 0);
  __syncthreads();
  // row `row` of bucket c at place `at`: its position, and its tile's record if it is the tile's first
  const auto record = [&](int32_t c, int32_t at) {
    p.tiles[first_tile[c] + at / kLoraTile] =
        make_int2(c < p.num_adapters ? c : -1, min(count[c] - at, kLoraTile));
  };
  for (int32_t row0 = 0; row0 < p.rows; row0 += kStep) {
    if (!one_step) load_ids(row0);
#pragma unroll
    for (int i = 0; i < kPlanTurns; ++i) {
      const int32_t row = row0 + i * kTurn + my_row;
      if (!one_step) {
#pragma unroll
        for (int e = 0; e < 4; ++e) place[i][e] = p.place[min(row + e, p.rows - 1)];
      }
      if (row >= p.rows) continue;
      if (row + 3 < p.rows && b[i][0] == b[i][1] && b[i][0] == b[i][2] && b[i][0] == b[i][3]) {
        // four places in a row (counted together)
        const int32_t at = place[i][0], first = (at + kLoraTile - 1) / kLoraTile * kLoraTile;
        *reinterpret_cast<i32x4_u*>(p.perm + (int64_t)first_tile[b[i][0]] * kLoraTile + at) =
            i32x4_u{row, row + 1, row + 2, row + 3};
        if (first < at + 4) record(b[i][0], first);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (row + e >= p.rows) continue;
          const int32_t c = b[i][e], at = place[i][e];
          p.perm[(int64_t)first_tile[c] * kLoraTile + at] = row + e;
          if (at % kLoraTile == 0) record(c, at);
        }
      }
    }
  }
}

// ---------------------------------------------------------------- launches --------------

int64_t lora_max_tiles(int32_t rows, int32_t num_adapters) {
  return rows / kLoraTile + std::min<int64_t>((int64_t)num_adapters + 1, rows);
}

int32_t col_groups(const LoraArgs& p, int32_t cols) {
  int32_t n = 0;
  for (int q = 0; q < p.num_slices; ++q) n += (p.slice_begin[q + 1] - p.slice_begin[q] + cols - 1) / cols;
  return n;
}

// Groups that 16 rows can have, and groups of all rows.
int32_t tile_slots(const LoraArgs& p) { return std::min(std::min(kLoraSmallTile, p.num_adapters + 1), p.rows); }
int32_t small_slots(const LoraArgs& p) { return (p.rows + kLoraSmallTile - 1) / kLoraSmallTile * tile_slots(p); }

template <int KP, int WAVES, int kBase>
void launch_expand_waves(LoraArgs p, hipStream_t stream) {
  p.col_groups = col_groups(p, 128 * WAVES);
  hipLaunchKernelGGL((lora_expand_small_kernel<KP, WAVES, kBase>), dim3((unsigned)(small_slots(p) * p.col_groups)),
                     dim3(WAVES * kWave), 0, stream, p);
}

// Above rank 32 two wavefronts have all of B's 64 (of 128, twice 64) elements in flight: 128 rows on 3072
// x 1024, rank 64 6.5 us; four wavefronts and twice 32 elements 7.2.
template <int kBase>
hipError_t launch_expand_small(const LoraArgs& p, hipStream_t stream) {
  if (p.rank <= 16) launch_expand_waves<16, 4, kBase>(p, stream);
  else if (p.rank <= 32) launch_expand_waves<32, 4, kBase>(p, stream);
  else if constexpr (kBase != kBaseRowsShrink) launch_expand_waves<64, 2, kBase>(p, stream);
  return hipGetLastError();
}

// Whether a small addition computes t in the expand's work-groups (one launch, but every group of
// 512 columns reads its adapter's A again): where all of them are on the GPU at once, three a CU up to
// rank 16, two up to 32 (two chunks ahead in the shrink, not four, for that many). Measured, us in a graph over
// eight sets of tensors in turn, one launch and two (work-groups): k = 2048, 1024 columns, rank 16, 300 rows of
// 100 adapters (608) 11.5 and 12.4, 400 rows (800) 14.8 and 13.4; k = 3072, 300 rows of 20 (608) 11.8 and 12.9,
// 400 rows (800) 15.6 and 13.3; qkv (k = 1024), 96 rows of 16 (768) 8.3 and 10.9, 128 rows (1024) 8.9 and 11.5: a
// short k gains beyond the line too; rank 32, gate/up, 64 rows of 8 (432) 9.3 and 10.6, 96 rows (648) 12.6 and
// 11.2; k = 2048, 900 rows of 3 (456) 12.5 and 14.3.
bool shrink_in_expand(const LoraArgs& p) {
  return p.rank <= 32 && (int64_t)small_slots(p) * col_groups(p, 128 * kLoraWaves) <= (p.rank <= 16 ? 768 : 512);
}

template <int R>
void launch_shrink_rows(const LoraArgs& p, int64_t tiles, int32_t cb, int32_t blocks, hipStream_t stream) {
  const int64_t parts = (tiles * (kLoraTile / R) + 7) / 8 * 8;  // whole rounds of the XCDs
  const dim3 grid((unsigned)(parts * blocks)), block(kLoraThreads);
  switch (cb) {
    case 1: hipLaunchKernelGGL((lora_shrink_kernel<R, 1>), grid, block, 0, stream, p); break;
    case 2: hipLaunchKernelGGL((lora_shrink_kernel<R, 2>), grid, block, 0, stream, p); break;
    case 3: hipLaunchKernelGGL((lora_shrink_kernel<R, 3>), grid, block, 0, stream, p); break;
    default: hipLaunchKernelGGL((lora_shrink_kernel<R, 4>), grid, block, 0, stream, p); break;
  }
}

// At most 64 columns of t a work-group, shared evenly. 64 rows a work-group read A half as often as
// 32, but are half as many. The line is where they fill the GPU one and a half times; around it the two
// are within 4 % of a call, either way. Us a call in a graph, 32 and 64 rows (work-groups of 64): gate/up, rank 64,
// 8192 rows (256) 76.8 and 76.0, 12288 (384) 97.1 and 95.8, 16384 (512) 122.1 and 121.5; qkv, rank 16, 16384 rows
// (256) 77.1 and 77.4, 24576 (384) 115.6 and 114.6, 32768 (512) 144.3 and 146.6; 2048 x 1024, rank 16, 16384 rows
// (256) 41.6 and 42.1, 24576 (384) 72.4 and 69.9, 32768 (512) 90.7 and 94.5.
void launch_shrink_sorted(const LoraArgs& p, int64_t tiles, hipStream_t stream) {
  const int32_t cols16 = (p.num_slices * p.rank + 15) / 16, n = (cols16 + 3) / 4, cb = (cols16 + n - 1) / n;
  const int32_t blocks = (cols16 + cb - 1) / cb;
  if ((int64_t)p.rows / 64 * blocks >= 384)
    launch_shrink_rows<64>(p, tiles, cb, blocks, stream);
  else
    launch_shrink_rows<32>(p, tiles, cb, blocks, stream);
}

hipError_t launch_expand_sorted(LoraArgs p, int64_t tiles, hipStream_t stream) {
  p.col_groups = col_groups(p, kSortedCols);
  const dim3 grid((unsigned)(tiles * p.col_groups)), block(kLoraThreads);
  if (p.rank <= 16)
    hipLaunchKernelGGL((lora_expand_kernel<16, 1>), grid, block, 0, stream, p);
  else if (p.rank <= 32)
    hipLaunchKernelGGL((lora_expand_kernel<32, 1>), grid, block, 0, stream, p);
  else if (p.rank <= 64)
    hipLaunchKernelGGL((lora_expand_kernel<64, 1>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((lora_expand_kernel<64, 2>), grid, block, 0, stream, p);
  return hipGetLastError();
}

// Whether an addition works on groups of 16 rows, unsorted. What it costs grows with the groups that
// there may be, each with its work-groups of the shrink and the expand and the time of about four more. Sorting
// costs a launch in front, 5-8 us up to 16384 rows and 9 for every 16384 more (one work-group does it). The line
// of 20 a CU, 5120, is below the first place where sorting was the faster one. Unsorted and sorted, us a call in a
// graph over eight sets of tensors in turn, ids at random (count): qkv, rank 16, 512 rows of 8 adapters (4320) 18.3
// and 22.7, 768 (6480) 24.4 and 23.0; gate/up, rank 16, 768 rows of 4 (4320) 20.3 and 22.6, 1024 (5760) 24.2 and
// 23.4; rank 64, 128 rows of 20 (4608) 22.4 and 24.1, 256 (9216) 35.7 and 24.7; 3072 x 1024, rank 32, 512 rows of 20
// (4096) 22.8 and 25.4, 768 (6144) 28.8 and 26.5. Others cross later and lose up to 4 us between: 2048 x 1024, rank
// 16, 768 rows of 100 (5376) 18.5 and 22.3, 1024 (7168) 20.8 and 22.7, 1280 (8960) 24.7 and 23.1. So do long runs
// of one adapter, which leave most groups empty (qkv, 1024 rows of 8, 8640: 17.2 and 23.5), but the host does not
// know the ids.
bool small_add(const LoraArgs& p) {
  if (p.num_adapters > kLoraMaxSorted) return true;  // the sort's counters would not fit its LDS
  const int32_t each = 4 + col_groups(p, p.rank <= 32 ? 512 : 256) + (p.num_slices * p.rank + 15) / 16;
  return (int64_t)small_slots(p) * each <= 20 * 256;
}

// Whether the projection's work-groups add the adapters themselves (the shrink before them) rather
// than leave partial sums to an expand. Measured, us of the two forms' kernels: 97 rows, 1024 x 6144, rank
// 16 15.2 and 16.7; 1 row, 1024 x 4096 8.9 and 9.7 (in two launches).
bool expand_in_linear(const LoraArgs& p, const LinCfg& c) { return c.ks == 1 && p.rank <= 16; }

size_t t_bytes(const LoraArgs& p) { return (size_t)p.rows * p.num_slices * p.rank * sizeof(float); }

}  // namespace

size_t lora_linear_workspace_bytes(const LoraArgs& p) {
  const LinCfg c = choose_config(p.rows, p.n_out / kLinTile, p.k, 1);
  if (expand_in_linear(p, c)) return p.rows <= kOneLaunchRows ? 0 : t_bytes(p);
  return t_bytes(p) + (size_t)c.ks * p.rows * p.n_out * sizeof(float);
}

size_t lora_add_workspace_bytes(const LoraArgs& p) {
  if (small_add(p)) return shrink_in_expand(p) ? 0 : t_bytes(p);
  return t_bytes(p) + (size_t)lora_max_tiles(p.rows, p.num_adapters) * (kLoraTile * sizeof(int32_t) + sizeof(int2)) +
         (size_t)p.rows * sizeof(int32_t);
}

int64_t lora_add_groups(const LoraArgs& p) {
  const bool small = small_add(p);
  const int64_t tiles = small ? small_slots(p) : lora_max_tiles(p.rows, p.num_adapters);
  // (an unsorted expand has 256 columns or more a work-group; a shrink 32 rows and 64 columns of t)
  return tiles * std::max<int64_t>(col_groups(p, small ? 256 : kSortedCols),
                                   2 * ((p.num_slices * p.rank + (small ? 15 : 63)) / (small ? 16 : 64)));
}

hipError_t launch_lora_linear(const LoraArgs& args, const void* w, int64_t w_stride, void* ws, hipStream_t stream) {
  LoraArgs p = args;
  p.tile_slots = tile_slots(p);
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
  const int32_t cols16 = (p.num_slices * p.rank + 15) / 16;
  if (expand_in_linear(p, c)) {
    a.y = p.out;
    a.y_stride = p.out_stride;
    const bool here = p.rows <= kOneLaunchRows;
    if (p.num_adapters > 0 && !here) {
      hipLaunchKernelGGL(lora_shrink_small_kernel, dim3(small_slots(p) * cols16), dim3(kLoraThreads), 0, stream, p);
      if (hipError_t err = hipGetLastError(); err != hipSuccess) return err;
    }
    const auto launch = [&](auto nb) {
      if (here)
        hipLaunchKernelGGL((lora_linear_expand_kernel<nb.value, true>), dim3(lin_groups), dim3(kLinThreads), 0, stream,
                           a, p);
      else
        hipLaunchKernelGGL((lora_linear_expand_kernel<nb.value, false>), dim3(lin_groups), dim3(kLinThreads), 0, stream,
                           a, p);
    };
    switch (c.nb) {
      case 1: launch(std::integral_constant<int, 1>{}); break;
      case 2: launch(std::integral_constant<int, 2>{}); break;
      default: launch(std::integral_constant<int, 4>{}); break;
    }
    return hipGetLastError();
  }
  // 32 columns of t a work-group where there would be too many of 16 to be resident beside the
  // projection's (two a CU): 128 rows, rank 64, k = 3072 11.8 us instead of 13.4
  const bool wide = small_slots(p) * cols16 >= 512;
  const int32_t shrink = p.num_adapters > 0 ? small_slots(p) * (wide ? (cols16 + 1) / 2 : cols16) : 0;
  const dim3 grid(lin_groups + shrink), block(kLinThreads);
  const auto launch = [&](auto nb, auto cb) {
    hipLaunchKernelGGL((lora_linear_kernel<nb.value, cb.value>), grid, block, 0, stream, a, p, lin_groups);
  };
  const auto launch_nb = [&](auto nb) {
    if (wide) launch(nb, std::integral_constant<int, 2>{});
    else launch(nb, std::integral_constant<int, 1>{});
  };
  switch (c.nb) {
    case 1: launch_nb(std::integral_constant<int, 1>{}); break;
    case 2: launch_nb(std::integral_constant<int, 2>{}); break;
    default: launch_nb(std::integral_constant<int, 4>{}); break;
  }
  if (hipError_t err = hipGetLastError(); err != hipSuccess) return err;
  return launch_expand_small<kBasePartial>(p, stream);
}

hipError_t launch_lora_add(const LoraArgs& args, void* ws, hipStream_t stream) {
  LoraArgs p = args;
  p.tile_slots = tile_slots(p);
  p.t = static_cast<float*>(ws);
  const int32_t width = p.num_slices * p.rank;
  if (small_add(p)) {
    if (shrink_in_expand(p)) return launch_expand_small<kBaseRowsShrink>(p, stream);
    if (p.num_adapters > 0) {
      hipLaunchKernelGGL(lora_shrink_small_kernel, dim3(small_slots(p) * ((width + 15) / 16)), dim3(kLoraThreads), 0,
                         stream, p);
      if (hipError_t err = hipGetLastError(); err != hipSuccess) return err;
    }
    return launch_expand_small<kBaseRows>(p, stream);
  }
  const int64_t tiles = lora_max_tiles(p.rows, p.num_adapters);
  char* at = static_cast<char*>(ws) + t_bytes(p);
  p.max_tiles = (int32_t)tiles;
  p.perm = reinterpret_cast<int32_t*>(at);
  p.tiles = reinterpret_cast<int2*>(p.perm + tiles * kLoraTile);
  p.place = reinterpret_cast<int32_t*>(p.tiles + tiles);
  hipLaunchKernelGGL(lora_plan_kernel, dim3(1), dim3(kPlanThreads), 2 * (p.num_adapters + 1) * sizeof(int32_t), stream,
                     p);
  if (hipError_t err = hipGetLastError(); err != hipSuccess) return err;
  if (p.num_adapters > 0) {
    launch_shrink_sorted(p, tiles, stream);
    if (hipError_t err = hipGetLastError(); err != hipSuccess) return err;
  }
  return launch_expand_sorted(p, tiles, stream);
}

}  // namespace pk
