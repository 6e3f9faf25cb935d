// The weight-streaming tile of the decode-step linear layers (at most 128 token rows), shared by
// the plain layers (linear.hip) and the layers with per-row adapters beside them (lora.hip).
// linear.hip's header says how a launch is cut into work-groups and what the MFMA layout is.
#pragma once

#include "common.h"

namespace pk {
namespace {

constexpr int kLinThreads = 256;   // four wavefronts
constexpr int kLinTile = 32;       // weight rows (output columns) per tile
constexpr int kLinKBlock = 64;     // K elements per wavefront block (4 MFMA steps)
constexpr int kLinChunk = 4 * kLinKBlock;  // K elements per LDS stage (one block per wavefront)
#ifndef PK_LINEAR_TARGET_GROUPS
#define PK_LINEAR_TARGET_GROUPS 256
#endif
#ifndef PK_LINEAR_MIN_GROUPS
#define PK_LINEAR_MIN_GROUPS 64
#endif
#ifndef PK_LINEAR_MT2_ROWS
#define PK_LINEAR_MT2_ROWS 64
#endif
constexpr int kLinTargetGroups = PK_LINEAR_TARGET_GROUPS;  // work-groups a split launch aims for
constexpr int kLinMinGroups = PK_LINEAR_MIN_GROUPS;        // smallest grid left unsplit
constexpr int kLinMaxChunks = 4;                           // longest unsplit K walk (chunks)
constexpr int kLinMt2Rows = PK_LINEAR_MT2_ROWS;            // more rows: two row tiles per group

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 bf16x8_t;
// 16-byte register value for the staged loads (a native vector: HIP's uint4 struct is
// copied through private memory by the staging loops)
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float silu_mul(float g, float u) {
  const float gb = bf16_lo(pack_bf16x2(g, 0.f));  // g and u rounded to bf16 (the GEMM output)
  const float ub = bf16_lo(pack_bf16x2(u, 0.f));
  return gb / (1.0f + expf(-gb)) * ub;
}

enum Epi { kEpiStore = 0, kEpiSiluMul = 1, kEpiPartial = 2 };

struct LinArgs {
  const uint16_t* x;
  int64_t x_stride;
  const uint16_t* w;
  int64_t w_stride;
  int32_t rows;
  int32_t n_out;     // output columns (inter for SiLU * mul)
  int32_t k;
  int32_t ks;        // K splits
  uint16_t* y;       // bf16 output (store / SiLU epilogue)
  int64_t y_stride;
  float* part;       // [ks][rows][np * n_out] fp32 partial sums
};

// LDS of linear_tile: two stages of the operand tiles, or the four wavefronts' sums.
constexpr int lin_smem_bytes(int np, int mt) {
  const int stages = 2 * (np + mt) * 32 * kLinChunk * 2, sums = 4 * np * 4 * kWave * 16;
  return stages > sums ? stages : sums;
}

// Waits for this wavefront's LDS operations, then for every wavefront of the work-group.
// s_waitcnt lgkmcnt(0) on its own: __syncthreads() would also wait for vmcnt(0), i.e. for
// the global loads of later K chunks that are still in flight.
__device__ __forceinline__ void lin_lds_barrier() {
  __builtin_amdgcn_s_waitcnt((15 & 15) | ((63 >> 4) << 14) | (7 << 4) | (0 << 8));  // lgkmcnt(0) only
  asm volatile("s_barrier" ::: "memory");
}

// NP = weight tiles per work-group (2: gate rows n0.., up rows n_out + n0..); MT = 32-row x
// tiles per work-group; NB = 256-wide K chunks whose global loads are issued together.
//
// Loads: a 32-row x 256-column operand tile (16 KB) is read by the 256 threads as four
// instructions of 8 rows x 512 contiguous bytes (thread t: row 8 i + t / 32, 16-byte
// column t % 32), so every 4-lane quad reads 64 bytes of one row. (Loading the MFMA layout
// straight from memory puts 32 different rows in one instruction and 4 in every quad,
// which costs four L1 tag lookups per quad.) The tile goes to LDS with 16-byte column c of
// row r at r * 512 + ((c ^ r) & 31) * 16, so the stores and the MFMA operand reads
// (16 lanes = 16 rows of one column) are free of bank conflicts. Two LDS stages: chunk c
// is stored in stage c & 1 while the other stage may still be read for chunk c - 1.
// Wavefront w multiplies the 64 columns [64 w, 64 w + 64) of every chunk.
// What an epilogue adds to the sums of a work-group's 32 x 32 outputs (NP = MT = 1) before they are
// rounded: load is called before the K walk; after it prepare, which has all of the LDS, put and add, with
// barriers between the three and LDS of their own for the last two. Thread (c, q) adds to row c,
// columns 4 q .. 4 q + 3. Here: nothing.
struct NoAddend {
  __device__ __forceinline__ void load(int row0, int n0) {}
  __device__ __forceinline__ void prepare(char* lds) {}
  __device__ __forceinline__ void put(char* lds) const {}
  __device__ __forceinline__ void add(const char* lds, float4& v) const {}
};

// `block` is the work-group's index in the launch shape of choose_config, `smem` its
// lin_smem_bytes(NP, MT) bytes of LDS.
template <int NP, int MT, int NB, int EPI, class Addend>
__device__ __forceinline__ void linear_tile(const LinArgs a, const int block, char* smem, Addend addend) {
  constexpr int kOps = NP + MT;               // operand tiles per chunk
  constexpr int kTileBytes = 32 * kLinChunk * 2;
  constexpr int kStage = kOps * kTileBytes;
  constexpr int kSumBytes = 4 * NP * 4 * kWave * 16;  // the four wavefronts' sums of one x tile
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = threadIdx.x / kWave;
  const int r = lane & 31, h = lane >> 5;
  const int ntiles = a.n_out / kLinTile;
  const int per_group = ntiles * a.ks;  // work-groups of one row group
  const int mgroup = block / per_group;
  const int rem = block - mgroup * per_group;
  const int split = rem / ntiles;
  const int n0 = (rem - split * ntiles) * kLinTile;
  const int row0 = mgroup * MT * 32;
  const int kc = a.k / a.ks;
  const int kbeg = split * kc;

  // loader: thread row lr (+ 8 i), 16-byte column lc
  const int lr = threadIdx.x >> 5, lc = threadIdx.x & 31;
  const uint16_t* src[kOps][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int p = 0; p < NP; ++p)
      src[p][i] = a.w + (int64_t)(p * a.n_out + n0 + 8 * i + lr) * a.w_stride + kbeg + 8 * lc;
#pragma unroll
    for (int t = 0; t < MT; ++t)
      src[NP + t][i] =
          a.x + (int64_t)min(row0 + 32 * t + 8 * i + lr, a.rows - 1) * a.x_stride + kbeg + 8 * lc;
  }
  int wofs[4], rofs[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 8 * i + lr;
    wofs[i] = row * (2 * kLinChunk) + ((lc ^ row) & 31) * 16;
    const int cc = 8 * wave + 4 * h + i;  // MFMA step i reads 16-byte column cc of row r
    rofs[i] = r * (2 * kLinChunk) + ((cc ^ r) & 31) * 16;
  }

  addend.load(row0, n0);

  f32x16 acc[NP][MT];
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[p][t][i] = 0.f;

  const int nch = kc / kLinChunk;
  for (int j0 = 0; j0 < nch; j0 += NB) {
    u32x4_t st[NB][kOps][4];
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int o = 0; o < kOps; ++o)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          st[j][o][i] = *reinterpret_cast<const u32x4_t*>(src[o][i] + (j0 + j) * kLinChunk);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      char* stage = smem + ((j0 + j) & 1) * kStage;
#pragma unroll
      for (int o = 0; o < kOps; ++o)
#pragma unroll
        for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x4_t*>(stage + o * kTileBytes + wofs[i]) = st[j][o][i];
      lin_lds_barrier();
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        u32x4_t xv[MT];
#pragma unroll
        for (int t = 0; t < MT; ++t) xv[t] = *reinterpret_cast<const u32x4_t*>(stage + (NP + t) * kTileBytes + rofs[q]);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          const u32x4_t wv = *reinterpret_cast<const u32x4_t*>(stage + p * kTileBytes + rofs[q]);
#pragma unroll
          for (int t = 0; t < MT; ++t)
            acc[p][t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, wv),
                                                                __builtin_bit_cast(bf16x8_t, xv[t]),
                                                                acc[p][t], 0, 0, 0);
        }
      }
    }
  }
  __syncthreads();  // every wavefront is done with the stages before they hold the sums
  addend.prepare(smem);
  auto red = reinterpret_cast<float4 (*)[NP][4][kWave]>(smem);

  // Add the four wavefronts' accumulators one x-row tile at a time. Thread (c, q) then owns
  // x row 32 t + c and the 4 output columns n0 + 4 q .. + 3: D elements 4 (q >> 1) .. + 3 of
  // lane c + 32 (q & 1), stored as one float4 per lane and element quad.
  const int c = threadIdx.x >> 3, q = threadIdx.x & 7;
  const int n = n0 + 4 * q;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    if (t) __syncthreads();
#pragma unroll
    for (int p = 0; p < NP; ++p)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        red[wave][p][j][lane] = make_float4(acc[p][t][4 * j], acc[p][t][4 * j + 1], acc[p][t][4 * j + 2],
                                            acc[p][t][4 * j + 3]);
    addend.put(smem + kSumBytes);
    __syncthreads();
    const int m = row0 + 32 * t + c;
    float4 v[NP];
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const float4 a0 = red[0][p][q >> 1][c + 32 * (q & 1)], a1 = red[1][p][q >> 1][c + 32 * (q & 1)];
      const float4 a2 = red[2][p][q >> 1][c + 32 * (q & 1)], a3 = red[3][p][q >> 1][c + 32 * (q & 1)];
      v[p] = make_float4(a0.x + a1.x + a2.x + a3.x, a0.y + a1.y + a2.y + a3.y, a0.z + a1.z + a2.z + a3.z,
                         a0.w + a1.w + a2.w + a3.w);
    }
    if (m < a.rows) {
      if constexpr (EPI == kEpiStore) {
        addend.add(smem + kSumBytes, v[0]);
        *reinterpret_cast<uint2*>(a.y + (int64_t)m * a.y_stride + n) =
            make_uint2(pack_bf16x2(v[0].x, v[0].y), pack_bf16x2(v[0].z, v[0].w));
      } else if constexpr (EPI == kEpiSiluMul) {
        *reinterpret_cast<uint2*>(a.y + (int64_t)m * a.y_stride + n) =
            make_uint2(pack_bf16x2(silu_mul(v[0].x, v[NP - 1].x), silu_mul(v[0].y, v[NP - 1].y)),
                       pack_bf16x2(silu_mul(v[0].z, v[NP - 1].z), silu_mul(v[0].w, v[NP - 1].w)));
      } else {
        float* pp = a.part + ((int64_t)split * a.rows + m) * (NP * a.n_out) + n;
#pragma unroll
        for (int p = 0; p < NP; ++p) *reinterpret_cast<float4*>(pp + p * a.n_out) = v[p];
      }
    }
  }
}

// Launch shape: MT row tiles per work-group, row groups, K splits, blocks per load batch.
struct LinCfg {
  int mt, mgroups, ks, nb;
};

// K is left unsplit when the grid of (weight tile x 32-row tile) work-groups has at least
// kLinMinGroups entries and a work-group then walks at most kLinMaxChunks 256-wide
// chunks; otherwise KS is the smallest divisor of K / 256 whose grid reaches
// kLinTargetGroups (K / 256 at most). KS does not depend on the epilogue, so every
// epilogue sums the same products in the same order and the fused entry points equal
// linear + the standalone epilogue kernels bit for bit. The merged gate / up weight
// (np = 2) takes two row tiles per work-group above kLinMt2Rows rows, which keeps its
// grid within one work-group per CU (its stages take 128 KB of LDS); row tiles do not
// change any sum. Wavefronts batch the loads of up to four chunks.
LinCfg choose_config(int rows, int tiles, int k, int np) {
  LinCfg c{};
  const int64_t base = (int64_t)tiles * ((rows + 31) / 32);
  const int blocks = k / kLinChunk;
  c.ks = blocks;
  if (base >= kLinMinGroups && blocks <= kLinMaxChunks) {
    c.ks = 1;
  } else {
    for (int s = 1; s < blocks; ++s)
      if (blocks % s == 0 && base * s >= kLinTargetGroups) {
        c.ks = s;
        break;
      }
  }
  c.mt = np == 2 && rows > kLinMt2Rows ? 2 : 1;
  c.mgroups = (rows + 32 * c.mt - 1) / (32 * c.mt);
  const int chunks = blocks / c.ks;  // 256-wide K chunks per work-group
  c.nb = chunks % 4 == 0 ? 4 : chunks % 2 == 0 ? 2 : 1;
  return c;
}

}  // namespace
}  // namespace pk
