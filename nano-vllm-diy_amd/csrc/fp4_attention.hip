// Attention over a paged K/V cache held in 4 bits (format: fp4.h), for any mixture of sequences: one query row, a
// few (drafted tokens), or chunks of a prompt.
//
// Reference: the flash_attn_varlen_func call over paged K/V (src/layers/attention.py:95-104), whose mask and GQA
// rules hold here; the reference has no 4-bit cache. For query row r of a sequence with Lq rows and Lk keys
//     o = sum_t p_t V[t] / sum_t p_t,   p_t = exp2(c q.K[t] - m),   t <= r + Lk - Lq,   c = scale log2(e)
// with K[t], V[t] the rows' values. One pass over the keys: m is a reference at most 8 below the largest score so
// far (in the exp2 domain); while it holds, nothing is rescaled, and p stays below 2^8. Scores, p's sum and the
// output are fp32; p is rounded to bf16 for the matrix product, as the 16-bit cache's kernels round it.
// Sums p V must stay in fp32's range where their mean does: below 6 x 2^64 (scale bytes below kLargeScale) 2^22 keys
// and weights of 2^8 do; a wavefront that meets a larger scale of V raises its reference by kRaise, and weights of at most
// 2^-24, over 2^22 keys of at most 6 x 2^125, stay below 2^126. Weights below 2^-94 of the largest then vanish, in place of 2^-126.
//
// Columns. A kv head's query heads and a sequence's query rows are the columns of one matrix product: column
// r G + i is query head i of the group and row r. A wavefront holds T tiles of 16 columns of one kv head:
//   S^T = K Q^T  v_mfma_f32_16x16x32_bf16, 16 keys x 16 columns: lane l holds key l % 16.
//   O^T += V^T P^T  lane l of S^T has column l % 16 and keys 16 t + 4 (l / 16) + i (tile t, i < 4): as the operand
//                P^T of the next product these are the 8 keys of its lane for two tiles, so P never changes lanes.
// Values convert to bf16 with their scale in one instruction for two. (The matrix instructions that read 4-bit
// values with their scales keep about 12 bits below the largest product of a sum, measured; scores here are
// held in 32, so they are not used.) The two kinds of work-groups differ in who converts:
//   few rows (rows x group <= 16): T = 1, a tile of work is all of a sequence's rows and up to 8 kv heads, and a
//       wavefront converts the keys that it takes, 32 of one head at once, straight into the products' operands. Of
//       K, lane l has of key l % 16 the 32 dimensions from 32 (l / 16): 16 consecutive bytes with one scale byte; the
//       product runs over them 8 at a time, and q is laid out in the same order of dimensions. Of V, lane l loads 4
//       bytes of each of its 8 keys, the dimensions 8 (l % 16) .. + 7, and dimension 8 (l % 16) + j is row l % 16 of
//       the j-th of 8 products: the output's rows are a permutation of the dimensions and V needs no transposition,
//       two keys' values of one dimension are put side by side by a byte permute.
//   more rows: T = 2, a tile of work is 256 columns of one kv head, a wavefront 32 of them, and the work-group
//       converts a step's rows once for its wavefronts.
//
// Work. The steps of every tile lie end to end on a line, which is cut into `runs` equal runs, one work-group each,
// whatever the lengths: a work-group takes the end of one tile, whole tiles and the beginning of another. A tile that
// a cut splits leaves fp32 partial results (o, m, sum), which a second kernel merges; a cut splits at most one tile,
// so there are at most two partial results a run. The lengths are on the GPU only, so a launch has work-groups of both
// kinds wherever the call's bounds allow sequences of more than 16 columns; those without any end at once.
#include <algorithm>

#include "fp4.h"

namespace pk {
namespace {

constexpr int kFewWaves = 8;          // wavefronts of a work-group over sequences of few rows
constexpr int kFewRing = 3;           // steps in LDS
constexpr int kManyWaves = 8;         // ... of more rows
constexpr int kManyTiles = 2;         // tiles of 16 columns a wavefront of the latter holds
constexpr int kManyCols = kManyWaves * kManyTiles * 16;
constexpr int kManyStep = 64;         // keys of its step
constexpr int kManyRing = 4;          // steps of 4-bit rows in LDS
constexpr int kSub = 32;              // keys a wavefront takes at once
constexpr int kGroups = 16;           // groups of 64 sequences that are in LDS at a time
constexpr int kChunk = kGroups * kWave;
constexpr float kLowest = -3.402823466e38f;
constexpr float kSlack = 8.f;         // the scores may exceed their reference by this (exp2 domain)
constexpr float kRaise = 32.f;        // what the reference is raised by for large rows of V
constexpr uint32_t kLargeScale = 192; // their scale bytes: the two highest bits set

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 frag;
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) uint32_t lds_u32;
typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) u32x2 lds_u32x2;
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
typedef __attribute__((address_space(3))) int lds_i32;
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) i32x4 lds_i32x4;
typedef __attribute__((address_space(3))) float lds_f32;
typedef __attribute__((address_space(3))) f32x2 lds_f32x2;

__device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(frag, a), __builtin_bit_cast(frag, b), c, 0, 0, 0);
}

// The maximum and the sum over the four lanes l, l ^ 16, l ^ 32, l ^ 48, in all of them.
__device__ __forceinline__ float quarters_max(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float quarters_sum(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// An entry of a list that no kernel here writes, at a position that is the same for the wavefront: a scalar load,
// which does not wait for the vector loads in flight as a vector load's use would.
__device__ __forceinline__ int scalar_i32(const int32_t* p) {
  typedef __attribute__((address_space(4))) const int32_t* constant;
  return uniform(*(constant)reinterpret_cast<uintptr_t>(p));
}

// a + b of counts, at most INT32_MAX: lengths that are no cumulative ones may add up to more steps than a call can
// have, which must not come back as few.
__device__ __forceinline__ int add_sat(int a, int b) { return __builtin_elementwise_add_sat(a, b); }

// Inclusive sum over the wavefront.
__device__ __forceinline__ int scan64(int v, int lane) {
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));  // row_shr:1, :2, :4, :8
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
  v = add_sat(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = __builtin_amdgcn_readlane(v, 31),
            r2 = __builtin_amdgcn_readlane(v, 47);
  const int row = lane >> 4;
  return add_sat(add_sat(add_sat(v, row >= 1 ? r0 : 0), row >= 2 ? r1 : 0), row >= 3 ? r2 : 0);
}

// A sequence of the call: its first query row, the rows that are computed, and the keys. causal rows are aligned by
// the true number of rows, which max_seqlen_q only cuts.
struct Seq {
  int q0, rows, shift, keys;  // row r sees keys t <= r + shift
};
__device__ __forceinline__ Seq make_seq(const Fp4AttnArgs& a, int q0, int q1, int k0, int k1) {
  Seq s;
  s.q0 = q0;
  s.keys = min(k1 - k0, a.max_seqlen_k);
  s.rows = s.keys > 0 && q0 >= 0 ? (int)min((int64_t)min(q1 - q0, a.max_seqlen_q), a.num_rows - q0) : 0;
  s.shift = a.causal ? s.keys - (q1 - q0) : s.keys;
  return s;
}
__device__ __forceinline__ Seq seq_of(const Fp4AttnArgs& a, int b) {
  return make_seq(a, a.cu_q[b], a.cu_q[b + 1], a.cu_k[b], a.cu_k[b + 1]);
}
// Steps of STEP keys of tile j of a sequence: up to the last key its last row sees, at least one.
template <bool MANY, int STEP>
__device__ __forceinline__ int tile_steps(const Fp4AttnArgs& a, const Seq& s, int j) {
  const int per_tile = MANY ? kManyCols >> a.group_shift : s.rows;
  const int last = min(s.rows, (j + 1) * per_tile) - 1;
  const int end = min(s.keys, last + s.shift + 1);
  return max(1, (end + STEP - 1) / STEP);
}

// Steps of a sequence on the line of one kv head (MANY) or of all kv heads; 0 where it is on the other line.
template <bool MANY, int STEP>
__device__ __forceinline__ int seq_steps(const Fp4AttnArgs& a, const Seq& s) {
  if (s.rows <= 0 || (s.rows << a.group_shift > 16) != MANY) return 0;
  if constexpr (!MANY) return tile_steps<false, STEP>(a, s, 0);
  const int tiles = ((s.rows << a.group_shift) + kManyCols - 1) / kManyCols;
  int n = 0;
  for (int j = 0; j < tiles; ++j) n += tile_steps<true, STEP>(a, s, j);
  return n;
}

// A tile of query rows on the line: steps [start, start + steps) of it.
struct Tile {
  Seq seq;
  int b, head, j;    // sequence, kv head (MANY), tile of it
  int64_t start;
  int steps;
};

// Waits until the wavefronts' reads and writes of LDS are over.
__device__ __forceinline__ void meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// n / d rounded down, of whole numbers below 2^53, the same for the wavefront: a quotient that is not whole is at least
// 1 / d below the next one, more than 2^-53 of it, so the rounding of 64-bit floating point does not reach it. (An
// eighth of the instructions of the division of 64-bit integers.)
__device__ __forceinline__ int64_t div_floor(int64_t n, int64_t d) {
  const int64_t q = (int64_t)((double)n / (double)d);
  return (int64_t)((uint64_t)(uint32_t)uniform((int)(q >> 32)) << 32 | (uint32_t)uniform((int)q));
}

// The line of steps: MANY: kv head by kv head, sequence by sequence, tile by tile; otherwise the sequences' steps,
// which the wavefronts take for a kv head each. A chunk's steps are summed up in LDS, a thread to a sequence, and looked
// up from there, the sequence's lengths with them. (With every wavefront keeping the steps of 512 sequences in
// registers, and beginning with the first of all sequences for every piece: 106 us in place of 74 for 1024 sequences of
// 100-400 keys, 5165 in place of 357 for 16384 of 16-64, 36.8 in place of 34.4 for 128 of 100-2048.)
template <bool MANY, int STEP>
struct Line {
  static constexpr int kBytes = kChunk * 20 + kGroups * 4;
  lds_i32x4* seqs;   // [kChunk] Seq
  lds_i32* sums;     // [kChunk] steps of a group of 64 sequences up to and with each of them, [kGroups] of whole groups
  int base, before;  // the chunk's first sequence, the steps before it
  int per_head;      // steps of all sequences
  int64_t total;

  // (every wavefront of the work-group comes here)
  __device__ __forceinline__ void load(const Fp4AttnArgs& a, int first, int steps_before, int wave, int lane) {
    base = first;
    before = steps_before;
    meet();  // the last chunk has been read
#pragma unroll 1
    for (int group = wave; group < kGroups; group += 8) {
      int sum = 0;
      if (first + 64 * group < a.num_seqs) {
        const int b = first + 64 * group + lane;
        if (b < a.num_seqs) {
          const Seq s = seq_of(a, b);
          seqs[64 * group + lane] = i32x4{s.q0, s.rows, s.shift, s.keys};
          sum = seq_steps<MANY, STEP>(a, s);
        }
        sum = scan64(sum, lane);
        sums[64 * group + lane] = sum;
      }
      if (lane == kWave - 1) sums[kChunk + group] = sum;
    }
    meet();
  }
  // Steps of the chunk's groups up to and with each, a lane a group (the same in all lanes past the last).
  __device__ __forceinline__ int group_ends(int lane) const { return scan64(lane < kGroups ? sums[kChunk + lane] : 0, lane); }
  __device__ __forceinline__ void init(const Fp4AttnArgs& a, lds_u8* lds, int wave, int lane) {
    seqs = (lds_i32x4*)lds;
    sums = (lds_i32*)(lds + kChunk * 16);
    int64_t sum = 0;
    for (int first = 0; first < a.num_seqs; first += kChunk) {
      load(a, first, (int)sum, wave, lane);
      sum = min(sum + __builtin_amdgcn_readlane(group_ends(lane), kWave - 1), (int64_t)INT32_MAX);
    }
    per_head = sum < INT32_MAX ? (int)sum : 0;  // (the call's bounds allow fewer steps: there is no work in such lengths)
    total = MANY ? (int64_t)per_head * a.num_kv_heads : per_head;
  }
  // The tile at position p < total. (Positions that grow walk the chunks once.)
  __device__ __forceinline__ Tile at(const Fp4AttnArgs& a, int64_t p, int wave, int lane) {
    Tile t;
    t.head = MANY ? (int)div_floor(p, per_head) : 0;
    t.j = 0;
    const int64_t head_start = (int64_t)t.head * per_head;
    const int want = (int)(p - head_start);
    if (want < before) load(a, 0, 0, wave, lane);
    int group_end = before + group_ends(lane);
    while (want >= __builtin_amdgcn_readlane(group_end, kWave - 1)) {
      load(a, base + kChunk, __builtin_amdgcn_readlane(group_end, kWave - 1), wave, lane);
      group_end = before + group_ends(lane);
    }
    const int group = __builtin_ctzll(__builtin_amdgcn_ballot_w64(want < group_end));
    const int group_start = group ? __builtin_amdgcn_readlane(group_end, group - 1) : before;
    const int end = group_start + sums[64 * group + lane];
    const int in_group = __builtin_ctzll(__builtin_amdgcn_ballot_w64(want < end));
    const int seq_start = in_group ? __builtin_amdgcn_readlane(end, in_group - 1) : group_start;
    const int b = base + 64 * group + in_group;
    const i32x4 of = seqs[64 * group + in_group];
    const Seq s = {uniform(of[0]), uniform(of[1]), uniform(of[2]), uniform(of[3])};
    t.seq = s;
    int start = seq_start, steps = tile_steps<MANY, STEP>(a, s, 0);
    if constexpr (MANY) {
      const int tiles = ((s.rows << a.group_shift) + kManyCols - 1) / kManyCols;
      for (int j0 = 0; j0 < tiles; j0 += kWave) {
        const int j = j0 + lane;
        const int mine = j < tiles ? tile_steps<true, STEP>(a, s, j) : 0;
        const int incl = start + scan64(mine, lane);
        const uint64_t m = __builtin_amdgcn_ballot_w64(want < incl);
        if (m) {
          const int w = __builtin_ctzll(m);
          t.j = j0 + w;
          steps = __builtin_amdgcn_readlane(mine, w);
          start = __builtin_amdgcn_readlane(incl, w) - steps;
          break;
        }
        start = __builtin_amdgcn_readlane(incl, kWave - 1);
      }
    }
    t.b = uniform(b);
    t.head = uniform(t.head);
    t.j = uniform(t.j);
    t.start = head_start + uniform(start);
    t.steps = uniform(steps);
    return t;
  }
};

// Runs that have work, the first step of run w, and the run of step p: run w has the steps from w total / runs
// (rounded down) on, so the runs differ by one step at most.
struct Cuts {
  int64_t total;
  int runs;
  __device__ __forceinline__ int64_t first(int w) const { return div_floor(w * total, runs); }
  __device__ __forceinline__ int run_of(int64_t p) const { return (int)div_floor((p + 1) * runs - 1, total); }
};
__device__ __forceinline__ Cuts cuts_of(int64_t total, int runs) { return {total, (int)(total < runs ? total : runs)}; }

// Partial result `slot` (2 run: a tile that began in an earlier run; 2 run + 1: one that goes on in the next),
// of a kv head (few rows) or of the tile's only one.
struct Partials {
  float* o;       // [slot][head][column][128]
  float2* ml;     // [slot][head][column]
  int32_t* live;  // runs that have work
  int4* split;    // [run] the tile that begins in it and goes on: first row of out, columns, partial results (0: none),
                  // kv head
  int heads, cols;
  __device__ __forceinline__ int64_t at(int64_t slot, int head, int col) const {
    return (slot * heads + head) * cols + col;
  }
};
template <bool MANY>
__host__ __device__ __forceinline__ size_t partial_rows(const Fp4AttnPlan& p, int num_kv_heads) {
  return MANY ? (size_t)2 * p.many_runs * kManyCols : (size_t)2 * p.few_runs * num_kv_heads * p.few_cols;
}

// ---- rows in LDS ---------------------------------------------------------------------------
//
// A step's rows of the work-group's kv heads, HEADS slots a row: [K values | K scales | V values | V scales], a row's
// values HEADS x 4 chunks of 16 bytes, its scales HEADS dwords. They come straight from memory (global_load_lds, 1
// KiB an instruction for the values), a ring of three steps. (With every wavefront reading its own head's bytes into
// registers the kernel was bound by its load instructions: 40 a step of 64 keys and head, most of them of 16 to 256
// bytes, 355 us for 256 sequences of 1k-8k keys.)
//
// Banks. Chunk c of row r lies in slot c ^ swizzle(r) of the row. 16 lanes read K chunk 4 h + g of 16 rows (16
// bytes each), and 4 x 16 lanes 64 bytes each of four rows of V: with these swizzles, and the rows of a tile in the
// order of row_of, both touch every bank once (twice for V with two heads).
template <int HEADS>
__device__ __forceinline__ int swizzle(int r) {
  return HEADS >= 4 ? r & 15 : HEADS == 2 ? (r >> 1) & 7 : (r >> 2) & 3;
}
// The row (key) of a tile of 16 that is row m of its matrix product.
template <int HEADS>
__device__ __forceinline__ int row_of(int m) {
  return HEADS == 1 ? 4 * (m & 3) + (m >> 2) : m;
}

template <int HEADS, int ROWS>
struct Stage {
  static constexpr int kValues = ROWS * HEADS * kFp4HeadBytes;
  static constexpr int kScales = ROWS * HEADS * kFp4HeadScales;
  static constexpr int kCache = kValues + kScales;
  static constexpr int kBytes = 2 * kCache;
};

// Waits until this wavefront's loads have arrived, then for the other wavefronts.
__device__ __forceinline__ void arrive_all() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Waits until at most N of this wavefront's loads are in flight (and arrive_but: for the other wavefronts).
template <int N>
__device__ __forceinline__ void arrive_but() {
  asm volatile("s_waitcnt vmcnt(%c0) lgkmcnt(0)\n\ts_barrier" : : "i"(N) : "memory");
}

template <int N>
__device__ __forceinline__ void wait_but() {
  asm volatile("s_waitcnt vmcnt(%c0)" : : "i"(N) : "memory");
}

// 16 or 4 bytes per active lane from base + off to lds + 16 or 4 lane, in flight until arrive_all.
__device__ __forceinline__ void stage16(const uint8_t* base, int off, int lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "m0", "memory");
}
__device__ __forceinline__ void stage4(const uint8_t* base, int off, int lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "m0", "memory");
}

__device__ __forceinline__ const uint8_t* uniform_ptr(const uint8_t* p) {
  const uint64_t u = reinterpret_cast<uintptr_t>(p);
  const uint64_t lo = (uint32_t)uniform((int)(uint32_t)u), hi = (uint32_t)uniform((int)(u >> 32));
  return reinterpret_cast<const uint8_t*>(hi << 32 | lo);
}

// The place of a sequence's keys in the pages, from key t on in steps of `step` keys: the table's entry is read one
// step ahead. An entry that is no block has no rows, and its keys are seen by nobody.
struct Cursor {
  const int32_t* table;
  int t, entry, off, last, blk;

  // From `ahead` keys (fewer than 256) behind key t0 on, which is in the page `page`; the last key is in `last_page`.
  __device__ __forceinline__ void init(const Fp4AttnArgs& a, const int32_t* row, int t0, int page, int last_page, int ahead) {
    table = row;
    t = t0 + ahead;
    entry = page;
    off = t - page * a.block_size;
    last = last_page;
    while (off >= a.block_size) {
      off -= a.block_size;
      ++entry;
    }
    blk = scalar_i32(table + min(entry, last));
  }
  // (the entry is waited for here, ahead of the reads of LDS that would otherwise be waited for together with it)
  __device__ __forceinline__ void arrive() { asm volatile("" : "+s"(blk)); }
  __device__ __forceinline__ bool good(const Fp4AttnArgs& a) const { return blk >= 0 && blk < a.num_blocks; }
  __device__ __forceinline__ int rows(const Fp4AttnArgs& a, int keys) const { return good(a) ? keys - t : 0; }
  // Rows from here on in a cache (any place of the cache where there are none).
  __device__ __forceinline__ const uint8_t* at(const Fp4AttnArgs& a, const uint8_t* cache, int64_t block) const {
    return good(a) ? cache + (blk * block + (int64_t)off * a.row_bytes) : cache;
  }
  __device__ __forceinline__ void next(const Fp4AttnArgs& a, int step) {
    t += step;
    off += step;
    if (off >= a.block_size) {
      do {
        off -= a.block_size;
        ++entry;
      } while (off >= a.block_size);
      blk = scalar_i32(table + min(entry, last));
    }
  }
};

// One wavefront's share of a step's loads: of each cache two KiB of values, of one cache a quarter of the scales
// (256 slots of a head and row, 8 wavefronts).
template <int HEADS, int ROWS>
struct Loader {
  typedef Stage<HEADS, ROWS> S;
  static constexpr int kJobs = ROWS * HEADS / 16 / kFewWaves;  // KiB of values of a cache
  static constexpr int kScaleJobs = ROWS * HEADS / 64;         // 256 bytes of scales of a cache
  static_assert(kJobs * kFewWaves * 16 == ROWS * HEADS && 2 * kScaleJobs == kFewWaves, "loads divide among the wavefronts");
  static constexpr int kLoads = 2 * kJobs + 1;                 // of a wavefront and step
  int row[kJobs], col[kJobs];  // the lane's row after the cursor, and its place in the row
  int scale_row, scale_col;
  int lds, scale_lds;
  bool scales_of_v;
  Cursor at, own_scale_at;
  // (all of a step of 32 rows is in one page)
  static constexpr bool kOnePage = ROWS == kSub;
  __device__ __forceinline__ Cursor& scale_at() { return kOnePage ? at : own_scale_at; }

  // (a slot that is no head reads the last one's bytes, which nobody looks at)
  __device__ __forceinline__ void init(const Fp4AttnArgs& a, const int32_t* table, int t0, int keys, int head0, int heads,
                                       int wave, int lane) {
    const int first = wave * kJobs * 64 / (4 * HEADS);  // the first row
#pragma unroll
    for (int j = 0; j < kJobs; ++j) {
      const int slot = (wave * kJobs + j) * 64 + lane;
      const int r = slot / (4 * HEADS), c = (slot % (4 * HEADS)) ^ swizzle<HEADS>(r);
      row[j] = r - (first & ~31);
      col[j] = (head0 + min(c >> 2, heads - 1)) * kFp4HeadBytes + 16 * (c & 3);
    }
    lds = wave * kJobs * 1024;
    const int part = wave % kScaleJobs;
    scales_of_v = wave >= kScaleJobs;
    const int s = part * 64 + lane, r = s / HEADS, h = s % HEADS;
    const int scale_first = part * 64 / HEADS & ~31;
    scale_row = r - scale_first;
    scale_col = a.num_kv_heads * kFp4HeadBytes + (head0 + min(h, heads - 1)) * kFp4HeadScales;
    scale_lds = (scales_of_v ? S::kCache : 0) + S::kValues + part * 256;
    const int page = t0 / a.block_size, last_page = (keys - 1) / a.block_size;
    at.init(a, table, t0, page, last_page, first & ~31);
    if constexpr (!kOnePage) own_scale_at.init(a, table, t0, page, last_page, scale_first);
  }

  // The next step's rows into a stage of LDS; whether the wavefront's own 32 keys among them are in a block. A row that
  // is no key reads the last one that is (or, where there is none, the cache's first row): the count of loads in
  // flight is the same in every step.
  __device__ __forceinline__ bool issue(const Fp4AttnArgs& a, int keys, int stage) {
    const bool good = at.good(a);
    const int last = max(at.rows(a, keys), 1) - 1;
    const uint8_t* k = uniform_ptr(at.at(a, a.k, a.k_block));
    const uint8_t* v = uniform_ptr(at.at(a, a.v, a.v_block));
#pragma unroll
    for (int j = 0; j < kJobs; ++j) {
      const int off = min(row[j], last) * a.row_bytes + col[j];
      stage16(k, off, uniform(stage + lds + 1024 * j));
      stage16(v, off, uniform(stage + S::kCache + lds + 1024 * j));
    }
    const int scale_last = max(scale_at().rows(a, keys), 1) - 1;
    const uint8_t* c = kOnePage ? (scales_of_v ? v : k)
                                : uniform_ptr(scales_of_v ? scale_at().at(a, a.v, a.v_block) : scale_at().at(a, a.k, a.k_block));
    stage4(c, min(scale_row, scale_last) * a.row_bytes + scale_col, uniform(stage + scale_lds));
    at.next(a, ROWS);
    if constexpr (!kOnePage) own_scale_at.next(a, ROWS);
    return good;
  }
};

// ---- one wavefront's 32 keys -----------------------------------------------------------------

// Running softmax of the wavefront's columns: lane l has column l % 16 of every tile.
template <int T>
struct State {
  u32x4 q[T][4];     // dimensions 32 (l / 16) + 8 c .. of the column
  f32x4 acc[T][8];   // [j][i]: dimension 32 (l / 16) + 8 i + j
  float m[T];        // reference, the same in the column's four lanes
  float l[T];        // this lane's keys' share of the sum
  float slack;       // by how much scores may exceed m: kSlack, or kSlack - kRaise (the same for the wavefront)
};

// Raises the reference of all columns, before the weights of the first large rows of V.
template <int T>
__device__ __forceinline__ void raise_reference(State<T>& st) {
  if (st.slack != kSlack) return;
  st.slack = kSlack - kRaise;
#pragma unroll
  for (int x = 0; x < T; ++x) {
    st.m[x] += kRaise;  // (kLowest stays what it is)
    st.l[x] *= 0x1p-32f;
#pragma unroll
    for (int j = 0; j < 8; ++j) st.acc[x][j] *= 0x1p-32f;
  }
}
static_assert(kRaise == 32.f, "raise_reference's factor");

struct Vals {
  uint32_t d[2][4];  // tile t, row row_of(4 (l / 16) + i): dimensions 8 (l % 16) .. + 7
  uint32_t s[2][4];  // their scale byte
};

// Where a lane's rows lie in a stage.
template <int HEADS, int ROWS>
struct Lanes {
  typedef Stage<HEADS, ROWS> S;
  static constexpr int kTile = 16 * HEADS * kFp4HeadBytes, kScaleTile = 16 * HEADS * kFp4HeadScales;
  int k, ks, v[4], vs;

  // first: the wavefront's first row, slot: its head's.
  __device__ __forceinline__ void init(int first, int slot, int lane) {
    const int n = lane & 15, g = lane >> 4;
    int r = row_of<HEADS>(n);
    k = ((first + r) * 4 * HEADS + ((4 * slot + g) ^ swizzle<HEADS>(r))) * 16;
    ks = S::kValues + ((first + r) * HEADS + slot) * 4 + g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r = row_of<HEADS>(4 * g + i);
      v[i] = S::kCache + ((first + r) * 4 * HEADS + ((4 * slot + (n >> 2)) ^ swizzle<HEADS>(r))) * 16 + 4 * (n & 3);
    }
    vs = S::kCache + S::kValues + ((first + row_of<HEADS>(4 * g)) * HEADS + slot) * 4 + (n >> 2);
  }
  __device__ __forceinline__ void values(Vals& x, const lds_u8* stage) const {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x.d[t][i] = *(const lds_u32*)(stage + v[i] + t * kTile);
        x.s[t][i] = *(const lds_u8*)(stage + vs + t * kScaleTile + row_of<HEADS>(i) * HEADS * 4);
      }
  }
};

struct Keys {
  u32x4 d[2];        // row row_of(l % 16) of a tile: dimensions 32 (l / 16) .. + 31
  uint32_t s[2];
};

// S^T of two tiles of 16 keys.
template <int T>
__device__ __forceinline__ void scores(f32x4 (&s)[2][T], const State<T>& st, const Keys& k) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const float scale = fp4_scale(k.s[t]);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint4 w = fp4_unpack8(k.d[t][c], scale);
#pragma unroll
      for (int x = 0; x < T; ++x)
        s[t][x] = mfma(u32x4{w.x, w.y, w.z, w.w}, st.q[x][c], c ? s[t][x] : f32x4{0.f, 0.f, 0.f, 0.f});
    }
  }
}

// a.x + a.y + c on a packed bf16 pair.
__device__ __forceinline__ float add_bf16x2(uint32_t a, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(fp4_bf16x2, a), __builtin_bit_cast(fp4_bf16x2, 0x3f803f80u), c,
                                         false);
}

// The weights of the columns over NT tiles of 16 keys, in bf16 pairs, as the operand of the product with V: two
// tiles an operand, tile by tile, i by i. The sum is of the rounded weights, which is what the product weighs V with.
// (Whether the reference holds is asked of each lane's own scores; the column's largest is formed only where it
// does not.) large: the lane has met a scale byte of V from kLargeScale on.
template <int T, int NT>
__device__ __forceinline__ void weights(u32x4 (&p)[T][NT / 2], const f32x4 (&s)[NT][T], State<T>& st, bool large, float c2) {
  float top[T];
  bool over = large;
#pragma unroll
  for (int x = 0; x < T; ++x) {
    float mx = fmaxf(s[0][x][0], s[0][x][1]);
    mx = fmaxf(fmaxf(mx, s[0][x][2]), s[0][x][3]);
#pragma unroll
    for (int t = 1; t < NT; ++t) {
      mx = fmaxf(fmaxf(mx, s[t][x][0]), s[t][x][1]);
      mx = fmaxf(fmaxf(mx, s[t][x][2]), s[t][x][3]);
    }
    top[x] = mx;
    over |= mx * c2 > st.m[x] + st.slack;
  }
  if (__builtin_amdgcn_ballot_w64(over)) {
    if (__builtin_amdgcn_ballot_w64(large)) raise_reference(st);
#pragma unroll
    for (int x = 0; x < T; ++x) {
      const float m = fmaxf(st.m[x], quarters_max(top[x]) * c2 + (kSlack - st.slack));
      const float f = exp2_fast(st.m[x] - m);
      st.m[x] = m;
      st.l[x] *= f;
#pragma unroll
      for (int j = 0; j < 8; ++j) st.acc[x][j] *= f;
    }
  }
#pragma unroll
  for (int x = 0; x < T; ++x) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = exp2_fast(fmaf(s[t][x][i], c2, -st.m[x]));
      const uint32_t lo = fp4_pack_bf16(e[0], e[1]), hi = fp4_pack_bf16(e[2], e[3]);
      p[x][t >> 1][2 * (t & 1)] = lo;
      p[x][t >> 1][2 * (t & 1) + 1] = hi;
      st.l[x] = add_bf16x2(hi, add_bf16x2(lo, st.l[x]));
    }
  }
}

template <int kByte, int T>
__device__ __forceinline__ void add_pair(State<T>& st, const u32x4 (&p)[T][1], const Vals& v) {
  u32x4 even, odd;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t x = fp4_pair<kByte>(v.d[t][2 * i], fp4_scale(v.s[t][2 * i]));
      const uint32_t y = fp4_pair<kByte>(v.d[t][2 * i + 1], fp4_scale(v.s[t][2 * i + 1]));
      even[2 * t + i] = __builtin_amdgcn_perm(y, x, 0x05040100u);
      odd[2 * t + i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
    }
  }
#pragma unroll
  for (int x = 0; x < T; ++x) {
    st.acc[x][2 * kByte] = mfma(even, p[x][0], st.acc[x][2 * kByte]);
    st.acc[x][2 * kByte + 1] = mfma(odd, p[x][0], st.acc[x][2 * kByte + 1]);
  }
}

template <int T>
__device__ __forceinline__ void add_values(State<T>& st, const u32x4 (&p)[T][1], const Vals& v) {
  add_pair<0>(st, p, v);
  add_pair<1>(st, p, v);
  add_pair<2>(st, p, v);
  add_pair<3>(st, p, v);
}

// NaN blocks among keys some of which some columns do not see: 0 x NaN would reach those columns through the
// matrix product. The blocks are taken as zeros there, and a column that does see such a key gets its NaN here.
// (Lane l's 32 outputs are the block l / 16 of its column. The scale bytes of one key and all four blocks are lanes
// 0, 4, 8, 12 of the row of 16 lanes that has the key.) Rows past the last key hold anything, scales that no cache
// has among it, whose values are infinite: this is also what keeps them out.
template <int T, int HEADS>
__device__ __forceinline__ void nan_values(State<T>& st, Vals& v, uint32_t most, const int (&rel)[T], int lane) {
  if (!__builtin_amdgcn_ballot_w64(most > kFp4MaxScale)) return;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool bad = v.s[t][i] > kFp4MaxScale;
      const uint64_t which = __builtin_amdgcn_ballot_w64(bad);
      if (!which) continue;
      if (bad) v.s[t][i] = v.d[t][i] = 0;
      for (int g = 0; g < 4; ++g) {
        const bool here = which >> (16 * g + 4 * (lane >> 4)) & 1;  // row row_of(4 g + i) of the tile, block lane / 16
#pragma unroll
        for (int x = 0; x < T; ++x)
          if (here && 16 * t + row_of<HEADS>(4 * g + i) <= rel[x])
#pragma unroll
            for (int j = 0; j < 8; ++j) st.acc[x][j] += __builtin_nanf("");
      }
    }
}

// 32 keys of a stage. rel: the last of them that a column sees, where some column does not see all.
// (Products go before the other wavefront's exponentials: 128 sequences 33.8 us in place of 34.7.)
template <int T, int HEADS, int ROWS>
__device__ __forceinline__ void take(State<T>& st, const lds_u8* stage, const Lanes<HEADS, ROWS>& at, bool masked,
                                     const int (&rel)[T], float c2, int lane) {
  // (all reads of LDS at once, ahead of everything that waits for them)
  Keys k;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    k.d[t] = *(const lds_u32x4*)(stage + at.k + t * at.kTile);
    k.s[t] = *(const lds_u8*)(stage + at.ks + t * at.kScaleTile);
  }
  Vals v;
  at.values(v, stage);
  __builtin_amdgcn_sched_barrier(0);
  f32x4 s[2][T];
  __builtin_amdgcn_s_setprio(1);
  scores(s, st, k);
  __builtin_amdgcn_s_setprio(0);
  if (masked) {
#pragma unroll
    for (int x = 0; x < T; ++x)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * t + row_of<HEADS>(4 * (lane >> 4) + i) > rel[x]) s[t][x][i] = -INFINITY;
  }
  uint32_t most = 0;  // the largest scale byte of V's
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) most = max(most, v.s[t][i]);
  u32x4 p[T][1];
  weights<T, 2>(p, s, st, most >= kLargeScale, c2);
  if (masked) nan_values<T, HEADS>(st, v, most, rel, lane);
  __builtin_amdgcn_s_setprio(1);
  add_values<T>(st, p, v);
  __builtin_amdgcn_s_setprio(0);
}

// The 16 columns of a wavefront over few rows, through LDS like the keys (4 KiB a wavefront, where the last stage of
// the ring will be): loads into registers would be waited for together with every row that is in flight. Columns
// past the last row hold the last row's q; nobody looks at what comes of them.
struct Queries {
  __device__ __forceinline__ void issue(const Fp4AttnArgs& a, const Seq& seq, int head, int wave, int lane, int lds) const {
    const int last = (seq.rows << a.group_shift) - 1, group = 1 << a.group_shift;
    const uint8_t* q = uniform_ptr(reinterpret_cast<const uint8_t*>(a.q + seq.q0 * a.q_stride + (int64_t)head * group * kHeadDim));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = 4 * i + (lane >> 4), real = min(col, last);
      const int off = (int)((real >> a.group_shift) * a.q_stride + (real & (group - 1)) * kHeadDim) * 2 + 16 * ((lane ^ col) & 15);
      stage16(q, off, uniform(lds + wave * 4096 + 1024 * i));
    }
  }
  __device__ __forceinline__ void read(u32x4 (&q)[4], const lds_u8* lds, int wave, int lane) const {
    const int n = lane & 15, g = lane >> 4;
#pragma unroll
    for (int c = 0; c < 4; ++c) q[c] = *(const lds_u32x4*)(lds + wave * 4096 + n * 256 + (((4 * g + c) ^ n) * 16));
  }
};

// ---- results ---------------------------------------------------------------------------------

// COUNT of a lane's 32 output values from value r on (value 8 i + j is dimension 8 i + j of the lane's block): to the
// output's row, scaled, or to a partial result.
template <int COUNT>
__device__ __forceinline__ void put_out(uint16_t* out, const float* x, float inv) {
  if constexpr (COUNT >= 8) {
#pragma unroll
    for (int i = 0; i < COUNT; i += 8) {
      u32x4 w;
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = fp4_pack_bf16(x[i + 2 * j] * inv, x[i + 2 * j + 1] * inv);
      *reinterpret_cast<u32x4*>(out + i) = w;
    }
  } else {
    *reinterpret_cast<u32x2*>(out) = u32x2{fp4_pack_bf16(x[0] * inv, x[1] * inv), fp4_pack_bf16(x[2] * inv, x[3] * inv)};
  }
}
template <int COUNT>
__device__ __forceinline__ void put_part(float* out, const float* x) {
#pragma unroll
  for (int i = 0; i < COUNT; i += 4) *reinterpret_cast<f32x4*>(out + i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
}

// The SLICES wavefronts of a kv head, which took different keys, put their states together in LDS: every one of them
// ends with the column's m and l and with 32 / SLICES values of each lane, those from (32 / SLICES) slice on.
template <int SLICES, int HEADS>
__device__ __forceinline__ void join_slices(float (&x)[32 / SLICES], float* m, float* l, const State<1>& st, lds_u8* lds,
                                            int wave, int lane) {
  lds_f32x2* ml = (lds_f32x2*)lds;
  lds_f32* o = (lds_f32*)(lds + kFewWaves * kWave * 8);
  const int slot = wave % HEADS, slice = wave / HEADS;
  const float mine = st.m[0];
  arrive_all();  // every wavefront is done with the rows in LDS
  ml[wave * kWave + lane] = f32x2{mine, *l};
  arrive_all();
  float top = kLowest, sum = 0.f;
#pragma unroll
  for (int s = 0; s < SLICES; ++s) top = fmaxf(top, ml[(s * HEADS + slot) * kWave + lane][0]);
#pragma unroll
  for (int s = 0; s < SLICES; ++s) {
    const f32x2 other = ml[(s * HEADS + slot) * kWave + lane];
    sum = fmaf(exp2_fast(other[0] - top), other[1], sum);
  }
  const float f = exp2_fast(mine - top);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) o[(wave * 32 + 8 * i + j) * kWave + lane] = st.acc[0][j][i] * f;
  arrive_all();
  constexpr int N = 32 / SLICES;
#pragma unroll
  for (int r = 0; r < N; ++r) {
    x[r] = 0.f;
#pragma unroll
    for (int s = 0; s < SLICES; ++s) x[r] += o[((s * HEADS + slot) * 32 + N * slice + r) * kWave + lane];
  }
  *m = top;
  *l = sum;
}

// ---- the work-groups -------------------------------------------------------------------------

// A work-group's part of the line, and what the merge has to know of it.
template <bool MANY, int STEP>
struct Run {
  Line<MANY, STEP> line;
  Cuts cuts;
  int run;
  int64_t p, end;         // the next step, the one after the last
  int4 split;
  Tile tile;
  Seq seq;
  int s0, s1;             // the steps of the tile that are this run's
  bool whole;
  int row0;

  // False if there is nothing to do. Neighbouring runs of MANY, whose tiles read the same keys, go to one XCD
  // (work-groups go to the 8 of them in turn).
  __device__ __forceinline__ bool init(const Fp4AttnArgs& a, const Partials& part, int num_runs, int index, bool recorder,
                                       lds_u8* lds, int wave, int lane) {
    line.init(a, lds, wave, lane);
    cuts = cuts_of(line.total, num_runs);
    if (index == 0 && recorder) *part.live = cuts.runs;
    if (line.total == 0) return false;
    run = index;
    if constexpr (MANY) {
      const int per_xcd = (cuts.runs + 7) >> 3;
      if ((index >> 3) >= per_xcd) return false;
      run = (index & 7) * per_xcd + (index >> 3);
    }
    if (run >= cuts.runs) return false;
    p = cuts.first(run);
    end = cuts.first(run + 1);
    split = make_int4(0, 0, 0, 0);
    return true;
  }
  __device__ __forceinline__ bool next(const Fp4AttnArgs& a, const Partials& part, int wave, int lane) {
    if (p >= end) return false;
    tile = line.at(a, p, wave, lane);
    seq = tile.seq;
    s0 = (int)(p - tile.start);
    s1 = (int)min((int64_t)tile.steps, end - tile.start);
    p = tile.start + s1;
    whole = s0 == 0 && s1 == tile.steps;
    row0 = MANY ? tile.j * (kManyCols >> a.group_shift) : 0;
    if (s0 == 0 && !whole)
      split = make_int4(seq.q0 + row0, min((seq.rows - row0) << a.group_shift, part.cols),
                        cuts.run_of(tile.start + tile.steps - 1) - run + 1, tile.head);
    return true;
  }
  __device__ __forceinline__ int64_t slot() const { return 2 * (int64_t)run + (s0 == 0 ? 1 : 0); }
};

// A lane's columns: their rows and the last keys that they see.
template <int T>
struct Columns {
  int row[T], head[T], last[T];  // row of the sequence, query head
  bool real[T];
  int lowest;                    // the last key that every column sees
  int furthest;                  // the last key that some column sees

  __device__ __forceinline__ void init(const Fp4AttnArgs& a, const Seq& seq, int row0, int kv_head, int first, bool live,
                                       int n) {
    lowest = a.max_seqlen_k;
    furthest = -1;
#pragma unroll
    for (int x = 0; x < T; ++x) {
      const int col = first + 16 * x + n;
      row[x] = row0 + (col >> a.group_shift);
      head[x] = (kv_head << a.group_shift) + (col & ((1 << a.group_shift) - 1));
      real[x] = row[x] < seq.rows && live;
      last[x] = real[x] ? min(seq.keys - 1, row[x] + seq.shift) : -1;
      if (real[x]) {
        lowest = min(lowest, last[x]);
        furthest = max(furthest, last[x]);
      }
    }
#pragma unroll
    for (int sh = 1; sh < 16; sh *= 2) {
      lowest = min(lowest, __shfl_xor(lowest, sh));
      furthest = max(furthest, __shfl_xor(furthest, sh));
    }
    lowest = uniform(lowest);
    furthest = uniform(furthest);
  }
};

// Few rows: HEADS slots of kv heads from head0 on, of which `heads` are heads, and 8 / HEADS wavefronts to each, which
// take 32 keys of every step in turn. Bound by HBM where there is enough to read: 217 us a call for 256 sequences of
// 1k-8k keys of 8 kv heads, 5.65 TB/s (the kernel 209 at best, where a stream that is only read reaches 6.34); 34 us for
// 128 of 100-2048 (4.2 TB/s), 5 of them before the first step is there. Sequences of at most 16 columns, what one tile holds, come here: 48 of 4 to 16 columns and 300-4000 keys of 4 kv
// heads took 22 us and 6 for the merge; with those of more than 8 columns in the other kernel 15 + 36 + 11, of more
// than 4 columns 8 + 50 + 12.
template <int HEADS>
struct FewLds {
  static constexpr int kRows = kSub * kFewWaves / HEADS;  // of a step
  static constexpr int kLine = kFewRing * Stage<HEADS, kRows>::kBytes;
  static constexpr int kBytes = kLine + Line<false, kRows>::kBytes;
};
// run: of `runs`, of the kv heads from head0 on.
template <int HEADS>
__device__ __forceinline__ void attend_few(const Fp4AttnArgs& a, const Partials& part, int runs, int heads, int index,
                                           int head0, lds_u8* lds) {
  constexpr int D = kHeadDim;
  constexpr int kSlices = kFewWaves / HEADS, ROWS = kSub * kSlices;
  typedef Stage<HEADS, ROWS> S;
  typedef Loader<HEADS, ROWS> L;
  const int lds0 = (int)(uintptr_t)lds;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = uniform(threadIdx.x / kWave);
  const int n = lane & 15, g = lane >> 4;
  const bool recorder = head0 == 0 && threadIdx.x == 0;
  Run<false, ROWS> run;
  if (!run.init(a, part, runs, index, recorder, lds + FewLds<HEADS>::kLine, wave, lane)) return;
  const int slot = wave % HEADS, slice = wave / HEADS;
  const bool live = slot < heads;
  const int head = head0 + min(slot, heads - 1);
  Queries queries;
  Lanes<HEADS, ROWS> at;
  at.init(slice * kSub, slot, lane);
  while (run.next(a, part, wave, lane)) {
    const Seq seq = run.seq;
    const int s0 = run.s0, s1 = run.s1;
    meet();  // the last piece has been read
    const int32_t* table = a.block_table + (int64_t)run.tile.b * a.bt_stride;
    L loader;
    loader.init(a, table, s0 * ROWS, seq.keys, head0, heads, wave, lane);
    uint32_t good = 0;  // bit i: step s + i's keys are in a block
    queries.issue(a, seq, head, wave, lane, lds0 + (kFewRing - 1) * S::kBytes);
#pragma unroll
    for (int i = 0; i < kFewRing - 1; ++i)
      if (i < s1 - s0) good |= (uint32_t)loader.issue(a, seq.keys, lds0 + i * S::kBytes) << i;

    Columns<1> cols;
    cols.init(a, seq, 0, head, 0, live, n);
    State<1> st;
    st.m[0] = kLowest;
    st.l[0] = 0.f;
    st.slack = kSlack;
#pragma unroll
    for (int j = 0; j < 8; ++j) st.acc[0][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (s1 - s0 >= kFewRing - 1)
      wait_but<(kFewRing - 1) * L::kLoads>();
    else
      wait_but<0>();
    queries.read(st.q[0], lds + (kFewRing - 1) * S::kBytes, wave, lane);

    int buf = 0, next_buf = kFewRing - 1;
    for (int s = s0; s < s1; ++s) {
      const lds_u8* stage = lds + buf * S::kBytes;
      // step s is there, and step s - 1 done with
      if (s + 1 < s1)
        arrive_but<(kFewRing - 2) * L::kLoads>();
      else
        arrive_but<0>();
      if (s + kFewRing - 1 < s1)
        good |= (uint32_t)loader.issue(a, seq.keys, lds0 + next_buf * S::kBytes) << (kFewRing - 1);
      loader.at.arrive();
      loader.scale_at().arrive();
      buf = buf + 1 == kFewRing ? 0 : buf + 1;
      next_buf = next_buf + 1 == kFewRing ? 0 : next_buf + 1;
      const int t0 = s * ROWS + slice * kSub;
      if (t0 <= cols.furthest && (uniform(good) & 1)) {  // (otherwise no column sees these keys)
        const int rel[1] = {cols.last[0] - t0};
        take(st, stage, at, t0 + kSub - 1 > cols.lowest, rel, a.scale_log2, lane);
      }
      good >>= 1;
    }

    constexpr int N = 32 / kSlices;
    float v[N], m = st.m[0], l = quarters_sum(st.l[0]);
    if constexpr (kSlices > 1) {
      join_slices<kSlices, HEADS>(v, &m, &l, st, lds, wave, lane);
    } else {
#pragma unroll
      for (int r = 0; r < 32; ++r) v[r] = st.acc[0][r & 7][r >> 3];
    }
    if (!cols.real[0]) continue;
    const int dim = 32 * g + N * slice;
    if (run.whole) {
      uint16_t* out = a.out + (int64_t)(seq.q0 + cols.row[0]) * a.out_stride + cols.head[0] * D + dim;
      put_out<N>(out, v, l == 0.f ? 0.f : 1.f / l);  // no key seen: zeros
    } else {
      const int64_t at_part = part.at(run.slot(), head, n);
      put_part<N>(part.o + at_part * D + dim, v);
      if (g == 0 && slice == 0) part.ml[at_part] = make_float2(m, l);
    }
  }
  if (recorder) part.split[run.run] = run.split;
}

// ---- more rows -------------------------------------------------------------------------------
//
// 256 columns of one kv head share its keys: a step's 64 rows come to LDS in 4 bits, the work-group's 512 threads
// convert them to bf16 tiles once (16 values of K and of V each), and its 8 wavefronts read these. (With each
// wavefront converting the rows for its own 32 columns the kernel was bound by its vector instructions, 282 for 32
// keys and 32 columns, 106 of them conversions.) Step s + 1 is converted after step s's products, in their shadow
// (before them 16 chunks of 1024 rows behind 4096 keys took 2% longer), steps s + 2 and s + 3 are on their way.
//
// Bound by the vector instructions and the products together: the matrix cores are busy for 43% of a SIMD's time,
// the vector units for 48%. The 16 chunks take 629 us a call, 985 TFLOP/s. Two other forms ran within 3% of this one: step s's exponentials between the products of
// step s + 1, and that with four wavefronts of 64 columns, half the reads of LDS.
//
// The tiles have 256-byte rows, 16 chunks of 16 bytes. K: chunk c of row r in slot c ^ (r & 15): the 16 lanes of a
// quarter wavefront read one chunk of 16 rows. V: slot c ^ v_swizzle(r): the transposing read takes four rows and 32
// bytes a quarter, two quarters at once, 16 different slots; and the conversion writes one chunk in two of each
// of two rows at once, 16 different slots again. Dimensions are in their own order here: lane l holds dimensions
// 32 c + 8 (l / 16) .. + 7 of key l % 16 (and of q), and dimension 16 j + l % 16 of V's four keys.
__device__ __forceinline__ int v_swizzle(int r) { return (2 * r & 14) | (r & 1); }

struct ManyLds {
  static constexpr int kRow = kHeadDim * 2;
  static constexpr int kTile = kManyStep * kRow;                   // bf16 rows of a cache
  static constexpr int kRawValues = kManyStep * kFp4HeadBytes;     // 4-bit rows of a cache
  static constexpr int kRawScales = kManyStep * kFp4HeadScales;
  static constexpr int kRawCache = kRawValues + kRawScales;
  static constexpr int kRaw = 2 * kRawCache;
  static constexpr int kTiles = kManyRing * kRaw;                  // after the ring: two pairs of tiles
  static constexpr int kBytes = kTiles + 4 * kTile;
  // A wavefront's loads of a step: 16 rows of one cache, 16 bytes a lane and four scales by its first 16 lanes.
  static constexpr int kLoads = 2;
};

struct ManyLoader {
  Cursor at;
  const uint8_t* cache;
  int64_t block;
  int row, col, scale_row, scale_col, lds, scale_lds;

  __device__ __forceinline__ void init(const Fp4AttnArgs& a, const int32_t* table, int t0, int keys, int head, int wave,
                                       int lane) {
    at.init(a, table, t0, t0 / a.block_size, (keys - 1) / a.block_size, 0);
    const bool is_v = wave >= kManyWaves / 2;
    cache = is_v ? a.v : a.k;
    block = is_v ? a.v_block : a.k_block;
    const int first = 16 * (wave % (kManyWaves / 2));
    row = first + (lane >> 2);
    col = head * kFp4HeadBytes + 16 * (lane & 3);
    scale_row = first + (lane & 15);
    scale_col = a.num_kv_heads * kFp4HeadBytes + head * kFp4HeadScales;
    lds = (is_v ? ManyLds::kRawCache : 0) + first * kFp4HeadBytes;
    scale_lds = (is_v ? ManyLds::kRawCache : 0) + ManyLds::kRawValues + first * kFp4HeadScales;
  }
  // (as Loader's)
  __device__ __forceinline__ bool issue(const Fp4AttnArgs& a, int keys, int stage, int lane) {
    const bool good = at.good(a);
    const int last = max(at.rows(a, keys), 1) - 1;
    const uint8_t* c = uniform_ptr(at.at(a, cache, block));
    stage16(c, min(row, last) * a.row_bytes + col, uniform(stage + lds));
    if (lane < 16) stage4(c, min(scale_row, last) * a.row_bytes + scale_col, uniform(stage + scale_lds));
    at.next(a, kManyStep);
    return good;
  }
};

// A step's rows from 4 bits to bf16: thread t has dimensions 16 (t % 8) .. of row t / 8. NaN blocks of V (and what
// lies past the last key) become zeros, which reach no column; columns that see a NaN block get theirs from
// many_nan. K's make their key's scores NaN.
__device__ __forceinline__ void convert_rows(const lds_u8* raw, lds_u8* tiles, int thread) {
  const int r = thread >> 3, part = thread & 7;
  const lds_u8* rk = raw + r * kFp4HeadBytes + 8 * part;
  const lds_u8* rs = raw + ManyLds::kRawValues + r * kFp4HeadScales + (part >> 1);
  const u32x2 k = *(const lds_u32x2*)rk;
  u32x2 v = *(const lds_u32x2*)(rk + ManyLds::kRawCache);
  const uint32_t ks = *rs;
  uint32_t vs = *(rs + ManyLds::kRawCache);
  if (vs > kFp4MaxScale) {
    vs = 0;
    v = u32x2{0, 0};
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = 2 * part + i;
    const uint4 wk = fp4_unpack8(k[i], fp4_scale(ks)), wv = fp4_unpack8(v[i], fp4_scale(vs));
    *(lds_u32x4*)(tiles + r * ManyLds::kRow + (c ^ (r & 15)) * 16) = u32x4{wk.x, wk.y, wk.z, wk.w};
    *(lds_u32x4*)(tiles + ManyLds::kTile + r * ManyLds::kRow + (c ^ v_swizzle(r)) * 16) = u32x4{wv.x, wv.y, wv.z, wv.w};
  }
}

// acc[x][j][i]: dimension 16 j + 4 (l / 16) + i. A column that sees a row of the step with NaN blocks of V gets NaN in
// their dimensions. s: the lane's row's scale bytes of V, rel: the last row that a column sees.
template <int T>
__device__ __forceinline__ void many_nan(State<T>& st, uint32_t s, const int (&rel)[T], int rows, int lane) {
  uint32_t bad = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b) bad |= (uint32_t)((s >> 8 * b & 0xff) > kFp4MaxScale) << b;
  uint64_t which = __builtin_amdgcn_ballot_w64(bad != 0 && lane < rows);
  while (which) {
    const int r = __builtin_ctzll(which);
    which &= which - 1;
    const uint32_t blocks = (uint32_t)__builtin_amdgcn_readlane((int)bad, r);
#pragma unroll
    for (int x = 0; x < T; ++x)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((blocks >> (j >> 1) & 1) && r <= rel[x]) st.acc[x][j] += __builtin_nanf("");
  }
}

// The 64 keys of a pair of tiles. k, v: the lane's places in them, for every chunk of K and every 16 dimensions of V.
// large: the lane's row has a scale byte of V from kLargeScale on.
// The reads are kept ahead of the products that use them (the compiler's own order reads each operand right before
// its product and waits for it.) A wavefront goes first while it has products: otherwise the two on a SIMD fall into step
// in some builds, and wait for the same units (16 chunks took 3 to 5% longer in those, with 3, 4, 5, 6 or 8 reads of K
// ahead, whichever way the registers came to lie; with the priorities 3 and 4 of them differ by less than 1%).
template <int T>
__device__ __forceinline__ void many_take(State<T>& st, const lds_u8* tiles, const int (&k)[4], const int (&v)[8],
                                          bool large, bool masked, const int (&rel)[T], float c2, int lane) {
  constexpr int kTile16 = 16 * ManyLds::kRow;
  constexpr int kAheadK = 4, kAheadV = 1;
  f32x4 s[4][T];
  u32x4 kw[kAheadK];
  u32x4 vw[kAheadV + 1][2];
  const auto read_k = [&](int i) { return *(const lds_u32x4*)(tiles + k[i & 3] + (i >> 2) * kTile16); };
  const auto read_v = [&](u32x4 (&w)[2], int j) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      lds_u8* at = const_cast<lds_u8*>(tiles + ManyLds::kTile + v[j] + t * kTile16);
      const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)at));
      w[t >> 1][2 * (t & 1)] = x[0];
      w[t >> 1][2 * (t & 1) + 1] = x[1];
    }
  };
#pragma unroll
  for (int i = 0; i < kAheadK; ++i) kw[i] = read_k(i);
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const u32x4 w = kw[i % kAheadK];
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int x = 0; x < T; ++x) s[i >> 2][x] = mfma(w, st.q[x][i & 3], i & 3 ? s[i >> 2][x] : f32x4{0.f, 0.f, 0.f, 0.f});
    if (i + kAheadK < 16) kw[i % kAheadK] = read_k(i + kAheadK);
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < kAheadV; ++j) read_v(vw[j], j);
  if (masked) {
#pragma unroll
    for (int x = 0; x < T; ++x)
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (16 * t + 4 * (lane >> 4) + i > rel[x]) s[t][x][i] = -INFINITY;
  }
  __builtin_amdgcn_s_setprio(0);
  u32x4 p[T][2];
  weights<T, 4>(p, s, st, large, c2);
  __builtin_amdgcn_s_setprio(1);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (j + kAheadV < 8) read_v(vw[(j + kAheadV) % (kAheadV + 1)], j + kAheadV);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int x = 0; x < T; ++x) st.acc[x][j] = mfma(vw[j % (kAheadV + 1)][h], p[x][h], st.acc[x][j]);
    __builtin_amdgcn_sched_barrier(0);
  }
  __builtin_amdgcn_s_setprio(0);
}

__device__ __forceinline__ void attend_many(const Fp4AttnArgs& a, const Partials& part, int runs, int index, lds_u8* lds) {
  constexpr int D = kHeadDim, T = kManyTiles;
  typedef ManyLds S;
  const int lds0 = (int)(uintptr_t)lds;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = uniform(threadIdx.x / kWave);
  const int n = lane & 15, g = lane >> 4;
  Run<true, kManyStep> run;
  if (!run.init(a, part, runs, index, threadIdx.x == 0, lds + S::kBytes, wave, lane)) return;
  int k_at[4], v_at[8];
#pragma unroll
  for (int c = 0; c < 4; ++c) k_at[c] = n * S::kRow + ((4 * c + g) ^ n) * 16;
  const int vr = 4 * g + (n >> 2);  // rows 4 g .. + 3, 8 bytes each
#pragma unroll
  for (int j = 0; j < 8; ++j) v_at[j] = vr * S::kRow + ((2 * j + ((n & 3) >> 1)) ^ v_swizzle(vr)) * 16 + 8 * (n & 1);
  while (run.next(a, part, wave, lane)) {
    const Seq seq = run.seq;
    const int s0 = run.s0, s1 = run.s1, head = run.tile.head;
    Columns<T> cols;
    cols.init(a, seq, run.row0, head, wave * T * 16, true, n);
    State<T> st;
    st.slack = kSlack;
#pragma unroll
    for (int x = 0; x < T; ++x) {
      const uint16_t* q = a.q + (int64_t)(seq.q0 + cols.row[x]) * a.q_stride + cols.head[x] * D + 8 * g;
#pragma unroll
      for (int c = 0; c < 4; ++c) st.q[x][c] = cols.real[x] ? *reinterpret_cast<const u32x4*>(q + 32 * c) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j) st.acc[x][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      st.m[x] = kLowest;
      st.l[x] = 0.f;
    }
    // (q is waited for here: in the loop the wait would be for every row in flight)
#pragma unroll
    for (int x = 0; x < T; ++x)
#pragma unroll
      for (int c = 0; c < 4; ++c) asm volatile("" : "+v"(st.q[x][c]));
    arrive_all();  // (the last piece's reads of LDS are over)
    const int32_t* table = a.block_table + (int64_t)run.tile.b * a.bt_stride;
    ManyLoader loader;
    loader.init(a, table, s0 * kManyStep, seq.keys, head, wave, lane);
    uint32_t good = 0;  // bit i: step s + i's keys are in a block
#pragma unroll
    for (int i = 0; i < kManyRing - 1; ++i)
      if (i < s1 - s0) good |= (uint32_t)loader.issue(a, seq.keys, lds0 + i * S::kRaw, lane) << i;
    if (s0 + 2 < s1)
      arrive_but<2 * S::kLoads>();
    else
      arrive_but<0>();
    convert_rows(lds, lds + S::kTiles, threadIdx.x);

    for (int s = s0; s < s1; ++s) {
      const int i = s - s0;
      // step s + 1's rows and step s's tiles are there, and step s - 1 is done with
      if (s + 2 < s1)
        arrive_but<S::kLoads>();
      else
        arrive_but<0>();
      if (s + 3 < s1) good |= (uint32_t)loader.issue(a, seq.keys, lds0 + ((i + 3) & 3) * S::kRaw, lane) << 3;
      loader.at.arrive();
      const int t0 = s * kManyStep;
      if (t0 <= cols.furthest && (uniform(good) & 1)) {  // (otherwise no column sees these keys)
        const lds_u8* tiles = lds + S::kTiles + (i & 1) * 2 * S::kTile;
        int rel[T];
#pragma unroll
        for (int x = 0; x < T; ++x) rel[x] = cols.last[x] - t0;
        const uint32_t scales = *(const lds_u32*)(lds + (i & 3) * S::kRaw + S::kRawCache + S::kRawValues + 4 * lane);
        const bool large = (scales & scales << 1 & 0x80808080u) != 0;  // (kLargeScale; NaN blocks are among them)
        many_take(st, tiles, k_at, v_at, large, t0 + kManyStep - 1 > cols.lowest, rel, a.scale_log2, lane);
        if (__builtin_amdgcn_ballot_w64(large)) many_nan(st, scales, rel, seq.keys - t0, lane);
      }
      if (s + 1 < s1) convert_rows(lds + ((i + 1) & 3) * S::kRaw, lds + S::kTiles + ((i + 1) & 1) * 2 * S::kTile, threadIdx.x);
      good >>= 1;
    }

#pragma unroll
    for (int x = 0; x < T; ++x) {
      const float l = quarters_sum(st.l[x]);
      if (!cols.real[x]) continue;
      if (run.whole) {
        uint16_t* out = a.out + (int64_t)(seq.q0 + cols.row[x]) * a.out_stride + cols.head[x] * D + 4 * g;
        const float inv = l == 0.f ? 0.f : 1.f / l;  // no key seen: zeros
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<u32x2*>(out + 16 * j) = u32x2{fp4_pack_bf16(st.acc[x][j][0] * inv, st.acc[x][j][1] * inv),
                                                          fp4_pack_bf16(st.acc[x][j][2] * inv, st.acc[x][j][3] * inv)};
      } else {
        const int64_t at_part = part.at(run.slot(), 0, wave * T * 16 + 16 * x + n);
#pragma unroll
        for (int j = 0; j < 8; ++j) *reinterpret_cast<f32x4*>(part.o + at_part * D + 16 * j + 4 * g) = st.acc[x][j];
        if (g == 0) part.ml[at_part] = make_float2(st.m[x], l);
      }
    }
  }
  if (threadIdx.x == 0) part.split[run.run] = run.split;
}

constexpr int kManyBytes = ManyLds::kBytes + Line<true, kManyStep>::kBytes;
static_assert(kFewWaves == kManyWaves, "one launch has work-groups of both");

template <int HEADS>
__global__ __launch_bounds__(kFewWaves* kWave, 2) void attend_few_kernel(const Fp4AttnArgs a, const Partials few, int few_runs,
                                                                         int heads) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[FewLds<HEADS>::kBytes];
  attend_few<HEADS>(a, few, few_runs, heads, blockIdx.x % few_runs, blockIdx.x / few_runs * heads, (lds_u8*)smem);
}

// Both kinds of sequences: the work-groups of one kind begin where those of the other end. (In two launches a mixed step's
// kernels took 38.3 and 37.4 us in place of 70.4; 16 chunks alone took 1% less.)
template <int HEADS>
__global__ __launch_bounds__(kFewWaves* kWave, 2) void attend_mixed_kernel(const Fp4AttnArgs a, const Partials few,
                                                                           const Partials many, int few_runs, int many_runs,
                                                                           int heads) {
  constexpr int kBytes = FewLds<HEADS>::kBytes > kManyBytes ? FewLds<HEADS>::kBytes : kManyBytes;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[kBytes];
  const int i = (int)blockIdx.x - many_runs;
  if (i < 0)
    attend_many(a, many, many_runs, blockIdx.x, (lds_u8*)smem);
  else
    attend_few<HEADS>(a, few, few_runs, heads, i % few_runs, i / few_runs * heads, (lds_u8*)smem);
}

// The tile that begins in a run and goes on, if there is one; its partial results are the run's second slot and the
// first ones of the runs after it. `groups` work-groups share a run's columns. 32 threads take a column (of a kv head),
// 4 dimensions each, and `slices` of them share a column's partial results, which meet in LDS. Work-groups of 512 and
// 1024 threads took 30 and 32 us behind 16 chunks in place of 17.
constexpr int kMergeThreads = 256;
constexpr int kMergeTeams = kMergeThreads / 32;
template <bool MANY>
__device__ __forceinline__ void merge(const Fp4AttnArgs& a, const Partials& part, int run, int first, int groups, int slices,
                                      f32x4 (&acc_of)[kMergeTeams][32], float2 (&ml_of)[kMergeTeams]) {
  constexpr int D = kHeadDim;
  const int4 split = part.split[run];
  if (run >= *part.live || split.z == 0) return;
  const int cols = split.y, pieces = split.z;
  const int pairs = MANY ? cols : cols * a.num_kv_heads;
  const int group = 1 << a.group_shift;
  const int t = threadIdx.x & 31, team = threadIdx.x >> 5;
  const int slice = team & (slices - 1);
  const int per_pass = kMergeTeams / slices;
  for (int base = first * per_pass; base < pairs; base += groups * per_pass) {
    const int pair = base + team / slices;
    const int head = MANY ? split.w : pair / cols;
    const int col = MANY ? pair : pair - head * cols;
    float m = kLowest, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (pair < pairs) {
      const auto at = [&](int j) { return part.at(2 * (int64_t)(run + j) + (j == 0 ? 1 : 0), MANY ? 0 : head, col); };
      // four at a time, all of their loads at once: a round trip less than with the maximum found ahead (a mixed step's
      // 42 MB 14.1 us in place of 17.3, 8 sequences 5.0 in place of 6.0)
      for (int j0 = slice; j0 < pieces; j0 += 4 * slices) {
        float2 ml[4];
        f32x4 o[4];
        float top = m;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t p = at(min(j0 + i * slices, pieces - 1));
          ml[i] = part.ml[p];
          o[i] = *reinterpret_cast<const f32x4*>(part.o + p * D + 4 * t);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, ml[i].x);  // (some of another team: it only moves the reference)
        const float f = exp2_fast(m - top);
        m = top;
        l *= f;
        acc *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool real = j0 + i * slices < pieces;
          const float w = real ? exp2_fast(ml[i].x - m) : 0.f;
          l = fmaf(w, real ? ml[i].y : 0.f, l);
          acc += w * (real ? o[i] : f32x4{0.f, 0.f, 0.f, 0.f});
        }
      }
    }
    if (slices > 1) {
      acc_of[team][t] = acc;
      if (t == 0) ml_of[team] = make_float2(m, l);
      __syncthreads();
      if (slice == 0 && pair < pairs) {
        float top = m;
        for (int i = 1; i < slices; ++i) top = fmaxf(top, ml_of[team + i].x);
        const float f = exp2_fast(m - top);
        l *= f;
        acc *= f;
        for (int i = 1; i < slices; ++i) {
          const float2 ml = ml_of[team + i];
          const float w = exp2_fast(ml.x - top);
          l = fmaf(w, ml.y, l);
          acc += w * acc_of[team + i][t];
        }
      }
      __syncthreads();
    }
    if (slice != 0 || pair >= pairs) continue;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t row = split.x + (col >> a.group_shift);
    uint16_t* out = a.out + row * a.out_stride + (head * group + (col & (group - 1))) * D + 4 * t;
    *reinterpret_cast<u32x2*>(out) = u32x2{fp4_pack_bf16(acc[0] * inv, acc[1] * inv), fp4_pack_bf16(acc[2] * inv, acc[3] * inv)};
  }
}

// One of the two kernels' merges.
struct Merge {
  Partials part;
  int runs, groups, slices;  // runs that may begin a split tile
};

// Work-groups of both merges: few's runs x groups, then many's.
__global__ __launch_bounds__(kMergeThreads) void merge_kernel(const Fp4AttnArgs a, const Merge few, const Merge many) {
  __shared__ f32x4 acc_of[kMergeTeams][32];
  __shared__ float2 ml_of[kMergeTeams];
  const int i = blockIdx.x, j = i - few.runs * few.groups;
  if (j < 0)
    merge<false>(a, few.part, i / few.groups, i % few.groups, few.groups, few.slices, acc_of, ml_of);
  else
    merge<true>(a, many.part, j / many.groups, j % many.groups, many.groups, many.slices, acc_of, ml_of);
}

template <bool MANY>
Partials partials_of(const Fp4AttnArgs& a, const Fp4AttnPlan& p, char* ws) {
  const size_t rows = partial_rows<MANY>(p, a.num_kv_heads);
  const int runs = MANY ? p.many_runs : p.few_runs;
  Partials r;
  r.split = reinterpret_cast<int4*>(ws);
  r.live = reinterpret_cast<int32_t*>(r.split + runs);
  r.o = reinterpret_cast<float*>(ws + ((size_t)runs + 1) * sizeof(int4));
  r.ml = reinterpret_cast<float2*>(r.o + rows * kHeadDim);
  r.heads = MANY ? 1 : a.num_kv_heads;
  r.cols = MANY ? kManyCols : p.few_cols;
  return r;
}

size_t partial_bytes(size_t rows, size_t runs) {
  return ((runs + 1) * sizeof(int4) + rows * (kHeadDim * sizeof(float) + sizeof(float2)) + 255) / 256 * 256;
}

// Teams of 32 threads for one column of a merge: one for every four of the partial results that a tile has if the
// call has as many tiles as its bounds say, 8 at most.
int merge_slices(int runs, int64_t tiles) {
  int slices = 1;
  while (slices < kMergeTeams && tiles * slices * 4 < runs) slices *= 2;
  return slices;
}

// Work-groups that share a split tile's passes: most runs have no such tile, and empty work-groups cost their launch.
int merge_groups(int runs, int passes) { return std::max(1, std::min(passes, 8192 / runs)); }

}  // namespace

Fp4AttnPlan fp4_attention_plan(int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads, int32_t max_seqlen_q,
                               int32_t max_seqlen_k, int64_t num_rows) {
  Fp4AttnPlan p{};
  const int group = num_heads / num_kv_heads;
  // a work-group has as many kv heads as divide them evenly, 8 at most, in 1, 2, 4 or 8 slots
  p.few_heads = std::min(num_kv_heads, kFewWaves);
  while (num_kv_heads % p.few_heads) --p.few_heads;
  p.few_slots = 1;
  while (p.few_slots < p.few_heads) p.few_slots *= 2;
  const int64_t few_steps = ((int64_t)max_seqlen_k * p.few_slots + kSub * kFewWaves - 1) / (kSub * kFewWaves);
  p.steps = num_seqs * few_steps;
  p.step_keys = kSub * kFewWaves / p.few_slots;
  p.few_cols = (int)std::min<int64_t>(16, (int64_t)max_seqlen_q * group);
  // a run to a compute unit, whose LDS a work-group fills (64, 128 and 512 runs: 708, 370 and 224 us in place of 215 for
  // 256 sequences of 1k-8k keys, 16, 14 and 15 in place of 11 for 8 of 256-2048)
  p.few_runs = (int)std::min<int64_t>(256, num_seqs * few_steps);
  p.few_bytes = partial_bytes(partial_rows<false>(p, num_kv_heads), p.few_runs);
  if ((int64_t)max_seqlen_q * group > 16) {
    const int64_t steps = ((int64_t)max_seqlen_k + kManyStep - 1) / kManyStep;
    const int64_t tiles = num_rows * group / kManyCols + num_seqs;  // of a kv head
    if (tiles * steps > p.steps) {
      p.steps = tiles * steps;
      p.step_keys = kManyStep;
    }
    p.many_tiles = std::max<int64_t>(1, num_rows * group / kManyCols) * num_kv_heads;
    p.many_runs = 256;
    p.many_bytes = partial_bytes(partial_rows<true>(p, num_kv_heads), p.many_runs);
  }
  return p;
}

namespace {
template <int HEADS>
void launch_attend(const Fp4AttnArgs& a, const Fp4AttnPlan& p, const Partials& few, const Partials& many, hipStream_t stream) {
  const unsigned few_groups = (unsigned)p.few_runs * (unsigned)(a.num_kv_heads / p.few_heads);
  if (p.many_runs)
    hipLaunchKernelGGL(attend_mixed_kernel<HEADS>, dim3(p.many_runs + few_groups), dim3(kFewWaves * kWave), 0, stream, a, few,
                       many, p.few_runs, p.many_runs, p.few_heads);
  else
    hipLaunchKernelGGL(attend_few_kernel<HEADS>, dim3(few_groups), dim3(kFewWaves * kWave), 0, stream, a, few, p.few_runs,
                       p.few_heads);
}
}  // namespace

hipError_t launch_fp4_attention(const Fp4AttnArgs& a, const Fp4AttnPlan& p, hipStream_t stream) {
  char* ws = static_cast<char*>(a.workspace);
  const Partials few = partials_of<false>(a, p, ws);
  const Partials many = p.many_runs ? partials_of<true>(a, p, ws + p.few_bytes) : few;
  switch (p.few_slots) {
    case 1: launch_attend<1>(a, p, few, many, stream); break;
    case 2: launch_attend<2>(a, p, few, many, stream); break;
    case 4: launch_attend<4>(a, p, few, many, stream); break;
    default: launch_attend<8>(a, p, few, many, stream); break;
  }
  if (hipError_t err = hipGetLastError()) return err;
  Merge merge_few{few, p.few_runs - 1, 1, 1}, merge_many{few, 0, 1, 1};
  if (merge_few.runs > 0) {
    merge_few.slices = merge_slices(p.few_runs, a.num_seqs);
    const int per_pass = kMergeTeams / merge_few.slices;
    merge_few.groups = merge_groups(p.few_runs, (a.num_kv_heads * p.few_cols + per_pass - 1) / per_pass);
  }
  if (p.many_runs) {
    const int slices = merge_slices(p.many_runs, p.many_tiles);
    merge_many = Merge{many, p.many_runs - 1, merge_groups(p.many_runs, kManyCols * slices / kMergeTeams), slices};
  }
  const int groups = merge_few.runs * merge_few.groups + merge_many.runs * merge_many.groups;
  if (groups) hipLaunchKernelGGL(merge_kernel, dim3((unsigned)groups), dim3(kMergeThreads), 0, stream, a, merge_few, merge_many);
  return hipGetLastError();
}

}  // namespace pk
