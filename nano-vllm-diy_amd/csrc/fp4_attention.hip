// Attention over a paged K/V cache held in 4 bits (format: fp4.h), for any mixture of sequences: one query row, a
// few (drafted tokens), or chunks of a prompt.
//
// Reference: the flash_attn_varlen_func call over paged K/V (src/layers/attention.py:95-104), whose mask and GQA
// rules hold here; the reference has no 4-bit cache. For query row r of a sequence with Lq rows and Lk keys
//     o = sum_t p_t V[t] / sum_t p_t,   p_t = exp2(c q.K[t] - m),   t <= r + Lk - Lq,   c = scale log2(e)
// with K[t], V[t] the rows' values. One pass over the keys: m is a reference at most 8 below the largest score so
// far (in the exp2 domain); while it holds, nothing is rescaled, and p stays below 2^8. Scores, p's sum and the
// output are fp32; p is rounded to bf16 for the matrix product, as the 16-bit cache's kernels round it.
//
// Columns. A kv head's query heads and a sequence's query rows are the columns of one matrix product: column
// r G + i is query head i of the group and row r. A wavefront holds T tiles of 16 columns of one kv head and takes
// 64 keys a step:
//   S^T = K Q^T  v_mfma_f32_16x16x32_bf16, 16 keys x 16 columns: lane l holds key l % 16 and, of its 128
//                dimensions, the 32 from 32 (l / 16) -- 16 consecutive bytes of the cache with one scale byte. The
//                product runs over them 8 at a time; q is laid out in the same order of dimensions.
//   O^T += V^T P^T  lane l of S^T has column l % 16 and keys 16 t + 4 (l / 16) + i (tile t, i < 4): as the operand
//                P^T of the next product these are the 8 keys of its lane for two tiles, so P never changes lanes.
//                V^T's operand needs, for those 8 keys, dimension n(l % 16): lane l loads 4 bytes of each of them,
//                the dimensions 8 (l % 16) .. + 7, and dimension 8 (l % 16) + j is row l % 16 of the j-th of 8
//                products. So the output's rows are a permutation of the dimensions and V needs no transposition
//                either: two keys' values of one dimension are put side by side by a byte permute.
// Values convert to bf16 with their scale in one instruction for two. (The matrix instructions that read 4-bit
// values with their scales keep about 12 bits below the largest product of a sum, measured; scores here are
// held in 32, so they are not used.)
//
// Work. The steps of 64 keys of every tile of query rows lie end to end on a line, which is cut into `runs` equal
// runs, one work-group each, whatever the lengths: a work-group takes the end of one tile, whole tiles and the
// beginning of another. A tile that a cut splits leaves fp32 partial results (o, m, sum), which a second kernel
// merges; a cut splits at most one tile, so there are at most two partial results a run.
//   few rows (rows x group <= 16): T = 1, a tile is all of a sequence's rows, a wavefront is one kv head and the
//       work-group reads whole token rows.
//   more rows: T = 2, a tile is 128 columns of one kv head, a wavefront 32 of them.
#include <algorithm>

#include "fp4.h"

namespace pk {
namespace {

constexpr int kStep = 64;             // keys of a step
constexpr int kManyWaves = 4;         // wavefronts of a work-group over sequences of more rows
constexpr int kManyTiles = 2;         // tiles of 16 columns a wavefront of it holds
constexpr int kManyCols = kManyWaves * kManyTiles * 16;
constexpr int kSlots = 8;             // sequences a lane keeps the steps of
constexpr int kChunk = kSlots * kWave;
constexpr float kLowest = -3.402823466e38f;
constexpr float kSlack = 8.f;         // the scores may exceed their reference by this (exp2 domain)

typedef __attribute__((__vector_size__(8 * sizeof(__bf16)))) __bf16 frag;

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

// Inclusive sum over the wavefront.
__device__ __forceinline__ int scan64(int v, int lane) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1, :2, :4, :8
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  const int r0 = __builtin_amdgcn_readlane(v, 15), r1 = __builtin_amdgcn_readlane(v, 31),
            r2 = __builtin_amdgcn_readlane(v, 47);
  const int row = lane >> 4;
  return v + (row >= 1 ? r0 : 0) + (row >= 2 ? r1 : 0) + (row >= 3 ? r2 : 0);
}

// A sequence of the call: its first query row, the rows that are computed, and the keys. causal rows are aligned by
// the true number of rows, which max_seqlen_q only cuts.
struct Seq {
  int q0, rows, shift, keys;  // row r sees keys t <= r + shift
};
__device__ __forceinline__ Seq seq_of(const Fp4AttnArgs& a, int b) {
  const int q0 = a.cu_q[b], q1 = a.cu_q[b + 1], k0 = a.cu_k[b], k1 = a.cu_k[b + 1];
  Seq s;
  s.q0 = q0;
  s.keys = min(k1 - k0, a.max_seqlen_k);
  s.rows = s.keys > 0 ? min(q1 - q0, a.max_seqlen_q) : 0;
  s.shift = a.causal ? s.keys - (q1 - q0) : s.keys;
  return s;
}

// Steps of tile j of a sequence: up to the last key its last row sees, at least one.
template <bool MANY>
__device__ __forceinline__ int tile_steps(const Fp4AttnArgs& a, const Seq& s, int j) {
  const int per_tile = MANY ? kManyCols >> a.group_shift : s.rows;
  const int last = min(s.rows, (j + 1) * per_tile) - 1;
  const int end = min(s.keys, last + s.shift + 1);
  return max(1, (end + kStep - 1) / kStep);
}

// Steps of a sequence on the line of one kv head (MANY) or of all kv heads; 0 where it is on the other line.
template <bool MANY>
__device__ __forceinline__ int seq_steps(const Fp4AttnArgs& a, const Seq& s) {
  if (s.rows <= 0 || (s.rows << a.group_shift > 16) != MANY) return 0;
  if constexpr (!MANY) return tile_steps<false>(a, s, 0);
  const int tiles = ((s.rows << a.group_shift) + kManyCols - 1) / kManyCols;
  int n = 0;
  for (int j = 0; j < tiles; ++j) n += tile_steps<true>(a, s, j);
  return n;
}

// A tile of query rows on the line: steps [start, start + steps) of it.
struct Tile {
  int b, head, j;    // sequence, kv head (MANY), tile of it
  int64_t start;
  int steps;
};

// The line of steps: MANY: kv head by kv head, sequence by sequence, tile by tile; otherwise the sequences' steps,
// which the wavefronts take for a kv head each.
template <bool MANY>
struct Line {
  int n[kSlots];     // steps of sequence `base` + 64 s + lane
  int base;
  int per_head;      // steps of all sequences
  int64_t total;

  __device__ __forceinline__ void load(const Fp4AttnArgs& a, int first, int lane) {
    base = first;
#pragma unroll
    for (int s = 0; s < kSlots; ++s) {
      n[s] = 0;
      const int b = first + 64 * s + lane;
      if (first + 64 * s < a.num_seqs && b < a.num_seqs) n[s] = seq_steps<MANY>(a, seq_of(a, b));
    }
  }
  __device__ __forceinline__ void init(const Fp4AttnArgs& a, int lane) {
    per_head = 0;
    for (int first = 0; first < a.num_seqs; first += kChunk) {
      load(a, first, lane);
#pragma unroll
      for (int s = 0; s < kSlots; ++s)
        if (first + 64 * s < a.num_seqs) per_head += __builtin_amdgcn_readlane(scan64(n[s], lane), kWave - 1);
    }
    total = MANY ? (int64_t)per_head * a.num_kv_heads : per_head;
  }
  // The tile at position p < total.
  __device__ __forceinline__ Tile at(const Fp4AttnArgs& a, int64_t p, int lane) {
    Tile t;
    t.head = MANY ? (int)(p / per_head) : 0;
    t.j = 0;
    const int64_t head_start = (int64_t)t.head * per_head;
    const int want = (int)(p - head_start);
    int before = 0, b = 0, seq_start = 0;
    bool found = false;
    for (int first = 0; first < a.num_seqs && !found; first += kChunk) {
      if (base != first) load(a, first, lane);
#pragma unroll
      for (int s = 0; s < kSlots; ++s) {
        if (!found && first + 64 * s < a.num_seqs) {
          const int incl = before + scan64(n[s], lane);
          const uint64_t m = __builtin_amdgcn_ballot_w64(want < incl);
          if (m) {
            const int j = __builtin_ctzll(m);
            b = first + 64 * s + j;
            seq_start = __builtin_amdgcn_readlane(incl - n[s], j);
            found = true;
          }
          before = __builtin_amdgcn_readlane(incl, kWave - 1);
        }
      }
    }
    t.b = b;
    const Seq s = seq_of(a, b);
    int start = seq_start, steps = tile_steps<MANY>(a, s, 0);
    if constexpr (MANY) {
      const int tiles = ((s.rows << a.group_shift) + kManyCols - 1) / kManyCols;
      for (int j0 = 0; j0 < tiles; j0 += kWave) {
        const int j = j0 + lane;
        const int mine = j < tiles ? tile_steps<true>(a, s, j) : 0;
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
    t.start = head_start + start;
    t.steps = steps;
    return t;
  }
};

// Runs that have work, the first step of run w, and the run of step p: run w has the steps from w total / runs
// (rounded down) on, so the runs differ by one step at most.
struct Cuts {
  int64_t total;
  int64_t runs;
  __device__ __forceinline__ int64_t first(int64_t w) const { return w * total / runs; }
  __device__ __forceinline__ int run_of(int64_t p) const { return (int)(((p + 1) * runs - 1) / total); }
};
__device__ __forceinline__ Cuts cuts_of(int64_t total, int runs) { return {total, total < runs ? total : runs}; }

// Partial result `slot` (2 run: a tile that began in an earlier run; 2 run + 1: one that goes on in the next),
// of a kv head (few rows) or of the tile's only one.
struct Partials {
  float* o;       // [slot][head][column][128]
  float2* ml;     // [slot][head][column]
  int heads, cols;
  __device__ __forceinline__ int64_t at(int64_t slot, int head, int col) const {
    return (slot * heads + head) * cols + col;
  }
};
template <bool MANY>
__host__ __device__ __forceinline__ size_t partial_rows(const Fp4AttnPlan& p, int num_kv_heads) {
  return MANY ? (size_t)2 * p.many_runs * kManyCols : (size_t)2 * p.few_runs * num_kv_heads * p.few_cols;
}

// What a wavefront reads of a page's 64 rows. Four resources a cache, one for 16 rows: a row past the sequence's
// end is out of its range and reads as zeros (the range check covers the lane's offset alone), so no key needs a
// clamp, and a value behind the end is zero whatever the page holds.
struct Offsets {
  int k, ks;         // key l % 16: its 16 bytes, its scale
  int v[4], vs[4];   // key 4 (l / 16) + i: its 4 bytes, their scale
};
struct Keys {
  u32x4 d[4];
  uint32_t s[4];
};
struct Vals {
  uint32_t d[4][4];
  uint32_t s[4][4];
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const uint8_t* page, int rows, int row_bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(page), (short)0, max(rows, 0) * row_bytes, 0x00020000);
}

__device__ __forceinline__ void load_keys(Keys& k, const uint8_t* page, int rows, int row_bytes, const Offsets& o) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const __amdgpu_buffer_rsrc_t r = rows_of(page + 16 * t * row_bytes, min(rows - 16 * t, 16), row_bytes);
    k.d[t] = __builtin_amdgcn_raw_buffer_load_b128(r, o.k, 0, 0);
    k.s[t] = __builtin_amdgcn_raw_buffer_load_b8(r, o.ks, 0, 0);
  }
}

__device__ __forceinline__ void load_vals(Vals& v, const uint8_t* page, int rows, int row_bytes, const Offsets& o) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const __amdgpu_buffer_rsrc_t r = rows_of(page + 16 * t * row_bytes, min(rows - 16 * t, 16), row_bytes);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v.d[t][i] = __builtin_amdgcn_raw_buffer_load_b32(r, o.v[i], 0, 0);
      v.s[t][i] = __builtin_amdgcn_raw_buffer_load_b8(r, o.vs[i], 0, 0);
    }
  }
}

// Running softmax of the wavefront's columns: lane l has column l % 16 of every tile.
template <int T>
struct State {
  u32x4 q[T][4];     // dimensions 32 (l / 16) + 8 c .. of the column
  f32x4 acc[T][8];   // [j][i]: dimension 32 (l / 16) + 8 i + j
  float m[T];        // reference, the same in the column's four lanes
  float l[T];        // this lane's keys' share of the sum
};

template <int T>
__device__ __forceinline__ void scores(f32x4 (&s)[4][T], const State<T>& st, const Keys& k) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const float scale = fp4_scale(k.s[t]);
#pragma unroll
    for (int x = 0; x < T; ++x) s[t][x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint4 w = fp4_unpack8(k.d[t][c], scale);
#pragma unroll
      for (int x = 0; x < T; ++x) s[t][x] = mfma(u32x4{w.x, w.y, w.z, w.w}, st.q[x][c], s[t][x]);
    }
  }
}

// The step's weights of the columns, in bf16 pairs: p[x][h] are keys 16 (2 h + t) + 4 (l / 16) + i in the order t, i.
template <int T>
__device__ __forceinline__ void weights(u32x4 (&p)[T][2], f32x4 (&s)[4][T], State<T>& st, float c2) {
  float top[T];
  bool over = false;
#pragma unroll
  for (int x = 0; x < T; ++x) {
    float mx = fmaxf(s[0][x][0], s[0][x][1]);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = t ? 0 : 2; i < 4; ++i) mx = fmaxf(mx, s[t][x][i]);
    top[x] = quarters_max(mx) * c2;
    over |= top[x] > st.m[x] + kSlack;
  }
  if (__builtin_amdgcn_ballot_w64(over)) {
#pragma unroll
    for (int x = 0; x < T; ++x) {
      const float m = fmaxf(st.m[x], top[x]);
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
    for (int t = 0; t < 4; ++t) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        e[i] = exp2_fast(fmaf(s[t][x][i], c2, -st.m[x]));
        st.l[x] += e[i];
      }
      p[x][t >> 1][2 * (t & 1)] = pack_bf16x2(e[0], e[1]);
      p[x][t >> 1][2 * (t & 1) + 1] = pack_bf16x2(e[2], e[3]);
    }
  }
}

template <int kByte, int T>
__device__ __forceinline__ void add_pair(State<T>& st, const u32x4 (&p)[T][2], const Vals& v, int h) {
  u32x4 even, odd;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t x = fp4_pair<kByte>(v.d[2 * h + t][2 * i], fp4_scale(v.s[2 * h + t][2 * i]));
      const uint32_t y = fp4_pair<kByte>(v.d[2 * h + t][2 * i + 1], fp4_scale(v.s[2 * h + t][2 * i + 1]));
      even[2 * t + i] = __builtin_amdgcn_perm(y, x, 0x05040100u);
      odd[2 * t + i] = __builtin_amdgcn_perm(y, x, 0x07060302u);
    }
  }
#pragma unroll
  for (int x = 0; x < T; ++x) {
    st.acc[x][2 * kByte] = mfma(even, p[x][h], st.acc[x][2 * kByte]);
    st.acc[x][2 * kByte + 1] = mfma(odd, p[x][h], st.acc[x][2 * kByte + 1]);
  }
}

template <int T>
__device__ __forceinline__ void add_values(State<T>& st, const u32x4 (&p)[T][2], const Vals& v) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    add_pair<0>(st, p, v, h);
    add_pair<1>(st, p, v, h);
    add_pair<2>(st, p, v, h);
    add_pair<3>(st, p, v, h);
  }
}

// Whether a value block of the step is NaN (the lanes' scale bytes).
__device__ __forceinline__ bool any_nan(const Vals& v) {
  uint32_t m = 0;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, v.s[t][i]);
  return __builtin_amdgcn_ballot_w64(m == kFp4ScaleNaN) != 0;
}

// NaN blocks of a step some of whose keys some columns do not see: 0 x NaN would reach those columns through the
// matrix product. The blocks are taken as zeros there, and a column that does see such a key gets its NaN here.
// (Lane l's 32 outputs are the block l / 16 of its column. The scale bytes of one key and all four blocks are lanes
// 0, 4, 8, 12 of the row of 16 lanes that loaded the key.)
template <int T>
__device__ __forceinline__ void nan_values(State<T>& st, Vals& v, const int (&rel)[T], int lane) {
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int bad = v.s[t][i] == kFp4ScaleNaN;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int here = __shfl(bad, 16 * g + 4 * (lane >> 4));  // key 16 t + 4 g + i, block lane / 16
#pragma unroll
        for (int x = 0; x < T; ++x)
          if (here && 16 * t + 4 * g + i <= rel[x])
#pragma unroll
            for (int j = 0; j < 8; ++j) st.acc[x][j] += __builtin_nanf("");
      }
      if (bad) v.s[t][i] = v.d[t][i] = 0;
    }
}

// Work-group `index` of the line's. head0: the first kv head of its wavefronts (few rows). Neighbouring runs of
// MANY, whose tiles read the same keys, go to one XCD (work-groups go to the 8 of them in turn).
template <bool MANY, int T>
__device__ __forceinline__ void attend_run(const Fp4AttnArgs& a, const Partials& part, int num_runs, int index, int head0) {
  constexpr int D = kHeadDim;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = uniform(threadIdx.x / kWave);
  const int n = lane & 15, g = lane >> 4;
  Line<MANY> line;
  line.init(a, lane);
  if (line.total == 0) return;
  const Cuts cuts = cuts_of(line.total, num_runs);
  int run = index;
  if constexpr (MANY) {
    const int per_xcd = ((int)cuts.runs + 7) >> 3;
    if ((index >> 3) >= per_xcd) return;
    run = (index & 7) * per_xcd + (index >> 3);
  }
  if (run >= cuts.runs) return;
  const int64_t end = cuts.first(run + 1);
  for (int64_t p = cuts.first(run); p < end;) {
    const Tile tile = line.at(a, p, lane);
    const Seq seq = seq_of(a, tile.b);
    const int s0 = (int)(p - tile.start);
    const int s1 = (int)min((int64_t)tile.steps, end - tile.start);
    p = tile.start + s1;
    const int head = MANY ? tile.head : head0 + wave;
    const int group = 1 << a.group_shift;
    const int row0 = MANY ? tile.j * (kManyCols >> a.group_shift) : 0;

    // The columns: their rows, their last keys, q.
    State<T> st;
    int col[T], row[T], last[T];
    int lowest = a.max_seqlen_k;  // the last key that every column sees
    int furthest = -1;            // the last key that some column sees
#pragma unroll
    for (int x = 0; x < T; ++x) {
      col[x] = (MANY ? wave * T * 16 : 0) + 16 * x + n;
      row[x] = row0 + (col[x] >> a.group_shift);
      const bool real = row[x] < seq.rows;
      last[x] = real ? min(seq.keys - 1, row[x] + seq.shift) : -1;
      if (real) {
        lowest = min(lowest, last[x]);
        furthest = max(furthest, last[x]);
      }
      const uint16_t* q = a.q + (int64_t)(seq.q0 + row[x]) * a.q_stride + (head * group + (col[x] & (group - 1))) * D + 32 * g;
#pragma unroll
      for (int c = 0; c < 4; ++c) st.q[x][c] = real ? *reinterpret_cast<const u32x4*>(q + 8 * c) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < 8; ++j) st.acc[x][j] = f32x4{0.f, 0.f, 0.f, 0.f};
      st.m[x] = kLowest;
      st.l[x] = 0.f;
    }
#pragma unroll
    for (int sh = 1; sh < 16; sh *= 2) {
      lowest = min(lowest, __shfl_xor(lowest, sh));
      furthest = max(furthest, __shfl_xor(furthest, sh));
    }
    lowest = uniform(lowest);
    furthest = uniform(furthest);

    Offsets o;
    o.k = n * a.row_bytes + head * kFp4HeadBytes + 16 * g;
    o.ks = n * a.row_bytes + a.num_kv_heads * kFp4HeadBytes + head * kFp4HeadScales + g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o.v[i] = (4 * g + i) * a.row_bytes + head * kFp4HeadBytes + 4 * n;
      o.vs[i] = (4 * g + i) * a.row_bytes + a.num_kv_heads * kFp4HeadBytes + head * kFp4HeadScales + (n >> 2);
    }
    const int32_t* table = a.block_table + (int64_t)tile.b * a.bt_stride;
    // Step s's rows in the caches; a table entry that is no block has none, and its keys are seen by nobody.
    const uint8_t *kp, *vp;
    int rows;
    const auto page = [&](int s) {
      const int t0 = s * kStep;
      const int blk = uniform(table[t0 / a.block_size]);
      const int64_t off = (int64_t)(t0 % a.block_size) * a.row_bytes;
      const bool good = blk >= 0 && blk < a.num_blocks;
      kp = a.k + (good ? blk * a.k_block + off : 0);
      vp = a.v + (good ? blk * a.v_block + off : 0);
      rows = good ? min(seq.keys - t0, kStep) : 0;
    };

    // (wavefronts of MANY whose columns see fewer keys than the tile's last end earlier)
    const int stop = MANY ? min(s1, furthest / kStep + 1) : s1;
    if (s0 < stop && furthest >= 0) {
      Keys k;
      Vals v;
      page(s0);
      load_keys(k, kp, rows, a.row_bytes, o);
      load_vals(v, vp, rows, a.row_bytes, o);
      for (int s = s0; s < stop; ++s) {
        const int t0 = s * kStep;
        const bool bad_page = rows == 0;
        f32x4 sc[4][T];
        scores<T>(sc, st, k);
        if (s + 1 < stop) {
          page(s + 1);
          load_keys(k, kp, rows, a.row_bytes, o);
        }
        if (t0 + kStep - 1 > lowest || bad_page) {
          int rel[T];
#pragma unroll
          for (int x = 0; x < T; ++x) {
            rel[x] = bad_page ? -1 : last[x] - t0;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (16 * t + 4 * g + i > rel[x]) sc[t][x][i] = -INFINITY;
          }
          if (any_nan(v)) nan_values<T>(st, v, rel, lane);
        }
        u32x4 pw[T][2];
        weights<T>(pw, sc, st, a.scale_log2);
        add_values<T>(st, pw, v);
        if (s + 1 < stop) load_vals(v, vp, rows, a.row_bytes, o);
      }
    }

    // A whole tile's output, or a partial result of a split one.
    const bool whole = s0 == 0 && s1 == tile.steps;
    const int64_t slot = 2 * (int64_t)run + (s0 == 0 ? 1 : 0);
#pragma unroll
    for (int x = 0; x < T; ++x) {
      const float l = quarters_sum(st.l[x]);
      if (row[x] >= seq.rows) continue;
      if (whole) {
        const float inv = l == 0.f ? 0.f : 1.f / l;  // no key seen: zeros
        uint16_t* out = a.out + (int64_t)(seq.q0 + row[x]) * a.out_stride + (head * group + (col[x] & (group - 1))) * D + 32 * g;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u32x4 w;
#pragma unroll
          for (int j = 0; j < 4; ++j) w[j] = pack_bf16x2(st.acc[x][2 * j][i] * inv, st.acc[x][2 * j + 1][i] * inv);
          *reinterpret_cast<u32x4*>(out + 8 * i) = w;
        }
      } else {
        const int64_t at = part.at(slot, MANY ? 0 : head, col[x]);
        float* po = part.o + at * D + 32 * g;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          *reinterpret_cast<f32x4*>(po + 8 * i) = f32x4{st.acc[x][0][i], st.acc[x][1][i], st.acc[x][2][i], st.acc[x][3][i]};
          *reinterpret_cast<f32x4*>(po + 8 * i + 4) = f32x4{st.acc[x][4][i], st.acc[x][5][i], st.acc[x][6][i], st.acc[x][7][i]};
        }
        if (g == 0) part.ml[at] = make_float2(st.m[x], l);
      }
    }
  }
}

__global__ __launch_bounds__(8 * kWave, 2) void attend_few_kernel(const Fp4AttnArgs a, const Partials part, int runs) {
  attend_run<false, 1>(a, part, runs, blockIdx.x, blockIdx.y * (blockDim.x / kWave));
}

__global__ __launch_bounds__(kManyWaves* kWave, 2) void attend_many_kernel(const Fp4AttnArgs a, const Partials part, int runs) {
  attend_run<true, kManyTiles>(a, part, runs, blockIdx.x, 0);
}

// Work-group i: the tile that the cut between runs i and i + 1 splits, if that is its first cut. Its partial results
// are run i's second slot and the first ones of the runs after it. 32 threads a column, 4 dimensions each.
constexpr int kMergeThreads = 256;
template <bool MANY>
__global__ __launch_bounds__(kMergeThreads) void merge_kernel(const Fp4AttnArgs a, const Partials part, int runs) {
  constexpr int D = kHeadDim;
  const int lane = threadIdx.x & (kWave - 1);
  Line<MANY> line;
  line.init(a, lane);
  if (line.total == 0) return;
  const Cuts cuts = cuts_of(line.total, runs);
  const int i = blockIdx.x;
  if (i + 1 >= cuts.runs) return;
  const int64_t cut = cuts.first(i + 1);
  const Tile tile = line.at(a, cut, lane);
  if (tile.start == cut || tile.start < cuts.first(i)) return;
  const Seq seq = seq_of(a, tile.b);
  const int pieces = cuts.run_of(tile.start + tile.steps - 1) - i + 1;
  const int head = MANY ? tile.head : (int)blockIdx.y;
  const int group = 1 << a.group_shift;
  const int row0 = MANY ? tile.j * (kManyCols >> a.group_shift) : 0;
  const int cols = min((seq.rows - row0) << a.group_shift, part.cols);
  const int t = threadIdx.x & 31;
  for (int col = threadIdx.x >> 5; col < cols; col += kMergeThreads / 32) {
    const auto at = [&](int j) { return part.at(2 * (int64_t)(i + j) + (j == 0 ? 1 : 0), MANY ? 0 : head, col); };
    float m = kLowest;
    for (int j = t; j < pieces; j += 32) m = fmaxf(m, part.ml[at(j)].x);
#pragma unroll
    for (int sh = 1; sh < 32; sh *= 2) m = fmaxf(m, __shfl_xor(m, sh, 32));
    float l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < pieces; ++j) {
      const float2 ml = part.ml[at(j)];
      const float w = exp2_fast(ml.x - m);
      l = fmaf(w, ml.y, l);
      acc += w * *reinterpret_cast<const f32x4*>(part.o + at(j) * D + 4 * t);
    }
    const int row = row0 + (col >> a.group_shift);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t* out = a.out + (int64_t)(seq.q0 + row) * a.out_stride + (head * group + (col & (group - 1))) * D + 4 * t;
    *reinterpret_cast<u32x2*>(out) = u32x2{pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv)};
  }
}

template <bool MANY>
Partials partials_of(const Fp4AttnArgs& a, const Fp4AttnPlan& p, char* ws) {
  const size_t rows = partial_rows<MANY>(p, a.num_kv_heads);
  Partials r;
  r.o = reinterpret_cast<float*>(ws);
  r.ml = reinterpret_cast<float2*>(ws + rows * kHeadDim * sizeof(float));
  r.heads = MANY ? 1 : a.num_kv_heads;
  r.cols = MANY ? kManyCols : p.few_cols;
  return r;
}

size_t partial_bytes(size_t rows) { return (rows * (kHeadDim * sizeof(float) + sizeof(float2)) + 255) / 256 * 256; }

}  // namespace

Fp4AttnPlan fp4_attention_plan(int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads, int32_t max_seqlen_q,
                               int32_t max_seqlen_k, int64_t num_rows) {
  Fp4AttnPlan p{};
  const int group = num_heads / num_kv_heads;
  const int64_t steps = ((int64_t)max_seqlen_k + kStep - 1) / kStep;
  // a work-group has as many kv heads as divide them evenly, 8 at most
  p.few_heads = std::min(num_kv_heads, 8);
  while (num_kv_heads % p.few_heads) --p.few_heads;
  p.few_cols = (int)std::min<int64_t>(16, (int64_t)max_seqlen_q * group);
  const int64_t waves = 4096;
  p.few_runs = (int)std::min<int64_t>(waves / p.few_heads, num_seqs * steps);
  p.too_long = num_seqs * steps > INT32_MAX;
  p.few_bytes = partial_bytes(partial_rows<false>(p, num_kv_heads));
  if ((int64_t)max_seqlen_q * group > 16) {
    const int64_t tiles = num_rows * group / kManyCols + num_seqs;  // of a kv head
    p.too_long |= tiles * steps > INT32_MAX;
    p.many_runs = 512;
    p.many_bytes = partial_bytes(partial_rows<true>(p, num_kv_heads));
  }
  return p;
}

hipError_t launch_fp4_attention(const Fp4AttnArgs& a, const Fp4AttnPlan& p, hipStream_t stream) {
  char* ws = static_cast<char*>(a.workspace);
  const Partials few = partials_of<false>(a, p, ws);
  const int head_groups = a.num_kv_heads / p.few_heads;
  hipLaunchKernelGGL(attend_few_kernel, dim3((unsigned)p.few_runs, (unsigned)head_groups),
                     dim3((unsigned)(p.few_heads * kWave)), 0, stream, a, few, p.few_runs);
  if (hipError_t err = hipGetLastError()) return err;
  if (p.few_runs > 1)
    hipLaunchKernelGGL((merge_kernel<false>), dim3((unsigned)(p.few_runs - 1), (unsigned)a.num_kv_heads),
                       dim3(kMergeThreads), 0, stream, a, few, p.few_runs);
  if (hipError_t err = hipGetLastError()) return err;
  if (p.many_runs) {
    const Partials many = partials_of<true>(a, p, ws + p.few_bytes);
    hipLaunchKernelGGL(attend_many_kernel, dim3((unsigned)p.many_runs), dim3(kManyWaves * kWave), 0, stream, a, many,
                       p.many_runs);
    if (hipError_t err = hipGetLastError()) return err;
    hipLaunchKernelGGL((merge_kernel<true>), dim3((unsigned)(p.many_runs - 1)), dim3(kMergeThreads), 0, stream, a, many,
                       p.many_runs);
  }
  return hipGetLastError();
}

}  // namespace pk
