// Rows of 4-bit K/V caches (format: fp4.h): tokens stored as given, appended with q/k norm and rotation, and read
// back as bf16 values.
//
// Reference: the 16-bit forms of the same steps, store_kvcache (src/layers/attention.py:10-61) and the producer in
// Qwen3Attention.forward (src/models/qwen3.py:80-89); the reference has no quantised cache.
//
// Lanes: a 16-lane DPP row owns one head row of 128 values, lane c the values [8c, 8c + 8), so 32 values with one
// scale are four neighbouring lanes (a quad): their largest magnitude is two quad permutes away, and a lane packs
// its 8 values into one dword (16 lanes write the head's 64 bytes).
//
// What bounds them: HBM. A head row costs 256 bytes read and 68 written.
#include "fp4.h"
#include "norm_rope.h"

namespace pk {
namespace {

constexpr int kRowThreads = 256;
constexpr int kRowsPerGroup = kRowThreads / 16;

// The largest magnitude (bf16 bits, sign cleared; infinities and NaN stay the largest) of the quad's 32 values.
__device__ __forceinline__ uint32_t quad_top(const uint4 w) {
  uint32_t m = 0;
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, max(x[i] & 0x7fffu, (x[i] >> 16) & 0x7fffu));
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, kDppXor1, 0xf, 0xf, false));
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, kDppXor2, 0xf, 0xf, false));
  return m;
}

// A head row's 8 values of this lane into 4 bits: the lane's dword, and the quad's scale byte.
__device__ __forceinline__ uint32_t quantise8(const uint4 w, uint32_t* scale_byte) {
  *scale_byte = fp4_scale_byte(quad_top(w));
  return fp4_pack8(w, *scale_byte);
}

// The dword and the scale byte of lane c into head h of a token's row.
__device__ __forceinline__ void put_head(uint8_t* row, int heads, int h, int c, uint32_t data, uint32_t scale_byte) {
  *reinterpret_cast<uint32_t*>(row + h * kFp4HeadBytes + c * 4) = data;
  if ((c & 3) == 0) row[heads * kFp4HeadBytes + h * kFp4HeadScales + (c >> 2)] = (uint8_t)scale_byte;
}

// Head rows that a 16-lane row has in flight: a work-group takes 64 head rows at once, whole tokens (`tokens` of them;
// one token where it has more). One row at a time, with its own division and its slot's load before its own, stored
// 11406 tokens of 8 kv heads in 14.7 us, this takes 11.8 (12.1 at a large copy's rate).
constexpr int kRowsAhead = 4;
constexpr int kRowsAtOnce = kRowsPerGroup * kRowsAhead;
inline int tokens_at_once(int rows) { return rows < kRowsAtOnce ? kRowsAtOnce / rows : 1; }

__global__ __launch_bounds__(kRowThreads) void store_fp4_kernel(const Fp4StoreArgs a, int tokens) {
  const int c = threadIdx.x & 15;
  const int per_token = 2 * a.num_kv_heads;
  const int64_t first = (int64_t)blockIdx.x * tokens;
  const int rows = (int)min((int64_t)tokens, a.num_tokens - first) * per_token;
  for (int base = threadIdx.x >> 4; base < rows; base += kRowsAtOnce) {
    uint4 w[kRowsAhead];
    int32_t slot[kRowsAhead];
    int of[kRowsAhead];  // head row of its token
#pragma unroll
    for (int i = 0; i < kRowsAhead; ++i) {
      const int r = min(base + kRowsPerGroup * i, rows - 1);
      const int64_t token = first + r / per_token;
      of[i] = r % per_token;
      const uint16_t* src = of[i] < a.num_kv_heads ? a.key + token * a.key_stride + of[i] * kHeadDim
                                                   : a.value + token * a.value_stride + (of[i] - a.num_kv_heads) * kHeadDim;
      slot[i] = a.slot_mapping[token];
      w[i] = *reinterpret_cast<const uint4*>(src + c * 8);
    }
#pragma unroll
    for (int i = 0; i < kRowsAhead; ++i) {
      if (base + kRowsPerGroup * i >= rows || slot[i] < 0 || slot[i] >= a.num_slots) continue;
      const bool is_v = of[i] >= a.num_kv_heads;
      uint32_t s;
      const uint32_t d = quantise8(w[i], &s);
      put_head((is_v ? a.v_cache : a.k_cache) + (int64_t)slot[i] * a.row_bytes, a.num_kv_heads,
               is_v ? of[i] - a.num_kv_heads : of[i], c, d, s);
    }
  }
}

// Sum of a double over the 16 lanes of a DPP row, in every lane of it.
template <int kCtrl>
__device__ __forceinline__ double dpp64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, kCtrl, 0xf, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), kCtrl, 0xf, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double row16_sum64(double v) {
  v += dpp64<kDppXor1>(v);
  v += dpp64<kDppXor2>(v);
  v += dpp64<kDppHalfMirror>(v);
  v += dpp64<kDppMirror>(v);
  return v;
}

// 1 / sqrt(x) to the last bits of 64: the hardware's estimate and two steps of Newton's iteration.
__device__ __forceinline__ float inverse_root(double x) {
  double y = __builtin_amdgcn_rsq(x);
#pragma unroll
  for (int i = 0; i < 2; ++i) y = y * (1.5 - 0.5 * x * y * y);
  return x > 1.7e308 ? 0.f : (float)y;
}

// RMSNorm and rotation of one head row (norm_rope.h's steps and rounding points) with every operation rounded by
// itself and the root taken in 64 bits: which of two neighbouring 4-bit values a key gets must not hang on how a
// compiler fuses products, or on the order of a sum.
__device__ __forceinline__ uint4 norm_rope_exact(const uint4 w, const uint16_t* wt, float eps, const float cv[8],
                                                 const float sv[8], bool lower, int c) {
#pragma clang fp contract(off)
  float f[8];
  unpack8(w, f);
  if (wt != nullptr) {
    double ss = 0.;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double d = f[e];
      ss = __builtin_fma(d, d, ss);
    }
    ss = row16_sum64(ss);
    const float rs = inverse_root(ss * (1.0 / kHeadDim) + (double)eps);
    float wf[8];
    unpack8(*reinterpret_cast<const uint4*>(wt + c * 8), wf);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = round_bf16(wf[e] * (f[e] * rs));
  }
  float o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float p = dpp_ror8(f[e]);  // element d +- 64
    const float t1 = lower ? f[e] : p;
    const float t2 = lower ? p : f[e];
    const float a = t1 * (lower ? cv[e] : sv[e]);
    const float b = t2 * (lower ? sv[e] : cv[e]);
    o[e] = lower ? a - b : a + b;
  }
  return pack8(o);
}

// One wavefront per share of a token: its position, slot and cos/sin row are read once, DPP row j of it takes head
// rows 4 (part + parts i) + j, with kAppendRows of them in flight.
constexpr int kAppendRows = 8;
__global__ __launch_bounds__(kRowThreads) void append_fp4_kernel(const Fp4AppendArgs a, int parts) {
  constexpr int D = kHeadDim;
  constexpr int kWaves = kRowThreads / kWave;
  const int lane = threadIdx.x & (kWave - 1);
  const int c = lane & 15;
  const bool lower = c < 8;
  const int rows = a.num_heads + 2 * a.num_kv_heads;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t item = (int64_t)blockIdx.x * kWaves + wave;
  if (item >= (int64_t)a.num_tokens * parts) return;
  const int32_t token = (int32_t)(item / parts);
  const int part = (int)(item - (int64_t)token * parts);
  const uint16_t* src = a.qkv + (int64_t)token * a.qkv_stride + c * 8;
  const int32_t slot = a.slot_mapping[token];
  const bool stored = slot >= 0 && slot < a.num_slots;
  float cv[8], sv[8];
  rope_cos_sin_row(a.cos_sin, a.max_position, a.positions[token], c, cv, sv);
  const int stride = 4 * parts;
  for (int base = 4 * part + (lane >> 4); base < rows; base += stride * kAppendRows) {
    uint4 w[kAppendRows];
#pragma unroll
    for (int i = 0; i < kAppendRows; ++i) {
      const int r = base + stride * i;
      w[i] = *reinterpret_cast<const uint4*>(src + (r < rows ? r : base) * D);
    }
#pragma unroll
    for (int i = 0; i < kAppendRows; ++i) {
      const int r = base + stride * i;
      if (r >= rows) break;
      if (r < a.num_heads) {
        *reinterpret_cast<uint4*>(a.q_out + (int64_t)token * a.q_out_stride + r * D + c * 8) =
            norm_rope_exact(w[i], a.q_weight, a.eps, cv, sv, lower, c);
        continue;
      }
      const bool is_v = r >= a.num_heads + a.num_kv_heads;
      const int h = r - a.num_heads - (is_v ? a.num_kv_heads : 0);
      const uint4 x = is_v ? w[i] : norm_rope_exact(w[i], a.k_weight, a.eps, cv, sv, lower, c);
      uint32_t s;
      const uint32_t d = quantise8(x, &s);
      if (stored)
        put_head((is_v ? a.v_cache : a.k_cache) + (int64_t)slot * a.row_bytes, a.num_kv_heads, h, c, d, s);
      uint16_t* out = is_v ? a.v_out : a.k_out;
      if (out != nullptr)
        *reinterpret_cast<uint4*>(out + (int64_t)token * (is_v ? a.v_out_stride : a.k_out_stride) + h * D + c * 8) =
            fp4_unpack8(d, fp4_scale(s));
    }
  }
}

// Sequence blockIdx.y's rows through its table, `tokens` keys at once as store_fp4_kernel takes tokens (one head row at
// a time: 9.3 us for 11406 keys of 8 kv heads in five sequences, this: 8.4 to 8.7; 6.0 at a large copy's rate. What is over
// is the start of the launch and the chain of lengths, table entry and row.)
__global__ __launch_bounds__(kRowThreads) void gather_fp4_kernel(const Fp4GatherArgs a, int tokens) {
  const int b = blockIdx.y;
  const int c = threadIdx.x & 15;
  const int k0 = a.cu_k[b];
  if (k0 < 0) return;
  const int64_t len = min((int64_t)min(a.cu_k[b + 1] - k0, a.max_seqlen_k), a.num_rows - k0);
  const int32_t* table = a.block_table + (int64_t)b * a.bt_stride;
  for (int64_t first = (int64_t)blockIdx.x * tokens; first < len; first += (int64_t)gridDim.x * tokens) {
    const int rows = (int)min((int64_t)tokens, len - first) * a.num_kv_heads;
    for (int base = threadIdx.x >> 4; base < rows; base += kRowsAtOnce) {
      uint32_t d[kRowsAhead], s[kRowsAhead];
      int t[kRowsAhead], h[kRowsAhead], blk[kRowsAhead];
#pragma unroll
      for (int i = 0; i < kRowsAhead; ++i) {
        const int r = min(base + kRowsPerGroup * i, rows - 1);
        t[i] = (int)first + r / a.num_kv_heads;
        h[i] = r % a.num_kv_heads;
        blk[i] = table[t[i] / a.block_size];
      }
#pragma unroll
      for (int i = 0; i < kRowsAhead; ++i) {
        d[i] = s[i] = 0;  // rows of no block: zeros
        if (blk[i] < 0 || blk[i] >= a.num_blocks) continue;
        const uint8_t* row = a.cache + (int64_t)blk[i] * a.block_stride + (int64_t)(t[i] % a.block_size) * a.row_bytes;
        d[i] = *reinterpret_cast<const uint32_t*>(row + h[i] * kFp4HeadBytes + c * 4);
        s[i] = row[a.num_kv_heads * kFp4HeadBytes + h[i] * kFp4HeadScales + (c >> 2)];
      }
#pragma unroll
      for (int i = 0; i < kRowsAhead; ++i)
        if (base + kRowsPerGroup * i < rows)
          *reinterpret_cast<uint4*>(a.dst + ((int64_t)(k0 + t[i]) * a.num_kv_heads + h[i]) * kHeadDim + c * 8) =
              fp4_unpack8(d[i], fp4_scale(s[i]));
    }
  }
}

}  // namespace

hipError_t launch_store_fp4(const Fp4StoreArgs& a, hipStream_t stream) {
  const int tokens = tokens_at_once(2 * a.num_kv_heads);
  hipLaunchKernelGGL(store_fp4_kernel, dim3((unsigned)(((int64_t)a.num_tokens + tokens - 1) / tokens)), dim3(kRowThreads),
                     0, stream, a, tokens);
  return hipGetLastError();
}

hipError_t launch_append_fp4(const Fp4AppendArgs& a, hipStream_t stream) {
  const int quads = (a.num_heads + 2 * a.num_kv_heads + 3) / 4;  // 4 head rows per wavefront step
  // A token's head rows are shared by up to 8 wavefronts while that fills an idle card and not after: with 1, 2, 4
  // and 8 of them, 16 + 8 + 8 head rows took, us
  //     1 token 5.4 3.8 3.2 2.8    256  6.2  4.4  3.7  3.7    2048 12.7 11.8 11.6 14.8    16384 67 69 86 120
  //     97      6.0 4.2 3.5 3.1    512  6.5  4.9  4.6  5.1    4096 19.1 18.6 20.1 26.3
  int parts = 1;
  while (parts < 8 && (int64_t)a.num_tokens * parts * 2 <= (parts < 4 ? 8192 : 2048)) parts *= 2;
  parts = parts < quads ? parts : quads;
  const int64_t items = (int64_t)a.num_tokens * parts;
  constexpr int kWaves = kRowThreads / kWave;
  hipLaunchKernelGGL(append_fp4_kernel, dim3((unsigned)((items + kWaves - 1) / kWaves)), dim3(kRowThreads), 0, stream,
                     a, parts);
  return hipGetLastError();
}

hipError_t launch_gather_fp4(const Fp4GatherArgs& a, hipStream_t stream) {
  const int tokens = tokens_at_once(a.num_kv_heads);
  const int64_t bx = ((int64_t)a.max_seqlen_k + tokens - 1) / tokens;
  hipLaunchKernelGGL(gather_fp4_kernel, dim3((unsigned)(bx > 4096 ? 4096 : bx), (unsigned)a.num_seqs),
                     dim3(kRowThreads), 0, stream, a, tokens);
  return hipGetLastError();
}

}  // namespace pk
