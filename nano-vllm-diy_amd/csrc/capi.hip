// extern "C" entry points of libpagedkv.so (declared in include/pagedkv.h).
//
// Each entry point validates its arguments on the host (shapes, strides, 16-byte
// alignment of every vector-loaded pointer), fills the kernel argument block and
// enqueues on the caller's stream. Nothing here allocates, synchronises or reads
// device memory, so every call can be recorded into a hipGraph.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <mutex>
#include <numeric>
#include <string>

#include "../../include/pagedkv.h"
#include "common.h"
#include "fp4.h"

namespace {

thread_local std::string g_last_error;

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return code;
}

int hip_status(hipError_t err, const char* what) {
  if (err == hipSuccess) return PK_OK;
  return fail(PK_ERR_HIP, "%s: %s", what, hipGetErrorString(err));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

constexpr size_t kWorkspaceAlign = 256;
constexpr int kMaxSeqs = 65535;
constexpr int kMaxSeqlen = 65535 * 64;  // key tiles of 64 keys fit in 16 bits

size_t round_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

struct WorkspaceLayout {
  int split_tokens;
  int max_splits;
  size_t part_o_bytes;
  size_t part_ml_bytes;
  // chunked-prefill plan region (only when max_seqlen_q > 1)
  int64_t pf_item_cap;
  size_t pf_queue_off, pf_items_off, pf_merges_off, pf_part_o_off, pf_part_ml_off;
  pk::FlatDecodePlan flat;  // flat decode grid (flat.groups == 0: split grid only)
  size_t flat_meta_off;
  size_t total;
};

// [decode: partial numerators | partial (max, sum) | flat-grid record]
// (empty when no sequence can have more than one split: those write their output directly).
// Partial units: the split grid's num_seqs x max_splits (shared-prefix chunks in the first
// slots of each sequence); with the flat grid, the shared-prefix chunks (num_seqs x
// prefix_slots <= num_seqs x max_splits) followed by the grid's num_seqs + groups pieces.
// [prefill: queue header | work items | merge list | partial numerators | (max, sum)]
WorkspaceLayout workspace_layout(int num_seqs, int num_heads, int head_dim, int max_seqlen_q, int max_seqlen_k) {
  WorkspaceLayout w{};
  w.split_tokens = pk::decode_split_tokens(num_seqs, max_seqlen_k);
  w.max_splits = max_seqlen_k > 0 ? (max_seqlen_k + w.split_tokens - 1) / w.split_tokens : 0;
  w.flat = pk::decode_flat_plan(num_seqs, max_seqlen_k);  // groups > 0 only when max_splits > 1
  if (w.max_splits > 1) {  // single-split sequences write their output directly
    size_t seq_units = (size_t)num_seqs * (size_t)w.max_splits;
    if (w.flat.groups > 0) seq_units += (size_t)num_seqs + (size_t)w.flat.groups;
    const size_t units = seq_units * (size_t)num_heads;
    w.part_o_bytes = round_up(units * (size_t)head_dim * sizeof(uint16_t), kWorkspaceAlign);  // bf16
    w.part_ml_bytes = round_up(units * 2 * sizeof(float), kWorkspaceAlign);
  }
  size_t off = w.part_o_bytes + w.part_ml_bytes;
  if (w.flat.groups > 0) {  // the flat grid's run length and key-line positions, for the combine
    w.flat_meta_off = off;
    off += round_up(((size_t)num_seqs + 2) * sizeof(int32_t), kWorkspaceAlign);
  }
  if (max_seqlen_q > 1) {
    w.pf_item_cap = pk::prefill_item_cap(num_seqs, num_heads, max_seqlen_q);
    w.pf_queue_off = off;
    off += round_up(pk::kPrefillQueueInts * sizeof(int32_t), kWorkspaceAlign);
    w.pf_items_off = off;
    off += round_up((size_t)w.pf_item_cap * 16, kWorkspaceAlign);
    w.pf_merges_off = off;
    off += round_up((size_t)pk::kPrefillMergeCap * 16, kWorkspaceAlign);
    w.pf_part_o_off = off;
    off += (size_t)pk::kPrefillPartCap * 32 * pk::kPrefillRows * 4 * sizeof(uint16_t);
    w.pf_part_ml_off = off;
    off += round_up((size_t)pk::kPrefillPartCap * pk::kPrefillRows * 2 * sizeof(float), kWorkspaceAlign);
  }
  w.total = off;
  return w;
}

// The one-launch decode steps write the token's row at block * block_stride + offset *
// row_stride, where pk_store_kvcache / pk_qk_norm_rope_store write at slot * row: the two
// agree only for caches whose rows and blocks are contiguous, which both entry points
// therefore require (the reference's runner allocates the cache that way,
// model_runner.py:159-165, and asserts the row stride, attention.py:53).
int check_contiguous_cache(const char* what, int64_t k_row_stride, int64_t v_row_stride, int64_t k_block_stride,
                           int64_t v_block_stride, int32_t block_size, int32_t num_kv_heads, int32_t head_dim) {
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  if (k_row_stride != row || v_row_stride != row || k_block_stride != (int64_t)block_size * row ||
      v_block_stride != (int64_t)block_size * row)
    return fail(PK_ERR_INVALID_ARG,
                "%s: caches must have contiguous rows and blocks (row stride %lld, block stride %lld; got %lld/%lld, "
                "%lld/%lld)",
                what, (long long)row, (long long)block_size * row, (long long)k_row_stride, (long long)v_row_stride,
                (long long)k_block_stride, (long long)v_block_stride);
  return PK_OK;
}

// Shared argument checks of the decode-step linear entry points; 0 when valid.
int check_linear(const char* what, const void* x, int64_t x_row_stride, const void* weight,
                 int64_t weight_row_stride, int32_t rows, int32_t n_out, int32_t k,
                 const void* out, int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                 size_t need) {
  if (rows < 0) return fail(PK_ERR_INVALID_ARG, "%s: rows=%d < 0", what, rows);
  if (rows > pk::kLinearMaxRows)
    return fail(PK_ERR_UNSUPPORTED, "%s: rows=%d above %d (a decode-step kernel)", what, rows, pk::kLinearMaxRows);
  if (n_out <= 0 || n_out % 32 != 0)
    return fail(PK_ERR_UNSUPPORTED, "%s: n_out=%d must be a positive multiple of 32", what, n_out);
  if (k <= 0 || k % 256 != 0) return fail(PK_ERR_UNSUPPORTED, "%s: k=%d must be a positive multiple of 256", what, k);
  if (!x || !weight || !out) return fail(PK_ERR_INVALID_ARG, "%s: null x / weight / out", what);
  if (x_row_stride < k || x_row_stride % 8 || weight_row_stride < k || weight_row_stride % 8 ||
      out_row_stride < n_out || out_row_stride % 8)
    return fail(PK_ERR_INVALID_ARG, "%s: row strides must cover their rows and be multiples of 8", what);
  if (!aligned16(x) || !aligned16(weight) || !aligned16(out))
    return fail(PK_ERR_INVALID_ARG, "%s: x / weight / out must be 16-byte aligned", what);
  // out is written while other work-groups still read x: the two must not overlap
  const auto xb = reinterpret_cast<uintptr_t>(x), ob = reinterpret_cast<uintptr_t>(out);
  const uintptr_t x_end = xb + ((uintptr_t)(rows - 1) * x_row_stride + k) * 2;
  const uintptr_t o_end = ob + ((uintptr_t)(rows - 1) * out_row_stride + n_out) * 2;
  if (rows > 0 && xb < o_end && ob < x_end) return fail(PK_ERR_INVALID_ARG, "%s: out overlaps x", what);
  if (workspace_bytes < need)
    return fail(PK_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, need, workspace_bytes);
  if (need && (!workspace || !aligned16(workspace)))
    return fail(PK_ERR_WORKSPACE, "%s: workspace must be non-null and 16-byte aligned", what);
  return PK_OK;
}

// ---- pages of the cache ------------------------------------------------------------------

// Caches of the page operators: a block is block_size * row_elems contiguous elements.
int page_caches(const char* what, pk::PageCaches* c, void* k, void* v, int64_t k_layer, int64_t v_layer,
                int64_t k_block, int64_t v_block, int32_t layers, int32_t num_blocks, int32_t block_size,
                int32_t row_elems, int64_t pairs) {
  if (layers <= 0 || num_blocks <= 0 || block_size <= 0 || row_elems <= 0)
    return fail(PK_ERR_INVALID_ARG, "%s: layers=%d, num_blocks=%d, block_size=%d, row_elems=%d", what, layers,
                num_blocks, block_size, row_elems);
  if (row_elems % 8) return fail(PK_ERR_UNSUPPORTED, "%s: row_elems=%d must be a multiple of 8", what, row_elems);
  if (!k || !v || !aligned16(k) || !aligned16(v))
    return fail(PK_ERR_INVALID_ARG, "%s: caches must be non-null and 16-byte aligned", what);
  const int64_t block = (int64_t)block_size * row_elems;
  if (block > INT32_MAX) return fail(PK_ERR_UNSUPPORTED, "%s: block of %lld elements", what, (long long)block);
  if (k_block < block || v_block < block || k_block % 8 || v_block % 8 || k_layer % 8 || v_layer % 8 ||
      (layers > 1 && (k_layer < block || v_layer < block)))
    return fail(PK_ERR_INVALID_ARG, "%s: block and layer strides must be >= block_size * row_elems and multiples of 8",
                what);
  *c = pk::PageCaches{static_cast<uint4*>(k), static_cast<uint4*>(v), k_layer / 8, v_layer / 8, k_block / 8,
                      v_block / 8, layers, num_blocks, block_size, row_elems / 8};
  if (pk::copy_pieces(*c, pairs) > pk::kCopyMaxPieces)
    return fail(PK_ERR_UNSUPPORTED, "%s: %lld pages of %d layers in one call", what, (long long)pairs, layers);
  return PK_OK;
}

int page_tables(const char* what, pk::PageTables* t, int32_t* tables, int64_t stride, int32_t rows, int32_t width,
                int32_t* lens, int32_t* ref_counts, int32_t num_blocks, int32_t block_size) {
  if (rows < 0 || width < 0 || num_blocks <= 0 || block_size <= 0)
    return fail(PK_ERR_INVALID_ARG, "%s: rows=%d, table_width=%d, num_blocks=%d, block_size=%d", what, rows, width,
                num_blocks, block_size);
  if (num_blocks > (1 << 30))  // the kernels step over them in 32 bits
    return fail(PK_ERR_UNSUPPORTED, "%s: num_blocks=%d (at most 2^30)", what, num_blocks);
  if (rows > 0 && width > 0 && (!tables || stride < width))
    return fail(PK_ERR_INVALID_ARG, "%s: block_tables null, or its row stride %lld below the width %d", what,
                (long long)stride, width);
  if ((rows > 0 && !lens) || !ref_counts)
    return fail(PK_ERR_INVALID_ARG, "%s: null context_lens / ref_counts", what);
  *t = pk::PageTables{tables, stride, rows, width, lens, ref_counts, num_blocks, block_size,
                      (int32_t)std::min<int64_t>((int64_t)width * block_size, INT32_MAX)};
  return PK_OK;
}

int check_list(const char* what, int32_t n) {
  if (n < 0) return fail(PK_ERR_INVALID_ARG, "%s: %d sequences listed", what, n);
  if (n > pk::kPoolMaxList)
    return fail(PK_ERR_UNSUPPORTED, "%s: %d sequences in one call (at most %d)", what, n, pk::kPoolMaxList);
  return PK_OK;
}

int check_scratch(const char* what, const void* ws, size_t bytes, size_t need) {
  if (bytes < need || (need > 0 && !ws))
    return fail(PK_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", what, bytes, need);
  if (need > 0 && !aligned16(ws)) return fail(PK_ERR_WORKSPACE, "%s: workspace must be 16-byte aligned", what);
  return PK_OK;
}

// ---- adapters beside a projection ---------------------------------------------------------

// The slices of an operator's output columns.
int lora_slices(const char* what, pk::LoraArgs* p, int32_t n_out, const int32_t* slices, int32_t num_slices) {
  if (num_slices < 1 || num_slices > pk::kLoraMaxSlices || (num_slices > 1 && !slices))
    return fail(PK_ERR_INVALID_ARG, "%s: num_slices=%d (1 to %d, with their widths)", what, num_slices,
                pk::kLoraMaxSlices);
  int64_t sum = 0;
  for (int q = 0; q < num_slices; ++q) {
    const int32_t w = slices ? slices[q] : n_out;
    if (w <= 0) return fail(PK_ERR_INVALID_ARG, "%s: slice %d has %d columns", what, q, w);
    if (w % 32) return fail(PK_ERR_UNSUPPORTED, "%s: slice of %d columns, must be a multiple of 32", what, w);
    sum += w;
    if (sum > n_out) break;
    p->slice_begin[q + 1] = (int32_t)sum;
  }
  if (sum != n_out) return fail(PK_ERR_INVALID_ARG, "%s: the slices' widths do not add up to n_out=%d", what, n_out);
  p->num_slices = num_slices;
  return PK_OK;
}

// Whether the rows of two tensors of 16-bit elements share memory; with one stride, columns of one buffer
// beside each other do not.
bool rows_overlap(const void* a, int64_t a_stride, int64_t a_width, const void* b, int64_t b_stride, int64_t b_width,
                  int64_t rows) {
  const auto ab = reinterpret_cast<uintptr_t>(a), bb = reinterpret_cast<uintptr_t>(b);
  const uintptr_t a_end = ab + ((uintptr_t)(rows - 1) * a_stride + a_width) * 2;
  const uintptr_t b_end = bb + ((uintptr_t)(rows - 1) * b_stride + b_width) * 2;
  if (ab >= b_end || bb >= a_end) return false;
  if (a_stride != b_stride) return true;
  const int64_t s = a_stride * 2, d = (int64_t)((intptr_t)(bb - ab) % s);
  const int64_t at = d < 0 ? d + s : d;  // b's columns in a's row
  return at < a_width * 2 || at + b_width * 2 > s;
}

int lora_args(const char* what, pk::LoraArgs* p, const void* x, int64_t x_row_stride, int32_t rows, int32_t n_out,
              int32_t k, const void* lora_a, int64_t a_adapter_stride, int64_t a_row_stride, const void* lora_b,
              int64_t b_adapter_stride, int64_t b_row_stride, int32_t num_adapters, int32_t rank,
              const int32_t* adapter_ids, const float* scales, const int32_t* slices, int32_t num_slices, void* out,
              int64_t out_row_stride) {
  if (rows < 0 || n_out <= 0 || k <= 0 || num_adapters < 0)
    return fail(PK_ERR_INVALID_ARG, "%s: rows=%d, n_out=%d, k=%d, num_adapters=%d", what, rows, n_out, k, num_adapters);
  if (k % 8) return fail(PK_ERR_UNSUPPORTED, "%s: k=%d must be a multiple of 8", what, k);
  if (rows > pk::kLoraMaxRows || n_out > pk::kLoraMaxOut)
    return fail(PK_ERR_UNSUPPORTED, "%s: rows=%d, n_out=%d (at most %d and %d)", what, rows, n_out, pk::kLoraMaxRows,
                pk::kLoraMaxOut);
  if (rank <= 0 || rank % 8 || rank > pk::kLoraMaxRank)
    return fail(PK_ERR_UNSUPPORTED, "%s: rank=%d must be a multiple of 8 up to %d", what, rank, pk::kLoraMaxRank);
  *p = pk::LoraArgs{};
  if (int rc = lora_slices(what, p, n_out, slices, num_slices)) return rc;
  if (rows > 0) {
    if (!x || !out || !adapter_ids || (num_adapters > 0 && (!lora_a || !lora_b)))
      return fail(PK_ERR_INVALID_ARG, "%s: null pointer argument", what);
    if (!aligned16(x) || !aligned16(out) || (num_adapters > 0 && (!aligned16(lora_a) || !aligned16(lora_b))))
      return fail(PK_ERR_INVALID_ARG, "%s: x, lora_a, lora_b and out must be 16-byte aligned", what);
    if (x_row_stride < k || x_row_stride % 8 || out_row_stride < n_out || out_row_stride % 8)
      return fail(PK_ERR_INVALID_ARG, "%s: row strides must cover a row and be multiples of 8", what);
    if (num_adapters > 0 && (a_row_stride < k || a_row_stride % 8 || b_row_stride < rank || b_row_stride % 8 ||
                             a_adapter_stride < 0 || a_adapter_stride % 8 || b_adapter_stride < 0 ||
                             b_adapter_stride % 8))
      return fail(PK_ERR_INVALID_ARG, "%s: adapter strides must cover a row and be multiples of 8", what);
  }
  p->x = static_cast<const uint16_t*>(x);
  p->x_stride = x_row_stride;
  p->rows = rows;
  p->n_out = n_out;
  p->k = k;
  p->a = static_cast<const uint16_t*>(lora_a);
  p->a_adapter = a_adapter_stride;
  p->a_row = a_row_stride;
  p->b = static_cast<const uint16_t*>(lora_b);
  p->b_adapter = b_adapter_stride;
  p->b_row = b_row_stride;
  p->num_adapters = num_adapters;
  p->rank = rank;
  p->ids = adapter_ids;
  p->scales = scales;
  p->out = static_cast<uint16_t*>(out);
  p->out_stride = out_row_stride;
  return PK_OK;
}

}  // namespace

extern "C" {

int pk_abi_version(void) { return 12; }

const char* pk_last_error(void) { return g_last_error.c_str(); }

int pk_store_kvcache(const void* key, int64_t key_row_stride, const void* value,
                     int64_t value_row_stride, void* k_cache, void* v_cache,
                     const int32_t* slot_mapping, int32_t num_tokens, int32_t row_elems,
                     int64_t num_slots, pk_stream_t stream) {
  g_last_error.clear();
  if (num_tokens < 0) return fail(PK_ERR_INVALID_ARG, "store_kvcache: num_tokens=%d < 0", num_tokens);
  if (num_tokens == 0) return PK_OK;
  if (!key || !value || !k_cache || !v_cache || !slot_mapping)
    return fail(PK_ERR_INVALID_ARG, "store_kvcache: null pointer argument");
  if (row_elems <= 0 || row_elems % 8 != 0)
    return fail(PK_ERR_INVALID_ARG, "store_kvcache: row_elems=%d must be a positive multiple of 8", row_elems);
  if (key_row_stride < row_elems || value_row_stride < row_elems)
    return fail(PK_ERR_INVALID_ARG, "store_kvcache: row strides (%lld, %lld) smaller than row_elems=%d",
                (long long)key_row_stride, (long long)value_row_stride, row_elems);
  if (key_row_stride % 8 != 0 || value_row_stride % 8 != 0)
    return fail(PK_ERR_INVALID_ARG, "store_kvcache: row strides (%lld, %lld) must be multiples of 8 elements",
                (long long)key_row_stride, (long long)value_row_stride);
  if (!aligned16(key) || !aligned16(value) || !aligned16(k_cache) || !aligned16(v_cache))
    return fail(PK_ERR_INVALID_ARG, "store_kvcache: key/value/cache pointers must be 16-byte aligned");
  if (num_slots < 0) return fail(PK_ERR_INVALID_ARG, "store_kvcache: num_slots < 0");
  return hip_status(pk::launch_store_kvcache(key, key_row_stride, value, value_row_stride, k_cache,
                                             v_cache, slot_mapping, num_tokens, row_elems,
                                             num_slots, reinterpret_cast<hipStream_t>(stream)),
                    "store_kvcache launch");
}

int pk_gather_kv(const void* cache, int64_t block_stride, int32_t block_size,
                 const int32_t* block_table, int32_t block_table_stride,
                 const int32_t* cu_seqlens_k, int32_t num_seqs, int32_t max_seqlen_k,
                 int32_t row_elems, void* dst, pk_stream_t stream) {
  g_last_error.clear();
  if (num_seqs < 0 || max_seqlen_k < 0)
    return fail(PK_ERR_INVALID_ARG, "gather_kv: negative num_seqs or max_seqlen_k");
  if (num_seqs == 0 || max_seqlen_k == 0) return PK_OK;
  if (num_seqs > 65535) return fail(PK_ERR_INVALID_ARG, "gather_kv: num_seqs=%d > 65535", num_seqs);
  if (!cache || !block_table || !cu_seqlens_k || !dst)
    return fail(PK_ERR_INVALID_ARG, "gather_kv: null pointer argument");
  if (row_elems <= 0 || row_elems % 8 != 0 || block_stride % 8 != 0 || block_size <= 0 ||
      block_stride < (int64_t)block_size * row_elems)
    return fail(PK_ERR_INVALID_ARG, "gather_kv: bad row_elems=%d / block_size=%d / block_stride=%lld",
                row_elems, block_size, (long long)block_stride);
  if (!aligned16(cache) || !aligned16(dst))
    return fail(PK_ERR_INVALID_ARG, "gather_kv: cache and dst must be 16-byte aligned");
  return hip_status(pk::launch_gather_kv(cache, block_stride, block_size, block_table,
                                         block_table_stride, cu_seqlens_k, num_seqs, max_seqlen_k,
                                         row_elems, dst, reinterpret_cast<hipStream_t>(stream)),
                    "gather_kv launch");
}

size_t pk_varlen_attention_workspace_bytes(int32_t num_seqs, int32_t num_heads, int32_t head_dim,
                                           int32_t max_seqlen_q, int32_t max_seqlen_k) {
  if (num_seqs <= 0 || num_heads <= 0 || head_dim <= 0 || max_seqlen_k <= 0 || max_seqlen_q < 0) return 0;
  return workspace_layout(num_seqs, num_heads, head_dim, max_seqlen_q, max_seqlen_k).total;
}

int pk_varlen_attention(const void* q, int64_t q_row_stride, const void* k, const void* v,
                        int64_t k_row_stride, int64_t v_row_stride, int64_t k_block_stride,
                        int64_t v_block_stride, const int32_t* block_table,
                        int32_t block_table_stride, int32_t block_size,
                        const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int32_t num_seqs,
                        int32_t max_seqlen_q, int32_t max_seqlen_k, int32_t num_heads,
                        int32_t num_kv_heads, int32_t head_dim, float softmax_scale,
                        int32_t causal, void* out, int64_t out_row_stride, void* workspace,
                        size_t workspace_bytes, pk_stream_t stream) {
  return pk_varlen_attention_ex(q, q_row_stride, k, v, k_row_stride, v_row_stride, k_block_stride,
                                v_block_stride, block_table, block_table_stride, block_size, cu_seqlens_q,
                                cu_seqlens_k, num_seqs, max_seqlen_q, max_seqlen_k, num_heads, num_kv_heads,
                                head_dim, softmax_scale, causal, out, out_row_stride, workspace,
                                workspace_bytes, PK_CACHED_PREFIX_KEYS_DEFAULT, stream);
}

namespace {

// Inputs of the fused decode step's producer (pk_qkv_decode_attention).
struct FusedProducer {
  const void* qkv;
  int64_t qkv_row_stride;
  const int64_t* positions;
  const float* cos_sin;
  int64_t max_position;
  const void* q_norm;
  const void* k_norm;
  float eps;
  const int32_t* slot_mapping;
  int64_t num_slots;
  const void* new_k;            // store + decode: the tokens' K / V rows (qkv == nullptr)
  int64_t new_k_stride;
  const void* new_v;
  int64_t new_v_stride;
};

// Shared body of pk_varlen_attention_ex and pk_qkv_decode_attention (fp != nullptr: q comes
// from the fused producer, q itself is unused).
int attention_impl(const void* q, int64_t q_row_stride, const void* k, const void* v, int64_t k_row_stride,
                   int64_t v_row_stride, int64_t k_block_stride, int64_t v_block_stride,
                   const int32_t* block_table, int32_t block_table_stride, int32_t block_size,
                   const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int32_t num_seqs,
                   int32_t max_seqlen_q, int32_t max_seqlen_k, int32_t num_heads, int32_t num_kv_heads,
                   int32_t head_dim, float softmax_scale, int32_t causal, void* out, int64_t out_row_stride,
                   void* workspace, size_t workspace_bytes, int32_t cached_prefix_keys, const FusedProducer* fp,
                   int32_t shared_prefix_keys, int64_t num_rows, pk_stream_t stream) {
  if (head_dim != pk::kHeadDim)
    return fail(PK_ERR_UNSUPPORTED, "varlen_attention: head_dim=%d not built (only %d)", head_dim, pk::kHeadDim);
  if (num_seqs < 0 || max_seqlen_q < 0 || max_seqlen_k < 0)
    return fail(PK_ERR_INVALID_ARG, "varlen_attention: negative num_seqs / max_seqlen");
  if (num_seqs > kMaxSeqs) return fail(PK_ERR_INVALID_ARG, "varlen_attention: num_seqs=%d > %d", num_seqs, kMaxSeqs);
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
    return fail(PK_ERR_INVALID_ARG, "varlen_attention: num_heads=%d not a multiple of num_kv_heads=%d",
                num_heads, num_kv_heads);
  const int group = num_heads / num_kv_heads;
  if (group != 1 && group != 2 && group != 4 && group != 8)
    return fail(PK_ERR_UNSUPPORTED, "varlen_attention: GQA group %d not built (1, 2, 4, 8)", group);
  if (num_seqs == 0 || max_seqlen_q == 0 || max_seqlen_k == 0) return PK_OK;
  if ((!q && !(fp && fp->qkv)) || !k || !v || !out || !cu_seqlens_q || !cu_seqlens_k)
    return fail(PK_ERR_INVALID_ARG, "varlen_attention: null pointer argument");
  // the prefill work list packs key-tile indices in 16 bits and the kv head in 8
  if (max_seqlen_k > kMaxSeqlen || max_seqlen_q > kMaxSeqlen)
    return fail(PK_ERR_UNSUPPORTED, "varlen_attention: max_seqlen_q=%d / max_seqlen_k=%d above %d",
                max_seqlen_q, max_seqlen_k, kMaxSeqlen);
  if (num_kv_heads > 255)
    return fail(PK_ERR_UNSUPPORTED, "varlen_attention: num_kv_heads=%d above 255", num_kv_heads);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return fail(PK_ERR_INVALID_ARG, "varlen_attention: q/k/v/out must be 16-byte aligned");
  if (fp && fp->qkv) q_row_stride = (int64_t)num_heads * head_dim;  // unused: q comes from qkv
  const int64_t kv_row = (int64_t)num_kv_heads * head_dim;
  if (q_row_stride < (int64_t)num_heads * head_dim || out_row_stride < (int64_t)num_heads * head_dim ||
      k_row_stride < kv_row || v_row_stride < kv_row)
    return fail(PK_ERR_INVALID_ARG, "varlen_attention: a row stride is smaller than its row");
  if (q_row_stride % 8 || out_row_stride % 8 || k_row_stride % 8 || v_row_stride % 8)
    return fail(PK_ERR_INVALID_ARG, "varlen_attention: row strides must be multiples of 8 elements");
  if (k_row_stride >= (1 << 22) || v_row_stride >= (1 << 22))
    return fail(PK_ERR_INVALID_ARG, "varlen_attention: K/V row strides must be below 2^22 elements");
  const bool paged = block_table != nullptr;
  if (paged) {
    if (block_size <= 0 || block_size % 64 != 0)
      return fail(PK_ERR_INVALID_ARG, "varlen_attention: block_size=%d must be a positive multiple of 64",
                  block_size);
    if (block_table_stride < (max_seqlen_k + block_size - 1) / block_size)
      return fail(PK_ERR_INVALID_ARG,
                  "varlen_attention: block_table_stride=%d < ceil(max_seqlen_k=%d / block_size=%d)",
                  block_table_stride, max_seqlen_k, block_size);
    if (k_block_stride % 8 || v_block_stride % 8 || k_block_stride < (int64_t)block_size * k_row_stride ||
        v_block_stride < (int64_t)block_size * v_row_stride)
      return fail(PK_ERR_INVALID_ARG, "varlen_attention: bad cache block strides (%lld, %lld)",
                  (long long)k_block_stride, (long long)v_block_stride);
  }
  if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale))
    return fail(PK_ERR_INVALID_ARG, "varlen_attention: softmax_scale must be positive and finite");
  if (fp) {  // a one-launch decode step stores into the cache it reads
    if (int rc = check_contiguous_cache(fp->qkv ? "qkv_decode_attention" : "store_decode_attention", k_row_stride,
                                        v_row_stride, k_block_stride, v_block_stride, block_size, num_kv_heads,
                                        head_dim))
      return rc;
  }

  const WorkspaceLayout ws = workspace_layout(num_seqs, num_heads, head_dim, max_seqlen_q, max_seqlen_k);
  if (ws.total > 0) {
    if (!workspace || workspace_bytes < ws.total)
      return fail(PK_ERR_WORKSPACE, "varlen_attention: workspace of %zu bytes needed, %zu given",
                  ws.total, workspace ? workspace_bytes : (size_t)0);
    if ((reinterpret_cast<uintptr_t>(workspace) % kWorkspaceAlign) != 0)
      return fail(PK_ERR_WORKSPACE, "varlen_attention: workspace must be %zu-byte aligned", kWorkspaceAlign);
  }

  if (max_seqlen_q > 1 && ws.pf_item_cap > INT32_MAX)
    return fail(PK_ERR_UNSUPPORTED, "varlen_attention: prefill work list of %lld items too large",
                (long long)ws.pf_item_cap);

  pk::AttnArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_row_stride = q_row_stride;
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.k_row_stride = k_row_stride;
  a.v_row_stride = v_row_stride;
  a.k_block_stride = paged ? k_block_stride : 0;
  a.v_block_stride = paged ? v_block_stride : 0;
  a.block_table = block_table;
  a.bt_stride = paged ? block_table_stride : 0;
  a.block_size = paged ? block_size : 0;
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.num_seqs = num_seqs;
  a.max_seqlen_k = max_seqlen_k;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.out = static_cast<uint16_t*>(out);
  a.out_row_stride = out_row_stride;
  a.stream_from = cached_prefix_keys;
  if (fp) {
    a.qkv = static_cast<const uint16_t*>(fp->qkv);
    a.qkv_row_stride = fp->qkv_row_stride;
    a.positions = fp->positions;
    a.cos_sin = fp->cos_sin;
    a.max_position = fp->max_position;
    a.q_norm = static_cast<const uint16_t*>(fp->q_norm);
    a.k_norm = static_cast<const uint16_t*>(fp->k_norm);
    a.norm_eps = fp->eps;
    a.slot_mapping = fp->slot_mapping;
    a.num_slots = fp->num_slots;
    a.new_k = static_cast<const uint16_t*>(fp->new_k);
    a.new_k_stride = fp->new_k_stride;
    a.new_v = static_cast<const uint16_t*>(fp->new_v);
    a.new_v_stride = fp->new_v_stride;
  }
  a.split_tokens = ws.split_tokens;
  a.max_splits = ws.max_splits > 0 ? ws.max_splits : 1;
  a.grid_splits = a.max_splits;
  a.prefix_chunk = 1;
  a.prefix_stride = a.max_splits;
  if (shared_prefix_keys > 0 && paged && !fp && ws.max_splits > 1 && num_seqs <= pk::kSharedPrefixMaxSeqs) {
    // Shared-prefix decode. Chunks of CK = lcm(block_size, split) keys and a prefix of a
    // whole number of chunks keep the partial slots within the workspace's: P / CK prefix
    // slots + ceil((max_k - P) / split) split slots <= ceil(max_k / split).
    const int s = ws.split_tokens;
    const int ck = block_size / std::gcd(block_size, s) * s;
    const int P = std::min(shared_prefix_keys, max_seqlen_k) / ck * ck;
    if (P > 0 && ck / block_size <= pk::kSharedPrefixMaxChunkBlocks) {
      a.prefix_keys = P;
      a.prefix_chunk = ck;
      a.prefix_slots = P / ck;
      a.grid_splits = (max_seqlen_k - P + s - 1) / s;
      if (a.prefix_slots + a.grid_splits > a.max_splits)
        return fail(PK_ERR_HIP, "varlen_attention: shared-prefix slots %d + %d exceed %d", a.prefix_slots,
                    a.grid_splits, a.max_splits);
    }
  }
  char* const wsb = static_cast<char*>(workspace);
  if (ws.part_o_bytes > 0) {
    a.part_o = reinterpret_cast<uint16_t*>(wsb);
    a.part_ml = reinterpret_cast<float*>(wsb + ws.part_o_bytes);
  }
  if (ws.flat.groups > 0) {  // the flat decode grid: pieces after the shared-prefix chunks, if any
    a.flat_groups = ws.flat.groups;
    a.flat_min_chunk = ws.flat.min_chunk;
    a.flat_meta = reinterpret_cast<int32_t*>(wsb + ws.flat_meta_off);
    if (a.prefix_keys > 0) {
      a.prefix_stride = a.prefix_slots;
      a.flat_unit0 = num_seqs * a.prefix_slots;
    }
  }
  if (max_seqlen_q > 1) {
    a.pf_queue = reinterpret_cast<int32_t*>(wsb + ws.pf_queue_off);
    a.pf_items = reinterpret_cast<int4*>(wsb + ws.pf_items_off);
    a.pf_merges = reinterpret_cast<int4*>(wsb + ws.pf_merges_off);
    a.pf_part_o = reinterpret_cast<uint16_t*>(wsb + ws.pf_part_o_off);
    a.pf_part_ml = reinterpret_cast<float*>(wsb + ws.pf_part_ml_off);
    a.pf_item_cap = (int32_t)std::min<int64_t>(ws.pf_item_cap, INT32_MAX);
    a.pf_merge_cap = pk::kPrefillMergeCap;
    a.pf_part_cap = pk::kPrefillPartCap;
  }

  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  // with prefill rows the decode partials are merged by the prefill merge kernel, which the
  // call launches anyway (one launch fewer)
  a.combine_in_merge = max_seqlen_q > 1;
  int rc = PK_OK;
  hipError_t e = hipSuccess;
  if (a.prefix_keys > 0 && pk::launch_shared_prefix_flat(a, group, s, &e)) {
    // the shared-prefix work and the flat decode grid in one launch, then the combine
    rc = hip_status(e, "shared-prefix + flat decode launch");
    if (rc != PK_OK) return rc;
    rc = hip_status(pk::launch_decode_combine(a, group, s), "decode combine launch");
  } else {
    if (a.prefix_keys > 0) {
      rc = hip_status(pk::launch_shared_prefix(a, group, s), "shared-prefix launch");
      if (rc != PK_OK) return rc;
    }
    rc = hip_status(pk::launch_decode(a, group, paged, max_seqlen_k, s), "decode launch");
  }
  if (rc != PK_OK) return rc;
  if (max_seqlen_q > 1)
    rc = hip_status(pk::launch_prefill(a, group, paged, causal != 0, max_seqlen_q, num_rows, s), "prefill launch");
  return rc;
}

}  // namespace

int pk_varlen_attention_ex(const void* q, int64_t q_row_stride, const void* k, const void* v,
                           int64_t k_row_stride, int64_t v_row_stride, int64_t k_block_stride,
                           int64_t v_block_stride, const int32_t* block_table,
                           int32_t block_table_stride, int32_t block_size,
                           const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int32_t num_seqs,
                           int32_t max_seqlen_q, int32_t max_seqlen_k, int32_t num_heads,
                           int32_t num_kv_heads, int32_t head_dim, float softmax_scale,
                           int32_t causal, void* out, int64_t out_row_stride, void* workspace,
                           size_t workspace_bytes, int32_t cached_prefix_keys, pk_stream_t stream) {
  g_last_error.clear();
  return attention_impl(q, q_row_stride, k, v, k_row_stride, v_row_stride, k_block_stride, v_block_stride,
                        block_table, block_table_stride, block_size, cu_seqlens_q, cu_seqlens_k, num_seqs,
                        max_seqlen_q, max_seqlen_k, num_heads, num_kv_heads, head_dim, softmax_scale, causal, out,
                        out_row_stride, workspace, workspace_bytes, cached_prefix_keys, nullptr, 0, 0, stream);
}

int pk_varlen_attention_shared_prefix(const void* q, int64_t q_row_stride, const void* k, const void* v,
                                      int64_t k_row_stride, int64_t v_row_stride, int64_t k_block_stride,
                                      int64_t v_block_stride, const int32_t* block_table,
                                      int32_t block_table_stride, int32_t block_size,
                                      const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int32_t num_seqs,
                                      int32_t max_seqlen_q, int32_t max_seqlen_k, int32_t num_heads,
                                      int32_t num_kv_heads, int32_t head_dim, float softmax_scale, int32_t causal,
                                      void* out, int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                                      int32_t cached_prefix_keys, int32_t shared_prefix_keys, pk_stream_t stream) {
  return pk_varlen_attention_rows(q, q_row_stride, k, v, k_row_stride, v_row_stride, k_block_stride, v_block_stride,
                                  block_table, block_table_stride, block_size, cu_seqlens_q, cu_seqlens_k, num_seqs,
                                  max_seqlen_q, max_seqlen_k, num_heads, num_kv_heads, head_dim, softmax_scale,
                                  causal, out, out_row_stride, workspace, workspace_bytes, cached_prefix_keys,
                                  shared_prefix_keys, 0, stream);
}

int pk_varlen_attention_rows(const void* q, int64_t q_row_stride, const void* k, const void* v,
                             int64_t k_row_stride, int64_t v_row_stride, int64_t k_block_stride,
                             int64_t v_block_stride, const int32_t* block_table,
                             int32_t block_table_stride, int32_t block_size,
                             const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int32_t num_seqs,
                             int32_t max_seqlen_q, int32_t max_seqlen_k, int32_t num_heads,
                             int32_t num_kv_heads, int32_t head_dim, float softmax_scale, int32_t causal,
                             void* out, int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                             int32_t cached_prefix_keys, int32_t shared_prefix_keys,
                             int64_t num_rows, pk_stream_t stream) {
  g_last_error.clear();
  if (shared_prefix_keys < 0)
    return fail(PK_ERR_INVALID_ARG, "varlen_attention: shared_prefix_keys=%d < 0", shared_prefix_keys);
  if (block_table == nullptr && shared_prefix_keys > 0)
    return fail(PK_ERR_INVALID_ARG, "varlen_attention: a shared prefix needs paged K/V (block_table)");
  if (num_rows < 0) return fail(PK_ERR_INVALID_ARG, "varlen_attention: num_rows=%lld < 0", (long long)num_rows);
  return attention_impl(q, q_row_stride, k, v, k_row_stride, v_row_stride, k_block_stride, v_block_stride,
                        block_table, block_table_stride, block_size, cu_seqlens_q, cu_seqlens_k, num_seqs,
                        max_seqlen_q, max_seqlen_k, num_heads, num_kv_heads, head_dim, softmax_scale, causal, out,
                        out_row_stride, workspace, workspace_bytes, cached_prefix_keys, nullptr, shared_prefix_keys,
                        num_rows, stream);
}

int pk_qkv_decode_attention(const void* qkv, int64_t qkv_row_stride, const int64_t* positions,
                            const float* cos_sin, int64_t max_position, const void* q_norm_weight,
                            const void* k_norm_weight, float eps, void* k_cache, void* v_cache,
                            int64_t k_row_stride, int64_t v_row_stride, int64_t k_block_stride,
                            int64_t v_block_stride, const int32_t* slot_mapping, int64_t num_slots,
                            const int32_t* block_table, int32_t block_table_stride, int32_t block_size,
                            const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int32_t num_seqs,
                            int32_t max_seqlen_k, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                            float softmax_scale, void* out, int64_t out_row_stride, void* workspace,
                            size_t workspace_bytes, int32_t cached_prefix_keys, pk_stream_t stream) {
  g_last_error.clear();
  if (num_seqs <= 0 || max_seqlen_k <= 0) return num_seqs < 0 || max_seqlen_k < 0 ?
      fail(PK_ERR_INVALID_ARG, "qkv_decode_attention: negative num_seqs / max_seqlen_k") : PK_OK;
  if (!qkv || !positions || !cos_sin || !slot_mapping || !block_table)
    return fail(PK_ERR_INVALID_ARG, "qkv_decode_attention: null qkv / positions / cos_sin / slot_mapping / block_table");
  if (max_position <= 0) return fail(PK_ERR_INVALID_ARG, "qkv_decode_attention: max_position must be positive");
  if (!(eps >= 0.f)) return fail(PK_ERR_INVALID_ARG, "qkv_decode_attention: eps must be >= 0");
  if (num_slots < 0) return fail(PK_ERR_INVALID_ARG, "qkv_decode_attention: num_slots < 0");
  const int64_t row = (int64_t)(num_heads + 2 * num_kv_heads) * head_dim;
  if (qkv_row_stride < row || qkv_row_stride % 8 != 0)
    return fail(PK_ERR_INVALID_ARG, "qkv_decode_attention: qkv_row_stride=%lld must be >= %lld and a multiple of 8",
                (long long)qkv_row_stride, (long long)row);
  if (!aligned16(qkv) || !aligned16(cos_sin) || (q_norm_weight && !aligned16(q_norm_weight)) ||
      (k_norm_weight && !aligned16(k_norm_weight)))
    return fail(PK_ERR_INVALID_ARG, "qkv_decode_attention: qkv / cos_sin / norm weights must be 16-byte aligned");
  const FusedProducer fp{qkv, qkv_row_stride, positions, cos_sin, max_position, q_norm_weight, k_norm_weight,
                         eps, slot_mapping, num_slots, nullptr, 0, nullptr, 0};
  return attention_impl(nullptr, 0, k_cache, v_cache, k_row_stride, v_row_stride, k_block_stride, v_block_stride,
                        block_table, block_table_stride, block_size, cu_seqlens_q, cu_seqlens_k, num_seqs, 1,
                        max_seqlen_k, num_heads, num_kv_heads, head_dim, softmax_scale, 1, out, out_row_stride,
                        workspace, workspace_bytes, cached_prefix_keys, &fp, 0, 0, stream);
}

int pk_store_decode_attention(const void* q, int64_t q_row_stride, const void* key, int64_t key_row_stride,
                              const void* value, int64_t value_row_stride, void* k_cache, void* v_cache,
                              int64_t k_row_stride, int64_t v_row_stride, int64_t k_block_stride,
                              int64_t v_block_stride, const int32_t* slot_mapping, int64_t num_slots,
                              const int32_t* block_table, int32_t block_table_stride, int32_t block_size,
                              const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int32_t num_seqs,
                              int32_t max_seqlen_k, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                              float softmax_scale, void* out, int64_t out_row_stride, void* workspace,
                              size_t workspace_bytes, int32_t cached_prefix_keys, pk_stream_t stream) {
  g_last_error.clear();
  if (num_seqs <= 0 || max_seqlen_k <= 0) return num_seqs < 0 || max_seqlen_k < 0 ?
      fail(PK_ERR_INVALID_ARG, "store_decode_attention: negative num_seqs / max_seqlen_k") : PK_OK;
  if (!key || !value || !slot_mapping || !block_table)
    return fail(PK_ERR_INVALID_ARG, "store_decode_attention: null key / value / slot_mapping / block_table");
  if (num_slots < 0) return fail(PK_ERR_INVALID_ARG, "store_decode_attention: num_slots < 0");
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  if (key_row_stride < row || value_row_stride < row || key_row_stride % 8 || value_row_stride % 8)
    return fail(PK_ERR_INVALID_ARG, "store_decode_attention: key/value row strides must be >= %lld and multiples of 8",
                (long long)row);
  if (!aligned16(key) || !aligned16(value))
    return fail(PK_ERR_INVALID_ARG, "store_decode_attention: key / value must be 16-byte aligned");
  const FusedProducer fp{nullptr, 0, nullptr, nullptr, 0, nullptr, nullptr, 0.f, slot_mapping, num_slots,
                         key, key_row_stride, value, value_row_stride};
  return attention_impl(q, q_row_stride, k_cache, v_cache, k_row_stride, v_row_stride, k_block_stride,
                        v_block_stride, block_table, block_table_stride, block_size, cu_seqlens_q, cu_seqlens_k,
                        num_seqs, 1, max_seqlen_k, num_heads, num_kv_heads, head_dim, softmax_scale, 1, out,
                        out_row_stride, workspace, workspace_bytes, cached_prefix_keys, &fp, 0, 0, stream);
}

int pk_qk_norm_rope_store(const void* qkv, int64_t qkv_row_stride, const int64_t* positions,
                          const float* cos_sin, int64_t max_position, const void* q_norm_weight,
                          const void* k_norm_weight, float eps, int32_t num_tokens,
                          int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, void* q_out,
                          int64_t q_out_row_stride, void* k_out, int64_t k_out_row_stride,
                          void* k_cache, void* v_cache, const int32_t* slot_mapping,
                          int64_t num_slots, pk_stream_t stream) {
  g_last_error.clear();
  if (head_dim != pk::kHeadDim)
    return fail(PK_ERR_UNSUPPORTED, "qk_norm_rope_store: head_dim=%d not built (only %d)", head_dim, pk::kHeadDim);
  if (num_tokens < 0) return fail(PK_ERR_INVALID_ARG, "qk_norm_rope_store: num_tokens=%d < 0", num_tokens);
  if (num_heads <= 0 || num_kv_heads <= 0)
    return fail(PK_ERR_INVALID_ARG, "qk_norm_rope_store: num_heads=%d, num_kv_heads=%d must be positive",
                num_heads, num_kv_heads);
  if (num_tokens == 0) return PK_OK;
  if (!qkv || !positions || !cos_sin || !q_out)
    return fail(PK_ERR_INVALID_ARG, "qk_norm_rope_store: null qkv / positions / cos_sin / q_out");
  if ((k_cache == nullptr) != (v_cache == nullptr))
    return fail(PK_ERR_INVALID_ARG, "qk_norm_rope_store: pass both caches or neither");
  if (k_cache && !slot_mapping) return fail(PK_ERR_INVALID_ARG, "qk_norm_rope_store: null slot_mapping");
  if (max_position <= 0) return fail(PK_ERR_INVALID_ARG, "qk_norm_rope_store: max_position must be positive");
  if (!(eps >= 0.f)) return fail(PK_ERR_INVALID_ARG, "qk_norm_rope_store: eps must be >= 0");
  if (num_slots < 0) return fail(PK_ERR_INVALID_ARG, "qk_norm_rope_store: num_slots < 0");
  const int64_t row = (int64_t)(num_heads + 2 * num_kv_heads) * head_dim;
  if (qkv_row_stride < row || qkv_row_stride % 8 != 0)
    return fail(PK_ERR_INVALID_ARG, "qkv_row_stride=%lld must be >= %lld and a multiple of 8",
                (long long)qkv_row_stride, (long long)row);
  if (q_out_row_stride < (int64_t)num_heads * head_dim || q_out_row_stride % 8 != 0)
    return fail(PK_ERR_INVALID_ARG, "q_out_row_stride=%lld must be >= %d and a multiple of 8",
                (long long)q_out_row_stride, num_heads * head_dim);
  if (k_out && (k_out_row_stride < (int64_t)num_kv_heads * head_dim || k_out_row_stride % 8 != 0))
    return fail(PK_ERR_INVALID_ARG, "k_out_row_stride=%lld must be >= %d and a multiple of 8",
                (long long)k_out_row_stride, num_kv_heads * head_dim);
  if (!aligned16(qkv) || !aligned16(q_out) || (k_out && !aligned16(k_out)) ||
      (k_cache && (!aligned16(k_cache) || !aligned16(v_cache))) || !aligned16(cos_sin) ||
      (q_norm_weight && !aligned16(q_norm_weight)) || (k_norm_weight && !aligned16(k_norm_weight)))
    return fail(PK_ERR_INVALID_ARG, "qk_norm_rope_store: tensors must be 16-byte aligned");
  return hip_status(pk::launch_qk_norm_rope_store(qkv, qkv_row_stride, positions, cos_sin, max_position,
                                                  q_norm_weight, k_norm_weight, eps, num_tokens,
                                                  num_heads, num_kv_heads, q_out, q_out_row_stride,
                                                  k_out, k_out_row_stride, k_cache, v_cache,
                                                  slot_mapping, num_slots,
                                                  reinterpret_cast<hipStream_t>(stream)),
                    "qk_norm_rope_store launch");
}

int pk_add_rmsnorm(const void* x, int64_t x_row_stride, const void* residual,
                   int64_t residual_row_stride, const void* weight, float eps, int32_t rows,
                   int32_t hidden, void* out, int64_t out_row_stride, void* residual_out,
                   int64_t residual_out_row_stride, pk_stream_t stream) {
  g_last_error.clear();
  if (rows < 0) return fail(PK_ERR_INVALID_ARG, "add_rmsnorm: rows=%d < 0", rows);
  if (rows == 0) return PK_OK;
  if (hidden <= 0 || hidden % 8 != 0 || hidden > 4096)
    return fail(PK_ERR_UNSUPPORTED, "add_rmsnorm: hidden=%d must be a multiple of 8 and <= 4096", hidden);
  if (!x || !weight || !out || (residual && !residual_out))
    return fail(PK_ERR_INVALID_ARG, "add_rmsnorm: null x / weight / out, or residual without residual_out");
  if (x_row_stride < hidden || out_row_stride < hidden || x_row_stride % 8 || out_row_stride % 8 ||
      (residual && (residual_row_stride < hidden || residual_row_stride % 8 ||
                    residual_out_row_stride < hidden || residual_out_row_stride % 8)))
    return fail(PK_ERR_INVALID_ARG, "add_rmsnorm: row strides must be >= hidden and multiples of 8");
  if (!aligned16(x) || !aligned16(weight) || !aligned16(out) ||
      (residual && (!aligned16(residual) || !aligned16(residual_out))))
    return fail(PK_ERR_INVALID_ARG, "add_rmsnorm: tensors must be 16-byte aligned");
  return hip_status(pk::launch_add_rmsnorm(x, x_row_stride, residual, residual_row_stride, weight, eps,
                                           rows, hidden, out, out_row_stride, residual_out,
                                           residual_out_row_stride, reinterpret_cast<hipStream_t>(stream)),
                    "add_rmsnorm launch");
}

int pk_silu_and_mul(const void* x, int64_t x_row_stride, int32_t rows, int32_t inter, void* out,
                    int64_t out_row_stride, pk_stream_t stream) {
  g_last_error.clear();
  if (rows < 0) return fail(PK_ERR_INVALID_ARG, "silu_and_mul: rows=%d < 0", rows);
  if (rows == 0) return PK_OK;
  if (inter <= 0 || inter % 8 != 0)
    return fail(PK_ERR_UNSUPPORTED, "silu_and_mul: width %d must be a positive multiple of 8", inter);
  if (!x || !out) return fail(PK_ERR_INVALID_ARG, "silu_and_mul: null pointer argument");
  if (x_row_stride < 2 * (int64_t)inter || x_row_stride % 8 || out_row_stride < inter || out_row_stride % 8)
    return fail(PK_ERR_INVALID_ARG, "silu_and_mul: bad row strides");
  if (!aligned16(x) || !aligned16(out)) return fail(PK_ERR_INVALID_ARG, "silu_and_mul: tensors must be 16-byte aligned");
  return hip_status(pk::launch_silu_and_mul(x, x_row_stride, rows, inter, out, out_row_stride,
                                            reinterpret_cast<hipStream_t>(stream)),
                    "silu_and_mul launch");
}

int pk_lm_head_greedy(const void* hidden_states, int64_t row_stride, const int32_t* cu_seqlens_q,
                      const void* weight, int64_t weight_row_stride, int32_t rows, int32_t vocab,
                      int32_t hidden, uint64_t* keys, int32_t* token_ids, pk_stream_t stream) {
  g_last_error.clear();
  if (rows < 0 || vocab <= 0) return fail(PK_ERR_INVALID_ARG, "lm_head_greedy: rows=%d, vocab=%d", rows, vocab);
  if (rows == 0) return PK_OK;
  if (hidden <= 0 || hidden % 128 != 0)
    return fail(PK_ERR_UNSUPPORTED, "lm_head_greedy: hidden=%d must be a positive multiple of 128", hidden);
  if (!hidden_states || !weight || !keys || !token_ids)
    return fail(PK_ERR_INVALID_ARG, "lm_head_greedy: null pointer argument");
  if (row_stride < hidden || row_stride % 8 || weight_row_stride < hidden || weight_row_stride % 8)
    return fail(PK_ERR_INVALID_ARG, "lm_head_greedy: row strides must be >= hidden and multiples of 8");
  if (!aligned16(hidden_states) || !aligned16(weight) || (reinterpret_cast<uintptr_t>(keys) & 7u))
    return fail(PK_ERR_INVALID_ARG, "lm_head_greedy: hidden_states / weight 16-byte, keys 8-byte aligned");
  return hip_status(pk::launch_lm_head_greedy(hidden_states, row_stride, cu_seqlens_q, weight,
                                              weight_row_stride, rows, vocab, hidden,
                                              reinterpret_cast<unsigned long long*>(keys), token_ids,
                                              reinterpret_cast<hipStream_t>(stream)),
                    "lm_head_greedy launch");
}

size_t pk_linear_workspace_bytes(int32_t rows, int32_t n_out, int32_t k, int32_t epilogue) {
  if (rows <= 0 || rows > pk::kLinearMaxRows || n_out <= 0 || n_out % 32 || k <= 0 || k % 256) return 0;
  return pk::linear_workspace_bytes(rows, n_out, k, epilogue);
}

int pk_linear(const void* x, int64_t x_row_stride, const void* weight, int64_t weight_row_stride,
              int32_t rows, int32_t n_out, int32_t k, int32_t epilogue, void* out, int64_t out_row_stride,
              void* workspace, size_t workspace_bytes, pk_stream_t stream) {
  g_last_error.clear();
  if (epilogue != PK_LINEAR_STORE && epilogue != PK_LINEAR_SILU_MUL)
    return fail(PK_ERR_INVALID_ARG, "linear: epilogue=%d is not PK_LINEAR_STORE or PK_LINEAR_SILU_MUL", epilogue);
  const size_t need = pk_linear_workspace_bytes(rows, n_out, k, epilogue);
  if (int rc = check_linear("linear", x, x_row_stride, weight, weight_row_stride, rows, n_out, k, out,
                            out_row_stride, workspace, workspace_bytes, need))
    return rc;
  if (rows == 0) return PK_OK;
  return hip_status(pk::launch_linear(x, x_row_stride, weight, weight_row_stride, rows, n_out, k, epilogue, out,
                                      out_row_stride, workspace, reinterpret_cast<hipStream_t>(stream)),
                    "linear launch");
}

int pk_linear_add_rmsnorm(const void* x, int64_t x_row_stride, const void* weight, int64_t weight_row_stride,
                          int32_t rows, int32_t hidden, int32_t k, const void* residual,
                          int64_t residual_row_stride, const void* norm_weight, float eps, void* out,
                          int64_t out_row_stride, void* residual_out, int64_t residual_out_row_stride,
                          void* workspace, size_t workspace_bytes, pk_stream_t stream) {
  g_last_error.clear();
  if (hidden > 4096) return fail(PK_ERR_UNSUPPORTED, "linear_add_rmsnorm: hidden=%d above 4096", hidden);
  const size_t need = pk_linear_workspace_bytes(rows, hidden, k, PK_LINEAR_ADD_RMSNORM);
  if (int rc = check_linear("linear_add_rmsnorm", x, x_row_stride, weight, weight_row_stride, rows, hidden, k, out,
                            out_row_stride, workspace, workspace_bytes, need))
    return rc;
  if (!residual || !residual_out || !norm_weight)
    return fail(PK_ERR_INVALID_ARG, "linear_add_rmsnorm: null residual / residual_out / norm_weight");
  if (residual_row_stride < hidden || residual_row_stride % 8 || residual_out_row_stride < hidden ||
      residual_out_row_stride % 8)
    return fail(PK_ERR_INVALID_ARG, "linear_add_rmsnorm: residual row strides must be >= hidden and multiples of 8");
  if (!aligned16(residual) || !aligned16(residual_out) || !aligned16(norm_weight))
    return fail(PK_ERR_INVALID_ARG, "linear_add_rmsnorm: residual / residual_out / norm_weight must be 16-byte aligned");
  if (!(eps >= 0.f)) return fail(PK_ERR_INVALID_ARG, "linear_add_rmsnorm: eps must be >= 0");
  if (rows == 0) return PK_OK;
  return hip_status(pk::launch_linear_add_rmsnorm(x, x_row_stride, weight, weight_row_stride, rows, hidden, k,
                                                  residual, residual_row_stride, norm_weight, eps, out,
                                                  out_row_stride, residual_out, residual_out_row_stride,
                                                  workspace, reinterpret_cast<hipStream_t>(stream)),
                    "linear_add_rmsnorm launch");
}

size_t pk_lora_linear_workspace_bytes(int32_t rows, int32_t n_out, int32_t k, int32_t rank, int32_t num_slices) {
  if (rows <= 0 || rows > pk::kLinearMaxRows || n_out <= 0 || n_out % 32 || k <= 0 || k % 256 || rank <= 0 ||
      rank > pk::kLoraMaxRank || num_slices <= 0 || num_slices > pk::kLoraMaxSlices)
    return 0;
  pk::LoraArgs p{};
  p.rows = rows, p.n_out = n_out, p.k = k, p.rank = rank, p.num_slices = num_slices;
  return pk::lora_linear_workspace_bytes(p);
}

int pk_lora_linear(const void* x, int64_t x_row_stride, const void* weight, int64_t weight_row_stride, int32_t rows,
                   int32_t n_out, int32_t k, const void* lora_a, int64_t a_adapter_stride, int64_t a_row_stride,
                   const void* lora_b, int64_t b_adapter_stride, int64_t b_row_stride, int32_t num_adapters,
                   int32_t rank, const int32_t* adapter_ids, const float* scales, const int32_t* slices,
                   int32_t num_slices, void* out, int64_t out_row_stride, void* workspace, size_t workspace_bytes,
                   pk_stream_t stream) {
  g_last_error.clear();
  pk::LoraArgs p;
  if (int rc = lora_args("lora_linear", &p, x, x_row_stride, rows, n_out, k, lora_a, a_adapter_stride, a_row_stride,
                         lora_b, b_adapter_stride, b_row_stride, num_adapters, rank, adapter_ids, scales, slices,
                         num_slices, out, out_row_stride))
    return rc;
  if (rows == 0) return PK_OK;
  const size_t need = pk_lora_linear_workspace_bytes(rows, n_out, k, rank, num_slices);
  if (int rc = check_linear("lora_linear", x, x_row_stride, weight, weight_row_stride, rows, n_out, k, out,
                            out_row_stride, workspace, workspace_bytes, need))
    return rc;
  return hip_status(pk::launch_lora_linear(p, weight, weight_row_stride, workspace,
                                           reinterpret_cast<hipStream_t>(stream)),
                    "lora_linear launch");
}

size_t pk_lora_add_workspace_bytes(int32_t rows, int32_t n_out, int32_t rank, const int32_t* slices,
                                   int32_t num_slices, int32_t num_adapters) {
  pk::LoraArgs p{};
  if (rows <= 0 || rank <= 0 || rank > pk::kLoraMaxRank || num_adapters < 0 ||
      lora_slices("lora_add", &p, n_out, slices, num_slices) != PK_OK)
    return 0;
  p.rows = rows, p.n_out = n_out, p.rank = rank, p.num_adapters = num_adapters;
  return pk::lora_add_workspace_bytes(p);
}

int pk_lora_add(const void* y, int64_t y_row_stride, const void* x, int64_t x_row_stride, int32_t rows, int32_t n_out,
                int32_t k, const void* lora_a, int64_t a_adapter_stride, int64_t a_row_stride, const void* lora_b,
                int64_t b_adapter_stride, int64_t b_row_stride, int32_t num_adapters, int32_t rank,
                const int32_t* adapter_ids, const float* scales, const int32_t* slices, int32_t num_slices, void* out,
                int64_t out_row_stride, void* workspace, size_t workspace_bytes, pk_stream_t stream) {
  g_last_error.clear();
  pk::LoraArgs p;
  if (int rc = lora_args("lora_add", &p, x, x_row_stride, rows, n_out, k, lora_a, a_adapter_stride, a_row_stride,
                         lora_b, b_adapter_stride, b_row_stride, num_adapters, rank, adapter_ids, scales, slices,
                         num_slices, out, out_row_stride))
    return rc;
  if (rows == 0) return PK_OK;
  if (!y || !aligned16(y) || y_row_stride < n_out || y_row_stride % 8)
    return fail(PK_ERR_INVALID_ARG, "lora_add: y null, not 16-byte aligned, or its row stride no multiple of 8 >= n_out");
  if (y == out && y_row_stride != out_row_stride)
    return fail(PK_ERR_INVALID_ARG, "lora_add: out may be y only with y's row stride");
  if (pk::lora_add_groups(p) > pk::kLoraMaxGroups)
    return fail(PK_ERR_UNSUPPORTED, "lora_add: rows=%d of n_out=%d are too many for one launch", rows, n_out);
  // out is written while other work-groups still read x and y
  if (rows_overlap(out, out_row_stride, n_out, x, x_row_stride, k, rows))
    return fail(PK_ERR_INVALID_ARG, "lora_add: out overlaps x");
  if (y != out && rows_overlap(out, out_row_stride, n_out, y, y_row_stride, n_out, rows))
    return fail(PK_ERR_INVALID_ARG, "lora_add: out overlaps y without being y");
  if (int rc = check_scratch("lora_add", workspace, workspace_bytes,
                             pk::lora_add_workspace_bytes(p)))
    return rc;
  p.y = static_cast<const uint16_t*>(y);
  p.y_stride = y_row_stride;
  return hip_status(pk::launch_lora_add(p, workspace, reinterpret_cast<hipStream_t>(stream)), "lora_add launch");
}

int pk_copy_blocks(void* k_caches, void* v_caches, int64_t k_layer_stride, int64_t v_layer_stride,
                   int64_t k_block_stride, int64_t v_block_stride, int32_t num_layers, int32_t num_blocks,
                   int32_t block_size, int32_t row_elems, const int32_t* src_blocks, const int32_t* dst_blocks,
                   const int32_t* num_tokens, int32_t num_pairs, pk_stream_t stream) {
  g_last_error.clear();
  if (num_pairs < 0) return fail(PK_ERR_INVALID_ARG, "copy_blocks: num_pairs=%d < 0", num_pairs);
  pk::PageCaches c{};
  if (int rc = page_caches("copy_blocks", &c, k_caches, v_caches, k_layer_stride, v_layer_stride, k_block_stride,
                           v_block_stride, num_layers, num_blocks, block_size, row_elems, num_pairs))
    return rc;
  if (num_pairs == 0) return PK_OK;
  if (!src_blocks || !dst_blocks) return fail(PK_ERR_INVALID_ARG, "copy_blocks: null src_blocks / dst_blocks");
  return hip_status(pk::launch_copy_blocks(c, src_blocks, dst_blocks, num_tokens, num_pairs,
                                           reinterpret_cast<hipStream_t>(stream)),
                    "copy_blocks launch");
}

size_t pk_fork_workspace_bytes(int32_t num_forks) { return pk::fork_workspace_bytes(num_forks); }

int pk_fork_sequences(void* k_caches, void* v_caches, int64_t k_layer_stride, int64_t v_layer_stride,
                      int64_t k_block_stride, int64_t v_block_stride, int32_t num_layers, int32_t num_blocks,
                      int32_t block_size, int32_t row_elems, int32_t* block_tables, int64_t block_table_stride,
                      int32_t num_rows, int32_t table_width, int32_t* context_lens, int32_t* ref_counts,
                      const int32_t* parents, const int32_t* children, int32_t num_forks, int32_t* new_blocks,
                      void* workspace, size_t workspace_bytes, pk_stream_t stream) {
  g_last_error.clear();
  if (int rc = check_list("fork_sequences", num_forks)) return rc;
  pk::PageCaches c{};
  pk::PageTables t{};
  if (int rc = page_caches("fork_sequences", &c, k_caches, v_caches, k_layer_stride, v_layer_stride, k_block_stride,
                           v_block_stride, num_layers, num_blocks, block_size, row_elems, num_forks))
    return rc;
  if (int rc = page_tables("fork_sequences", &t, block_tables, block_table_stride, num_rows, table_width,
                           context_lens, ref_counts, num_blocks, block_size))
    return rc;
  if (num_forks == 0) return PK_OK;
  if (!parents || !children || !new_blocks)
    return fail(PK_ERR_INVALID_ARG, "fork_sequences: null parents / children / new_blocks");
  if (int rc = check_scratch("fork_sequences", workspace, workspace_bytes, pk_fork_workspace_bytes(num_forks)))
    return rc;
  return hip_status(pk::launch_fork_sequences(t, c, parents, children, num_forks, new_blocks, workspace,
                                              reinterpret_cast<hipStream_t>(stream)),
                    "fork_sequences launch");
}

int pk_extend_sequences(int32_t* block_tables, int64_t block_table_stride, int32_t num_rows, int32_t table_width,
                        int32_t* context_lens, int32_t* ref_counts, int32_t num_blocks, int32_t block_size,
                        const int32_t* rows, int32_t num_listed, int32_t* slot_mapping, pk_stream_t stream) {
  g_last_error.clear();
  if (int rc = check_list("extend_sequences", num_listed)) return rc;
  pk::PageTables t{};
  if (int rc = page_tables("extend_sequences", &t, block_tables, block_table_stride, num_rows, table_width,
                           context_lens, ref_counts, num_blocks, block_size))
    return rc;
  if ((int64_t)num_blocks * block_size > INT32_MAX)
    return fail(PK_ERR_UNSUPPORTED, "extend_sequences: %lld slots do not fit 32-bit slot numbers",
                (long long)num_blocks * block_size);
  if (num_listed == 0) return PK_OK;
  if (!rows || !slot_mapping) return fail(PK_ERR_INVALID_ARG, "extend_sequences: null rows / slot_mapping");
  return hip_status(pk::launch_extend_sequences(t, rows, num_listed, slot_mapping,
                                                reinterpret_cast<hipStream_t>(stream)),
                    "extend_sequences launch");
}

int pk_free_sequences(int32_t* block_tables, int64_t block_table_stride, int32_t num_rows, int32_t table_width,
                      int32_t* context_lens, int32_t* ref_counts, int32_t num_blocks, int32_t block_size,
                      const int32_t* rows, int32_t num_listed, pk_stream_t stream) {
  g_last_error.clear();
  if (num_listed < 0) return fail(PK_ERR_INVALID_ARG, "free_sequences: %d sequences listed", num_listed);
  if (num_listed > (1 << 24))
    return fail(PK_ERR_UNSUPPORTED, "free_sequences: %d sequences in one call (at most 2^24)", num_listed);
  pk::PageTables t{};
  if (int rc = page_tables("free_sequences", &t, block_tables, block_table_stride, num_rows, table_width,
                           context_lens, ref_counts, num_blocks, block_size))
    return rc;
  if (num_listed == 0) return PK_OK;
  if (!rows) return fail(PK_ERR_INVALID_ARG, "free_sequences: null rows");
  return hip_status(pk::launch_free_sequences(t, rows, num_listed, reinterpret_cast<hipStream_t>(stream)),
                    "free_sequences launch");
}

size_t pk_compact_workspace_bytes(int32_t num_blocks) { return pk::compact_workspace_bytes(num_blocks); }

int pk_compact_blocks(void* k_caches, void* v_caches, int64_t k_layer_stride, int64_t v_layer_stride,
                      int64_t k_block_stride, int64_t v_block_stride, int32_t num_layers, int32_t num_blocks,
                      int32_t block_size, int32_t row_elems, int32_t* block_tables, int64_t block_table_stride,
                      int32_t num_rows, int32_t table_width, const int32_t* context_lens, int32_t* ref_counts,
                      int32_t* block_map, int32_t* num_live, void* workspace, size_t workspace_bytes,
                      pk_stream_t stream) {
  g_last_error.clear();
  pk::PageCaches c{};
  pk::PageTables t{};
  if (int rc = page_caches("compact_blocks", &c, k_caches, v_caches, k_layer_stride, v_layer_stride, k_block_stride,
                           v_block_stride, num_layers, num_blocks, block_size, row_elems, num_blocks))
    return rc;
  if (int rc = page_tables("compact_blocks", &t, block_tables, block_table_stride, num_rows, table_width,
                           const_cast<int32_t*>(context_lens), ref_counts, num_blocks, block_size))
    return rc;
  if (!block_map || !num_live) return fail(PK_ERR_INVALID_ARG, "compact_blocks: null block_map / num_live");
  if (int rc = check_scratch("compact_blocks", workspace, workspace_bytes, pk_compact_workspace_bytes(num_blocks)))
    return rc;
  return hip_status(pk::launch_compact_blocks(t, c, block_map, num_live, workspace,
                                              reinterpret_cast<hipStream_t>(stream)),
                    "compact_blocks launch");
}

// ---- caches held in 4 bits -----------------------------------------------------------------

namespace {

// A pair of 4-bit caches' head geometry; 0 when it is built.
int fp4_heads(const char* what, int32_t num_kv_heads, int32_t head_dim) {
  if (head_dim != pk::kHeadDim)
    return fail(PK_ERR_UNSUPPORTED, "%s: head_dim=%d not built (only %d)", what, head_dim, pk::kHeadDim);
  if (num_kv_heads <= 0 || num_kv_heads > pk::kFp4MaxHeads)
    return fail(PK_ERR_UNSUPPORTED, "%s: num_kv_heads=%d (1 to %d)", what, num_kv_heads, pk::kFp4MaxHeads);
  return PK_OK;
}

// Tokens and head rows of a call are counted in 32 bits, up to 8 wavefronts to a token.
int fp4_tokens(const char* what, int64_t tokens, int64_t head_rows) {
  if (tokens < 0) return fail(PK_ERR_INVALID_ARG, "%s: %lld tokens", what, (long long)tokens);
  if (tokens * head_rows >= (1ll << 27))
    return fail(PK_ERR_UNSUPPORTED, "%s: %lld tokens of %lld head rows in one call (below 2^27)", what,
                (long long)tokens, (long long)head_rows);
  return PK_OK;
}

// A (tokens, heads, 128) bf16 tensor with contiguous heads.
int fp4_rows(const char* what, const char* name, const void* p, int64_t stride, int64_t heads) {
  if (!p) return fail(PK_ERR_INVALID_ARG, "%s: null %s", what, name);
  if (!aligned16(p) || stride < heads * pk::kHeadDim || stride % 8)
    return fail(PK_ERR_INVALID_ARG, "%s: %s must be 16-byte aligned, its row stride %lld a multiple of 8 that covers a row",
                what, name, (long long)stride);
  return PK_OK;
}

int fp4_caches(const char* what, const void* k, const void* v) {
  if (!k || !v || !aligned16(k) || !aligned16(v))
    return fail(PK_ERR_INVALID_ARG, "%s: caches must be non-null and 16-byte aligned", what);
  return PK_OK;
}

int fp4_blocks(const char* what, int64_t block_stride, int32_t num_blocks, int32_t block_size, int32_t row_bytes) {
  if (num_blocks <= 0 || block_size <= 0)
    return fail(PK_ERR_INVALID_ARG, "%s: num_blocks=%d, block_size=%d", what, num_blocks, block_size);
  if (block_stride < (int64_t)block_size * row_bytes || block_stride % 16)
    return fail(PK_ERR_INVALID_ARG, "%s: block stride of %lld bytes, must be a multiple of 16 and cover %d rows of %d",
                what, (long long)block_stride, block_size, row_bytes);
  return PK_OK;
}

}  // namespace

size_t pk_fp4_row_bytes(int32_t num_kv_heads) {
  return num_kv_heads > 0 && num_kv_heads <= pk::kFp4MaxHeads ? (size_t)pk::fp4_row_bytes(num_kv_heads) : 0;
}

int pk_store_kvcache_fp4(const void* key, int64_t key_row_stride, const void* value, int64_t value_row_stride,
                         void* k_cache, void* v_cache, const int32_t* slot_mapping, int32_t num_tokens,
                         int32_t num_kv_heads, int32_t head_dim, int64_t num_slots, pk_stream_t stream) {
  g_last_error.clear();
  const char* what = "store_kvcache_fp4";
  if (int rc = fp4_heads(what, num_kv_heads, head_dim)) return rc;
  if (int rc = fp4_tokens(what, num_tokens, 2 * num_kv_heads)) return rc;
  if (num_slots < 0) return fail(PK_ERR_INVALID_ARG, "%s: num_slots < 0", what);
  if (num_tokens == 0) return PK_OK;
  if (int rc = fp4_rows(what, "key", key, key_row_stride, num_kv_heads)) return rc;
  if (int rc = fp4_rows(what, "value", value, value_row_stride, num_kv_heads)) return rc;
  if (int rc = fp4_caches(what, k_cache, v_cache)) return rc;
  if (!slot_mapping) return fail(PK_ERR_INVALID_ARG, "%s: null slot_mapping", what);
  pk::Fp4StoreArgs a{};
  a.key = static_cast<const uint16_t*>(key);
  a.key_stride = key_row_stride;
  a.value = static_cast<const uint16_t*>(value);
  a.value_stride = value_row_stride;
  a.k_cache = static_cast<uint8_t*>(k_cache);
  a.v_cache = static_cast<uint8_t*>(v_cache);
  a.slot_mapping = slot_mapping;
  a.num_tokens = num_tokens;
  a.num_kv_heads = num_kv_heads;
  a.row_bytes = pk::fp4_row_bytes(num_kv_heads);
  a.num_slots = num_slots;
  return hip_status(pk::launch_store_fp4(a, reinterpret_cast<hipStream_t>(stream)), "store_kvcache_fp4 launch");
}

int pk_qk_norm_rope_store_fp4(const void* qkv, int64_t qkv_row_stride, const int64_t* positions, const float* cos_sin,
                              int64_t max_position, const void* q_norm_weight, const void* k_norm_weight, float eps,
                              int32_t num_tokens, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                              void* q_out, int64_t q_out_row_stride, void* k_out, int64_t k_out_row_stride,
                              void* v_out, int64_t v_out_row_stride, void* k_cache, void* v_cache,
                              const int32_t* slot_mapping, int64_t num_slots, pk_stream_t stream) {
  g_last_error.clear();
  const char* what = "qk_norm_rope_store_fp4";
  if (int rc = fp4_heads(what, num_kv_heads, head_dim)) return rc;
  if (num_heads <= 0 || num_heads > 65535) return fail(PK_ERR_INVALID_ARG, "%s: num_heads=%d", what, num_heads);
  if (int rc = fp4_tokens(what, num_tokens, num_heads + 2 * num_kv_heads)) return rc;
  if (num_slots < 0 || max_position <= 0)
    return fail(PK_ERR_INVALID_ARG, "%s: num_slots=%lld, max_position=%lld", what, (long long)num_slots,
                (long long)max_position);
  if (!(eps >= 0.f) || !std::isfinite(eps)) return fail(PK_ERR_INVALID_ARG, "%s: eps must be finite and not negative", what);
  if (num_tokens == 0) return PK_OK;
  if (int rc = fp4_rows(what, "qkv", qkv, qkv_row_stride, num_heads + 2 * num_kv_heads)) return rc;
  if (int rc = fp4_rows(what, "q_out", q_out, q_out_row_stride, num_heads)) return rc;
  if (k_out)
    if (int rc = fp4_rows(what, "k_out", k_out, k_out_row_stride, num_kv_heads)) return rc;
  if (v_out)
    if (int rc = fp4_rows(what, "v_out", v_out, v_out_row_stride, num_kv_heads)) return rc;
  if (int rc = fp4_caches(what, k_cache, v_cache)) return rc;
  if (!positions || !cos_sin || !slot_mapping)
    return fail(PK_ERR_INVALID_ARG, "%s: null positions / cos_sin / slot_mapping", what);
  if (!aligned16(cos_sin) || (q_norm_weight && !aligned16(q_norm_weight)) || (k_norm_weight && !aligned16(k_norm_weight)))
    return fail(PK_ERR_INVALID_ARG, "%s: cos_sin and norm weights must be 16-byte aligned", what);
  pk::Fp4AppendArgs a{};
  a.qkv = static_cast<const uint16_t*>(qkv);
  a.qkv_stride = qkv_row_stride;
  a.positions = positions;
  a.cos_sin = cos_sin;
  a.max_position = max_position;
  a.q_weight = static_cast<const uint16_t*>(q_norm_weight);
  a.k_weight = static_cast<const uint16_t*>(k_norm_weight);
  a.eps = eps;
  a.num_tokens = num_tokens;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.row_bytes = pk::fp4_row_bytes(num_kv_heads);
  a.q_out = static_cast<uint16_t*>(q_out);
  a.q_out_stride = q_out_row_stride;
  a.k_out = static_cast<uint16_t*>(k_out);
  a.k_out_stride = k_out_row_stride;
  a.v_out = static_cast<uint16_t*>(v_out);
  a.v_out_stride = v_out_row_stride;
  a.k_cache = static_cast<uint8_t*>(k_cache);
  a.v_cache = static_cast<uint8_t*>(v_cache);
  a.slot_mapping = slot_mapping;
  a.num_slots = num_slots;
  return hip_status(pk::launch_append_fp4(a, reinterpret_cast<hipStream_t>(stream)), "qk_norm_rope_store_fp4 launch");
}

int pk_gather_kv_fp4(const void* cache, int64_t block_stride, int32_t num_blocks, int32_t block_size,
                     int32_t num_kv_heads, int32_t head_dim, const int32_t* block_table, int32_t block_table_stride,
                     const int32_t* cu_seqlens_k, int32_t num_seqs, int32_t max_seqlen_k, int64_t num_rows, void* dst,
                     pk_stream_t stream) {
  g_last_error.clear();
  const char* what = "gather_kv_fp4";
  if (int rc = fp4_heads(what, num_kv_heads, head_dim)) return rc;
  if (num_rows < 0) return fail(PK_ERR_INVALID_ARG, "%s: num_rows=%lld", what, (long long)num_rows);
  if (num_seqs < 0 || num_seqs > kMaxSeqs || max_seqlen_k < 0 || max_seqlen_k > kMaxSeqlen)
    return fail(PK_ERR_INVALID_ARG, "%s: num_seqs=%d (at most %d), max_seqlen_k=%d (at most %d)", what, num_seqs,
                kMaxSeqs, max_seqlen_k, kMaxSeqlen);
  if (num_seqs == 0 || max_seqlen_k == 0 || num_rows == 0) return PK_OK;
  if (int rc = fp4_blocks(what, block_stride, num_blocks, block_size, pk::fp4_row_bytes(num_kv_heads))) return rc;
  if (!cache || !block_table || !cu_seqlens_k || !dst) return fail(PK_ERR_INVALID_ARG, "%s: null pointer argument", what);
  if (!aligned16(cache) || !aligned16(dst))
    return fail(PK_ERR_INVALID_ARG, "%s: cache and dst must be 16-byte aligned", what);
  if (block_table_stride < (max_seqlen_k - 1) / block_size + 1)
    return fail(PK_ERR_INVALID_ARG, "%s: block_table_stride=%d does not cover max_seqlen_k=%d in blocks of %d", what,
                block_table_stride, max_seqlen_k, block_size);
  pk::Fp4GatherArgs a{};
  a.cache = static_cast<const uint8_t*>(cache);
  a.block_stride = block_stride;
  a.num_blocks = num_blocks;
  a.block_size = block_size;
  a.num_kv_heads = num_kv_heads;
  a.row_bytes = pk::fp4_row_bytes(num_kv_heads);
  a.block_table = block_table;
  a.bt_stride = block_table_stride;
  a.cu_k = cu_seqlens_k;
  a.num_seqs = num_seqs;
  a.max_seqlen_k = max_seqlen_k;
  a.num_rows = num_rows;
  a.dst = static_cast<uint16_t*>(dst);
  return hip_status(pk::launch_gather_fp4(a, reinterpret_cast<hipStream_t>(stream)), "gather_kv_fp4 launch");
}

size_t pk_varlen_attention_fp4_workspace_bytes(int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads,
                                               int32_t max_seqlen_q, int32_t max_seqlen_k) {
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || max_seqlen_q <= 0 ||
      max_seqlen_k <= 0)
    return 0;
  const pk::Fp4AttnPlan p = pk::fp4_attention_plan(num_seqs, num_heads, num_kv_heads, max_seqlen_q, max_seqlen_k, 0);
  return p.few_bytes + p.many_bytes;
}

int pk_varlen_attention_fp4(const void* q, int64_t q_row_stride, const void* k_cache, const void* v_cache,
                            int64_t k_block_stride, int64_t v_block_stride, int32_t num_blocks, int32_t block_size,
                            const int32_t* block_table, int32_t block_table_stride, const int32_t* cu_seqlens_q,
                            const int32_t* cu_seqlens_k, int32_t num_seqs, int64_t num_rows, int32_t max_seqlen_q,
                            int32_t max_seqlen_k, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                            float softmax_scale, int32_t causal, void* out, int64_t out_row_stride, void* workspace,
                            size_t workspace_bytes, pk_stream_t stream) {
  g_last_error.clear();
  const char* what = "varlen_attention_fp4";
  if (int rc = fp4_heads(what, num_kv_heads, head_dim)) return rc;
  if (num_seqs < 0 || num_rows < 0 || max_seqlen_q < 0 || max_seqlen_k < 0)
    return fail(PK_ERR_INVALID_ARG, "%s: negative num_seqs / num_rows / max_seqlen", what);
  if (num_seqs > kMaxSeqs) return fail(PK_ERR_INVALID_ARG, "%s: num_seqs=%d > %d", what, num_seqs, kMaxSeqs);
  if (num_heads <= 0 || num_heads % num_kv_heads)
    return fail(PK_ERR_INVALID_ARG, "%s: num_heads=%d not a multiple of num_kv_heads=%d", what, num_heads, num_kv_heads);
  const int group = num_heads / num_kv_heads;
  if (group != 1 && group != 2 && group != 4 && group != 8)
    return fail(PK_ERR_UNSUPPORTED, "%s: GQA group %d not built (1, 2, 4, 8)", what, group);
  if (num_seqs == 0 || num_rows == 0 || max_seqlen_q == 0 || max_seqlen_k == 0) return PK_OK;
  if (max_seqlen_k > kMaxSeqlen || max_seqlen_q > kMaxSeqlen)
    return fail(PK_ERR_UNSUPPORTED, "%s: max_seqlen_q=%d / max_seqlen_k=%d above %d", what, max_seqlen_q, max_seqlen_k,
                kMaxSeqlen);
  if (int rc = fp4_rows(what, "q", q, q_row_stride, num_heads)) return rc;
  if (q_row_stride >= (1ll << 25))  // (16 rows' offsets in bytes are 32 bits)
    return fail(PK_ERR_UNSUPPORTED, "%s: q row stride of %lld elements (below 2^25)", what, (long long)q_row_stride);
  if (int rc = fp4_rows(what, "out", out, out_row_stride, num_heads)) return rc;
  if (int rc = fp4_caches(what, k_cache, v_cache)) return rc;
  if (!block_table || !cu_seqlens_q || !cu_seqlens_k)
    return fail(PK_ERR_INVALID_ARG, "%s: null block_table / cu_seqlens", what);
  const int32_t row_bytes = pk::fp4_row_bytes(num_kv_heads);
  if (int rc = fp4_blocks(what, k_block_stride, num_blocks, block_size, row_bytes)) return rc;
  if (int rc = fp4_blocks(what, v_block_stride, num_blocks, block_size, row_bytes)) return rc;
  if (block_size % 64) return fail(PK_ERR_INVALID_ARG, "%s: block_size=%d must be a multiple of 64", what, block_size);
  if (block_table_stride < (max_seqlen_k - 1) / block_size + 1)
    return fail(PK_ERR_INVALID_ARG, "%s: block_table_stride=%d does not cover max_seqlen_k=%d in blocks of %d", what,
                block_table_stride, max_seqlen_k, block_size);
  if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale))
    return fail(PK_ERR_INVALID_ARG, "%s: softmax_scale must be positive and finite", what);
  const pk::Fp4AttnPlan p =
      pk::fp4_attention_plan(num_seqs, num_heads, num_kv_heads, max_seqlen_q, max_seqlen_k, num_rows);
  if (p.steps > INT32_MAX)  // (a line of them is counted in 32 bits)
    return fail(PK_ERR_UNSUPPORTED, "%s: %d sequences of up to %d keys, %lld rows: up to %lld steps of %d keys (below 2^31)",
                what, num_seqs, max_seqlen_k, (long long)num_rows, (long long)p.steps, p.step_keys);
  const size_t need = p.few_bytes + p.many_bytes;
  if (!workspace || workspace_bytes < need)
    return fail(PK_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, need,
                workspace ? workspace_bytes : (size_t)0);
  if (reinterpret_cast<uintptr_t>(workspace) % kWorkspaceAlign)
    return fail(PK_ERR_WORKSPACE, "%s: workspace must be %zu-byte aligned", what, kWorkspaceAlign);
  pk::Fp4AttnArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.q_stride = q_row_stride;
  a.k = static_cast<const uint8_t*>(k_cache);
  a.v = static_cast<const uint8_t*>(v_cache);
  a.k_block = k_block_stride;
  a.v_block = v_block_stride;
  a.row_bytes = row_bytes;
  a.block_size = block_size;
  a.num_blocks = num_blocks;
  a.block_table = block_table;
  a.bt_stride = block_table_stride;
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.num_seqs = num_seqs;
  a.max_seqlen_q = max_seqlen_q;
  a.max_seqlen_k = max_seqlen_k;
  a.num_rows = num_rows;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.group_shift = __builtin_ctz((unsigned)group);
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.causal = causal;
  a.out = static_cast<uint16_t*>(out);
  a.out_stride = out_row_stride;
  a.workspace = workspace;
  return hip_status(pk::launch_fp4_attention(a, p, reinterpret_cast<hipStream_t>(stream)), "varlen_attention_fp4 launch");
}

}  // extern "C"

// ---- allocation-free entry point --------------------------------------------------------
// pk_varlen_attention_noalloc runs the kernels of pk_varlen_attention_ex on this file-scope
// device array instead of a caller's workspace. Each GPU holds its own copy
// (PK_NOALLOC_SCRATCH_BYTES) from the first call of this entry point on it until the process
// ends: the array is the only device content of this file's code object, which loads at the
// symbol lookup below, not at the library's other launches. In host
// code `scratch` names a host-side stand-in, not device memory: its device address comes from
// hipGetSymbolAddress, once per device with that device current, and only that address is
// ever passed to a kernel.
static __device__ __align__(256) unsigned char scratch[PK_NOALLOC_SCRATCH_BYTES];

namespace {

constexpr int kMaxDevices = 64;
std::mutex g_scratch_mu;
void* g_scratch_ptr[kMaxDevices] = {};  // device address of `scratch` per device ordinal

// Device address of the current device's scratch, looked up on its first use (no allocation).
int device_scratch(pk_stream_t stream, void** out) {
  int dev = -1;
  if (hipError_t e = hipGetDevice(&dev); e != hipSuccess) return hip_status(e, "varlen_attention_noalloc: hipGetDevice");
  if (dev < 0 || dev >= kMaxDevices)
    return fail(PK_ERR_UNSUPPORTED, "varlen_attention_noalloc: device ordinal %d above %d", dev, kMaxDevices - 1);
  if (stream != nullptr) {  // the kernels run on the stream's device: it must own this scratch
    int sdev = -1;
    if (hipError_t e = hipStreamGetDevice(reinterpret_cast<hipStream_t>(stream), &sdev); e != hipSuccess)
      return hip_status(e, "varlen_attention_noalloc: hipStreamGetDevice");
    if (sdev != dev)
      return fail(PK_ERR_INVALID_ARG, "varlen_attention_noalloc: stream belongs to device %d, current device is %d",
                  sdev, dev);
  }
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (g_scratch_ptr[dev] == nullptr) {
    void* p = nullptr;
    if (hipError_t e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)); e != hipSuccess)
      return hip_status(e, "varlen_attention_noalloc: hipGetSymbolAddress(scratch)");
    if (p == nullptr || (reinterpret_cast<uintptr_t>(p) % kWorkspaceAlign) != 0)
      return fail(PK_ERR_HIP, "varlen_attention_noalloc: scratch address %p unusable", p);
    g_scratch_ptr[dev] = p;
  }
  *out = g_scratch_ptr[dev];
  return PK_OK;
}

}  // namespace

extern "C" int pk_varlen_attention_noalloc(const void* q, int64_t q_row_stride, const void* k, const void* v,
                                           int64_t k_row_stride, int64_t v_row_stride, int64_t k_block_stride,
                                           int64_t v_block_stride, const int32_t* block_table,
                                           int32_t block_table_stride, int32_t block_size,
                                           const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                                           int32_t num_seqs, int32_t max_seqlen_q, int32_t max_seqlen_k,
                                           int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                           float softmax_scale, int32_t causal, void* out, int64_t out_row_stride,
                                           int32_t cached_prefix_keys, pk_stream_t stream) {
  g_last_error.clear();
  const size_t need = pk_varlen_attention_workspace_bytes(num_seqs, num_heads, head_dim, max_seqlen_q, max_seqlen_k);
  if (need > (size_t)PK_NOALLOC_SCRATCH_BYTES)
    return fail(PK_ERR_WORKSPACE,
                "varlen_attention_noalloc: these launch bounds (num_seqs=%d, max_seqlen_q=%d, max_seqlen_k=%d) need "
                "%zu bytes of scratch; the static scratch holds %zu (use pk_varlen_attention_ex with a workspace)",
                num_seqs, max_seqlen_q, max_seqlen_k, need, (size_t)PK_NOALLOC_SCRATCH_BYTES);
  void* ws = nullptr;
  if (need > 0) {
    if (int rc = device_scratch(stream, &ws)) return rc;
  }
  return attention_impl(q, q_row_stride, k, v, k_row_stride, v_row_stride, k_block_stride, v_block_stride, block_table,
                        block_table_stride, block_size, cu_seqlens_q, cu_seqlens_k, num_seqs, max_seqlen_q,
                        max_seqlen_k, num_heads, num_kv_heads, head_dim, softmax_scale, causal, out, out_row_stride,
                        ws, need > 0 ? (size_t)PK_NOALLOC_SCRATCH_BYTES : 0, cached_prefix_keys, nullptr, 0, 0, stream);
}
