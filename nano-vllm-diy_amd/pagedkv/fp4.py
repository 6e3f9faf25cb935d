"""A paged K/V cache held in 4 bits: rows stored, appended with norm and rotation, read back, and attended over
(csrc/fp4_rows.hip and fp4_attention.hip through the C-ABI).

A cache is a uint8 tensor (NB, BS, row) of token rows, or (L, NB, BS, row) with the layers' views used one by one,
row = fp4_row_bytes(num_kv_heads): Hkv x 64 bytes of values, two to a byte (the lower dimension in the low four
bits), Hkv x 4 scale bytes, one per 32 dimensions, and up to a multiple of 16 bytes that nothing touches. A value is
0, 0.5, 1, 1.5, 2, 3, 4 or 6 with a sign, times 2^(scale byte - 127): exact in bf16. Of 32 values with the largest
magnitude a, the scale is the smallest power of two s with a <= 7 s (2^-126 .. 2^125), and values are rounded to
nearest, ties to even, at most 6 s; with an infinity or NaN among them all 32 are NaN. Pages, tables and slots are
those of the 16-bit caches (num_kv_heads is what the row's bytes say).

Everything runs on the current stream, reads nothing back and can be captured into a HIP graph.
"""
from __future__ import annotations

import torch

from ._call import call, scratch
from ._lib import lib
from .ops import _given_workspace, _req_i32

_BF16, _U8, _I32 = torch.bfloat16, torch.uint8, torch.int32
HEAD_DIM = 128
_HEAD_BYTES = 68  # of a kv head in a row: 64 of values, 4 scales


def fp4_row_bytes(num_kv_heads: int) -> int:
    """Bytes of a token's row, K or V: 68 per kv head, rounded up to 16."""
    if not 0 < num_kv_heads <= 255:
        raise ValueError(f"num_kv_heads must be 1 to 255, got {num_kv_heads}")
    return (_HEAD_BYTES * num_kv_heads + 15) // 16 * 16


def is_fp4_cache(cache: torch.Tensor) -> bool:
    """Whether a bound cache is held in 4 bits."""
    return cache.dtype is _U8


def _cache(name: str, c: torch.Tensor, device: torch.device) -> int:
    """The kv heads of one layer's cache, after its checks."""
    shape, stride = c.shape, c.stride()
    if c.dtype is not _U8 or len(shape) != 3 or stride[2] != 1 or stride[1] != shape[2]:
        raise ValueError(f"{name} must be a (NB, BS, row) uint8 tensor with contiguous token rows")
    heads = shape[2] // _HEAD_BYTES
    if not 0 < heads <= 255 or fp4_row_bytes(heads) != shape[2]:
        raise ValueError(f"{name}: rows of {shape[2]} bytes are no 4-bit rows (fp4_row_bytes(num_kv_heads))")
    if c.device != device:
        raise ValueError(f"{name} is on {c.device}, expected {device}")
    return heads


def _caches(k_cache: torch.Tensor, v_cache: torch.Tensor, device: torch.device) -> int:
    heads = _cache("k_cache", k_cache, device)
    if _cache("v_cache", v_cache, device) != heads or v_cache.shape != k_cache.shape:
        raise ValueError(f"k_cache {tuple(k_cache.shape)} and v_cache {tuple(v_cache.shape)} must have one shape")
    return heads


def _slot_caches(k_cache: torch.Tensor, v_cache: torch.Tensor, device: torch.device) -> tuple[int, int]:
    """(kv heads, slots) of caches whose slot s is row s: contiguous blocks."""
    shape = k_cache.shape
    if len(shape) == 3 and v_cache.shape == shape and k_cache.dtype is v_cache.dtype is _U8 and \
            k_cache.is_contiguous() and v_cache.is_contiguous() and k_cache.device == v_cache.device == device:
        blocks, block_size, row = shape
        heads = row // _HEAD_BYTES
        if 0 < heads <= 255 and (_HEAD_BYTES * heads + 15) // 16 * 16 == row:
            return heads, blocks * block_size
    # (which of them it was)
    heads = _caches(k_cache, v_cache, device)
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("rows are stored into caches with contiguous blocks")
    return heads, k_cache.shape[0] * k_cache.shape[1]


def _rows(name: str, t: torch.Tensor, n: int, heads: int, device: torch.device) -> int:
    """Row stride of a (n, heads, 128) bf16 tensor with contiguous heads."""
    stride = t.stride()
    if t.dtype is not _BF16 or t.shape != (n, heads, HEAD_DIM) or stride[2] != 1 or (heads > 1 and stride[1] != HEAD_DIM):
        raise ValueError(f"{name} must be a ({n}, {heads}, {HEAD_DIM}) bf16 tensor with contiguous heads, got "
                         f"{tuple(t.shape)} {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    # (neither a single row nor a single head has a stride of its own)
    return stride[0] if n > 1 else heads * HEAD_DIM


def _i32(name: str, t: torch.Tensor, n: int, device: torch.device) -> int:
    if t.dtype is not _I32 or t.device != device:
        _req_i32(name, t, device)
    if t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous ({n},) tensor, got {tuple(t.shape)}")
    return t.data_ptr()


def _table(block_table: torch.Tensor, num_seqs: int, max_seqlen_k: int, block_size: int, device: torch.device):
    if block_table.dtype is not _I32 or block_table.device != device:
        _req_i32("block_table", block_table, device)
    shape, stride = block_table.shape, block_table.stride()
    if len(shape) != 2 or shape[0] < num_seqs or (shape[1] > 1 and stride[1] != 1):
        raise ValueError("block_table must be (S, W) with contiguous rows, one per sequence")
    if shape[1] * block_size < max_seqlen_k:
        raise ValueError(f"block_table of {shape[1]} blocks of {block_size} does not cover max_seqlen_k={max_seqlen_k}")
    # (the kernels step from row to row by the stride that is given to them: an expanded table has none)
    if num_seqs > 1 and stride[0] * block_size < max_seqlen_k:
        raise ValueError(f"block_table rows are {stride[0]} entries apart, which does not cover max_seqlen_k={max_seqlen_k} "
                         f"in blocks of {block_size} (every sequence needs a row of its own)")
    return block_table.data_ptr(), stride[0] if num_seqs > 1 else max(stride[0], shape[1])


def store_kvcache_fp4(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      slot_mapping: torch.Tensor) -> None:
    """store_kvcache into 4-bit caches: key, value (N, Hkv, 128) bf16 with contiguous heads (any row stride), caches
    (NB, BS, row) uint8, slot_mapping (N,) int32. Slots outside the cache are passed over (-1: padding)."""
    dev = key.device
    heads, slots = _slot_caches(k_cache, v_cache, dev)
    n = key.shape[0]
    k_stride, v_stride = _rows("key", key, n, heads, dev), _rows("value", value, n, heads, dev)
    slot_ptr = _i32("slot_mapping", slot_mapping, n, dev)
    if n:
        call(lib().pk_store_kvcache_fp4, "pk_store_kvcache_fp4", dev, key.data_ptr(), k_stride, value.data_ptr(),
             v_stride, k_cache.data_ptr(), v_cache.data_ptr(), slot_ptr, n, heads, HEAD_DIM, slots)


def qk_norm_rope_store_fp4(qkv: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, num_heads: int,
                           num_kv_heads: int, head_dim: int, q_norm_weight: torch.Tensor | None,
                           k_norm_weight: torch.Tensor | None, eps: float, k_cache: torch.Tensor,
                           v_cache: torch.Tensor, slot_mapping: torch.Tensor, return_kv: bool = False,
                           q_out: torch.Tensor | None = None):
    """qk_norm_rope_store into 4-bit caches: q/k RMSNorm, rotation and the store from the fused qkv projection,
    qkv (N, (Hq + 2 Hkv) 128) bf16, positions (N,) int64, cos_sin from rope_cos_sin, in one kernel.

    Returns (q, k, v): q (N, Hq, 128) and, with return_kv, the values that the stored rows hold, (N, Hkv, 128) bf16
    (attention over fresh keys then sees what later steps read); otherwise k and v are None. Slots outside the cache
    are passed over; q, k and v are computed for every token. k is rounded to bf16 before it is quantised, so its row
    is what store_kvcache_fp4 makes of that bf16 row."""
    dev = qkv.device
    heads, slots = _slot_caches(k_cache, v_cache, dev)
    width = (num_heads + 2 * num_kv_heads) * head_dim
    if heads != num_kv_heads or head_dim != HEAD_DIM:
        raise ValueError(f"caches hold {heads} kv heads of {HEAD_DIM}, got {num_kv_heads} of {head_dim}")
    shape, stride = qkv.shape, qkv.stride()
    if len(shape) != 2 or qkv.dtype is not _BF16 or shape[1] != width or stride[1] != 1:
        raise ValueError(f"qkv must be (N, {width}) bf16 with contiguous rows")
    n = shape[0]
    if positions.dtype is not torch.int64 or positions.device != dev or positions.shape != (n,) or \
            not positions.is_contiguous():
        raise ValueError("positions must be a contiguous (N,) int64 tensor on the qkv device")
    if cos_sin.dim() == 3:
        cos_sin = cos_sin.squeeze(1)
    table = cos_sin.shape
    if cos_sin.dtype is not torch.float32 or len(table) != 2 or table[1] != HEAD_DIM or \
            not cos_sin.is_contiguous() or cos_sin.device != dev:
        raise ValueError("cos_sin must be a contiguous (P, 128) float32 table on the qkv device")
    for name, w in (("q_norm_weight", q_norm_weight), ("k_norm_weight", k_norm_weight)):
        if w is not None and (w.dtype is not _BF16 or w.shape != (HEAD_DIM,) or not w.is_contiguous() or
                              w.device != dev):
            raise ValueError(f"{name} must be a contiguous ({HEAD_DIM},) bf16 tensor on the qkv device")
    slot_ptr = _i32("slot_mapping", slot_mapping, n, dev)
    q_stride, row = num_heads * HEAD_DIM, heads * HEAD_DIM
    if q_out is None:
        q_out = torch.empty(n, num_heads, HEAD_DIM, dtype=_BF16, device=dev)
    else:
        q_stride = _rows("q_out", q_out, n, num_heads, dev)
    k = v = None
    if return_kv:
        k = torch.empty(n, heads, HEAD_DIM, dtype=_BF16, device=dev)
        v = torch.empty_like(k)
    if n:
        call(lib().pk_qk_norm_rope_store_fp4, "pk_qk_norm_rope_store_fp4", dev, qkv.data_ptr(),
             stride[0] if n > 1 else width, positions.data_ptr(), cos_sin.data_ptr(), table[0],
             0 if q_norm_weight is None else q_norm_weight.data_ptr(),
             0 if k_norm_weight is None else k_norm_weight.data_ptr(), float(eps), n, num_heads, heads, HEAD_DIM,
             q_out.data_ptr(), q_stride, 0 if k is None else k.data_ptr(), row, 0 if v is None else v.data_ptr(), row,
             k_cache.data_ptr(), v_cache.data_ptr(), slot_ptr, slots)
    return q_out, k, v


def gather_kv_fp4(cache: torch.Tensor, block_table: torch.Tensor, cu_seqlens_k: torch.Tensor, max_seqlen_k: int,
                  total_k: int | None = None) -> torch.Tensor:
    """The values of every sequence's rows of a 4-bit cache, (sum Lk, Hkv, 128) bf16, through its block table (rows
    of entries that are no block are 0).

    total_k (= cu_seqlens_k[-1]) sizes the output; pass it to avoid a device read. max_seqlen_k must bound every
    length (rows past it, or past total_k, are not written)."""
    dev = cache.device
    heads = _cache("cache", cache, dev)
    num_seqs = cu_seqlens_k.numel() - 1
    if num_seqs < 0:
        raise ValueError("cu_seqlens_k must have one more entry than there are sequences")
    cu_ptr = _i32("cu_seqlens_k", cu_seqlens_k, num_seqs + 1, dev)
    bt_ptr, bt_stride = _table(block_table, num_seqs, max_seqlen_k, cache.shape[1], dev)
    if total_k is None:
        total_k = int(cu_seqlens_k[-1].item())
    dst = torch.empty(total_k, heads, HEAD_DIM, dtype=_BF16, device=dev)
    if total_k and num_seqs:
        call(lib().pk_gather_kv_fp4, "pk_gather_kv_fp4", dev, cache.data_ptr(), cache.stride(0), cache.shape[0],
             cache.shape[1], heads, HEAD_DIM, bt_ptr, bt_stride, cu_ptr, num_seqs, int(max_seqlen_k), total_k, dst.data_ptr())
    return dst


def fp4_workspace_bytes(num_seqs: int, num_heads: int, num_kv_heads: int, max_seqlen_q: int, max_seqlen_k: int) -> int:
    """Scratch bytes of one varlen_attention_fp4 call."""
    return int(lib().pk_varlen_attention_fp4_workspace_bytes(num_seqs, num_heads, num_kv_heads, max_seqlen_q,
                                                             max_seqlen_k))


def varlen_attention_fp4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cu_seqlens_q: torch.Tensor,
                         cu_seqlens_k: torch.Tensor, max_seqlen_q: int, max_seqlen_k: int, block_table: torch.Tensor,
                         softmax_scale: float | None = None, causal: bool = True, out: torch.Tensor | None = None,
                         workspace: torch.Tensor | None = None) -> torch.Tensor:
    """varlen_attention over 4-bit paged caches: q (N, Hq, 128) bf16, caches (NB, BS, row) uint8 read through
    block_table (S, W) int32, lengths from cu_seqlens_q / cu_seqlens_k (S + 1,) int32; bottom-right-aligned causal
    mask, GQA h -> h // (Hq / Hkv). One call takes any mixture of sequences with one query row, a few or many.
    Returns out (N, Hq, 128) bf16. A row that sees no key is 0; rows of no sequence, and of sequences without keys
    (graph padding, as varlen_attention takes it), are left as they are in a given out and hold anything in a new one.

    workspace: optional caller-owned uint8 scratch of fp4_workspace_bytes(...) bytes; calls that may overlap must not
    share one. Without it every call, captured ones too, takes its own."""
    dev = q.device
    if q.dim() != 3:
        raise ValueError("q must be (N, Hq, 128)")
    n, num_heads = q.shape[:2]
    heads = _caches(k_cache, v_cache, dev)
    q_stride = _rows("q", q, n, num_heads, dev)
    num_seqs = cu_seqlens_q.numel() - 1
    if num_seqs < 0:
        raise ValueError("cu_seqlens_q must have one more entry than there are sequences")
    cu_q, cu_k = _i32("cu_seqlens_q", cu_seqlens_q, num_seqs + 1, dev), _i32("cu_seqlens_k", cu_seqlens_k, num_seqs + 1, dev)
    bt_ptr, bt_stride = _table(block_table, num_seqs, max_seqlen_k, k_cache.shape[1], dev)
    out_stride = num_heads * HEAD_DIM
    if out is None:
        out = torch.empty(n, num_heads, HEAD_DIM, dtype=_BF16, device=dev)
    else:
        out_stride = _rows("out", out, n, num_heads, dev)
    if not n or not num_seqs:
        return out
    nbytes = fp4_workspace_bytes(num_seqs, num_heads, heads, max_seqlen_q, max_seqlen_k)
    ws = scratch(nbytes, dev) if workspace is None else _given_workspace(workspace, nbytes, dev)
    call(lib().pk_varlen_attention_fp4, "pk_varlen_attention_fp4", dev, q.data_ptr(), q_stride, k_cache.data_ptr(),
         v_cache.data_ptr(), k_cache.stride(0), v_cache.stride(0), k_cache.shape[0], k_cache.shape[1], bt_ptr,
         bt_stride, cu_q, cu_k, num_seqs, n, int(max_seqlen_q), int(max_seqlen_k), num_heads, heads, HEAD_DIM,
         HEAD_DIM ** -0.5 if softmax_scale is None else float(softmax_scale), 1 if causal else 0, out.data_ptr(),
         out_stride, ws.data_ptr(), nbytes)
    return out
