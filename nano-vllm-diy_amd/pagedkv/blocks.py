"""Pages of the paged KV cache: copied, and for sequences whose tables live on the device forked,
grown, freed and compacted (csrc/kv_pages.hip through the C-ABI).

The pool is three int32 tensors on the device: block_tables (R, W), -1 padded; context_lens (R,),
the tokens of every row, 0 for an empty one; ref_counts (NB,), the holders of every block, 0 for a
free one -- what the reference's BlockManager keeps in host lists (src/engine/block_manager.py:
75-246). A row of n tokens holds its first ceil(n / block_size) entries. Blocks are given out
lowest number first, in the order of the call's list, so every result is reproducible. Nothing is
read back to the host, so all of it can run under torch.cuda.graph capture; calls on one pool have
to be ordered (one stream, or events between streams).

Caches are (L, NB, BS, Hkv, D) tensors as the runner keeps them, or one layer's (NB, BS, Hkv, D); held in
4 bits they are (L, NB, BS, row) or (NB, BS, row), uint8 (fp4.py).
"""
from __future__ import annotations

import torch

from ._call import call, scratch
from ._lib import lib
from .fp4 import _cache as check_fp4_cache
from .ops import _req_i32


_I32 = torch.int32


def _list_i32(name: str, t: torch.Tensor, device: torch.device) -> int:
    shape = t.shape
    if t.dtype is not _I32 or t.device != device:
        _req_i32(name, t, device)
    if len(shape) != 1 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 1-D tensor")
    return shape[0]


def _fp4_as_16bit(name: str, c: torch.Tensor) -> torch.Tensor:
    """A cache held in 4 bits as one of 16-bit elements, with a head dimension: pages are copied as bytes."""
    if c.dim() not in (3, 4):
        raise ValueError(f"{name} cache of 4 bits must be (L, NB, BS, row) or (NB, BS, row), got {tuple(c.shape)}")
    one_layer = c if c.dim() == 3 else c[0] if c.shape[0] else c.new_empty(c.shape[1:])
    check_fp4_cache(f"{name} cache", one_layer, c.device)
    return c.view(torch.int16).unsqueeze(-2)


def _cache_args(k: torch.Tensor, v: torch.Tensor):
    """(pointers, strides, sizes) of the C-ABI for a pair of caches, and their device."""
    if k.dtype is torch.uint8 and v.dtype is torch.uint8:
        k, v = _fp4_as_16bit("k", k), _fp4_as_16bit("v", v)
    shape, ks, vs = k.shape, k.stride(), v.stride()
    if v.shape != shape or len(shape) not in (4, 5):
        raise ValueError("caches must be two (L, NB, BS, Hkv, D) or (NB, BS, Hkv, D) tensors of one shape")
    if k.dtype != v.dtype or k.element_size() != 2:
        raise TypeError("caches must share one 16-bit dtype")
    dev = k.device
    if v.device != dev or dev.type != "cuda":
        raise ValueError(f"caches must be on one GPU, got {dev} and {v.device}")
    if len(shape) == 4:
        shape, ks, vs = (1, *shape), (0, *ks), (0, *vs)
    layers, blocks, block_size, heads, head_dim = shape
    row = heads * head_dim
    if ks[2:] != (row, head_dim, 1) or vs[2:] != (row, head_dim, 1):
        raise ValueError("a block's rows must be contiguous (block_size x heads x head_dim)")
    return (k.data_ptr(), v.data_ptr(), ks[0], vs[0], ks[1], vs[1], layers, blocks, block_size, row), dev


def _pool_args(block_tables: torch.Tensor, context_lens: torch.Tensor, ref_counts: torch.Tensor,
               device: torch.device):
    if block_tables.dtype is not _I32 or block_tables.device != device:
        _req_i32("block_tables", block_tables, device)
    shape, stride = block_tables.shape, block_tables.stride()
    if len(shape) != 2 or (shape[1] > 1 and stride[1] != 1):
        raise ValueError("block_tables must be (R, W) with contiguous rows")
    rows, width = shape
    if rows > 1 and stride[0] < width:
        raise ValueError("block_tables' rows must not overlap")
    if _list_i32("context_lens", context_lens, device) != rows:
        raise ValueError(f"context_lens must have one length per row of block_tables ({rows})")
    _list_i32("ref_counts", ref_counts, device)
    return block_tables.data_ptr(), max(stride[0], width), rows, width, context_lens.data_ptr(), ref_counts.data_ptr()


def copy_blocks(k_caches: torch.Tensor, v_caches: torch.Tensor, src_blocks: torch.Tensor,
                dst_blocks: torch.Tensor, num_tokens: torch.Tensor | None = None) -> None:
    """Copy pages in every layer, K and V, in one launch: for every pair i the first num_tokens[i]
    token rows (None: whole pages) of block src_blocks[i] to block dst_blocks[i].

    src_blocks, dst_blocks and num_tokens are (P,) int32 on the caches' device. Pairs with a block
    outside the cache (-1: none), one block twice or no tokens are passed over. A target may be
    neither the target nor the source of another pair of the call.
    """
    args, dev = _cache_args(k_caches, v_caches)
    pairs = _list_i32("src_blocks", src_blocks, dev)
    if _list_i32("dst_blocks", dst_blocks, dev) != pairs or \
            (num_tokens is not None and _list_i32("num_tokens", num_tokens, dev) != pairs):
        raise ValueError("src_blocks, dst_blocks and num_tokens must have one entry per pair")
    call(lib().pk_copy_blocks, "pk_copy_blocks", dev, *args, src_blocks.data_ptr(), dst_blocks.data_ptr(),
         0 if num_tokens is None else num_tokens.data_ptr(), pairs)


def fork_sequences(k_caches: torch.Tensor, v_caches: torch.Tensor, block_tables: torch.Tensor,
                   context_lens: torch.Tensor, ref_counts: torch.Tensor, parents: torch.Tensor,
                   children: torch.Tensor) -> torch.Tensor:
    """Rows children[i] of the tables become copies of rows parents[i].

    A child shares its parent's full pages (ref_counts + 1) and, where the parent's last page is
    not full, gets a new page with that page's tokens, copied in every layer, so parent and child
    both grow without seeing each other's tokens. Returns new_blocks (n,) int32: that page's
    number; -1 where none was needed; -2 where the pool had none left; -3 where children[i] is no
    row of the tables, is not empty or was listed before. With -2 and -3 the child stays as it
    was. Parents are read as they are before the call: one that the call makes a child is empty.
    At most 1024 forks a call.
    """
    args, dev = _cache_args(k_caches, v_caches)
    pool = _pool_args(block_tables, context_lens, ref_counts, dev)
    if ref_counts.numel() != args[7]:
        raise ValueError(f"ref_counts must have one count per block ({args[7]})")
    n = _list_i32("parents", parents, dev)
    if _list_i32("children", children, dev) != n:
        raise ValueError("parents and children must have one entry per fork")
    new_blocks = torch.empty(n, dtype=torch.int32, device=dev)
    nbytes = lib().pk_fork_workspace_bytes(n)
    ws = scratch(nbytes, dev)
    call(lib().pk_fork_sequences, "pk_fork_sequences", dev, *args, *pool, parents.data_ptr(), children.data_ptr(), n,
         new_blocks.data_ptr(), ws.data_ptr(), nbytes)
    return new_blocks


def extend_sequences(block_tables: torch.Tensor, context_lens: torch.Tensor, ref_counts: torch.Tensor,
                     block_size: int, rows: torch.Tensor) -> torch.Tensor:
    """One more token for every listed row of the tables; returns slot_mapping (n,) int32.

    The token's slot is the one store_kvcache and the decode calls take; a row whose last page is
    full gets a new page, and its length grows by one (a last page that is not full has to be the
    row's alone, as forks leave it). -1, and nothing changed, where the row is
    no row of the tables or was listed before, its table is full or the pool has no page left.
    At most 1024 rows a call.
    """
    dev = block_tables.device
    pool = _pool_args(block_tables, context_lens, ref_counts, dev)
    n = _list_i32("rows", rows, dev)
    slots = torch.empty(n, dtype=torch.int32, device=dev)
    call(lib().pk_extend_sequences, "pk_extend_sequences", dev, *pool, ref_counts.numel(), int(block_size),
         rows.data_ptr(), n, slots.data_ptr())
    return slots


def free_sequences(block_tables: torch.Tensor, context_lens: torch.Tensor, ref_counts: torch.Tensor,
                   block_size: int, rows: torch.Tensor) -> None:
    """Free the listed rows: their pages lose a holder (a page without one is free), their table
    entries become -1 and their lengths 0. A row listed twice is freed once; entries that are no
    row of the tables (-1) are passed over."""
    dev = block_tables.device
    pool = _pool_args(block_tables, context_lens, ref_counts, dev)
    n = _list_i32("rows", rows, dev)
    call(lib().pk_free_sequences, "pk_free_sequences", dev, *pool, ref_counts.numel(), int(block_size),
         rows.data_ptr(), n)


def compact_blocks(k_caches: torch.Tensor, v_caches: torch.Tensor, block_tables: torch.Tensor,
                   context_lens: torch.Tensor, ref_counts: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Move the live pages to the front of the cache with the fewest moves: with M live pages, those
    at M and above go, in order, to the free ones below M, in every layer, and ref_counts and the
    tables follow. Returns block_map (NB,) int32, every page's new number (-1: it was free), and
    num_live (1,) int32, M. Tables kept elsewhere are renamed by the map."""
    args, dev = _cache_args(k_caches, v_caches)
    pool = _pool_args(block_tables, context_lens, ref_counts, dev)
    if ref_counts.numel() != args[7]:
        raise ValueError(f"ref_counts must have one count per block ({args[7]})")
    block_map = torch.empty_like(ref_counts)
    num_live = torch.empty(1, dtype=torch.int32, device=dev)
    nbytes = lib().pk_compact_workspace_bytes(args[7])
    ws = scratch(nbytes, dev)
    call(lib().pk_compact_blocks, "pk_compact_blocks", dev, *args, *pool, block_map.data_ptr(), num_live.data_ptr(),
         ws.data_ptr(), nbytes)
    return block_map, num_live
