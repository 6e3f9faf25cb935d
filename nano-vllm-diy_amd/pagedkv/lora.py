"""Low-rank adapters of many requests at once beside a shared projection (csrc/lora.hip through the
C-ABI): every token row carries the number of its own adapter, on the device.

    out[m, c] = base[m, c] + scales[a] * sum_j (sum_k x[m, k] lora_a[a, q r + j, k]) * lora_b[a, c, j]

with a = adapter_ids[m] (outside [0, L): no adapter, e.g. -1), r the rank and q the slice of column
c. A merged projection (qkv, gate/up) has one slice per layer merged in it: its output widths are
`slices`, the layers' A matrices are stacked in lora_a (L, len(slices) * r, k), their B matrices,
one after the other in lora_b (L, n_out, r). Adapters of smaller rank are padded with zeros;
scales (L,) float32 holds alpha / r of each. Everything is bf16, summed in fp32 and rounded once.
Infinities and NaN act as in the formula, but an infinite element of lora_b may give NaN for an infinity.

lora_linear computes the projection as well (decode steps, at most 128 rows); lora_add adds to a
projection's output, for prefill steps, whose projections are library products. No call reads
the device from the host, so both run under torch.cuda.graph capture.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache

import torch

from ._call import call, scratch
from ._lib import lib
from .ops import LINEAR_MAX_ROWS, _given_workspace, _req_i32


@lru_cache(maxsize=256)
def _slices(slices: tuple[int, ...] | None, n_out: int):
    widths = (n_out,) if slices is None else slices
    if not widths or sum(widths) != n_out:
        raise ValueError(f"slices {slices} do not add up to the projection's {n_out} outputs")
    return (ctypes.c_int32 * len(widths))(*widths), len(widths)


_BF16, _F32 = torch.bfloat16, torch.float32


def _rows2d(name: str, t: torch.Tensor, device: torch.device) -> tuple[torch.Size, int]:
    """(shape, row stride) of a 2-D bf16 tensor with contiguous rows on the device."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or t.dtype is not _BF16 or stride[1] != 1:
        raise ValueError(f"{name} must be a 2-D bf16 tensor with contiguous rows")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return shape, stride[0]


def _adapter(name: str, t: torch.Tensor, device: torch.device) -> tuple[torch.Size, tuple[int, ...]]:
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or t.dtype is not _BF16 or stride[2] != 1:
        raise ValueError(f"{name} must be a 3-D bf16 tensor with contiguous rows")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return shape, stride


def _adapter_args(rows, k, n_out, dev, lora_a, lora_b, adapter_ids, scales, slices):
    """The adapter arguments of the C-ABI, after the checks both operators share."""
    arr, num_slices = _slices(slices, n_out)
    a_shape, a_stride = _adapter("lora_a", lora_a, dev)
    (adapters, b_rows, rank), b_stride = _adapter("lora_b", lora_b, dev)
    if b_rows != n_out or a_shape != (adapters, num_slices * rank, k):
        raise ValueError(f"lora_a {tuple(a_shape)} and lora_b {tuple(lora_b.shape)} must be (L, {num_slices} * r, {k}) "
                         f"and (L, {n_out}, r)")
    if adapter_ids.dtype is not torch.int32 or adapter_ids.device != dev:
        _req_i32("adapter_ids", adapter_ids, dev)
    if adapter_ids.shape != (rows,) or not adapter_ids.is_contiguous():
        raise ValueError(f"adapter_ids must be a contiguous ({rows},) tensor")
    if scales is not None and (scales.dtype is not _F32 or scales.shape != (adapters,) or scales.device != dev or
                               not scales.is_contiguous()):
        raise ValueError(f"scales must be a contiguous ({adapters},) float32 tensor on {dev}")
    return (lora_a.data_ptr(), a_stride[0], a_stride[1], lora_b.data_ptr(), b_stride[0], b_stride[1], adapters, rank,
            adapter_ids.data_ptr(), 0 if scales is None else scales.data_ptr(), arr, num_slices)


def _out(out, rows, n_out, dev):
    if out is None:
        return torch.empty(rows, n_out, dtype=torch.bfloat16, device=dev), n_out
    shape, stride = _rows2d("out", out, dev)
    if shape != (rows, n_out):
        raise ValueError(f"out must be a ({rows}, {n_out}) tensor")
    return out, stride


def lora_workspace_bytes(rows: int, n_out: int, k: int, rank: int, slices=None, num_adapters: int = 0,
                         linear: bool = False) -> int:
    """Scratch bytes of one lora_add call, or with linear=True of one lora_linear call (0: none)."""
    return _workspace_bytes(rows, n_out, k, rank, None if slices is None else tuple(slices), num_adapters, linear)


@lru_cache(maxsize=4096)
def _workspace_bytes(rows: int, n_out: int, k: int, rank: int, slices: tuple[int, ...] | None, num_adapters: int,
                     linear: bool) -> int:
    arr, num_slices = _slices(slices, n_out)
    if linear:
        return int(lib().pk_lora_linear_workspace_bytes(rows, n_out, k, rank, num_slices))
    return int(lib().pk_lora_add_workspace_bytes(rows, n_out, rank, arr, num_slices, num_adapters))


def _workspace(workspace, nbytes, dev):
    """(pointer, bytes, the tensor) of the scratch of a call"""
    if nbytes == 0:
        return 0, 0, None
    ws = scratch(nbytes, dev) if workspace is None else _given_workspace(workspace, nbytes, dev)
    return ws.data_ptr(), nbytes, ws


def lora_linear(x: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                adapter_ids: torch.Tensor, scales: torch.Tensor | None = None, slices=None,
                out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """F.linear(x, weight) of a decode step plus every row's own adapter: x (rows <= 128, k) bf16,
    weight (n_out, k) bf16, adapter_ids (rows,) int32. The projection's sums are not rounded before
    the adapter is added. workspace: optional caller-owned uint8 scratch of
    lora_workspace_bytes(..., linear=True) bytes; calls that may overlap must not share one."""
    dev = x.device
    (rows, k), x_stride = _rows2d("x", x, dev)
    (n_out, w_k), w_stride = _rows2d("weight", weight, dev)
    if w_k != k:
        raise ValueError(f"weight {tuple(weight.shape)} does not match x {tuple(x.shape)}")
    if rows > LINEAR_MAX_ROWS:
        raise ValueError(f"decode-step linear layers take at most {LINEAR_MAX_ROWS} rows, got {rows}")
    slices = None if slices is None else tuple(slices)
    args = _adapter_args(rows, k, n_out, dev, lora_a, lora_b, adapter_ids, scales, slices)
    out, out_stride = _out(out, rows, n_out, dev)
    ws, nbytes, _keep = _workspace(workspace, _workspace_bytes(rows, n_out, k, args[7], slices, 0, True), dev)
    call(lib().pk_lora_linear, "pk_lora_linear", dev, x.data_ptr(), x_stride, weight.data_ptr(), w_stride, rows, n_out,
         k, *args, out.data_ptr(), out_stride, ws, nbytes)
    return out


def lora_add(y: torch.Tensor, x: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
             adapter_ids: torch.Tensor, scales: torch.Tensor | None = None, slices=None,
             out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """y plus every row's own adapter applied to x: y (rows, n_out) bf16 is the projection's output,
    x (rows, k) bf16 its input. out may be y (in place); otherwise rows without an adapter are
    copied. workspace: optional caller-owned uint8 scratch of lora_workspace_bytes(...) bytes."""
    dev = x.device
    (rows, k), x_stride = _rows2d("x", x, dev)
    (y_rows, n_out), y_stride = _rows2d("y", y, dev)
    if y_rows != rows:
        raise ValueError(f"y {tuple(y.shape)} does not match x {tuple(x.shape)}")
    slices = None if slices is None else tuple(slices)
    args = _adapter_args(rows, k, n_out, dev, lora_a, lora_b, adapter_ids, scales, slices)
    out, out_stride = _out(out, rows, n_out, dev)
    ws, nbytes, _keep = _workspace(workspace, _workspace_bytes(rows, n_out, k, args[7], slices, args[6], False), dev)
    call(lib().pk_lora_add, "pk_lora_add", dev, y.data_ptr(), y_stride, x.data_ptr(), x_stride, rows, n_out, k, *args,
         out.data_ptr(), out_stride, ws, nbytes)
    return out
