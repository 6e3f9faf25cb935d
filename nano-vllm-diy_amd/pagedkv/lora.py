"""Low-rank adapters of many requests at once beside a shared projection (csrc/lora.hip through the
C-ABI): every token row carries the number of its own adapter, on the device.

    out[m, c] = base[m, c] + scales[a] * sum_j (sum_k x[m, k] lora_a[a, q r + j, k]) * lora_b[a, c, j]

with a = adapter_ids[m] (outside [0, L): no adapter, e.g. -1), r the rank and q the slice of column
c. A merged projection (qkv, gate/up) has one slice per layer merged in it: its output widths are
`slices`, the layers' A matrices are stacked in lora_a (L, len(slices) * r, k), their B matrices,
one after the other in lora_b (L, n_out, r). Adapters of smaller rank are padded with zeros;
scales (L,) float32 holds alpha / r of each. Everything is bf16, summed in fp32 and rounded once.

lora_linear computes the projection as well (decode steps, at most 128 rows); lora_add adds to a
projection's output, for prefill steps, whose projections are library products. No call reads
the device from the host, so both run under torch.cuda.graph capture.
"""
from __future__ import annotations

import ctypes
from functools import lru_cache

import torch

from ._lib import check, lib
from .ops import LINEAR_MAX_ROWS, _given_workspace, _req_i32, _rows2d, _stream


@lru_cache(maxsize=256)
def _slices(slices: tuple[int, ...] | None, n_out: int):
    widths = (n_out,) if slices is None else slices
    if not widths or sum(widths) != n_out:
        raise ValueError(f"slices {slices} do not add up to the projection's {n_out} outputs")
    return (ctypes.c_int32 * len(widths))(*widths), len(widths)


def _adapter_args(x, n_out, lora_a, lora_b, adapter_ids, scales, slices):
    """The adapter arguments of the C-ABI, after the checks both operators share."""
    _rows2d("x", x)
    rows, k = x.shape
    dev = x.device
    arr, num_slices = _slices(None if slices is None else tuple(slices), n_out)
    for name, t in (("lora_a", lora_a), ("lora_b", lora_b)):
        if t.dim() != 3 or t.dtype != torch.bfloat16 or t.stride(2) != 1:
            raise ValueError(f"{name} must be a 3-D bf16 tensor with contiguous rows")
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, expected {dev}")
    adapters, _, rank = lora_b.shape
    if lora_b.shape[1] != n_out or lora_a.shape != (adapters, num_slices * rank, k):
        raise ValueError(f"lora_a {tuple(lora_a.shape)} and lora_b {tuple(lora_b.shape)} must be (L, {num_slices} * r, "
                         f"{k}) and (L, {n_out}, r)")
    _req_i32("adapter_ids", adapter_ids, dev)
    if adapter_ids.shape != (rows,) or not adapter_ids.is_contiguous():
        raise ValueError(f"adapter_ids must be a contiguous ({rows},) tensor")
    if scales is not None and (scales.dtype != torch.float32 or scales.shape != (adapters,) or scales.device != dev or
                               not scales.is_contiguous()):
        raise ValueError(f"scales must be a contiguous ({adapters},) float32 tensor on {dev}")
    return (lora_a.data_ptr(), lora_a.stride(0), lora_a.stride(1), lora_b.data_ptr(), lora_b.stride(0),
            lora_b.stride(1), adapters, rank, adapter_ids.data_ptr(), 0 if scales is None else scales.data_ptr(), arr,
            num_slices)


def _out(out, rows, n_out, dev):
    if out is None:
        return torch.empty(rows, n_out, dtype=torch.bfloat16, device=dev)
    _rows2d("out", out)
    if out.shape != (rows, n_out) or out.device != dev:
        raise ValueError(f"out must be a ({rows}, {n_out}) tensor on {dev}")
    return out


def lora_workspace_bytes(rows: int, n_out: int, k: int, rank: int, num_slices: int = 1, num_adapters: int = 0,
                         linear: bool = False) -> int:
    """Scratch bytes of one lora_add call, or with linear=True of one lora_linear call."""
    if linear:
        return int(lib().pk_lora_linear_workspace_bytes(rows, n_out, k, rank, num_slices))
    return int(lib().pk_lora_add_workspace_bytes(rows, rank, num_slices, num_adapters))


def _scratch(workspace, nbytes, dev):
    # one buffer per call, from the capture's own pool under capture: no two graphs share it
    if workspace is None:
        return torch.empty(nbytes, dtype=torch.uint8, device=dev)
    return _given_workspace(workspace, nbytes, dev)


def lora_linear(x: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                adapter_ids: torch.Tensor, scales: torch.Tensor | None = None, slices=None,
                out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """F.linear(x, weight) of a decode step plus every row's own adapter: x (rows <= 128, k) bf16,
    weight (n_out, k) bf16, adapter_ids (rows,) int32. The projection's sums are not rounded before
    the adapter is added. workspace: optional caller-owned uint8 scratch of
    lora_workspace_bytes(..., linear=True) bytes; calls that may overlap must not share one."""
    _rows2d("weight", weight)
    n_out = weight.shape[0]
    args = _adapter_args(x, n_out, lora_a, lora_b, adapter_ids, scales, slices)
    rows, k = x.shape
    dev = x.device
    if weight.shape[1] != k or weight.device != dev:
        raise ValueError(f"weight {tuple(weight.shape)} on {weight.device} does not match x {tuple(x.shape)} on {dev}")
    if rows > LINEAR_MAX_ROWS:
        raise ValueError(f"decode-step linear layers take at most {LINEAR_MAX_ROWS} rows, got {rows}")
    out = _out(out, rows, n_out, dev)
    nbytes = lib().pk_lora_linear_workspace_bytes(rows, n_out, k, args[7], args[11])
    ws = _scratch(workspace, nbytes, dev)
    with torch.cuda.device(dev):
        check(lib().pk_lora_linear(x.data_ptr(), x.stride(0), weight.data_ptr(), weight.stride(0), rows, n_out, k,
                                   *args, out.data_ptr(), out.stride(0), ws.data_ptr(), nbytes, _stream(x)),
              "pk_lora_linear")
    return out


def lora_add(y: torch.Tensor, x: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
             adapter_ids: torch.Tensor, scales: torch.Tensor | None = None, slices=None,
             out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """y plus every row's own adapter applied to x: y (rows, n_out) bf16 is the projection's output,
    x (rows, k) bf16 its input. out may be y (in place); otherwise rows without an adapter are
    copied. workspace: optional caller-owned uint8 scratch of lora_workspace_bytes(...) bytes."""
    _rows2d("y", y)
    n_out = y.shape[1]
    args = _adapter_args(x, n_out, lora_a, lora_b, adapter_ids, scales, slices)
    rows, k = x.shape
    dev = x.device
    if y.shape[0] != rows or y.device != dev:
        raise ValueError(f"y {tuple(y.shape)} on {y.device} does not match x {tuple(x.shape)} on {dev}")
    out = _out(out, rows, n_out, dev)
    nbytes = lib().pk_lora_add_workspace_bytes(rows, args[7], args[11], args[6])
    ws = _scratch(workspace, nbytes, dev)
    with torch.cuda.device(dev):
        check(lib().pk_lora_add(y.data_ptr(), y.stride(0), x.data_ptr(), x.stride(0), rows, n_out, k, *args,
                                out.data_ptr(), out.stride(0), ws.data_ptr(), nbytes, _stream(x)), "pk_lora_add")
    return out
