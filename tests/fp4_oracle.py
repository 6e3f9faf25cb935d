"""Plain 64-bit statements of the 4-bit cache's format, its rows and the attention over it (not a test module)."""
from __future__ import annotations

import torch

D = 128
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def row_bytes(kv: int) -> int:
    return -(-68 * kv // 16) * 16


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes (..., 128), scale bytes (..., 4)) of bf16 values (..., 128)."""
    blocks = x.double().unflatten(-1, (4, 32))
    top = blocks.abs().amax(-1)
    # the smallest power of two s with top <= 7 s: candidates from the exponent, no logarithms
    byte = torch.ones_like(top, dtype=torch.int64)
    for b in range(1, 252):
        byte += (top > 7 * 2.0 ** (b - 127)).long()
    a = blocks.abs() * torch.pow(2.0, 127.0 - byte.double()).unsqueeze(-1)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    dist = (a.unsqueeze(-1) - grid).abs()
    best = dist.amin(-1, keepdim=True)
    # of two equally near values the one with an even code
    order = dist + torch.where(dist == best, torch.tensor([0.0, 1e-9] * 4, dtype=torch.float64, device=x.device), 0.0)
    code = order.argmin(-1)
    code = torch.where(a >= 6, 7, code) + 8 * torch.signbit(blocks).long()
    bad = ~torch.isfinite(blocks).all(-1)
    byte = torch.where(bad, 255, byte)
    code = torch.where(bad.unsqueeze(-1), 0, code)
    return code.flatten(-2), byte


def pack(x: torch.Tensor) -> torch.Tensor:
    """Rows of bytes, without the last ones that nothing touches, of (..., Hkv, 128) bf16 values."""
    code, byte = quantise(x)
    data = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8).flatten(-2)
    return torch.cat((data, byte.to(torch.uint8).flatten(-2)), -1)


def values(rows: torch.Tensor, kv: int) -> torch.Tensor:
    """(..., Hkv, 128) fp64 values of rows of bytes."""
    data = rows[..., :64 * kv].long().unflatten(-1, (kv, 64))
    code = torch.stack((data & 15, data >> 4), -1).flatten(-2)
    byte = rows[..., 64 * kv:68 * kv].long().unflatten(-1, (kv, 4))
    grid = torch.tensor(GRID + [-g for g in GRID], dtype=torch.float64, device=rows.device)
    scale = torch.where(byte == 255, float("nan"), torch.pow(2.0, byte.double() - 127)).repeat_interleave(32, -1)
    return grid[code] * scale


def norm_rope(x: torch.Tensor, weight, eps: float, positions: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """RMSNorm (root in 64 bits) and rotation of (N, heads, 128) bf16 with every operation rounded by itself."""
    f = x.float()
    if weight is not None:
        ms = x.double().pow(2).mean(-1, keepdim=True) + torch.tensor(eps, dtype=torch.float32).double()
        f = (weight.float() * (f * (1.0 / ms.sqrt()).float())).to(torch.bfloat16).float()
    pos = positions.clamp(0, table.shape[0] - 1)
    cos, sin = table[pos].unsqueeze(1).split(D // 2, -1)
    a, b = f.split(D // 2, -1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1).to(torch.bfloat16)


def attention(q, k_cache, v_cache, tables, q_lens, k_lens, scale: float, causal: bool = True):
    """(out, bound) in 64 bits, (N, Hq, 128): the attention and how far a kernel's bf16 output may be from it.

    The bound, with A = sum p |v| / sum p: half a step of the output's bf16 (2^-8 of the value), half a step of
    every weight's bf16 (2^-8 A), and what fp32 scores and sums lose: a score is off by at most 2^-16 of
    scale sum |q| |k| (128 products and their sums at 2^-24 each, taken four times as many), exp2 and the fp32
    sums of n terms by (n + 64) 2^-24, all of them relative to a weight and twice over (numerator, denominator).
    A weight below the smallest normal fp32 and bf16 value, 2^-126, may be lost altogether, against a sum that is at
    least 1 (the largest weight is between 1 and 2^8): n keys lose at most n 2^-126 max |v|, and an output below
    2^-126 as much as itself."""
    kv = k_cache.shape[-1] // 68
    h, bs, nb = q.shape[1], k_cache.shape[1], k_cache.shape[0]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    at = 0
    for i, (lq, lk) in enumerate(zip(q_lens, k_lens)):
        if lq > 0 and lk > 0:
            row = tables[i, :-(-lk // bs)].long()
            good = ((row >= 0) & (row < nb)).repeat_interleave(bs)[:lk]
            row = row.clamp(0, nb - 1)
            k = values(k_cache[row].flatten(0, 1)[:lk], kv).transpose(0, 1)
            v = values(v_cache[row].flatten(0, 1)[:lk], kv).transpose(0, 1)
            x = q[at:at + lq].double().transpose(0, 1).reshape(kv, -1, lq, D)
            s = torch.matmul(x, k.unsqueeze(1).transpose(-1, -2)) * scale
            seen = good.expand(lq, lk).clone()
            if causal:
                seen &= torch.ones(lq, lk, dtype=torch.bool, device=q.device).tril(lk - lq)
            p = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
            p = p.masked_fill(~seen, 0.0)  # rows that see nothing
            # keys that a row does not see take no part, whatever they hold
            vis = v.unsqueeze(1).unsqueeze(2).expand(kv, 1, lq, lk, D) if not torch.isfinite(v).all() else None
            if vis is None:
                o = torch.matmul(p, v.unsqueeze(1))
            else:
                vis = vis.masked_fill(~seen[None, None, :, :, None], 0.0)
                o = (p.unsqueeze(-1) * vis).sum(-2)
            out[at:at + lq] = o.reshape(h, lq, D).transpose(0, 1)
            av = v.abs().nan_to_num(0.0)
            mean = torch.matmul(p.nan_to_num(0.0), av.unsqueeze(1))
            reach = (torch.matmul(x.abs(), k.abs().nan_to_num(0.0).unsqueeze(1).transpose(-1, -2)) * scale).amax(-1, keepdim=True)
            loose = 2.0 ** -16 * reach + (lk + 64) * 2.0 ** -24
            lost = 2.0 ** -126 * (lk * av.amax() + 1)
            bound[at:at + lq] = (2.0 ** -8 * o.abs().nan_to_num(0.0) + mean * (2.0 ** -8 + 2 * loose) + lost).reshape(h, lq, D).transpose(0, 1)
        at += max(lq, 0)
    return out, bound * (1 + 2.0 ** -7)


def make_cache(kv: int, nb: int, bs: int, g: torch.Generator, device, spread: float = 1.0):
    """Caches (NB, BS, row) of normal values, their last bytes random."""
    out = []
    for _ in range(2):
        x = (torch.randn(nb, bs, kv, D, generator=g) * spread).to(torch.bfloat16).to(device)
        c = torch.randint(0, 256, (nb, bs, row_bytes(kv)), generator=g, dtype=torch.uint8).to(device)
        c[..., :68 * kv] = pack(x)
        out.append(c)
    return out
