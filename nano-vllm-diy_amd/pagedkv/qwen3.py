"""Qwen3 decoder (the reference's model, src/models/qwen3.py) assembled from the gfx950
kernels of this package; the dense projections are hipBLASLt GEMMs through torch.

Per layer (qwen3.py:155-169):
    x, residual = add_rmsnorm(h, input_layernorm, residual)        layernorm.py:18-28
    qkv = x W_qkv^T                                                 linear.py:190-228
    q, k = qk_norm_rope_store(qkv, ...)  (norms, RoPE, K/V store)   qwen3.py:80-88
    o = varlen_attention(q, k | k_cache, v | v_cache, ...)          attention.py:89-105
    h = o W_o^T                                                     qwen3.py:90
    x, residual = add_rmsnorm(h, post_attention_layernorm, residual)
    h = silu_and_mul(x W_gate_up^T) W_down^T                        qwen3.py:119-123
and the final norm (qwen3.py:194). Weights are random (the serving benchmark runs a
random-init model of the Qwen3-0.6B geometry); the LM head is tied to the embedding
(qwen3.py:215-216). With adapters bound (an addition), every token's own low-rank adapter is
added to each of the four projections.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import fp4, lora, ops
from .context import Context


@dataclass(frozen=True)
class Qwen3Config:
    """Qwen3-0.6B geometry (the HF config the reference loads, model_config.py:3-4)."""
    vocab_size: int = 151936
    hidden_size: int = 1024
    num_hidden_layers: int = 28
    num_attention_heads: int = 16
    num_key_value_heads: int = 8
    head_dim: int = 128
    intermediate_size: int = 3072
    rms_norm_eps: float = 1e-6
    rope_theta: float = 1000000.0
    max_position_embeddings: int = 40960


class Qwen3Weights:
    """All parameters, bf16 on one device, random-normal (std 0.02) with unit norms."""

    def __init__(self, cfg: Qwen3Config, device: torch.device, seed: int = 5, std: float = 0.02):
        g = torch.Generator(device=device).manual_seed(seed)
        bf = dict(dtype=torch.bfloat16, device=device)

        def randn(*shape):
            return (torch.randn(*shape, generator=g, device=device) * std).to(torch.bfloat16)

        H, D = cfg.hidden_size, cfg.head_dim
        qkv_out = (cfg.num_attention_heads + 2 * cfg.num_key_value_heads) * D
        self.embed = randn(cfg.vocab_size, H)                    # tied with the LM head
        self.layers = []
        for _ in range(cfg.num_hidden_layers):
            self.layers.append(dict(
                input_norm=torch.ones(H, **bf), post_norm=torch.ones(H, **bf),
                q_norm=torch.ones(D, **bf), k_norm=torch.ones(D, **bf),
                qkv=randn(qkv_out, H), o=randn(H, cfg.num_attention_heads * D),
                gate_up=randn(2 * cfg.intermediate_size, H), down=randn(H, cfg.intermediate_size)))
        self.final_norm = torch.ones(H, **bf)


class Qwen3Adapters:
    """Low-rank adapters for all four projections of every layer, as lora_linear / lora_add take them:
    per layer and projection (A, B) of num_adapters adapters, bf16, random-normal; scales (alpha / r)
    in fp32. The merged projections' slices are the layers merged in them (q, k, v; gate, up)."""

    def __init__(self, cfg: Qwen3Config, num_adapters: int, rank: int, device: torch.device, seed: int = 6,
                 std: float = 0.02, scale: float = 2.0):
        g = torch.Generator(device=device).manual_seed(seed)
        H, D, inter = cfg.hidden_size, cfg.head_dim, cfg.intermediate_size
        qd, kvd = cfg.num_attention_heads * D, cfg.num_key_value_heads * D
        self.slices = dict(qkv=(qd, kvd, kvd), o=(H,), gate_up=(inter, inter), down=(H,))
        width = dict(qkv=H, o=qd, gate_up=H, down=inter)

        def randn(*shape):
            return (torch.randn(*shape, generator=g, device=device) * std).to(torch.bfloat16)

        self.layers = [{name: (randn(num_adapters, len(s) * rank, width[name]), randn(num_adapters, sum(s), rank))
                        for name, s in self.slices.items()} for _ in range(cfg.num_hidden_layers)]
        self.scales = torch.full((num_adapters,), scale, dtype=torch.float32, device=device)


class Qwen3Model:
    """Forward over one step's tokens; K/V caches are (L, NB, BS, Hkv, D) per operand, or held in
    4 bits (L, NB, BS, fp4_row_bytes(Hkv)) uint8."""

    def __init__(self, cfg: Qwen3Config, weights: Qwen3Weights, k_caches: torch.Tensor | None,
                 v_caches: torch.Tensor | None, max_position: int):
        """k_caches / v_caches None: no cache yet (the warmup pass before the cache is sized,
        as the reference's Attention skips the store while k_cache is empty,
        attention.py:87-88); bind_caches attaches them later."""
        self.cfg = cfg
        self.w = weights
        self.bind_caches(k_caches, v_caches)
        dev = weights.embed.device
        self.cos_sin = ops.rope_cos_sin(max_position, cfg.head_dim, cfg.rope_theta, dev)
        self.scale = cfg.head_dim ** -0.5
        self.adapters: Qwen3Adapters | None = None

    def bind_adapters(self, adapters: Qwen3Adapters | None) -> None:
        """Adapters for the tokens whose Context names one (ctx.adapter_ids); None: none. For callers of
        forward: the engine, whose requests name no adapters, refuses a step while some are bound."""
        self.adapters = adapters

    def bind_caches(self, k_caches: torch.Tensor | None, v_caches: torch.Tensor | None) -> None:
        """Per-layer K/V cache views, (L, NB, BS, Hkv, D) per operand (model_runner.py:161-165), or
        (L, NB, BS, row) uint8 of a cache held in 4 bits."""
        if (k_caches is None) != (v_caches is None):
            raise ValueError("bind both caches or neither")
        if k_caches is not None and (fp4.is_fp4_cache(k_caches) or fp4.is_fp4_cache(v_caches)):
            cfg = self.cfg
            row = fp4.fp4_row_bytes(cfg.num_key_value_heads)
            for c in (k_caches, v_caches):
                if not fp4.is_fp4_cache(c) or cfg.head_dim != fp4.HEAD_DIM or c.dim() != 4 or \
                        c.shape[0] != cfg.num_hidden_layers or c.shape[3] != row:
                    raise ValueError(f"caches held in 4 bits must both be ({cfg.num_hidden_layers}, NB, BS, {row}) uint8 "
                                     f"for {cfg.num_key_value_heads} kv heads of {fp4.HEAD_DIM}, got "
                                     f"{tuple(c.shape)} {c.dtype} for heads of {cfg.head_dim}")
        self.k_caches = k_caches
        self.v_caches = v_caches

    def linear_workspace_bytes(self, max_rows: int) -> int:
        """Scratch the decode-step linear layers need for any batch of up to `max_rows`
        tokens (the launch shape, and so the scratch, depends on the row count)."""
        cfg = self.cfg
        H, qd, inter = cfg.hidden_size, cfg.num_attention_heads * cfg.head_dim, cfg.intermediate_size
        qkv_out = (cfg.num_attention_heads + 2 * cfg.num_key_value_heads) * cfg.head_dim
        need = 0
        for rows in range(1, min(max_rows, ops.LINEAR_MAX_ROWS) + 1):
            need = max(need, ops.linear_workspace_bytes(rows, qkv_out, H, ops.LINEAR_STORE),
                       ops.linear_workspace_bytes(rows, H, qd, ops.LINEAR_ADD_RMSNORM),
                       ops.linear_workspace_bytes(rows, inter, H, ops.LINEAR_SILU_MUL),
                       ops.linear_workspace_bytes(rows, H, inter, ops.LINEAR_ADD_RMSNORM))
        return need

    def forward(self, input_ids: torch.Tensor, positions: torch.Tensor, ctx: Context) -> torch.Tensor:
        """Steps of at most 128 tokens (decode batches) run every projection on the library's
        decode-step linear kernels, each fused with the op after it: qkv_proj; o_proj + the
        post-attention RMSNorm; gate_up_proj + SiluAndMul; down_proj + the next layer's input
        RMSNorm (the final norm after the last layer). Larger steps use F.linear (a library
        GEMM) and the separate norm / activation kernels. Rounding points are the same.
        With adapters (bind_adapters and ctx.adapter_ids) every projection is lora_linear, or
        F.linear and lora_add, followed by the separate kernels.
        ctx.cached_prefix_keys has Attention.forward's meaning, and None states, as 0 does, that no
        block is shared (the engine has no prefix cache): decode reads stream, and a decode step
        stores inside the attention launch. Forks share full blocks, which the one launch may read
        too; with the bound stated (above 0) they are computed once, after a store of its own.
        Caches held in 4 bits: every step is the 4-bit append and attention, whatever the bound; a fresh
        prompt attends over the values that its stored rows hold, so what is computed does not hang on how
        a prompt is cut into steps."""
        cfg, W = self.cfg, self.w
        Hq, Hkv, D = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
        eps = cfg.rms_norm_eps
        flat = ctx.block_tables is None
        small = input_ids.shape[0] <= ops.LINEAR_MAX_ROWS
        hint = getattr(ctx, "cached_prefix_keys", None) or 0  # absent on the reference Context
        # a decode step without a stated shared prefix: every sequence has one new token
        # (cu_seqlens_q = arange), read through block tables; the producer then runs inside the
        # attention launch
        decode = not flat and hint == 0 and ctx.max_seqlen_q == 1 and \
            input_ids.shape[0] == ctx.cu_seqlens_q.numel() - 1
        adapter_ids = getattr(ctx, "adapter_ids", None)  # absent on the reference Context
        ad = self.adapters if adapter_ids is not None else None

        def project(x, L, li, name):
            """x through a projection and its adapters, or the projection alone"""
            if ad is None:
                return ops.linear(x, L[name]) if small else F.linear(x, L[name])
            args = (*ad.layers[li][name], adapter_ids, ad.scales, ad.slices[name])
            if small:
                return lora.lora_linear(x, L[name], *args)
            y = F.linear(x, L[name])
            return lora.lora_add(y, x, *args, out=y)

        h = F.embedding(input_ids, W.embed)
        residual = None
        nl = len(W.layers)
        for li, L in enumerate(W.layers):
            if residual is None:
                x = ops.add_rmsnorm(h, L["input_norm"], eps)
                residual = h
            elif not small:
                x, residual = ops.add_rmsnorm(h, L["input_norm"], eps, residual=residual)
            qkv = project(x, L, li, "qkv")
            kc, vc = (None, None) if self.k_caches is None else (self.k_caches[li], self.v_caches[li])
            if kc is not None and fp4.is_fp4_cache(kc):
                q, k, v = fp4.qk_norm_rope_store_fp4(qkv, positions, self.cos_sin, Hq, Hkv, D, L["q_norm"], L["k_norm"],
                                                     eps, kc, vc, ctx.slot_mapping, return_kv=flat)
                lens = (ctx.cu_seqlens_q, ctx.cu_seqlens_k, ctx.max_seqlen_q, ctx.max_seqlen_k)
                if flat:
                    o = ops.varlen_attention(q, k, v, *lens, self.scale, True)
                else:
                    o = fp4.varlen_attention_fp4(q, kc, vc, *lens, ctx.block_tables, self.scale)
            elif decode:
                # one launch: q/k norm + RoPE, the K/V store and paged decode attention; no
                # block is stated to be shared, so every decode read streams
                o = ops.qkv_decode_attention(qkv, positions, self.cos_sin, Hq, Hkv, D, L["q_norm"], L["k_norm"],
                                             eps, kc, vc, ctx.slot_mapping, ctx.cu_seqlens_q, ctx.cu_seqlens_k,
                                             ctx.max_seqlen_k, self.scale, ctx.block_tables, cached_prefix_keys=0)
            else:
                q, k = ops.qk_norm_rope_store(qkv, positions, self.cos_sin, Hq, Hkv, D, L["q_norm"],
                                              L["k_norm"], eps, kc, vc, ctx.slot_mapping, return_k=flat)
                if flat:
                    v = qkv[:, (Hq + Hkv) * D:].view(-1, Hkv, D)
                    o = ops.varlen_attention(q, k, v, ctx.cu_seqlens_q, ctx.cu_seqlens_k,
                                             ctx.max_seqlen_q, ctx.max_seqlen_k, self.scale, True)
                else:
                    o = ops.varlen_attention(q, kc, vc, ctx.cu_seqlens_q, ctx.cu_seqlens_k,
                                             ctx.max_seqlen_q, ctx.max_seqlen_k, self.scale, True,
                                             ctx.block_tables, cached_prefix_keys=hint,
                                             shared_prefix_keys=hint if hint > 0 else None)
            if small and ad is None:
                x, residual = ops.linear_add_rmsnorm(o.view(-1, Hq * D), L["o"], residual,
                                                     L["post_norm"], eps, residual_out=residual)
                nxt = W.layers[li + 1]["input_norm"] if li + 1 < nl else W.final_norm
                x, residual = ops.linear_add_rmsnorm(ops.linear_silu_mul(x, L["gate_up"]), L["down"],
                                                     residual, nxt, eps, residual_out=residual)
            else:
                h = project(o.view(-1, Hq * D), L, li, "o")
                x, residual = ops.add_rmsnorm(h, L["post_norm"], eps, residual=residual)
                h = project(ops.silu_and_mul(project(x, L, li, "gate_up")), L, li, "down")
                if small and li + 1 < nl:
                    x, residual = ops.add_rmsnorm(h, W.layers[li + 1]["input_norm"], eps, residual=residual)
        if not small or ad is not None:
            x, _ = ops.add_rmsnorm(h, W.final_norm, eps, residual=residual)
        return x

    def greedy(self, hidden: torch.Tensor, ctx: Context, out: torch.Tensor | None = None) -> torch.Tensor:
        """Next tokens: the last row of each sequence for prefill batches (llm_head.py:61-63)."""
        cu = ctx.cu_seqlens_q if ctx.is_prefill else None
        return ops.lm_head_greedy(hidden, self.w.embed, cu, out=out)
