"""CPU tests of the 4-bit cache: the oracle's format against closed forms, and the refusals of the C entry points
(which return before any GPU work) and of the Python wrappers."""
import ctypes

import pytest
import torch

import fp4_oracle as ref
import pagedkv
from pagedkv import _lib

BUF = (ctypes.c_char * 65536)()
PTR = (ctypes.addressof(BUF) + 255) // 256 * 256
ARG, UNSUPPORTED, SPACE = _lib.PK_ERR_INVALID_ARG, _lib.PK_ERR_UNSUPPORTED, _lib.PK_ERR_WORKSPACE

CALLS = {
    "pk_store_kvcache_fp4": dict(key=PTR, key_stride=1024, value=PTR, value_stride=1024, k=PTR, v=PTR, slots=PTR, n=4,
                                 kv=8, d=128, num_slots=64, stream=None),
    "pk_qk_norm_rope_store_fp4": dict(qkv=PTR, qkv_stride=4096, positions=PTR, cos_sin=PTR, max_position=64, qw=PTR,
                                      kw=PTR, eps=1e-6, n=4, heads=16, kv=8, d=128, q_out=PTR, q_out_stride=2048,
                                      k_out=None, k_out_stride=0, v_out=None, v_out_stride=0, k=PTR, v=PTR, slots=PTR,
                                      num_slots=64, stream=None),
    "pk_gather_kv_fp4": dict(cache=PTR, block_stride=64 * 544, nb=4, bs=64, kv=8, d=128, table=PTR, table_stride=4,
                             cu_k=PTR, num_seqs=2, max_k=200, rows=300, dst=PTR, stream=None),
    "pk_varlen_attention_fp4": dict(q=PTR, q_stride=2048, k=PTR, v=PTR, k_block=64 * 544, v_block=64 * 544, nb=4, bs=64,
                                    table=PTR, table_stride=4, cu_q=PTR, cu_k=PTR, num_seqs=2, rows=2, max_q=1,
                                    max_k=200, heads=16, kv=8, d=128, scale=0.1, causal=1, out=PTR, out_stride=2048,
                                    ws=PTR, ws_bytes=1 << 40, stream=None),
}


def _call(name, **kw):
    args = dict(CALLS[name])
    assert set(kw) <= set(args), kw
    args.update(kw)
    return getattr(_lib.lib(), name)(*args.values())


@pytest.mark.parametrize("name,kw,code", [
    ("pk_store_kvcache_fp4", dict(d=64), UNSUPPORTED), ("pk_store_kvcache_fp4", dict(kv=0), UNSUPPORTED),
    ("pk_store_kvcache_fp4", dict(kv=256), UNSUPPORTED), ("pk_store_kvcache_fp4", dict(n=-1), ARG),
    ("pk_store_kvcache_fp4", dict(n=1 << 23), UNSUPPORTED), ("pk_store_kvcache_fp4", dict(num_slots=-1), ARG),
    ("pk_store_kvcache_fp4", dict(key=None), ARG), ("pk_store_kvcache_fp4", dict(value=PTR + 8), ARG),
    ("pk_store_kvcache_fp4", dict(key_stride=1016), ARG), ("pk_store_kvcache_fp4", dict(value_stride=1028), ARG),
    ("pk_store_kvcache_fp4", dict(k=PTR + 4), ARG), ("pk_store_kvcache_fp4", dict(slots=None), ARG),
    ("pk_qk_norm_rope_store_fp4", dict(d=96), UNSUPPORTED), ("pk_qk_norm_rope_store_fp4", dict(heads=0), ARG),
    ("pk_qk_norm_rope_store_fp4", dict(n=1 << 22), UNSUPPORTED), ("pk_qk_norm_rope_store_fp4", dict(max_position=0), ARG),
    ("pk_qk_norm_rope_store_fp4", dict(eps=-1e-6), ARG), ("pk_qk_norm_rope_store_fp4", dict(eps=float("nan")), ARG),
    ("pk_qk_norm_rope_store_fp4", dict(qkv_stride=4088), ARG), ("pk_qk_norm_rope_store_fp4", dict(q_out=None), ARG),
    ("pk_qk_norm_rope_store_fp4", dict(k_out=PTR, k_out_stride=1000), ARG),
    ("pk_qk_norm_rope_store_fp4", dict(v_out=PTR + 2, v_out_stride=1024), ARG),
    ("pk_qk_norm_rope_store_fp4", dict(positions=None), ARG), ("pk_qk_norm_rope_store_fp4", dict(qw=PTR + 2), ARG),
    ("pk_qk_norm_rope_store_fp4", dict(v=None), ARG),
    ("pk_gather_kv_fp4", dict(num_seqs=-1), ARG), ("pk_gather_kv_fp4", dict(num_seqs=70000), ARG),
    ("pk_gather_kv_fp4", dict(block_stride=64 * 544 - 16), ARG), ("pk_gather_kv_fp4", dict(block_stride=64 * 544 + 8), ARG),
    ("pk_gather_kv_fp4", dict(nb=0), ARG), ("pk_gather_kv_fp4", dict(bs=0), ARG), ("pk_gather_kv_fp4", dict(max_k=257), ARG),
    ("pk_gather_kv_fp4", dict(max_k=-1), ARG), ("pk_gather_kv_fp4", dict(dst=None), ARG),
    ("pk_gather_kv_fp4", dict(cache=PTR + 8), ARG), ("pk_gather_kv_fp4", dict(rows=-1), ARG),
    ("pk_varlen_attention_fp4", dict(d=64), UNSUPPORTED), ("pk_varlen_attention_fp4", dict(heads=20), ARG),
    ("pk_varlen_attention_fp4", dict(heads=24), UNSUPPORTED), ("pk_varlen_attention_fp4", dict(num_seqs=-1), ARG),
    ("pk_varlen_attention_fp4", dict(num_seqs=70000), ARG), ("pk_varlen_attention_fp4", dict(rows=-1), ARG),
    ("pk_varlen_attention_fp4", dict(max_q=-1), ARG), ("pk_varlen_attention_fp4", dict(max_k=1 << 23), UNSUPPORTED),
    ("pk_varlen_attention_fp4", dict(q=None), ARG), ("pk_varlen_attention_fp4", dict(q_stride=2040), ARG),
    ("pk_varlen_attention_fp4", dict(q_stride=1 << 25), UNSUPPORTED),
    ("pk_varlen_attention_fp4", dict(out=PTR + 8), ARG), ("pk_varlen_attention_fp4", dict(out_stride=2050), ARG),
    ("pk_varlen_attention_fp4", dict(bs=96, k_block=96 * 544, v_block=96 * 544), ARG),
    ("pk_varlen_attention_fp4", dict(k_block=64 * 543), ARG), ("pk_varlen_attention_fp4", dict(v_block=8), ARG),
    ("pk_varlen_attention_fp4", dict(table=None), ARG), ("pk_varlen_attention_fp4", dict(table_stride=3), ARG),
    ("pk_varlen_attention_fp4", dict(cu_k=None), ARG), ("pk_varlen_attention_fp4", dict(scale=0.0), ARG),
    ("pk_varlen_attention_fp4", dict(scale=float("inf")), ARG), ("pk_varlen_attention_fp4", dict(ws=None), SPACE),
    ("pk_varlen_attention_fp4", dict(ws_bytes=100), SPACE), ("pk_varlen_attention_fp4", dict(ws=PTR + 128), SPACE),
    ("pk_varlen_attention_fp4", dict(num_seqs=65535, max_k=65535 * 64, table_stride=65535), UNSUPPORTED),
    ("pk_varlen_attention_fp4", dict(rows=1 << 22, max_q=1 << 22, max_k=65535 * 64, table_stride=65535), UNSUPPORTED)])
def test_refusals(name, kw, code):
    assert _call(name, **kw) == code, _lib.lib().pk_last_error()
    assert name[3:].encode() in _lib.lib().pk_last_error()


def test_nothing_to_do_touches_no_pointer():
    assert _call("pk_store_kvcache_fp4", n=0, key=None, k=None) == 0
    assert _call("pk_qk_norm_rope_store_fp4", n=0, qkv=None) == 0
    assert _call("pk_gather_kv_fp4", num_seqs=0, cache=None) == 0
    assert _call("pk_gather_kv_fp4", rows=0, cache=None) == 0
    for kw in (dict(num_seqs=0), dict(rows=0), dict(max_q=0), dict(max_k=0)):
        assert _call("pk_varlen_attention_fp4", q=None, out=None, **kw) == 0


def test_row_bytes():
    for kv in (1, 2, 3, 4, 7, 8, 16, 255):
        assert pagedkv.fp4_row_bytes(kv) == _lib.lib().pk_fp4_row_bytes(kv) == ref.row_bytes(kv)
        assert pagedkv.fp4_row_bytes(kv) // 68 == kv  # the row's bytes say how many heads it has
    assert _lib.lib().pk_fp4_row_bytes(0) == _lib.lib().pk_fp4_row_bytes(256) == 0
    for kv in (0, -1, 256):
        with pytest.raises(ValueError):
            pagedkv.fp4_row_bytes(kv)


def test_workspace_bytes():
    one = pagedkv.fp4_workspace_bytes(256, 16, 8, 1, 8192)
    assert 0 < one <= 5 << 20
    assert one < pagedkv.fp4_workspace_bytes(256, 16, 8, 512, 8192) <= 105 << 20
    for bad in ((0, 16, 8, 1, 64), (1, 16, 0, 1, 64), (1, 15, 8, 1, 64), (1, 16, 8, 0, 64), (1, 16, 8, 1, 0)):
        assert pagedkv.fp4_workspace_bytes(*bad) == 0


# ------------------------------------------------------------------------------ the oracle ---
def test_oracle_scales_and_rounding():
    x = torch.zeros(1, 128)
    x[0, :9] = torch.tensor([7.0, 5.0, -5.0, 0.25, 0.75, 1.25, -1.75, 2.5, 3.5])
    x[0, 32] = 7.03125      # just over 7: the next scale
    x[0, 64:66] = torch.tensor([float("inf"), 1.0])
    code, byte = ref.quantise(x.to(torch.bfloat16))
    assert byte.tolist() == [[127, 128, 255, 1]]
    assert code[0, :9].tolist() == [7, 6, 14, 0, 2, 2, 12, 4, 6]
    assert code[0, 32].item() == 6  # 3.516 -> 4, of a scale of 2
    assert code[0, 64:96].abs().sum().item() == 0
    got = ref.values(ref.pack(x.to(torch.bfloat16).view(1, 1, 128)), 1)
    assert got[0, 0, :9].tolist() == [6, 4, -4, 0, 1, 1, -2, 2, 4] and got[0, 0, 32].item() == 8
    assert torch.isnan(got[0, 0, 64:96]).all() and got[0, 0, 96:].abs().sum().item() == 0


def test_oracle_error_and_range():
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(64, 128, generator=g) * torch.pow(10.0, torch.randint(-30, 30, (64, 1), generator=g))).to(torch.bfloat16)
    got = ref.values(ref.pack(x.view(64, 1, 128)), 1).view(64, 4, 32)
    top = x.double().view(64, 4, 32).abs().amax(-1, keepdim=True)
    assert ((got - x.double().view(64, 4, 32)).abs() <= top / 5).all()
    big = torch.full((1, 1, 128), torch.finfo(torch.bfloat16).max).to(torch.bfloat16)
    assert (ref.values(ref.pack(big), 1) == 6 * 2.0 ** 125).all()


# ------------------------------------------------------------------------------ the wrappers ---
def _tensors(n=4, kv=8, heads=16):
    c = [torch.zeros(4, 64, ref.row_bytes(kv), dtype=torch.uint8) for _ in range(2)]
    rows = torch.zeros(n, kv, 128, dtype=torch.bfloat16)
    return c[0], c[1], rows, torch.zeros(n, dtype=torch.int32), torch.zeros(n, heads, 128, dtype=torch.bfloat16)


def test_store_wrapper_refusals():
    kc, vc, rows, slots, _ = _tensors()
    bad = [(rows.float(), rows, kc, vc, slots), (rows, rows[:3], kc, vc, slots), (rows, rows, kc[:, :, :528], vc, slots),
           (rows, rows, kc.to(torch.int8), vc, slots), (rows, rows, kc, vc[:2], slots), (rows, rows, kc[::2], vc[::2], slots),
           (rows, rows, kc, vc, slots[:3]), (rows[:, :4], rows[:, :4], kc, vc, slots),
           (rows.transpose(1, 2), rows, kc, vc, slots), (rows, rows, kc[:, :, :480].contiguous()[:, :, 1:], vc, slots)]
    for args in bad:
        with pytest.raises(ValueError):
            pagedkv.store_kvcache_fp4(*args)
    with pytest.raises(TypeError):
        pagedkv.store_kvcache_fp4(rows, rows, kc, vc, slots.long())
    with pytest.raises(ValueError, match="GPU"):
        pagedkv.store_kvcache_fp4(rows, rows, kc, vc, slots)


def test_append_wrapper_refusals():
    kc, vc, _, slots, _ = _tensors()
    qkv, pos = torch.zeros(4, 4096, dtype=torch.bfloat16), torch.zeros(4, dtype=torch.int64)
    table, w = torch.zeros(16, 128), torch.ones(128, dtype=torch.bfloat16)
    ok = dict(qkv=qkv, positions=pos, cos_sin=table, num_heads=16, num_kv_heads=8, head_dim=128, q_norm_weight=w,
              k_norm_weight=w, eps=1e-6, k_cache=kc, v_cache=vc, slot_mapping=slots)
    for kw in (dict(num_kv_heads=4), dict(head_dim=64), dict(qkv=qkv[:, :4000]), dict(qkv=qkv.float()),
               dict(positions=pos.int()), dict(positions=pos[:2]), dict(cos_sin=table.double()),
               dict(cos_sin=table[:, :64]), dict(q_norm_weight=w[:64]), dict(k_norm_weight=w.float()),
               dict(slot_mapping=slots[:1]), dict(q_out=torch.zeros(4, 8, 128, dtype=torch.bfloat16)),
               dict(k_cache=kc.transpose(0, 1))):
        with pytest.raises(ValueError):
            pagedkv.qk_norm_rope_store_fp4(**{**ok, **kw})
    with pytest.raises(ValueError, match="GPU"):
        pagedkv.qk_norm_rope_store_fp4(**ok)


def test_attention_and_gather_wrapper_refusals():
    kc, vc, _, _, q = _tensors()
    cu = torch.arange(5, dtype=torch.int32)
    table = torch.zeros(4, 2, dtype=torch.int32)
    ok = dict(q=q, k_cache=kc, v_cache=vc, cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=1, max_seqlen_k=100,
              block_table=table)
    for kw in (dict(q=q[0]), dict(q=q.float()), dict(k_cache=kc[0]), dict(v_cache=vc[:, :32]), dict(cu_seqlens_k=cu[:4]),
               dict(block_table=table[:3]), dict(block_table=table[0]), dict(max_seqlen_k=129),
               dict(out=torch.zeros(4, 16, 64, dtype=torch.bfloat16)), dict(cu_seqlens_q=cu[:0]),
               dict(workspace=torch.zeros(8, dtype=torch.uint8))):
        with pytest.raises(ValueError):
            pagedkv.varlen_attention_fp4(**{**ok, **kw})
    with pytest.raises(TypeError):
        pagedkv.varlen_attention_fp4(**{**ok, "block_table": table.long()})
    for kw in (dict(max_seqlen_k=129), dict(block_table=table[:1]), dict(cache=kc.float())):
        with pytest.raises(ValueError):
            pagedkv.gather_kv_fp4(**{**dict(cache=kc, block_table=table, cu_seqlens_k=cu, max_seqlen_k=100, total_k=4), **kw})
    with pytest.raises(ValueError, match="GPU"):
        pagedkv.varlen_attention_fp4(**ok)


def test_page_operators_refuse_what_is_no_fp4_cache():
    one = torch.zeros(1, dtype=torch.int32)
    k = torch.zeros(2, 4, 64, 544, dtype=torch.uint8)
    with pytest.raises(ValueError, match="one GPU"):  # (the shapes are taken)
        pagedkv.copy_blocks(k, k.clone(), one, one)
    with pytest.raises(ValueError, match="one GPU"):
        pagedkv.copy_blocks(k[0], k[1], one, one)
    for bad in (k[..., :540], k[..., :528].contiguous(), k[0, 0], k.unsqueeze(0)):
        with pytest.raises(ValueError, match="4 bits|4-bit rows|contiguous"):
            pagedkv.copy_blocks(bad, bad.clone(), one, one)
    with pytest.raises(ValueError, match="one shape"):
        pagedkv.copy_blocks(k, k[:1].clone(), one, one)
    with pytest.raises((TypeError, ValueError)):
        pagedkv.copy_blocks(k, torch.zeros(2, 4, 64, 2, 128, dtype=torch.bfloat16), one, one)


def test_model_and_runner_refusals():
    from pagedkv.qwen3 import Qwen3Config, Qwen3Model, Qwen3Weights
    from pagedkv.runner import ModelRunner
    cfg = Qwen3Config(vocab_size=32, hidden_size=64, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1,
                      intermediate_size=96, max_position_embeddings=64)
    model = Qwen3Model(cfg, Qwen3Weights(cfg, torch.device("cpu")), None, None, 64)
    good = torch.zeros(2, 4, 64, 80, dtype=torch.uint8)
    model.bind_caches(good, good.clone())
    wide = torch.zeros(2, 4, 64, 1, 128, dtype=torch.bfloat16)
    model.bind_caches(wide, wide.clone())
    for k, v in ((good, wide), (wide, good), (good[:1], good[:1]), (good[..., :64], good[..., :64]),
                 (torch.zeros(2, 4, 64, 144, dtype=torch.uint8),) * 2, (good[0], good[0])):
        with pytest.raises(ValueError, match="4 bits"):
            model.bind_caches(k, v)
    with pytest.raises(ValueError, match="kv_cache_dtype"):
        ModelRunner(cfg, "cpu", 4, kv_cache_dtype="fp8")
    with pytest.raises(ValueError, match="64 tokens"):
        ModelRunner(cfg, "cpu", 4, block_size=32, kv_cache_dtype="fp4")


@pytest.mark.parametrize("flat", [True, False])
@pytest.mark.parametrize("hint", [None, 0, 64])
def test_attention_layer_takes_the_4_bit_operators(monkeypatch, flat, hint):
    from pagedkv import attention
    calls = []
    monkeypatch.setattr(attention.fp4, "store_kvcache_fp4", lambda k, v, kc, vc, slots: calls.append("store"))
    monkeypatch.setattr(attention.fp4, "varlen_attention_fp4", lambda q, *a: calls.append("paged") or q)
    monkeypatch.setattr(attention, "varlen_attention", lambda q, *a, **kw: calls.append("flat") or q)
    layer = pagedkv.Attention(128, 2, 1, 0.1)
    layer.k_cache = layer.v_cache = torch.zeros(4, 64, 80, dtype=torch.uint8)
    q, k = torch.zeros(3, 2, 128, dtype=torch.bfloat16), torch.zeros(3, 1, 128, dtype=torch.bfloat16)
    cu = torch.arange(4, dtype=torch.int32)
    layer(q, k, k, pagedkv.Context(cu_seqlens_q=cu, cu_seqlens_k=cu, max_seqlen_q=1, max_seqlen_k=1, slot_mapping=cu[:3],
                                   block_tables=None if flat else cu[:3, None], cached_prefix_keys=hint))
    assert calls == ["store", "flat" if flat else "paged"]
