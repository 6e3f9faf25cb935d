"""CPU tests of what Qwen3Model.forward makes of its Context: which of the package's operators it calls,
and with what. The operators themselves are replaced by recorders that return zeros of the right shape."""
from types import SimpleNamespace

import pytest
import torch

import pagedkv
from pagedkv import lora, ops
from pagedkv.engine import LLMEngine
from pagedkv.runner import ModelRunner
from pagedkv.qwen3 import Qwen3Adapters, Qwen3Config, Qwen3Model, Qwen3Weights

CFG = Qwen3Config(vocab_size=32, hidden_size=64, num_hidden_layers=2, num_attention_heads=2, num_key_value_heads=1,
                  head_dim=32, intermediate_size=96, max_position_embeddings=64)
BS = 4


@pytest.fixture
def calls(monkeypatch):
    """[(operator, keyword arguments other than tensors)] of a forward pass, in order."""
    log = []

    def record(module, name, result):
        def stub(*args, **kw):
            log.append((name, {k: v for k, v in kw.items() if not isinstance(v, torch.Tensor)}))
            return result(*args, **kw)
        monkeypatch.setattr(module, name, stub)

    def rows(x, n):
        return x.new_zeros(x.shape[0], n)

    heads, dim = CFG.num_attention_heads, CFG.head_dim
    record(ops, "add_rmsnorm", lambda x, w, eps, residual=None: x if residual is None else (x, residual))
    record(ops, "linear", lambda x, w: rows(x, w.shape[0]))
    record(ops, "linear_silu_mul", lambda x, w: rows(x, w.shape[0] // 2))
    record(ops, "linear_add_rmsnorm",
           lambda x, w, residual, norm, eps, residual_out=None: (rows(x, w.shape[0]), residual))
    record(ops, "silu_and_mul", lambda x: rows(x, x.shape[1] // 2))
    record(ops, "qk_norm_rope_store", lambda qkv, *a, **kw: (qkv.new_zeros(qkv.shape[0], heads, dim),
                                                             qkv.new_zeros(qkv.shape[0], 1, dim)))
    record(ops, "varlen_attention", lambda q, *a, **kw: torch.zeros_like(q))
    record(ops, "qkv_decode_attention", lambda qkv, *a, **kw: qkv.new_zeros(qkv.shape[0], heads, dim))
    record(lora, "lora_linear", lambda x, w, *a, **kw: rows(x, w.shape[0]))
    record(lora, "lora_add", lambda y, x, *a, **kw: y)
    return log


def _model():
    cpu = torch.device("cpu")
    caches = torch.zeros(2, CFG.num_hidden_layers, 8, BS, CFG.num_key_value_heads, CFG.head_dim, dtype=torch.bfloat16)
    return Qwen3Model(CFG, Qwen3Weights(CFG, cpu), caches[0], caches[1], 64)


def _fields(kind):
    """The eight fields of the reference's Context (src/utils/context.py:5-14) for a step of three
    sequences: fresh prompts, a chunk beside decodes, or a decode step."""
    lens_q = {"prefill": (2, 3, 1), "mixed": (1, 4, 1), "decode": (1, 1, 1)}[kind]
    lens_k = lens_q if kind == "prefill" else (5, 7, 3)

    def cu(lens):
        return torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32)

    return dict(is_prefill=kind != "decode", cu_seqlens_q=cu(lens_q), cu_seqlens_k=cu(lens_k), max_seqlen_q=max(lens_q),
                max_seqlen_k=max(lens_k), slot_mapping=torch.arange(sum(lens_q), dtype=torch.int32), context_lens=None,
                block_tables=None if kind == "prefill" else torch.arange(6, dtype=torch.int32).view(3, 2))


def _forward(model, ctx):
    n = int(ctx.cu_seqlens_q[-1])
    out = model.forward(torch.zeros(n, dtype=torch.int64), torch.zeros(n, dtype=torch.int64), ctx)
    assert out.shape == (n, CFG.hidden_size)


@pytest.mark.parametrize("adapters", [False, True])
@pytest.mark.parametrize("kind", ["prefill", "mixed", "decode"])
def test_context_of_eight_fields(calls, kind, adapters):
    """The reference's Context class, which has none of this package's optional fields, runs the base
    model: the same calls as a Context that leaves them out."""
    model = _model()
    if adapters:
        model.bind_adapters(Qwen3Adapters(CFG, 2, 8, torch.device("cpu")))
    _forward(model, SimpleNamespace(**_fields(kind)))
    eight = list(calls)
    calls.clear()
    _forward(model, pagedkv.Context(**_fields(kind)))
    assert eight == calls and eight
    assert not any(name.startswith("lora") for name, _ in eight)


@pytest.mark.parametrize("kind", ["prefill", "mixed", "decode"])
def test_adapter_ids_reach_all_four_projections(calls, kind):
    model = _model()
    model.bind_adapters(Qwen3Adapters(CFG, 2, 8, torch.device("cpu")))
    fields = _fields(kind)
    ids = torch.zeros(int(fields["cu_seqlens_q"][-1]), dtype=torch.int32)
    _forward(model, pagedkv.Context(**fields, adapter_ids=ids))
    assert sum(name == "lora_linear" for name, _ in calls) == 4 * CFG.num_hidden_layers
    assert not any(name in ("linear", "linear_silu_mul", "linear_add_rmsnorm") for name, _ in calls)


def test_engine_refuses_adapters(calls):
    """The engine's requests and steps name no adapters: with adapters bound to its model they would all be
    answered by the base model, so a step is refused, before anything is scheduled, and goes on once
    the adapters are unbound. The runner refuses both kinds of step by itself."""
    runner = object.__new__(ModelRunner)
    runner.model, runner.dev, runner.graphs = _model(), torch.device("cpu"), {}
    runner.model.greedy = lambda hidden, ctx: torch.zeros(1, dtype=torch.int32)
    done = []
    eng = object.__new__(LLMEngine)
    eng.runner = runner
    step = SimpleNamespace(**_fields("prefill"), input_ids=torch.zeros(6, dtype=torch.int64),
                           positions=torch.zeros(6, dtype=torch.int64), num_seqs=3)
    eng.scheduler = SimpleNamespace(schedule=lambda: done.append("schedule") or step,
                                    postprocess=lambda toks: done.append("postprocess") or 1)
    runner.model.bind_adapters(Qwen3Adapters(CFG, 2, 8, torch.device("cpu")))
    for refused in (eng.step, lambda: runner.run(step), lambda: runner.run_eager(step), lambda: runner.run_graph(step)):
        with pytest.raises(RuntimeError, match="adapters"):
            refused()
    assert not done and not calls
    runner.model.bind_adapters(None)
    assert eng.step() == (step, 1) and done == ["schedule", "postprocess"]


@pytest.mark.parametrize("kind", ["prefill", "mixed", "decode"])
@pytest.mark.parametrize("hint", [None, 0, 8, -1])
def test_cached_prefix_keys_reach_the_attention(calls, kind, hint):
    """What a Context states of shared blocks (forks share their parent's full pages): the attention gets
    the bound, a shared prefix (above 0) is computed once, and only a decode step without
    shared blocks stores inside the launch that reads the cache."""
    _forward(_model(), pagedkv.Context(**_fields(kind), cached_prefix_keys=hint))
    attention = [(n, kw) for n, kw in calls if n in ("varlen_attention", "qkv_decode_attention")]
    assert len(attention) == CFG.num_hidden_layers
    want = hint or 0
    for name, kw in attention:
        assert (name == "qkv_decode_attention") == (kind == "decode" and want == 0)
        if kind != "prefill":
            assert kw.get("cached_prefix_keys") == want
            assert (kw.get("shared_prefix_keys") or 0) == max(want, 0)
