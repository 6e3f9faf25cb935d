"""GPU tests of the framework's paths over caches held in 4 bits: the attention layer, the page operators, the model and
the engine, each against the 64-bit statement of its arithmetic (tests/fp4_oracle.py) or byte by byte."""
import random

import pytest
import torch

import fp4_oracle as ref
import pagedkv
import pagedkv.engine as E
from oracle import qwen3 as Q
from pagedkv.qwen3 import Qwen3Config
from pagedkv.runner import kv_cache_num_blocks
from pool_oracle import Pool, make_pool
from test_engine_gpu import LOGIT_TOL, _cpu_weights

pytestmark = pytest.mark.gpu
D, BS = 128, 64


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _cu(lens, dev):
    return _i32([0, *torch.tensor(lens).cumsum(0).tolist()], dev)


def _bf16(g, dev, *shape):
    return torch.randn(*shape, generator=g).to(torch.bfloat16).to(dev)


def _within(got, want, bound):
    over = (got.double() - want).abs() - bound
    assert over.max().item() <= 0, f"over the bound by {over.max().item():.3e} at {int(over.argmax())}"


def _random_cache(g, dev, kv, nb):
    return torch.randint(0, 256, (nb, BS, ref.row_bytes(kv)), generator=g, dtype=torch.uint8).to(dev)


def _slots(tables, first, new):
    """Slots of new[i] tokens from first[i] on of every sequence."""
    out = []
    for i, (f, n) in enumerate(zip(first, new)):
        out += [int(tables[i, t // BS]) * BS + t % BS for t in range(f, f + n)]
    return torch.tensor(out, dtype=torch.int32)


@pytest.mark.parametrize("heads,kv", [(16, 8), (8, 1)])
@pytest.mark.parametrize("hint", [None, 0, 64])
def test_attention_layer(gpu, heads, kv, hint):
    """Fresh prompts, a chunk beside single rows, a decode step: rows stored byte for byte, attention over them.
    On a stream of its own."""
    g = torch.Generator().manual_seed(heads + kv)
    tables = torch.tensor([[4, 1, 7], [2, 6, -1], [0, 5, 3]], dtype=torch.int32)
    kc, vc = _random_cache(g, gpu, kv, 9), _random_cache(g, gpu, kv, 9)
    want_k, want_v = kc.clone(), vc.clone()
    layer = pagedkv.Attention(D, heads, kv, D ** -0.5)
    layer.k_cache, layer.v_cache = kc, vc
    have = [0, 0, 0]
    stream = torch.cuda.Stream(gpu)
    stream.wait_stream(torch.cuda.current_stream(gpu))
    with torch.cuda.stream(stream):
        for new, flat in (([70, 1, 33], True), ([1, 60, 1], False), ([1, 1, 1], False), ([4, 2, 90], False)):
            n = sum(new)
            q, k, v = _bf16(g, gpu, n, heads, D), _bf16(g, gpu, n, kv, D), _bf16(g, gpu, n, kv, D)
            slots = _slots(tables, have, new)
            have = [h + a for h, a in zip(have, new)]
            ctx = pagedkv.Context(cu_seqlens_q=_cu(new, gpu), cu_seqlens_k=_cu(have, gpu), max_seqlen_q=max(new),
                                  max_seqlen_k=max(have), slot_mapping=slots.to(gpu),
                                  block_tables=None if flat else tables.to(gpu), cached_prefix_keys=hint)
            got = layer(q, k, v, ctx)
            for c, x in ((want_k, k), (want_v, v)):
                c.view(-1, c.shape[-1])[slots.long().to(gpu), :68 * kv] = ref.pack(x)
            assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
            if flat:  # attention over the fresh keys as given, which is what the 16-bit layer computes
                assert torch.equal(got, pagedkv.varlen_attention(q, k, v, ctx.cu_seqlens_q, ctx.cu_seqlens_k, max(new),
                                                                 max(have), D ** -0.5, True))
            else:
                _within(got, *ref.attention(q, kc, vc, tables.to(gpu), new, have, D ** -0.5))
    torch.cuda.current_stream(gpu).wait_stream(stream)


def test_attention_layer_padded_decode_in_a_graph(gpu):
    """A captured decode step of 6 rows, replayed for fewer sequences with the padding of the runner's graphs (slots -1,
    cumulative lengths 0, tables -1), eager work between the replays."""
    heads, kv, most = 16, 8, 6
    g = torch.Generator().manual_seed(5)
    kc, vc = ref.make_cache(kv, 20, BS, g, gpu)
    layer = pagedkv.Attention(D, heads, kv, D ** -0.5)
    layer.k_cache, layer.v_cache = kc, vc
    q, k, v = (torch.zeros(most, h, D, dtype=torch.bfloat16, device=gpu) for h in (heads, kv, kv))
    cu_q, cu_k = (torch.zeros(most + 1, dtype=torch.int32, device=gpu) for _ in range(2))
    slots, tables = torch.full((most,), -1, dtype=torch.int32, device=gpu), torch.full((most, 3), -1, dtype=torch.int32, device=gpu)
    ctx = pagedkv.Context(cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, max_seqlen_q=1, max_seqlen_k=3 * BS, slot_mapping=slots,
                          block_tables=tables)
    layer(q, k, v, ctx)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(q, k, v, ctx)
    for lens in ([5, 130, 64], [1, 1, 192, 65, 100, 7], [40], [77, 128]):
        s = len(lens)
        ids = torch.randperm(20, generator=g)[:3 * s].view(s, 3).to(torch.int32)
        for t, x in ((q, heads), (k, kv), (v, kv)):
            t.copy_(_bf16(g, gpu, most, x, D))
        cu_q.zero_(), cu_k.zero_(), slots.fill_(-1), tables.fill_(-1)
        cu_q[:s + 1], cu_k[:s + 1] = _cu([1] * s, gpu), _cu(lens, gpu)
        slots[:s] = _slots(ids, [n - 1 for n in lens], [1] * s).to(gpu)
        tables[:s] = ids.to(gpu)
        want_k, want_v = kc.clone(), vc.clone()
        graph.replay()
        for c, x in ((want_k, k), (want_v, v)):
            c.view(-1, c.shape[-1])[slots[:s].long(), :68 * kv] = ref.pack(x[:s])
        assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
        _within(out[:s], *ref.attention(q[:s], kc, vc, tables, [1] * s, lens, D ** -0.5))


def _bytes(c):
    """(L, NB, BS, 1, X) 16-bit elements as (L, NB, BS, 2 X) bytes of the same memory."""
    return c.view(torch.uint8).squeeze(-2)


@pytest.mark.parametrize("kv", [1, 3, 8])
def test_page_operators(gpu, kv):
    """Copy, fork, extend and compact on byte caches, against the pool in plain Python."""
    tables, lens, refs, k, v = make_pool(kv, [5, 0, 9, 0, 16], 4, 24, 6, head_dim=ref.row_bytes(kv) // 2)
    pool = Pool(tables, lens, refs, k, v, 4)
    tables, lens, refs, k, v = (t.to(gpu) for t in (tables, lens, refs, k, v))
    kb, vb = _bytes(k), _bytes(v)
    assert kb.shape == (2, 24, 4, ref.row_bytes(kv)) and kb.data_ptr() == k.data_ptr()
    used = [b for b, n in enumerate(refs.tolist()) if n]
    free = [b for b, n in enumerate(refs.tolist()) if not n]
    src, dst, tokens = used[:3] + [-1], free[:3] + [free[3]], [1, 4, 3, 2]
    pagedkv.copy_blocks(kb, vb, _i32(src, gpu), _i32(dst, gpu), _i32(tokens, gpu))
    pool.copy(src, dst, tokens)
    pool.same(tables, lens, refs, k, v)
    one_k, one_v = kb[1], vb[1]  # one layer alone
    pagedkv.copy_blocks(one_k, one_v, _i32(used[:1], gpu), _i32(free[4:5], gpu))
    for c in (pool.k, pool.v):
        c[1, free[4]] = c[1, used[0]]
    pool.same(tables, lens, refs, k, v)
    new = pagedkv.fork_sequences(kb, vb, tables, lens, refs, _i32([0, 4], gpu), _i32([1, 3], gpu))
    assert new.tolist() == pool.fork([0, 4], [1, 3])
    assert pagedkv.extend_sequences(tables, lens, refs, 4, _i32([0, 1, 2], gpu)).tolist() == pool.extend([0, 1, 2])
    pool.same(tables, lens, refs, k, v)
    pagedkv.free_sequences(tables, lens, refs, 4, _i32([0], gpu))
    pool.free([0])
    block_map, live = pagedkv.compact_blocks(kb, vb, tables, lens, refs)
    want_map, want_live = pool.compact()
    assert block_map.tolist() == want_map and live.item() == want_live
    pool.same(tables, lens, refs, k, v)


def test_fork_then_decode_then_compact(gpu):
    """Two continuations of one prompt grow apart over 4-bit pages, and moving the pages changes no bit of the answer."""
    heads, kv, nb = 16, 8, 12
    g = torch.Generator().manual_seed(9)
    kc, vc = ref.make_cache(kv, nb, BS, g, gpu)
    tables = torch.full((2, 4), -1, dtype=torch.int32)
    tables[0, :3] = torch.tensor([7, 3, 11])
    tables = tables.to(gpu)
    lens, refs = _i32([150, 0], gpu), torch.zeros(nb, dtype=torch.int32, device=gpu)
    refs[[7, 3, 11]] = 1
    new = pagedkv.fork_sequences(kc, vc, tables, lens, refs, _i32([0], gpu), _i32([1], gpu))
    assert new.tolist() == [0]
    for step in range(3):
        slots = pagedkv.extend_sequences(tables, lens, refs, BS, _i32([0, 1], gpu))
        k, v, q = _bf16(g, gpu, 2, kv, D), _bf16(g, gpu, 2, kv, D), _bf16(g, gpu, 2, heads, D)
        pagedkv.store_kvcache_fp4(k, v, kc, vc, slots)
        n = lens.tolist()
        assert n == [151 + step] * 2
        args = (_cu([1, 1], gpu), _cu(n, gpu), 1, max(n), tables)
        got = pagedkv.varlen_attention_fp4(q, kc, vc, *args)
        _within(got, *ref.attention(q, kc, vc, tables, [1, 1], n, D ** -0.5))
    block_map, live = pagedkv.compact_blocks(kc, vc, tables, lens, refs)
    assert live.item() == 4 and sorted(set(tables[:, :3].flatten().tolist())) == [0, 1, 2, 3]
    assert torch.equal(pagedkv.varlen_attention_fp4(q, kc, vc, *args), got)


def test_fresh_prompts_attend_over_what_is_stored(gpu):
    """The values that the append returns, under attention over fresh keys, and its rows, under attention over the
    pages, are one computation: both within the bound of the 64-bit result."""
    heads, kv = 16, 8
    g = torch.Generator().manual_seed(12)
    lens = [130, 1, 64, 7]
    n = sum(lens)
    tables = torch.arange(12, dtype=torch.int32).view(4, 3).flip(0).contiguous()
    kc, vc = _random_cache(g, gpu, kv, 12), _random_cache(g, gpu, kv, 12)
    qkv = _bf16(g, gpu, n, (heads + 2 * kv) * D)
    pos = torch.cat([torch.arange(x) for x in lens]).to(gpu)
    w = torch.ones(D, dtype=torch.bfloat16, device=gpu)
    q, k, v = pagedkv.qk_norm_rope_store_fp4(qkv, pos, pagedkv.rope_cos_sin(256, D, device=gpu), heads, kv, D, w, w, 1e-6,
                                             kc, vc, _slots(tables, [0] * 4, lens).to(gpu), return_kv=True)
    cu = _cu(lens, gpu)
    want, bound = ref.attention(q, kc, vc, tables.to(gpu), lens, lens, D ** -0.5)
    _within(pagedkv.varlen_attention(q, k, v, cu, cu, max(lens), max(lens), D ** -0.5, True), want, bound)
    _within(pagedkv.varlen_attention_fp4(q, kc, vc, cu, cu, max(lens), max(lens), tables.to(gpu)), want, bound)


def _oracle_logits(W, cfg, tokens, monkeypatch, jitter=None):
    """The oracle's logits with keys and values rounded to 4 bits, after a change of each by up to a rounding of bf16
    either way where a generator is given."""
    attend = Q.causal_attention

    def rounded(x):
        if jitter is not None:
            x = (x.float() * (1 + 2.0 ** -8 * (2 * torch.rand(x.shape, generator=jitter) - 1))).to(torch.bfloat16)
        return ref.values(ref.pack(x), x.shape[1]).to(torch.bfloat16)

    with monkeypatch.context() as m:
        m.setattr(Q, "causal_attention", lambda q, k, v, scale: attend(q, rounded(k), rounded(v), scale))
        return Q.forward_logits(W, cfg, tokens)


@pytest.mark.parametrize("eager", [False, True])
def test_engine(gpu, eager, monkeypatch):
    """The engine over a 4-bit cache, teacher-forced: prompts, decode steps in padded graphs and across blocks. The
    engine's keys differ from the oracle's by roundings of bf16, which the 4-bit rounding may make whole steps of:
    a chosen token's logit may lie below the best by the 16-bit engine's tolerance and twice what such roundings
    move the oracle's logits by."""
    cfg = Qwen3Config(num_hidden_layers=2)
    eng = E.LLMEngine(cfg, device=gpu, num_blocks=64, block_size=64, max_live_seqs=4, max_seq_len=512,
                      enforce_eager=eager, kv_cache_dtype="fp4")
    assert eng.runner.kv_cache.dtype is torch.uint8 and eng.runner.kv_cache.shape == (2, 2, 64, 64, 544)
    rng = random.Random(11)
    prompts = [[rng.randrange(cfg.vocab_size) for _ in range(n)] for n in (62, 125, 9)]
    outs, stats = eng.generate(prompts, [6, 9, 4], ignore_eos=True)
    assert [len(o) for o in outs] == [6, 9, 4] and stats.decode_steps > 0
    assert eng.scheduler.num_free_blocks() == 64
    W = _cpu_weights(eng.runner.weights)
    for p, out in zip(prompts, outs):
        logits = _oracle_logits(W, cfg, p + out, monkeypatch)
        moved = _oracle_logits(W, cfg, p + out, monkeypatch, torch.Generator().manual_seed(1))
        for j, tok in enumerate(out):
            row = logits[len(p) - 1 + j]
            tol = LOGIT_TOL + 2 * float((moved[len(p) - 1 + j] - row).abs().max())
            assert tol < 2 * float(row.std())  # (a wrong token lies about four spreads below the best)
            assert float(row[tok]) >= float(row.max()) - tol, (j, tok, float(row[tok]), float(row.max()), tol)


def test_blocks_that_fit(gpu):
    """A 4-bit cache is sized by its rows: 2048 / 544 of the blocks in the same memory."""
    torch.cuda.empty_cache()
    free, total = torch.cuda.mem_get_info(gpu)
    util = (total - free) / total + 0.03
    wide = kv_cache_num_blocks(2, 256, 8, D, util, device=gpu)
    fp4 = kv_cache_num_blocks(2, 256, 8, D, util, device=gpu, row_bytes=pagedkv.fp4_row_bytes(8))
    # (the bytes in use are read twice; the cache's rows are 544 bytes in place of 2048)
    assert fp4 * 544 <= (wide + 1) * 2048 and (fp4 + 1) * 544 >= wide * 2048


def test_engine_sizes_its_cache(gpu):
    """num_blocks None with gpu_memory_utilization: as many 4-bit blocks as fit, and the engine serves from them."""
    cfg = Qwen3Config(num_hidden_layers=2)
    torch.cuda.empty_cache()
    free, total = torch.cuda.mem_get_info(gpu)
    util = (total - free) / total + 0.03
    eng = E.LLMEngine(cfg, device=gpu, max_live_seqs=8, max_seq_len=1024, enforce_eager=True, gpu_memory_utilization=util,
                      kv_cache_dtype="fp4")
    nb = eng.runner.num_blocks
    assert eng.runner.kv_cache.shape == (2, 2, nb, 256, 544) and nb * 2 * 2 * 256 * 544 <= total * util
    rng = random.Random(4)
    prompts = [[rng.randrange(cfg.vocab_size) for _ in range(n)] for n in (40, 700)]
    outs, _ = eng.generate(prompts, [4, 6], ignore_eos=True)
    assert [len(o) for o in outs] == [4, 6] and eng.scheduler.num_free_blocks() == nb
