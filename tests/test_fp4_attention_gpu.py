"""GPU tests of attention over 4-bit caches against the 64-bit statement (tests/fp4_oracle.py), element by element
within the bound that is derived there."""
import pytest
import torch

import fp4_oracle as ref
import pagedkv

pytestmark = pytest.mark.gpu
D = 128


def _case(device, heads, kv, lens, bs=64, seed=0, spread=1.0, pad_rows=0):
    """Caches, tables (blocks in random order, blocks of nobody among them) and q for sequences of (Lq, Lk)."""
    g = torch.Generator().manual_seed(seed)
    need = [max(0, -(-k // bs)) for _, k in lens]
    nb = sum(need) + 3
    kc, vc = ref.make_cache(kv, nb, bs, g, device)
    ids = torch.randperm(nb, generator=g).tolist()
    tables = torch.full((len(lens), max(need + [1])), -1, dtype=torch.int32)
    for i, n in enumerate(need):
        tables[i, :n] = torch.tensor([ids.pop() for _ in range(n)], dtype=torch.int32)
    q_lens, k_lens = [q for q, _ in lens], [k for _, k in lens]
    n = sum(max(q, 0) for q in q_lens)
    q = (torch.randn(n + pad_rows, heads, D, generator=g) * spread).to(torch.bfloat16).to(device)
    return dict(q=q, kc=kc, vc=vc, tables=tables.to(device), q_lens=q_lens, k_lens=k_lens, n=n)


def _cu(lens, device):
    return torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(device)


def _run(c, max_q=None, max_k=None, **kw):
    dev = c["q"].device
    return pagedkv.varlen_attention_fp4(c["q"], c["kc"], c["vc"], _cu(c["q_lens"], dev), _cu(c["k_lens"], dev),
                                        max(c["q_lens"]) if max_q is None else max_q,
                                        max(c["k_lens"]) if max_k is None else max_k, c["tables"], **kw)


def _check(c, got, scale=D ** -0.5, causal=True):
    want, bound = ref.attention(c["q"][:c["n"]], c["kc"], c["vc"], c["tables"], c["q_lens"], c["k_lens"], scale, causal)
    got = got[:c["n"]].double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    over = ((got - want).abs() - bound).masked_fill(nan, -1.0)
    assert over.max().item() <= 0, f"off by {(got - want).abs().nan_to_num(0).max().item():.3e}, over the bound at {int(over.argmax())}"


GEOMETRIES = [(16, 8), (8, 4), (4, 2), (2, 1), (8, 1), (4, 4), (16, 2), (3, 3), (32, 16)]


@pytest.mark.parametrize("heads,kv", GEOMETRIES)
def test_single_rows(gpu, heads, kv):
    c = _case(gpu, heads, kv, [(1, k) for k in (1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 700)], seed=heads + kv)
    _check(c, _run(c))


@pytest.mark.parametrize("heads,kv", GEOMETRIES)
def test_few_rows(gpu, heads, kv):
    most = 16 // (heads // kv)
    lens = [(max(1, most - i), max(1, most - i) + p) for i, p in enumerate((0, 1, 50, 64, 130, 500, 63))]
    c = _case(gpu, heads, kv, lens, seed=heads + kv)
    _check(c, _run(c))


@pytest.mark.parametrize("heads,kv", GEOMETRIES)
def test_many_rows(gpu, heads, kv):
    lens = [(17, 17), (64, 64), (33, 97), (130, 131), (200, 456), (65, 64 + 65)]
    c = _case(gpu, heads, kv, lens, seed=heads + kv)
    _check(c, _run(c))


@pytest.mark.parametrize("bs", [64, 128, 192, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_mixtures_and_empty_sequences(gpu, bs, causal):
    lens = [(1, 300), (0, 0), (90, 400), (1, 1), (5, 257), (0, 70), (40, 40), (3, 0), (1, 511), (16, 1000)]
    c = _case(gpu, 16, 8, lens, bs=bs, seed=bs, pad_rows=4)
    out = torch.full_like(c["q"], 7.0)
    _run(c, causal=causal, out=out)
    rows = torch.ones(c["q"].shape[0], dtype=torch.bool)
    at = 0
    for lq, lk in lens:
        if lk == 0:
            rows[at:at + lq] = False
        at += lq
    rows[c["n"]:] = False
    assert (out[~rows.to(gpu)] == 7).all()  # rows without keys, and behind the last sequence
    out[~rows.to(gpu)] = 0
    _check(c, out, causal=causal)


@pytest.mark.parametrize("heads,kv", [(16, 8), (4, 1), (8, 1)])
def test_rows_that_see_no_key(gpu, heads, kv):
    """More query rows than keys: the first rows see nothing and are zeros, in every form."""
    lens = [(3, 1), (2, 1), (100, 30), (300, 1), (16, 15)]
    c = _case(gpu, heads, kv, lens, seed=9)
    got = _run(c)
    assert (got[:2] == 0).all() and (got[5:5 + 70] == 0).all()
    _check(c, got)


@pytest.mark.parametrize("lens", [[(1, 20000)], [(4, 9000), (1, 64)], [(1, 5000), (150, 5100)], [(260, 8000)],
                                  [(1, 70)] * 3 + [(700, 1500)]])
def test_long_sequences_split_over_work_groups(gpu, lens):
    c = _case(gpu, 16, 8, lens, bs=256, seed=len(lens))
    _check(c, _run(c))


def test_more_sequences_than_a_wavefront_keeps(gpu):
    g = torch.Generator().manual_seed(4)
    lens = [(int(a), int(b)) for a, b in zip(torch.randint(0, 3, (1300,), generator=g), torch.randint(0, 90, (1300,), generator=g))]
    lens[700], lens[1299], lens[0] = (40, 200), (30, 90), (20, 70)
    c = _case(gpu, 4, 2, lens, seed=4)
    out = _run(c, out=torch.zeros_like(c["q"]))
    _check(c, out)


def test_scores_far_from_zero(gpu):
    """Scores in the hundreds: weights that all but vanish, and a reference that moves step by step."""
    for spread in (30.0, 0.0):
        c = _case(gpu, 8, 2, [(1, 1000), (3, 500), (60, 300)], seed=3, spread=spread)
        _check(c, _run(c))
    c = _case(gpu, 8, 2, [(1, 1000), (3, 500), (60, 300)], seed=3)
    _check(c, _run(c, softmax_scale=4.0), scale=4.0)
    # ascending scores: keys grow with their position
    for i in range(c["tables"].shape[1]):
        blk = int(c["tables"][0, i])
        if blk >= 0:
            c["kc"][blk, :, 128:136] = 120 + i // 2
    _check(c, _run(c))


def test_bad_table_entries_hide_their_keys(gpu):
    c = _case(gpu, 16, 8, [(1, 700), (2, 700), (50, 700), (1, 64)], seed=5)
    nb = c["kc"].shape[0]
    c["tables"][0, 3], c["tables"][1, 0], c["tables"][2, 10], c["tables"][2, 0], c["tables"][3, 0] = -1, nb, -9, 2 ** 31 - 1, -1
    got = _run(c)
    assert (got[-1] == 0).all()
    _check(c, got)


def test_behind_the_last_key_anything_may_lie(gpu):
    """Rows of the last page past the sequence's end with every byte 255 (NaN scales), and tables that are wider."""
    lens = [(1, 70), (1, 64), (4, 100), (50, 130), (70, 333)]
    c = _case(gpu, 8, 4, lens, bs=128, seed=6)
    clean = _run(c)
    for i, (_, k) in enumerate(lens):
        if k % 128:
            blk = int(c["tables"][i, k // 128])
            c["kc"][blk, k % 128:] = 255
            c["vc"][blk, k % 128:] = 255
    free = sorted(set(range(c["kc"].shape[0])) - set(c["tables"].flatten().tolist()))
    c["kc"][free], c["vc"][free] = 255, 255
    wide = torch.full((len(lens), c["tables"].shape[1] + 3), free[0], dtype=torch.int32, device=gpu)
    wide[:, :c["tables"].shape[1]] = torch.where(c["tables"] < 0, free[0], c["tables"])
    c["tables"] = wide
    got = _run(c, max_k=128 * 5)
    _check(c, got)
    # the launch bound changed, so the sums may be cut elsewhere; with the same bound the bits are the same
    assert torch.equal(_run(c), clean)


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("heads,kv", [(16, 8), (8, 1), (2, 2)])
def test_nan_blocks_reach_the_rows_that_see_them(gpu, which, heads, kv):
    lens = [(1, 100), (1, 64), (2, 90), (16 // (heads // kv), 70), (140, 170), (33, 200)]
    c = _case(gpu, heads, kv, lens, seed=7)
    cache = c[which + "c"]
    for i, keys in enumerate(([10], [], [89], [66, 69], [30, 31, 100, 169], [199])):
        for j, t in enumerate(keys):
            row = cache[int(c["tables"][i, t // 64]), t % 64]
            row[64 * kv + 4 * (j % kv) + (t + j) % 4] = 255
    _check(c, _run(c))


def test_launch_bounds_cut_rows_and_keys(gpu):
    c = _case(gpu, 16, 8, [(1, 500), (40, 300), (6, 200)], seed=8)
    out = torch.full_like(c["q"], 5.0)
    _run(c, max_q=8, max_k=256, out=out)
    assert (out[9:41] == 5).all()
    # rows keep their places, keys past the bound are ignored (the last row is aligned with the last key that counts)
    c["k_lens"] = [min(k, 256) for k in c["k_lens"]]
    want, bound = ref.attention(c["q"], c["kc"], c["vc"], c["tables"], c["q_lens"], c["k_lens"], D ** -0.5)
    rows = torch.tensor(list(range(9)) + list(range(41, 47)), device=gpu)
    assert ((out.double() - want).abs() <= bound)[rows].all()


def test_strides_layers_and_given_buffers(gpu):
    """q and out as parts of wider rows, the caches one layer of a stack with room between blocks, its own workspace."""
    lens = [(1, 130), (20, 300), (3, 64)]
    c = _case(gpu, 8, 4, lens, seed=10)
    n = c["n"]
    want = _run(c)
    wide = torch.zeros(n, 12, D, dtype=torch.bfloat16, device=gpu)
    wide[:, 2:10] = c["q"]
    stack = torch.full((3, c["kc"].shape[0], 66, 272), 255, dtype=torch.uint8, device=gpu)
    stack2 = torch.full((c["kc"].shape[0], 2, 64, 272), 255, dtype=torch.uint8, device=gpu)
    stack[1, :, :64] = c["kc"]
    stack2[:, 1] = c["vc"]
    out = torch.full((n, 10, D), 3.0, dtype=torch.bfloat16, device=gpu)
    ws = torch.full((pagedkv.fp4_workspace_bytes(3, 8, 4, 20, 300),), 255, dtype=torch.uint8, device=gpu)
    c2 = dict(c, q=wide[:, 2:10], kc=stack[1, :, :64], vc=stack2[:, 1])
    _run(c2, out=out[:, 1:9], workspace=ws)
    assert torch.equal(out[:, 1:9], want)
    assert (out[:, 0] == 3).all() and (out[:, 9] == 3).all()


def test_cache_past_four_gigabytes(gpu):
    kv, bs, heads = 8, 256, 16
    nb = 2 ** 32 // (bs * 544) + 40
    g = torch.Generator().manual_seed(11)
    small = ref.make_cache(kv, 6, bs, g, gpu)
    kc, vc = (torch.zeros(nb, bs, 544, dtype=torch.uint8, device=gpu) for _ in range(2))
    ids = [nb - 1, nb - 20, 3, nb - 35, nb // 2 + 1, nb - 2]
    for i, b in enumerate(ids):
        kc[b], vc[b] = small[0][i], small[1][i]
    lens = [(1, 700), (30, 600)]
    q = torch.randn(31, heads, D, generator=g).to(torch.bfloat16).to(gpu)
    near = dict(q=q, kc=small[0], vc=small[1], q_lens=[1, 30], k_lens=[700, 600], n=31,
                tables=torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=gpu))
    far = dict(near, kc=kc, vc=vc, tables=torch.tensor([ids[:3], ids[3:]], dtype=torch.int32, device=gpu))
    got = _run(far)
    _check(near, got)
    assert torch.equal(got, _run(near))


def test_equal_calls_give_equal_bits(gpu):
    c = _case(gpu, 16, 8, [(1, 1500), (7, 900), (200, 1300), (1, 33)], bs=256, seed=12)
    first = _run(c)
    for _ in range(5):
        assert torch.equal(_run(c), first)


def test_captured_and_replayed(gpu):
    """Decode rows with graph padding, and a mixed batch, captured together; lengths change between replays."""
    c = _case(gpu, 16, 8, [(1, 700), (1, 900), (1, 300), (1, 5)], bs=64, seed=13)
    d = _case(gpu, 16, 8, [(60, 500), (2, 600)], bs=64, seed=14)
    cu_q, cu_k = _cu(c["q_lens"], gpu), _cu(c["k_lens"], gpu)
    d_q, d_k = _cu(d["q_lens"], gpu), _cu(d["k_lens"], gpu)
    out, out_d = torch.zeros_like(c["q"]), torch.zeros_like(d["q"])

    def step():
        pagedkv.varlen_attention_fp4(c["q"], c["kc"], c["vc"], cu_q, cu_k, 1, 900, c["tables"], out=out)
        pagedkv.varlen_attention_fp4(d["q"], d["kc"], d["vc"], d_q, d_k, 60, 600, d["tables"], out=out_d)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k_lens, live in (([700, 900, 300, 5], 4), ([1, 64, 65, 5], 4), ([640, 899, 0, 0], 2), ([700, 900, 300, 5], 4)):
        cu_k.copy_(_cu(k_lens, "cpu"))
        q_lens = [1] * live + [0] * (4 - live)
        cu_q.copy_(_cu(q_lens, "cpu"))
        out.zero_(), out_d.zero_()
        graph.replay()
        torch.cuda.synchronize()
        _check(dict(c, q_lens=q_lens, k_lens=k_lens, n=live), out)
        _check(d, out_d)


def test_two_streams_at_once(gpu):
    cases = [_case(gpu, 16, 8, [(1, 1200 + 100 * i), (150, 700), (4, 2000)], bs=256, seed=20 + i) for i in range(2)]
    want = [_run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(3):
        outs = []
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                outs.append(_run(c))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_append_then_attend_as_a_step_does(gpu):
    """Prompts appended and attended over, chunk by chunk and token by token: rows, tables and attention together."""
    heads, kv, bs = 16, 8, 64
    g = torch.Generator().manual_seed(30)
    total = [150, 70, 201]
    nb = 12
    kc, vc = (torch.randint(0, 256, (nb, bs, 544), generator=g, dtype=torch.uint8).to(gpu) for _ in range(2))
    ids = torch.randperm(nb, generator=g).tolist()
    tables = torch.full((3, 4), -1, dtype=torch.int32)
    for i, n in enumerate(total):
        for j in range(-(-n // bs)):
            tables[i, j] = ids.pop()
    table = pagedkv.rope_cos_sin(256, D, device=gpu)
    w = torch.ones(D, dtype=torch.bfloat16, device=gpu)
    have = [0, 0, 0]
    keys = [torch.zeros(n, kv, D, dtype=torch.bfloat16, device=gpu) for n in total]
    for new in ([100, 3, 0], [40, 60, 150], [1, 1, 1], [9, 6, 50]):
        new = [min(a, t - h) for a, t, h in zip(new, total, have)]
        n = sum(new)
        qkv = torch.randn(n, (heads + 2 * kv) * D, generator=g).to(torch.bfloat16).to(gpu)
        pos = torch.cat([torch.arange(h, h + a) for h, a in zip(have, new)])
        slots = torch.cat([tables[i, pos_i // bs].long() * bs + pos_i % bs for i, pos_i in
                           enumerate(torch.arange(h, h + a) for h, a in zip(have, new))]).to(torch.int32)
        q, k, _ = pagedkv.qk_norm_rope_store_fp4(qkv, pos.to(gpu), table, heads, kv, D, w, w, 1e-6, kc, vc,
                                                 slots.to(gpu), return_kv=True)
        at = 0
        for i, a in enumerate(new):
            keys[i][have[i]:have[i] + a] = k[at:at + a]
            at += a
            have[i] += a
        c = dict(q=q, kc=kc, vc=vc, tables=tables.to(gpu), q_lens=new, k_lens=have, n=n)
        _check(c, _run(c))
    cu = _cu(have, gpu)
    assert torch.equal(pagedkv.gather_kv_fp4(kc, tables.to(gpu), cu, max(have), sum(have)), torch.cat(keys))


@pytest.mark.parametrize("heads,kv", [(22, 11), (24, 12), (40, 40), (112, 14)])
def test_head_counts_that_no_slot_count_divides(gpu, heads, kv):
    """Work-groups of 1, 6, 8 and 7 kv heads, more than one of them side by side."""
    c = _case(gpu, heads, kv, [(1, 200), (2, 90), (1, 1), (40, 130), (3, 64), (1, 700)], seed=heads)
    _check(c, _run(c))


def test_more_sequences_than_are_in_lds(gpu):
    """More than 4096 sequences: short ones, empty ones, chunks on both sides of the border, for several kv heads."""
    g = torch.Generator().manual_seed(41)
    lens = [(1, int(k)) for k in torch.randint(0, 90, (8500,), generator=g)]
    for i, x in ((0, (70, 90)), (4094, (3, 200)), (4095, (150, 300)), (4096, (33, 33)), (4500, (0, 40)), (8191, (1, 700)),
                 (8192, (20, 500)), (8499, (90, 90))):
        lens[i] = x
    c = _case(gpu, 4, 2, lens, seed=42)
    out = torch.zeros_like(c["q"])
    _run(c, out=out)
    _check(c, out)


def test_rows_past_the_tensors_are_not_touched(gpu):
    """Cumulative lengths that go on past q's rows: what is there is computed, in its place in the mask."""
    lens = [(1, 90), (7, 100), (60, 130), (1, 70), (40, 64)]
    c = _case(gpu, 8, 4, lens, seed=51)
    want, bound = ref.attention(c["q"], c["kc"], c["vc"], c["tables"], c["q_lens"], c["k_lens"], D ** -0.5)
    for n in (0, 1, 3, 30, 68, 69, 80):
        room = torch.full((n + 40, 8, D), 7.0, dtype=torch.bfloat16, device=gpu)
        out = pagedkv.varlen_attention_fp4(c["q"][:n], c["kc"], c["vc"], _cu(c["q_lens"], gpu), _cu(c["k_lens"], gpu), 60, 130,
                                           c["tables"], out=room[:n])
        assert (room[n:] == 7).all()
        assert ((out.double() - want[:n]).abs() <= bound[:n]).all()
