"""GPU tests of the page operators (pk_copy_blocks, pk_fork_sequences, pk_extend_sequences,
pk_free_sequences, pk_compact_blocks) against a page pool in Python lists. Everything they compute is
a whole number or a copy, so every comparison is for equality, over the whole caches: what a call may
not touch has to keep its bits."""
import random

import pytest
import torch

import pagedkv
from pool_oracle import Pool, make_pool

pytestmark = pytest.mark.gpu


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _bits(t):
    return t.cpu().view(torch.int16)


@pytest.mark.parametrize("layers,blocks,bs,heads,dim", [
    (1, 5, 64, 1, 8), (3, 9, 64, 8, 128), (2, 7, 256, 2, 128), (28, 4, 128, 1, 128), (2, 6, 3, 5, 8)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_copy_blocks_partial_and_padded(gpu, layers, blocks, bs, heads, dim, dtype):
    tables, lens, refs, k, v = make_pool(layers + bs, [], bs, blocks, 1, layers, heads, dim, dtype)
    want = Pool(tables, lens, refs, k, v, bs)
    kg, vg = k.to(gpu), v.to(gpu)
    # whole and partial pages, none, more than a page, padding, blocks outside the cache, one block twice
    src = [0, 1, -1, blocks, 0, 1, 2]
    dst = [blocks - 1, blocks - 2, 2, 2, -1, blocks + 3, 2]
    tok = [bs, 1, bs, bs, bs, bs, bs]
    print(f"[copy] layers={layers} blocks={blocks} bs={bs} heads={heads} dim={dim} {dtype}", flush=True)
    want.copy(src, dst, tok)
    pagedkv.copy_blocks(kg, vg, _i32(src, gpu), _i32(dst, gpu), _i32(tok, gpu))
    assert torch.equal(_bits(kg), want.k.view(torch.int16)) and torch.equal(_bits(vg), want.v.view(torch.int16))
    for n in (0, -4, bs + 7, bs // 2 + 1):
        want.copy([1], [blocks - 1], [n])
        pagedkv.copy_blocks(kg, vg, _i32([1], gpu), _i32([blocks - 1], gpu), _i32([n], gpu))
    assert torch.equal(_bits(kg), want.k.view(torch.int16)) and torch.equal(_bits(vg), want.v.view(torch.int16))
    want.copy([2], [0], [bs])
    pagedkv.copy_blocks(kg, vg, _i32([2], gpu), _i32([0], gpu))
    pagedkv.copy_blocks(kg, vg, _i32([], gpu), _i32([], gpu))
    assert torch.equal(_bits(kg), want.k.view(torch.int16)) and torch.equal(_bits(vg), want.v.view(torch.int16))


def test_copy_blocks_layouts(gpu):
    """One layer's caches, and layers inside the blocks (block-major), as views of larger tensors."""
    g = torch.Generator().manual_seed(3)
    one = torch.randn(2, 6, 64, 2, 16, generator=g).to(torch.bfloat16)
    kv = one.to(gpu)
    print("[copy] one layer", flush=True)
    pagedkv.copy_blocks(kv[0], kv[1], _i32([4], gpu), _i32([1], gpu), _i32([40], gpu))
    one[:, 1, :40] = one[:, 4, :40]
    assert torch.equal(_bits(kv), one.view(torch.int16))
    big = torch.randn(6, 2, 5, 64, 2, 16, generator=g).to(torch.bfloat16)  # (NB, K/V, L, BS, Hkv, D)
    bg = big.to(gpu)
    print("[copy] block-major layers", flush=True)
    pagedkv.copy_blocks(bg[:, 0, 1:4].transpose(0, 1), bg[:, 1, 1:4].transpose(0, 1), _i32([0], gpu), _i32([5], gpu))
    big[5, :, 1:4] = big[0, :, 1:4]
    assert torch.equal(_bits(bg), big.view(torch.int16))


def test_copy_blocks_past_32_bits(gpu):
    """Caches of more than 2^32 bytes each: the first and last pages of the last layer."""
    layers, blocks, bs = 3, 3000, 256
    k = torch.zeros(layers, blocks, bs, 8, 128, dtype=torch.bfloat16, device=gpu)
    v = torch.zeros_like(k)
    assert k.numel() > 2 ** 31
    k[:, 1] = 1
    v[:, blocks - 2] = 2
    print("[copy] past 32 bits", flush=True)
    pagedkv.copy_blocks(k, v, _i32([1, blocks - 2], gpu), _i32([blocks - 1, 0], gpu))
    assert bool((k[:, blocks - 1] == 1).all()) and bool((k[:, 0] == 0).all())
    assert bool((v[:, 0] == 2).all()) and bool((v[:, blocks - 1] == 0).all())
    assert int(k.count_nonzero()) == 2 * k[:, 0].numel() and int(v.count_nonzero()) == 2 * v[:, 0].numel()


def _on(gpu, *ts):
    return [t.to(gpu) for t in ts]


@pytest.mark.parametrize("seed", range(6))
def test_pool_random_walk(gpu, seed):
    """A random run of all operators: forks of forks, refused children, rows listed twice, full and empty
    rows, an exhausted pool, full tables."""
    r = random.Random(seed)
    bs, rows, width = r.choice([(4, 12, 6), (64, 9, 3), (5, 40, 9)])
    nb = r.choice([rows * 2, rows * width])
    lens = [r.choice([0, 0, 1, bs, bs + 1, r.randint(0, width * bs)]) for _ in range(rows)]
    while sum(-(-n // bs) for n in lens) > nb:
        lens[r.randrange(rows)] = 0
    state = make_pool(seed, lens, bs, nb, width)
    want = Pool(*state, bs)
    t, ln, rc, k, v = _on(gpu, *state)
    for step in range(60):
        op = r.choice(["fork", "extend", "extend", "free", "compact"])
        n = r.randint(0, rows)
        pick = [r.randrange(-1, rows + 1) for _ in range(n)]
        print(f"[pool] seed={seed} step={step} {op} {n}", flush=True)
        if op == "fork":
            kids = [r.randrange(-1, rows + 1) for _ in range(n)]
            got = pagedkv.fork_sequences(k, v, t, ln, rc, _i32(pick, gpu), _i32(kids, gpu))
            assert got.cpu().tolist() == want.fork(pick, kids)
        elif op == "extend":
            got = pagedkv.extend_sequences(t, ln, rc, bs, _i32(pick, gpu))
            assert got.cpu().tolist() == want.extend(pick)
        elif op == "free":
            pick = pick[:r.randint(0, 3)] * 2
            pagedkv.free_sequences(t, ln, rc, bs, _i32(pick, gpu))
            want.free(pick)
        else:
            m, live = pagedkv.compact_blocks(k, v, t, ln, rc)
            wm, wl = want.compact()
            assert m.cpu().tolist() == wm and live.cpu().tolist() == [wl]
        want.same(t, ln, rc, k, v)
    held = torch.bincount(t[t >= 0].long().cpu(), minlength=nb)
    assert torch.equal(held, rc.cpu().long())  # every table entry is one holder


@pytest.mark.parametrize("n,nb", [(1, 1), (1024, 3000), (1000, 1700), (64, 70000)])
def test_largest_lists_and_pools(gpu, n, nb):
    """The longest lists, pools larger than one scan step of the allocator, and one whose only free blocks
    are its last ones."""
    bs, width = 2, 3
    half = n // 2
    lens = [3] * half + [0] * (n - half)
    state = make_pool(n, lens, bs, nb, width, layers=1)
    want = Pool(*state, bs)
    if nb > 60000:  # everything but the last 40 blocks has a holder outside the tables
        free = [b for b in range(nb) if want.refs[b] == 0]
        for b in free[:-40]:
            want.refs[b] = 1
            state[2][b] = 1
    t, ln, rc, k, v = _on(gpu, *state)
    parents = [i % max(half, 1) for i in range(n - half)]
    kids = list(range(half, n))
    print(f"[pool] n={n} nb={nb} fork", flush=True)
    got = pagedkv.fork_sequences(k, v, t, ln, rc, _i32(parents, gpu), _i32(kids, gpu))
    assert got.cpu().tolist() == want.fork(parents, kids)
    want.same(t, ln, rc, k, v)
    rows = list(range(n))
    for _ in range(2):
        print(f"[pool] n={n} nb={nb} extend", flush=True)
        got = pagedkv.extend_sequences(t, ln, rc, bs, _i32(rows, gpu))
        assert got.cpu().tolist() == want.extend(rows)
    pagedkv.free_sequences(t, ln, rc, bs, _i32(rows[::3], gpu))
    want.free(rows[::3])
    print(f"[pool] n={n} nb={nb} compact", flush=True)
    m, live = pagedkv.compact_blocks(k, v, t, ln, rc)
    wm, wl = want.compact()
    assert m.cpu().tolist() == wm and live.cpu().tolist() == [wl]
    want.same(t, ln, rc, k, v)


def test_strided_tables_and_lengths_past_the_table(gpu):
    """Tables that are columns of a wider tensor, and a length that runs past its table's width."""
    bs, width = 4, 3
    state = make_pool(5, [9, 12, 0, 0, 4], bs, 20, width)
    want = Pool(*state, bs)
    t, ln, rc, k, v = _on(gpu, *state)
    wide = torch.full((5, 8), 77, dtype=torch.int32, device=gpu)
    wide[:, 2:2 + width] = t
    t = wide[:, 2:2 + width]
    print("[pool] strided tables", flush=True)
    got = pagedkv.fork_sequences(k, v, t, ln, rc, _i32([0, 1], gpu), _i32([2, 3], gpu))
    assert got.cpu().tolist() == want.fork([0, 1], [2, 3])
    assert pagedkv.extend_sequences(t, ln, rc, bs, _i32([1, 2, 4], gpu)).cpu().tolist() == want.extend([1, 2, 4])
    want.same(t, ln, rc, k, v)
    ln[1] = 1000
    want.lens[1] = 1000
    pagedkv.free_sequences(t, ln, rc, bs, _i32([1], gpu))
    want.free([1])
    want.same(t, ln, rc, k, v)
    assert bool((wide[:, :2] == 77).all()) and bool((wide[:, 5:] == 77).all())


def test_captured_step_replays(gpu):
    """fork, extend, free and compact captured into one graph: every replay, with eager work between the
    replays, leaves what the eager calls leave."""
    bs, width = 8, 4
    state = make_pool(9, [13, 8, 0, 0, 0, 0], bs, 24, width, layers=3, heads=2)
    orig = _on(gpu, *state)
    t, ln, rc, k, v = (x.clone() for x in orig)
    parents, kids, done = _i32([0, 1, 0, -1], gpu), _i32([3, 4, 5, 2], gpu), _i32([0, 1, -1], gpu)

    def step():
        new = pagedkv.fork_sequences(k, v, t, ln, rc, parents, kids)
        slots = pagedkv.extend_sequences(t, ln, rc, bs, kids)
        pagedkv.free_sequences(t, ln, rc, bs, done)
        m, live = pagedkv.compact_blocks(k, v, t, ln, rc)
        return new, slots, m, live

    def reset():
        for x, o in zip((t, ln, rc, k, v), orig):
            x.copy_(o)

    print("[pool] eager step", flush=True)
    eager = [x.cpu() for x in step()] + [x.cpu().clone() for x in (t, ln, rc, k, v)]
    reset()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for i in range(4):
        reset()
        print(f"[pool] replay {i}", flush=True)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip([*outs, t, ln, rc, k, v], eager):
            assert torch.equal(a.cpu(), b)
        (torch.randn(256, 256, device=gpu) @ torch.randn(256, 256, device=gpu)).sum().item()


def test_other_stream(gpu):
    bs = 16
    state = make_pool(2, [40, 0], bs, 9, 3)
    want = Pool(*state, bs)
    t, ln, rc, k, v = _on(gpu, *state)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    print("[pool] other stream", flush=True)
    with torch.cuda.stream(s):
        new = pagedkv.fork_sequences(k, v, t, ln, rc, _i32([0], gpu), _i32([1], gpu))
    s.synchronize()
    assert new.cpu().tolist() == want.fork([0], [1])
    want.same(t, ln, rc, k, v)
