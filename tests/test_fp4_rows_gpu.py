"""GPU tests of rows of 4-bit caches: stored, appended with norm and rotation, read back. Everything is compared
for equality with the plain statement of the format (tests/fp4_oracle.py)."""
import pytest
import torch

import fp4_oracle as ref
import pagedkv

pytestmark = pytest.mark.gpu
D = 128


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, device, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(torch.bfloat16).to(device)


def _bytes(g, *shape, device):
    return torch.randint(0, 256, shape, generator=g, dtype=torch.uint8).to(device)


def _expect(cache, slots, x):
    """What the cache has to be after rows x were stored at slots."""
    want = cache.cpu().clone().view(-1, cache.shape[-1])
    kv = x.shape[1]
    for i, s in enumerate(slots):
        if 0 <= s < want.shape[0]:
            want[s, :68 * kv] = ref.pack(x[i].cpu())
    return want.view(cache.shape)


def test_every_bf16_value(gpu):
    """All finite bf16 values, each as the largest of its 32 and beside larger ones; then infinities and NaN."""
    bits = torch.arange(65536, dtype=torch.int32)
    every = bits.to(torch.int16).view(torch.bfloat16)
    finite = every[torch.isfinite(every)]
    blocks = torch.zeros(finite.numel(), 32, dtype=torch.bfloat16)
    blocks[:, 0] = finite
    blocks[:, 1] = -(finite * 0.61)
    blocks[:, 2] = finite.abs() * 0.7109375
    blocks[:, 3:] = finite.flip(0).unsqueeze(1) * torch.linspace(-1, 1, 29).to(torch.bfloat16)
    ramp = finite.sort().values[torch.arange(0, finite.numel(), 61)]
    tops = finite[torch.arange(3, finite.numel(), 977)].abs()
    pairs = torch.cartesian_prod(tops, ramp)
    more = torch.zeros(-(-pairs.shape[0] // 31), 31, dtype=torch.bfloat16)
    more.view(-1)[:pairs.shape[0]] = torch.minimum(pairs[:, 1].abs(), pairs[:, 0]) * pairs[:, 1].sign()
    more = torch.cat((pairs[torch.arange(more.shape[0]) * 31, 0].unsqueeze(1), more), 1)
    odd = torch.zeros(6, 32, dtype=torch.bfloat16)
    odd[:, 5] = torch.tensor([float("inf"), float("-inf"), float("nan"), 1.0, 0.0, -0.0])
    odd[:, 9] = torch.tensor([1.0, float("inf"), 3.0, float("nan"), 0.0, -0.0])
    x = torch.cat((blocks, more, odd))
    x = torch.cat((x, x[: -x.shape[0] % 8])).view(-1, 2, D)
    n = x.shape[0]
    kc, vc = (torch.zeros(-(-n // 64), 64, ref.row_bytes(2), dtype=torch.uint8, device=gpu) for _ in range(2))
    slots = torch.randperm(kc.shape[0] * 64, generator=_gen(1))[:n].to(torch.int32)
    pagedkv.store_kvcache_fp4(x.to(gpu), x.flip(0).to(gpu), kc, vc, slots.to(gpu))
    for cache, y in ((kc, x), (vc, x.flip(0))):
        assert torch.equal(cache.cpu().view(-1, cache.shape[-1])[slots.long(), :136], ref.pack(y))


@pytest.mark.parametrize("kv", [1, 2, 3, 5, 8, 16])
@pytest.mark.parametrize("n", [1, 2, 37, 301])
def test_store(gpu, kv, n):
    g = _gen(10 * n + kv)
    nb, bs = 7, 64
    kc, vc = (_bytes(g, nb, bs, ref.row_bytes(kv), device=gpu) for _ in range(2))
    key = _randn(g, n, kv, D, device=gpu)
    value = _randn(g, n, (2 * kv + 3) * D, device=gpu, scale=30.0)[:, 2 * D:(2 + kv) * D].view(n, kv, D)  # strided rows
    slots = torch.randperm(nb * bs, generator=g)[:n].tolist()
    for i, s in ((0, -1), (3, nb * bs), (5, -7), (6, 2 ** 31 - 1)):  # padding and slots that are none
        if n > 6:
            slots[i] = s
    want = _expect(kc, slots, key), _expect(vc, slots, value)
    pagedkv.store_kvcache_fp4(key, value, kc, vc, torch.tensor(slots, dtype=torch.int32, device=gpu))
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])


def test_store_nothing(gpu):
    kc, vc = (torch.full((2, 64, 272), 7, dtype=torch.uint8, device=gpu) for _ in range(2))
    empty = torch.zeros(0, 4, D, dtype=torch.bfloat16, device=gpu)
    pagedkv.store_kvcache_fp4(empty, empty, kc, vc, torch.zeros(0, dtype=torch.int32, device=gpu))
    assert (kc == 7).all() and (vc == 7).all()


@pytest.mark.parametrize("heads,kv", [(16, 8), (8, 4), (4, 2), (2, 1), (8, 1), (3, 3), (5, 1), (32, 8)])
@pytest.mark.parametrize("n", [1, 5, 130, 1100])
@pytest.mark.parametrize("norm", [True, False])
def test_append(gpu, heads, kv, n, norm):
    if n == 1100 and heads not in (16, 2):
        pytest.skip("one size of the wide launch for two geometries")
    g = _gen(1000 * heads + 10 * kv + n)
    nb, bs = -(-n // 64) + 2, 64
    kc, vc = (_bytes(g, nb, bs, ref.row_bytes(kv), device=gpu) for _ in range(2))
    qkv = _randn(g, n, (heads + 2 * kv + 1) * D, device=gpu, scale=3.0)[:, :(heads + 2 * kv) * D]  # strided rows
    pos = torch.randint(0, 500, (n,), generator=g)
    pos[0] = 499
    if n > 2:
        pos[1], pos[2] = -4, 900  # clamped into the table
    table = pagedkv.rope_cos_sin(500, D, device="cpu")
    qw, kw = (_randn(g, D, device="cpu", scale=0.2) + 1 for _ in range(2))
    slots = torch.randperm(nb * bs, generator=g)[:n].tolist()
    if n > 4:
        slots[4], slots[3] = -1, nb * bs + 5
    x = qkv.cpu().view(n, heads + 2 * kv, D) if qkv.is_contiguous() else qkv.cpu().contiguous().view(n, heads + 2 * kv, D)
    q = ref.norm_rope(x[:, :heads], qw if norm else None, 1e-6, pos, table)
    k = ref.norm_rope(x[:, heads:heads + kv], kw if norm else None, 1e-6, pos, table)
    v = x[:, heads + kv:]
    want = _expect(kc, slots, k), _expect(vc, slots, v)
    args = (qkv, pos.to(gpu), table.to(gpu), heads, kv, D, qw.to(gpu) if norm else None, kw.to(gpu) if norm else None,
            1e-6, kc, vc, torch.tensor(slots, dtype=torch.int32, device=gpu))
    got = pagedkv.qk_norm_rope_store_fp4(*args, return_kv=True)
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])
    assert torch.equal(got[0].cpu().view(torch.int16), q.view(torch.int16))
    for y, z in ((got[1], k), (got[2], v)):
        assert torch.equal(y.cpu().double(), ref.values(ref.pack(z), kv))
    again = pagedkv.qk_norm_rope_store_fp4(*args, q_out=torch.empty_like(got[0]))
    assert torch.equal(again[0], got[0]) and again[1] is None and again[2] is None
    # within a bf16 step of the 16-bit producer, whose products may be fused
    near, near_k = pagedkv.qk_norm_rope_store(qkv, pos.to(gpu), table.to(gpu), heads, kv, D, *args[6:8], 1e-6, return_k=True)
    assert (near.double() - got[0].double()).abs().max() <= 2 ** -7 * near.double().abs().max()


def test_append_of_extreme_rows(gpu):
    """Rows of zeros, of the largest values, of values whose squares leave 32 bits, and of NaN."""
    n, heads, kv = 6, 2, 1
    x = torch.zeros(n, heads + 2 * kv, D)
    x[1] = 3.0e38
    x[2] = 1.0e30 * torch.randn(heads + 2 * kv, D, generator=_gen(2))
    x[3] = 1.0e-30 * torch.randn(heads + 2 * kv, D, generator=_gen(3))
    x[4, :, 7] = float("nan")
    x[5] = torch.randn(heads + 2 * kv, D, generator=_gen(4))
    x = x.to(torch.bfloat16)
    table = pagedkv.rope_cos_sin(16, D, device="cpu")
    pos, w = torch.arange(n), torch.ones(D, dtype=torch.bfloat16)
    kc, vc = (torch.zeros(1, 64, 80, dtype=torch.uint8, device=gpu) for _ in range(2))
    q, k, v = pagedkv.qk_norm_rope_store_fp4(x.view(n, -1).to(gpu), pos.to(gpu), table.to(gpu), heads, kv, D, w.to(gpu),
                                             w.to(gpu), 1e-6, kc, vc, torch.arange(n, dtype=torch.int32, device=gpu), True)
    for i in (0, 1, 2, 3, 5):
        want = ref.norm_rope(x[i:i + 1, :heads], w, 1e-6, pos[i:i + 1], table)
        assert torch.equal(q[i:i + 1].cpu().view(torch.int16), want.view(torch.int16)), i
        want = ref.norm_rope(x[i:i + 1, heads:heads + 1], w, 1e-6, pos[i:i + 1], table)
        assert torch.equal(k[i:i + 1].cpu().double(), ref.values(ref.pack(want), 1)), i
        assert torch.equal(v[i:i + 1].cpu().double(), ref.values(ref.pack(x[i:i + 1, heads + 1:]), 1)), i
    assert torch.isnan(q[4]).all() and torch.isnan(k[4]).all()
    assert torch.isnan(v[4, 0, :32]).all() and (v[4, 0, 32:] == 0).all()


@pytest.mark.parametrize("kv,bs", [(8, 256), (3, 64), (1, 100), (2, 1)])
def test_gather(gpu, kv, bs):
    g = _gen(kv)
    lens = [1, 0, bs, bs + 1, 3 * bs - 1, 17]
    nb = 16
    base = _bytes(g, nb, bs + 3, ref.row_bytes(kv), device=gpu)
    cache = base[:, :bs]  # blocks with room between them
    cache[..., 64 * kv:68 * kv] = cache[..., 64 * kv:68 * kv].clamp(100, 150)
    cache[3, :, 64 * kv] = 255
    table = torch.randint(0, nb, (len(lens) + 1, 17), generator=g, dtype=torch.int32)
    table[3, 1], table[4, 0] = -1, nb  # no blocks: zeros
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32)
    got = pagedkv.gather_kv_fp4(cache, table.to(gpu), cu.to(gpu), max(lens), int(cu[-1]))
    assert got.shape == (int(cu[-1]), kv, D)
    c = cache.cpu()
    for i, n in enumerate(lens):
        for t in range(n):
            blk = int(table[i, t // bs])
            want = ref.values(c[blk, t % bs], kv) if 0 <= blk < nb else torch.zeros(kv, D, dtype=torch.float64)
            y = got[int(cu[i]) + t].cpu().double()
            assert torch.equal(y.nan_to_num(9e9), want.nan_to_num(9e9)), (i, t)
    assert torch.equal(pagedkv.gather_kv_fp4(cache, table.to(gpu), cu.to(gpu), max(lens)).view(torch.int16), got.view(torch.int16))


def test_rows_in_a_cache_past_four_gigabytes(gpu):
    """Slots and pages whose bytes lie past 2^32."""
    kv, bs = 8, 256
    nb = 2 ** 32 // (bs * 544) + 40
    kc, vc = (torch.zeros(nb, bs, 544, dtype=torch.uint8, device=gpu) for _ in range(2))
    g = _gen(5)
    n = 5
    slots = torch.tensor([nb * bs - 1, (nb - 30) * bs, 0, (nb - 3) * bs + 77, 2 ** 31 // 544 + 1], dtype=torch.int32)
    key, value = _randn(g, n, kv, D, device=gpu), _randn(g, n, kv, D, device=gpu)
    pagedkv.store_kvcache_fp4(key, value, kc, vc, slots.to(gpu))
    for cache, x in ((kc, key), (vc, value)):
        assert torch.equal(cache.view(-1, 544)[slots.long().to(gpu)].cpu(), ref.pack(x.cpu()))
        table = (slots // bs).view(n, 1)
        cu = torch.cat((torch.zeros(1), (slots % bs + 1).cumsum(0))).to(torch.int32)
        got = pagedkv.gather_kv_fp4(cache, table.to(gpu), cu.to(gpu), bs, int(cu[-1]))
        assert torch.equal(got[(cu[1:] - 1).long().to(gpu)].cpu().double(), ref.values(ref.pack(x.cpu()), kv))


def test_captured_append_store_and_gather(gpu):
    """A graph of a step's append, a store and the read back, replayed with other inputs between eager work."""
    n, heads, kv, bs, nb = 9, 4, 2, 64, 5
    g = _gen(6)
    qkv = _randn(g, n, (heads + 2 * kv) * D, device=gpu)
    pos = torch.arange(n, device=gpu)
    table = pagedkv.rope_cos_sin(64, D, device=gpu)
    slots = torch.randperm(nb * bs, generator=g)[:n].to(torch.int32).to(gpu)
    bt = torch.arange(nb, dtype=torch.int32, device=gpu).view(1, nb)
    cu = torch.tensor([0, nb * bs], dtype=torch.int32, device=gpu)
    kc, vc = (torch.zeros(nb, bs, ref.row_bytes(kv), dtype=torch.uint8, device=gpu) for _ in range(2))

    def step():
        q, k, v = pagedkv.qk_norm_rope_store_fp4(qkv, pos, table, heads, kv, D, None, None, 1e-6, kc, vc, slots, True)
        pagedkv.store_kvcache_fp4(k, v, kc, vc, slots)  # values of the format store as themselves
        return q, pagedkv.gather_kv_fp4(kc, bt, cu, nb * bs, nb * bs), pagedkv.gather_kv_fp4(vc, bt, cu, nb * bs, nb * bs)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        qkv.copy_(_randn(g, *qkv.shape, device=gpu, scale=1.0 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        bytes_ = kc.clone(), vc.clone()
        kc.zero_(), vc.zero_()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(kc, bytes_[0]) and torch.equal(vc, bytes_[1])


@pytest.mark.parametrize("kv", [33, 70, 255])
def test_more_head_rows_than_a_work_group_takes_at_once(gpu, kv):
    """Store and read back of tokens of more than 64 head rows."""
    g = _gen(kv)
    n, nb, bs = 5, 2, 64
    kc, vc = (_bytes(g, nb, bs, ref.row_bytes(kv), device=gpu) for _ in range(2))
    key, value = _randn(g, n, kv, D, device=gpu), _randn(g, n, kv, D, device=gpu, scale=1e-3)
    slots = [70, -1, 3, 64, 127]
    want = _expect(kc, slots, key), _expect(vc, slots, value)
    pagedkv.store_kvcache_fp4(key, value, kc, vc, torch.tensor(slots, dtype=torch.int32, device=gpu))
    assert torch.equal(kc.cpu(), want[0]) and torch.equal(vc.cpu(), want[1])
    kc[..., 64 * kv:68 * kv] = kc[..., 64 * kv:68 * kv].clamp(100, 150)
    table = torch.tensor([[1], [0]], dtype=torch.int32, device=gpu)
    cu = torch.tensor([0, 64, 68], dtype=torch.int32, device=gpu)
    got = pagedkv.gather_kv_fp4(kc, table, cu, 64, 68)
    assert torch.equal(got.cpu().double(), ref.values(torch.cat((kc[1], kc[0, :4])).cpu(), kv))


def test_read_back_stops_at_its_output(gpu):
    """Lengths that end past the output's rows, and past max_seqlen_k: nothing is written there."""
    kv, bs = 2, 64
    kc, _ = ref.make_cache(kv, 4, bs, _gen(2), gpu)
    table = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32, device=gpu)
    cu = torch.tensor([0, 100, 228], dtype=torch.int32, device=gpu)
    room = torch.full((256, kv, D), 7.0, dtype=torch.bfloat16, device=gpu)
    rows = torch.cat((kc[2], kc[0, :36], kc[1], kc[3]))
    from pagedkv._call import call
    from pagedkv._lib import lib
    call(lib().pk_gather_kv_fp4, "pk_gather_kv_fp4", gpu, kc.data_ptr(), kc.stride(0), 4, bs, kv, D, table.data_ptr(), 2,
         cu.data_ptr(), 2, 120, 190, room.data_ptr())
    assert torch.equal(room[:190].double(), ref.values(rows, kv)[:190]) and (room[190:] == 7).all()
    room.fill_(7.0)
    call(lib().pk_gather_kv_fp4, "pk_gather_kv_fp4", gpu, kc.data_ptr(), kc.stride(0), 4, bs, kv, D, table.data_ptr(), 2,
         cu.data_ptr(), 2, 120, 256, room.data_ptr())
    assert torch.equal(room[:220].double(), ref.values(rows, kv)[:220]) and (room[220:] == 7).all()


@pytest.mark.parametrize("n", [300, 2100, 5000])
def test_append_does_not_hang_on_the_number_of_tokens(gpu, n):
    """A token's q, rows and values are the same bits alone among few tokens, which 8 wavefronts share, and among many."""
    heads, kv, bs = 16, 8, 64
    g = _gen(n)
    qkv = _randn(g, n, (heads + 2 * kv) * D, device=gpu)
    pos = torch.randint(0, 512, (n,), generator=g).to(gpu)
    table = pagedkv.rope_cos_sin(512, D, device=gpu)
    qw, kw = _randn(g, D, device=gpu), _randn(g, D, device=gpu)
    slots = torch.randperm(80 * bs, generator=g)[:n].to(torch.int32).to(gpu)
    caches = [torch.zeros(80, bs, 544, dtype=torch.uint8, device=gpu) for _ in range(4)]

    def append(a, b, kc, vc):
        return pagedkv.qk_norm_rope_store_fp4(qkv[a:b], pos[a:b], table, heads, kv, D, qw, kw, 1e-6, kc, vc, slots[a:b], True)

    whole = append(0, n, *caches[:2])
    for a in range(0, n, 100):
        for x, y in zip(append(a, min(n, a + 100), *caches[2:]), whole):
            assert torch.equal(x.view(torch.int16), y[a:a + 100].view(torch.int16))
    assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])
