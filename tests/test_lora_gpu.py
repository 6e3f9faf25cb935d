"""GPU tests of the per-row adapters (pk_lora_linear, pk_lora_add) against their formula in 64 bits.

Tolerance, for every element: one rounding of the output, 2^-8 |exact| (half a bf16 step), and what the
fp32 sums may lose: k 2^-24 sum |x w| for the projection, and for the adapter (k + 2 r + 8) 2^-24 for its
two sums in a row plus 2^-16 for t's split into two bf16, all of it relative to the sum of the
products' sizes, s sum_j (sum_k |x A|) |B|. A wrong row, adapter, slice, scale or k range is off by
the size of the delta itself, orders of magnitude more.
"""
import pytest
import torch

import pagedkv

pytestmark = pytest.mark.gpu

QKV, O, GATE_UP, DOWN = (1024, (2048, 1024, 1024)), (2048, (1024,)), (1024, (3072, 3072)), (3072, (1024,))


def _rand(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(torch.bfloat16)


def _case(seed, rows, k, widths, rank, adapters, ids="mixed"):
    g = torch.Generator().manual_seed(seed)
    n = sum(widths)
    c = dict(x=_rand(g, rows, k), w=_rand(g, n, k, std=0.05), y=_rand(g, rows, n),
             a=_rand(g, adapters, len(widths) * rank, k, std=k ** -0.5), b=_rand(g, adapters, n, rank, std=0.3),
             scales=torch.rand(adapters, generator=g) * 3 + 0.1, widths=widths)
    if ids == "mixed":       # every value, none and values outside [0, adapters) among them
        i = torch.randint(-1, adapters + 1, (rows,), generator=g)
        i[torch.rand(rows, generator=g) < 0.02] = -2 ** 31
    elif ids == "runs":      # long runs of one adapter, as the prompts of a prefill step
        cut = torch.sort(torch.randint(0, rows + 1, (6,), generator=g)).values.tolist()
        i = torch.cat([torch.full((b - a,), int(torch.randint(-1, adapters, (1,), generator=g)))
                       for a, b in zip([0] + cut, cut + [rows])])
    else:
        i = torch.full((rows,), ids)
    c["ids"] = i.to(torch.int32)
    return c


def _exact(c, base, base_mag, k):
    """(formula in 64 bits, what fp32 sums may lose) per element."""
    x, r = c["x"].double(), c["b"].shape[2]
    out, mag = base.clone(), torch.zeros_like(base)
    for i in set(c["ids"].tolist()):
        if not 0 <= i < c["a"].shape[0]:
            continue
        rows = (c["ids"] == i).nonzero().squeeze(1)
        a, b, s = c["a"][i].double(), c["b"][i].double(), c["scales"][i].double()
        t, tm, at = s * (x[rows] @ a.T), s * (x[rows].abs() @ a.abs().T), 0
        for q, n in enumerate(c["widths"]):
            cols = slice(at, at + n)
            out[rows, cols] += t[:, q * r:(q + 1) * r] @ b[cols].T
            mag[rows, cols] += tm[:, q * r:(q + 1) * r] @ b[cols].abs().T
            at += n
    loss = (k + 8) * 2.0 ** -24 * base_mag + ((k + 2 * r + 8) * 2.0 ** -24 + 2.0 ** -16) * mag
    return out, loss


def _check(got, exact, loss, what):
    got = got.cpu().double()
    bound = 2.0 ** -8 * exact.abs() + (1 + 2.0 ** -8) * loss + 2.0 ** -133
    over = (got - exact).abs() - bound
    assert torch.isfinite(got).all() and over.max().item() <= 0, f"{what}: over its bound by {over.max().item():.3e}"


def _gpu(c, gpu):
    return {n: t.to(gpu) if isinstance(t, torch.Tensor) else t for n, t in c.items()}


def _linear(d, **kw):
    return pagedkv.lora_linear(d["x"], d["w"], d["a"], d["b"], d["ids"], d["scales"], slices=d["widths"], **kw)


def _add(d, **kw):
    return pagedkv.lora_add(d["y"], d["x"], d["a"], d["b"], d["ids"], d["scales"], slices=d["widths"], **kw)


@pytest.mark.parametrize("rows,proj,rank,adapters,ids", [
    (1, QKV, 16, 4, 2), (1, DOWN, 8, 1, -1), (7, O, 64, 3, "mixed"), (16, QKV, 128, 5, "mixed"),
    (17, GATE_UP, 24, 2, "mixed"), (33, DOWN, 72, 40, "mixed"), (97, GATE_UP, 16, 8, "runs"), (128, QKV, 16, 1, 0),
    (128, DOWN, 64, 130, "mixed"), (128, O, 8, 3, -1), (65, (256, (32, 96, 64, 32)), 40, 6, "mixed"),
    (100, (512, (64,)), 104, 300, "mixed"), (2, QKV, 16, 4, "mixed"), (2, GATE_UP, 8, 1, 0), (1, QKV, 8, 3, -1),
    (3, QKV, 16, 4, "mixed"), (1, GATE_UP, 40, 2, 1)])
def test_linear_against_formula(gpu, rows, proj, rank, adapters, ids):
    k, widths = proj
    c = _case(rows + rank, rows, k, widths, rank, adapters, ids)
    print(f"[lora_linear] rows={rows} k={k} widths={widths} rank={rank} adapters={adapters} ids={ids}", flush=True)
    got = _linear(_gpu(c, gpu))
    x, w = c["x"].double(), c["w"].double()
    _check(got, *_exact(c, x @ w.T, x.abs() @ w.abs().T, k), f"lora_linear {rows} {proj} {rank}")


@pytest.mark.parametrize("rows,proj,rank,adapters,ids", [
    (1, QKV, 16, 4, 1), (2, (8, (32,)), 8, 2, "mixed"), (63, (40, (32, 32)), 16, 3, "mixed"),
    (64, (1000, (96,)), 32, 3, "mixed"), (65, (1032, (160, 32, 32, 64)), 128, 3, "mixed"), (300, O, 8, 24, "mixed"),
    (512, QKV, 16, 600, "mixed"), (513, QKV, 16, 8, "runs"), (513, (40, (32, 32)), 40, 1, 0),
    (600, (264, (288,)), 72, 4095, "mixed"), (700, (64, (288,)), 8, 5000, "mixed"), (2500, O, 16, 1, "runs"),
    (1200, QKV, 16, 2, "mixed"), (1500, QKV, 16, 14, "runs"), (700, (1000, (96, 64)), 24, 3, "mixed"),
    (1025, DOWN, 64, 7, "runs"),
    (2000, GATE_UP, 128, 5, "runs"), (30, QKV, 32, 7, "mixed"), (64, QKV, 24, 3, "runs"), (33, DOWN, 16, 9, "mixed"),
    (128, O, 32, 2, "mixed"), (17000, (64, (32, 32)), 8, 3, "runs"), (33000, (64, (32,)), 16, 40, "mixed"),
    (24700, (256, (64, 64)), 32, 2, "runs"), (3001, O, 16, 50, "mixed"), (1500, (64, (32,)), 8, 4, -1)])
def test_add_against_formula(gpu, rows, proj, rank, adapters, ids):
    k, widths = proj
    c = _case(rows + rank, rows, k, widths, rank, adapters, ids)
    print(f"[lora_add] rows={rows} k={k} widths={widths} rank={rank} adapters={adapters} ids={ids}", flush=True)
    d = _gpu(c, gpu)
    got = _add(d)
    exact, loss = _exact(c, c["y"].double(), torch.zeros(rows, sum(widths), dtype=torch.float64), k)
    _check(got, exact, loss, f"lora_add {rows} {proj} {rank}")
    none = (c["ids"] < 0) | (c["ids"] >= adapters)
    assert torch.equal(got.cpu()[none].view(torch.int16), c["y"][none].view(torch.int16))  # a copy, bit for bit
    in_place = _add(d, out=d["y"])
    assert in_place is d["y"] and torch.equal(in_place.view(torch.int16), got.view(torch.int16))


@pytest.mark.parametrize("rows", [100, 1900])
def test_row_does_not_depend_on_the_batch(gpu, rows):
    """A row's bits are the same alone, in a batch and in another order of it, on both sides of the size
    at which rows are sorted."""
    d = _gpu(_case(rows, rows, 1024, (256, 64), 16, 5), gpu)
    sorts = pagedkv.lora_workspace_bytes(rows, 320, 1024, 16, (256, 64), 5) > rows * 32 * 4
    assert sorts == (rows == 1900)
    print(f"[lora_add] rows={rows} alone / together / reversed", flush=True)
    whole = _add(d)
    for m in (0, rows // 2, rows - 1):
        one = {n: d[n][m:m + 1] if n in ("x", "y", "ids") else d[n] for n in d}
        assert torch.equal(_add(one)[0].view(torch.int16), whole[m].view(torch.int16))
    back = {n: d[n].flip(0).contiguous() if n in ("x", "y", "ids") else d[n] for n in d}
    assert torch.equal(_add(back).flip(0).view(torch.int16), whole.view(torch.int16))


@pytest.mark.parametrize("rows", [40, 2700])
def test_non_finite_values_stay_in_their_rows(gpu, rows):
    """NaN and infinity in one row's x or y, or in one adapter, reach only the rows they belong to."""
    c = _case(rows, rows, 512, (64, 64), 16, 4)
    d = _gpu(c, gpu)
    clean = _add(d)
    c["ids"][3], c["ids"][5] = 1, -1
    d = _gpu(c, gpu)
    clean = _add(d)
    d["x"][3] = float("nan")
    d["x"][5] = float("inf")       # a row without an adapter: its x is not used
    d["y"][7, 9] = float("-inf")
    d["a"][2, 0, 0], d["b"][2, 70, 1] = float("nan"), float("inf")
    print(f"[lora_add] rows={rows} non-finite", flush=True)
    got = _add(d)
    bad = (c["ids"] == 2)
    bad[3] = True
    keep = ~bad
    keep[7] = False
    assert torch.equal(got.cpu()[keep].view(torch.int16), clean.cpu()[keep].view(torch.int16))
    assert bool(got[3].isnan().all()) and got[bad.to(gpu)].isfinite().logical_not().any(1).all()
    if not bad[7]:
        assert float(got[7, 9]) == float("-inf") and torch.equal(got[7, 10:], clean[7, 10:])


@pytest.mark.parametrize("rows,adapters", [(1, 3), (17, 1), (33, 40), (70, 3), (125, 15), (800, 3), (900, 300),
                                           (2700, 5)])
def test_strides_and_what_lies_around_the_output(gpu, rows, adapters):
    """x, y, out, weight and both adapters as views of larger tensors; nothing beside out is written,
    the rows behind the last one of a tile of 16 or 64 among it."""
    k, n, rank = 256, 96, 16
    c = _case(rows, rows, k, (64, 32), rank, adapters)
    d = _gpu(c, gpu)

    def view(t, pad):
        big = torch.full((*t.shape[:-1], t.shape[-1] + pad), float("nan"), dtype=t.dtype, device=gpu)
        big[..., 8:8 + t.shape[-1]] = t
        return big[..., 8:8 + t.shape[-1]]

    v = dict(d, x=view(d["x"], 24), y=view(d["y"], 40), w=view(d["w"], 16), b=view(d["b"], 8))
    layers = torch.stack([torch.zeros_like(d["a"]), d["a"]], 1)  # (L, layers, S r, k): this layer's slice
    v["a"] = layers[:, 1]
    big = torch.full((rows + 80, n + 48), 7.0, dtype=torch.bfloat16, device=gpu)
    out = big[1:1 + rows, 16:16 + n]
    print(f"[lora] rows={rows} adapters={adapters} strides", flush=True)
    _add(v, out=out)
    assert torch.equal(out, _add(d))
    out.fill_(7.0)
    assert bool((big == 7.0).all())
    one = torch.cat([d["x"], d["y"], torch.zeros_like(d["y"])], 1)  # x, y and out as columns of one buffer
    _add(dict(d, x=one[:, :k], y=one[:, k:k + n]), out=one[:, k + n:])
    assert torch.equal(one, torch.cat([d["x"], d["y"], _add(d)], 1))
    if rows <= 128:
        _linear(v, out=out)
        assert torch.equal(out, _linear(d))
        out.fill_(7.0)
        assert bool((big == 7.0).all())


def test_nothing_to_do(gpu):
    d = _gpu(_case(1, 5, 256, (64,), 8, 2), gpu)
    empty = dict(d, a=d["a"][:0], b=d["b"][:0], scales=d["scales"][:0])
    print("[lora] no adapters, no rows", flush=True)
    assert torch.equal(_add(empty), d["y"])
    none = dict(d, ids=torch.full_like(d["ids"], -1))
    assert torch.equal(_linear(empty), _linear(none))
    big = _gpu(_case(2, 600, 64, (32,), 8, 2), gpu)
    assert torch.equal(_add(dict(big, a=big["a"][:0], b=big["b"][:0], scales=big["scales"][:0])), big["y"])
    zero = dict(d, x=d["x"][:0], y=d["y"][:0], ids=d["ids"][:0])
    assert _add(zero).shape == (0, 64) and _linear(zero).shape == (0, 64)
    one = pagedkv.lora_add(d["y"], d["x"], d["a"], d["b"], d["ids"])      # scales and slices left out
    assert torch.equal(one, _add(dict(d, scales=torch.ones(2, device=gpu))))


def test_linear_without_adapters_is_the_projection(gpu):
    """Rows without an adapter get pk_linear's bits: the same sums, rounded once."""
    d = _gpu(_case(4, 100, 1024, (2048, 1024, 1024), 16, 3), gpu)
    print("[lora_linear] none", flush=True)
    got, plain = _linear(d), pagedkv.linear(d["x"], d["w"])
    none = ((d["ids"] < 0) | (d["ids"] >= 3)).nonzero().squeeze(1)
    assert none.numel() > 5 and torch.equal(got[none].view(torch.int16), plain[none].view(torch.int16))


def test_offsets_past_32_bits(gpu):
    """Adapters, y and out of more than 2^31 elements: the last adapters, rows and columns."""
    n, rank, adapters, rows = 32768, 128, 520, 66000
    b = torch.zeros(adapters, n, rank, dtype=torch.bfloat16, device=gpu)
    a = torch.zeros(adapters, rank, 8, dtype=torch.bfloat16, device=gpu)
    y = torch.zeros(rows, n, dtype=torch.bfloat16, device=gpu)
    assert b.numel() > 2 ** 31 and y.numel() > 2 ** 31
    a[adapters - 1, 5, 7], b[adapters - 1, n - 1, 5], b[adapters - 1, 3, 5] = 2.0, 3.0, 5.0
    x = torch.zeros(rows, 8, dtype=torch.bfloat16, device=gpu)
    x[:, 7] = 1.0
    ids = torch.full((rows,), 4, dtype=torch.int32, device=gpu)
    ids[rows - 1], ids[7] = adapters - 1, adapters - 1
    print("[lora_add] past 32 bits", flush=True)
    pagedkv.lora_add(y, x, a, b, ids, out=y)
    assert int(y.count_nonzero()) == 4
    assert y[rows - 1, n - 1].item() == 6.0 and y[7, 3].item() == 10.0 and y[7, n - 1].item() == 6.0


@pytest.mark.parametrize("rows", [48, 640, 3000])
def test_captured_call_replays_with_new_rows(gpu, rows):
    """A captured call replayed with other rows and other adapters in the same buffers, with eager calls
    of another shape between the replays."""
    cases = [_case(s, rows, 512, (64, 96), 24, 6) for s in range(4)]
    d = _gpu(cases[0], gpu)
    other = _gpu(_case(9, 33, 256, (64,), 8, 2), gpu)

    def step():
        return _add(d), _linear(d) if rows <= 128 else None

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    print(f"[lora] rows={rows} capture", flush=True)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = step()
    for i, c in enumerate(cases):
        for n in ("x", "y", "ids", "a", "b", "scales"):
            d[n].copy_(c[n])
        print(f"[lora] replay {i}", flush=True)
        g.replay()
        torch.cuda.synchronize()
        for got, want in zip(outs, step()):
            assert got is None or torch.equal(got, want)
        _add(other)
        _linear(other)
        torch.cuda.synchronize()


def test_two_streams(gpu):
    """Calls on two streams at once, each with its own scratch."""
    ds = [_gpu(_case(s, 4000, 1024, (512,), 16, 4), gpu) for s in range(2)]
    want = [_add(d) for d in ds]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ds]
    outs = [[], []]
    print("[lora_add] two streams", flush=True)
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(_add(ds[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for o in outs[i]:
            assert torch.equal(o, want[i])


def test_given_workspace(gpu):
    d = _gpu(_case(3, 2700, 256, (64, 32), 16, 5), gpu)
    need = pagedkv.lora_workspace_bytes(2700, 96, 256, 16, (64, 32), 5)
    assert need > 2700 * 32 * 4  # sorted
    ws = torch.full((need + 64,), 255, dtype=torch.uint8, device=gpu)
    print("[lora_add] workspace", flush=True)
    assert torch.equal(_add(d, workspace=ws[:need]), _add(d))
    assert bool((ws[need:] == 255).all())
    small = {n: d[n][:100] if n in ("x", "y", "ids") else d[n] for n in d}
    need = pagedkv.lora_workspace_bytes(100, 96, 256, 16, (64, 32), linear=True)
    ws = torch.full((need + 64,), 255, dtype=torch.uint8, device=gpu)
    assert torch.equal(_linear(small, workspace=ws[:need]), _linear(small))
    assert bool((ws[need:] == 255).all())
