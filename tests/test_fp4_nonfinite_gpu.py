"""GPU tests of tokens with infinities and NaN appended to 4-bit caches, against the plain statement of the steps
(tests/fp4_oracle.py): every bit of what is finite, and NaN where it is NaN."""
import pytest
import torch

import fp4_oracle as ref
import pagedkv

pytestmark = pytest.mark.gpu
D, HEADS, KV = 128, 4, 2


def _same(got, want):
    got, want = got.cpu(), want.to(torch.bfloat16)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got.view(torch.int16)[~nan], want.view(torch.int16)[~nan])


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("what", [["inf"], ["-inf"], ["nan"], ["inf", "-inf"], ["inf", "inf", "nan"]])
def test_append_of_rows_with_infinities_and_nan(gpu, norm, what):
    """One such row of q, k or v per token, in dimensions of either half; what is stored, returned and read back."""
    dims = [[3], [70], [100, 36], [0, 64, 127]]  # 36 and 100, 0 and 64 are rotated with each other
    n = 3 * len(dims) + 1
    g = torch.Generator().manual_seed(len(what) + norm)
    x = torch.randn(n, HEADS + 2 * KV, D, generator=g)
    for i, at in enumerate(dims):
        for j, row in enumerate((1, HEADS, HEADS + KV + 1)):
            for d, value in zip(at, (what * 3)[:len(at)]):
                x[3 * i + j, row, d] = float(value)
    x = x.to(torch.bfloat16)
    table = pagedkv.rope_cos_sin(64, D, device="cpu")
    pos = torch.arange(n) * 3 % 61 + 1  # (at 0 the sines are 0)
    w = (torch.randn(D, generator=g) * 0.2 + 1).to(torch.bfloat16) if norm else None
    kc, vc = (torch.full((1, 64, ref.row_bytes(KV)), 7, dtype=torch.uint8, device=gpu) for _ in range(2))
    slots = torch.randperm(64, generator=g)[:n].to(torch.int32)
    wd = None if w is None else w.to(gpu)
    q, k, v = pagedkv.qk_norm_rope_store_fp4(x.view(n, -1).to(gpu), pos.to(gpu), table.to(gpu), HEADS, KV, D, wd, wd, 1e-6, kc, vc,
                                             slots.to(gpu), return_kv=True)
    _same(q, ref.norm_rope(x[:, :HEADS], w, 1e-6, pos, table))
    for cache, out, rows in ((kc, k, ref.norm_rope(x[:, HEADS:HEADS + KV], w, 1e-6, pos, table)), (vc, v, x[:, HEADS + KV:])):
        packed = ref.pack(rows)
        assert torch.equal(cache.cpu()[0, slots.long(), :68 * KV], packed)
        _same(out, ref.values(packed, KV))
        cu = torch.tensor([0, 64], dtype=torch.int32, device=gpu)
        back = pagedkv.gather_kv_fp4(cache, torch.zeros(1, 1, dtype=torch.int32, device=gpu), cu, 64, 64)
        _same(back[slots.long().to(gpu)], ref.values(packed, KV))


def test_what_an_infinity_leaves_of_a_normalised_row(gpu):
    """Its own dimension and the one that it is rotated with are NaN, the others 0; of the stored row their 32 each."""
    x = torch.ones(1, HEADS + 2 * KV, D)
    x[0, :, 40] = float("inf")
    table = pagedkv.rope_cos_sin(8, D, device=gpu)
    w = torch.ones(D, dtype=torch.bfloat16, device=gpu)
    kc, vc = (torch.zeros(1, 64, ref.row_bytes(KV), dtype=torch.uint8, device=gpu) for _ in range(2))
    q, k, v = pagedkv.qk_norm_rope_store_fp4(x.view(1, -1).to(torch.bfloat16).to(gpu), torch.full((1,), 5, device=gpu), table, HEADS, KV, D,
                                             w, w, 1e-6, kc, vc, torch.zeros(1, dtype=torch.int32, device=gpu), return_kv=True)
    bad = torch.zeros(D, dtype=torch.bool, device=gpu)
    bad[[40, 104]] = True
    assert torch.isnan(q[:, :, bad]).all() and (q[:, :, ~bad] == 0).all()
    blocks = bad.view(4, 32).any(1).repeat_interleave(32)
    assert torch.isnan(k[:, :, blocks]).all() and (k[:, :, ~blocks] == 0).all()
    assert torch.isnan(v[:, :, 32:64]).all() and (v[:, :, :32] == 1).all() and (v[:, :, 64:] == 1).all()
