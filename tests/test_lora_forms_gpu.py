"""The kernels' instantiations that the tests by size leave out, against the formula in 64 bits (same
bounds): the sorted shrink with 64 rows and two or three blocks of 16 columns a work-group, the projection
walking one or two chunks of k at a time with the adapters in its epilogue, and its partial sums beside a
shrink of 16 or 32 columns."""
import pytest
import torch

from test_lora_gpu import O, QKV, _add, _case, _check, _exact, _gpu, _linear

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,proj,rank,adapters,ids", [
    (12300, (64, (32, 32, 32)), 32, 5, "runs"),    # 64 rows, 3 blocks, twice (qkv at rank 32 from 12288 rows)
    (12300, (64, (32, 32)), 40, 3, "mixed"),       # the second time with an empty block
    (24700, (64, (32,)), 32, 4, "mixed"), (24700, (72, (32, 64)), 16, 3, "runs"),  # 64 rows, 2 blocks
    (2600, (520, (256, 64)), 16, 5, "mixed")])     # 32 rows, 2 blocks
def test_sorted_shrink(gpu, rows, proj, rank, adapters, ids):
    k, widths = proj
    c = _case(rows + rank, rows, k, widths, rank, adapters, ids)
    print(f"[lora_add] rows={rows} k={k} widths={widths} rank={rank}", flush=True)
    exact, loss = _exact(c, c["y"].double(), torch.zeros(rows, sum(widths), dtype=torch.float64), k)
    _check(_add(_gpu(c, gpu)), exact, loss, f"lora_add {rows} {proj} {rank}")


@pytest.mark.parametrize("rows,proj,rank,adapters", [
    (1, (256, (2048,)), 16, 3), (20, (256, (2048,)), 8, 3), (2, (512, (1024, 1024)), 16, 3),
    (50, (512, (1024, 1024)), 16, 3), (30, (768, (2048,)), 16, 3), (40, (1024, (2048, 32, 96)), 16, 9),
    (2, (1024, (32, 2048, 64)), 8, 9), (100, (512, (2048, 32)), 96, 12), (50, (512, (2048, 32)), 24, 4),
    (128, (256, (2048,)), 128, 40), (128, QKV, 64, 20), (128, O, 8, 3), (2, O, 16, 4), (33, O, 32, 9)])
def test_linear(gpu, rows, proj, rank, adapters):
    k, widths = proj
    c = _case(rows + rank, rows, k, widths, rank, adapters)
    c["ids"][0] = adapters - 1
    print(f"[lora_linear] rows={rows} k={k} widths={widths} rank={rank} adapters={adapters}", flush=True)
    x, w = c["x"].double(), c["w"].double()
    _check(_linear(_gpu(c, gpu)), *_exact(c, x @ w.T, x.abs() @ w.abs().T, k), f"lora_linear {rows} {proj} {rank}")
