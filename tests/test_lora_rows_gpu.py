"""What a row's bits depend on. lora_add: on nothing but the row itself, in any batch, sorted or not.
lora_linear: on the number of rows too, which picks the projection's K split (as in linear) and the
form that adds the adapters, but on no other row's values or adapters."""
import pytest
import torch

from test_lora_gpu import DOWN, GATE_UP, O, QKV, _add, _case, _gpu, _linear

pytestmark = pytest.mark.gpu


def _bits(t):
    return t.view(torch.int16)


@pytest.mark.parametrize("rank", [8, 24, 32, 64, 72, 128])
@pytest.mark.parametrize("rows", [100, 2600])
def test_add_row_alone_and_in_any_batch(gpu, rows, rank):
    d = _gpu(_case(rows + rank, rows, 520, (256, 64), rank, 5), gpu)
    print(f"[lora_add] rows={rows} rank={rank} alone / together / shuffled", flush=True)
    whole = _add(d)
    own = ("x", "y", "ids")
    for m in (0, 1, rows // 2, rows - 1):
        assert torch.equal(_bits(_add({n: d[n][m:m + 1] if n in own else d[n] for n in d})[0]), _bits(whole[m]))
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(rank)).to(gpu)
    mixed = {n: d[n][order] if n in own else d[n] for n in d}
    assert torch.equal(_bits(_add(mixed)), _bits(whole[order]))
    assert torch.equal(_bits(_add({n: mixed[n][:60] if n in own else mixed[n] for n in d})), _bits(whole[order[:60]]))


@pytest.mark.parametrize("rows,proj,rank", [
    (2, QKV, 16), (2, O, 16), (7, GATE_UP, 8), (40, QKV, 16), (40, QKV, 24), (17, O, 128), (128, DOWN, 64), (128, O, 8)])
def test_linear_row_beside_any_other_rows(gpu, rows, proj, rank):
    k, widths = proj
    c = _case(rows + rank, rows, k, widths, rank, 6)
    other = _case(rows + rank + 1, rows, k, widths, rank, 6)
    keep = torch.zeros(rows, dtype=torch.bool)
    keep[::3] = True
    changed = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in c.items()}
    for n in ("x", "ids"):
        changed[n][~keep] = other[n][~keep]
    changed["ids"][rows - 1] = 2 if not keep[rows - 1] else changed["ids"][rows - 1]
    print(f"[lora_linear] rows={rows} k={k} rank={rank} other rows", flush=True)
    a, b = _linear(_gpu(c, gpu)).cpu(), _linear(_gpu(changed, gpu)).cpu()
    assert torch.equal(_bits(a[keep]), _bits(b[keep]))
    assert not torch.equal(_bits(a[~keep]), _bits(b[~keep]))
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(rank))
    shuffled = {n: t[order] if n in ("x", "ids") else t for n, t in c.items()}
    assert torch.equal(_bits(_linear(_gpu(shuffled, gpu)).cpu()), _bits(a[order]))
