"""GPU tests of attention over 4-bit caches for more sequences than a work-group has in LDS, 1024 at a time in groups of
64: sequences of both kinds on either side of these borders, and stretches of them without any work."""
import pytest
import torch

from test_fp4_attention_gpu import _case, _check, _run

pytestmark = pytest.mark.gpu


def _attend(gpu, lens, heads, kv, seed):
    c = _case(gpu, heads, kv, lens, seed=seed)
    out = torch.zeros_like(c["q"])
    _run(c, out=out)
    _check(c, out)
    return out


@pytest.mark.parametrize("n", [1023, 1024, 1025, 2048, 2100])
@pytest.mark.parametrize("heads,kv", [(4, 2), (8, 1)])
def test_both_kinds_on_either_side_of_the_borders(gpu, n, heads, kv):
    g = torch.Generator().manual_seed(n)
    lens = [(1, int(k)) for k in torch.randint(0, 70, (n,), generator=g)]
    special = [(70, 90), (3, 200), (150, 300), (33, 33), (0, 40), (1, 700), (20, 500), (90, 90), (2, 0)]
    for i, at in enumerate((0, 63, 64, 65, 1022, 1023, 1024, 1025, 1087, 1088, 2047, 2048, 2049, n - 1)):
        if at < n:
            lens[at] = special[(i + n) % len(special)]
    _attend(gpu, lens, heads, kv, n)


@pytest.mark.parametrize("many", [True, False])
@pytest.mark.parametrize("where", [[0, 1023], [1024], [2047, 2048], [64, 3000]])
def test_work_between_stretches_without_any(gpu, where, many):
    """All sequences of some chunks are empty, or of the other kind: lookups go past them, and back for the next head."""
    lens = [(0, 0)] * 3100
    for at in where:
        lens[at] = (90, 333) if many else (1, 800)
    _attend(gpu, lens, 8, 4, len(where))
    other = [(1, 5) if many else (20, 20) if i % 400 == 7 else (0, 9) for i in range(3100)]
    for at in where:
        other[at] = (90, 333) if many else (1, 800)
    _attend(gpu, other, 8, 4, len(where) + 10)
