"""GPU tests of attention over 4-bit caches whose V rows go up to the format's largest values: sums of p V leave the
range of fp32 nowhere where their mean does not."""
import pytest
import torch

import fp4_oracle as ref
import pagedkv
from test_fp4_attention_gpu import D, _case, _run

pytestmark = pytest.mark.gpu


def _raise_v(c, heads, by, rows=None):
    """V's scale bytes `by` higher (at most 252) for some kv heads, in all rows or in the rows that a mask (NB, BS) selects."""
    kv = c["vc"].shape[-1] // 68
    for h in heads:
        part = c["vc"][..., 64 * kv + 4 * h:64 * kv + 4 * h + 4]
        up = (part.int() + by).clamp(max=252).to(torch.uint8)
        part.copy_(up if rows is None else torch.where(rows.unsqueeze(-1), up, part))


def _check(c, got, scale=D ** -0.5):
    """As test_fp4_attention_gpu's, with what the larger reference costs: weights and sums are held relative to a
    largest weight of at least 2^-32, so what vanishes below fp32's smallest normal value, 2^-126, is up to 2^-94 of
    max |v| a key. And with the weights' rounding in the sum below: p (1 + d), |d| <= 2^-8, moves o = sum p v / sum p by
    sum d p (v - o) / sum p, at most 2^-8 (A + |o|). One key's V far above the others' comes near to that: of two keys
    with weights w and 1 - w and V only at the first, 2^-7 |o| (1 - w)."""
    want, bound = ref.attention(c["q"], c["kc"], c["vc"], c["tables"], c["q_lens"], c["k_lens"], scale)
    top = ref.values(c["vc"], c["vc"].shape[-1] // 68).abs().amax()
    bound = bound + 2.0 ** -94 * max(c["k_lens"]) * top + 2.0 ** -8 * want.abs()
    over = (got.double() - want).abs() - bound
    assert torch.isfinite(got).all()
    assert over.max().item() <= 0, f"over the bound by {over.max().item():.3e} at {int(over.argmax())}"


LENS = {"single": [(1, 64), (1, 1), (1, 700), (1, 6000), (1, 130)],
        "few": [(2, 300), (8, 1000), (3, 3), (5, 64)],
        "many": [(17, 17), (200, 456), (130, 1500), (64, 64)],
        "mixed": [(1, 500), (90, 400), (2, 70), (40, 40), (1, 3000)]}


@pytest.mark.parametrize("kind", list(LENS))
@pytest.mark.parametrize("by", [60, 64, 66, 98, 126])
def test_values_of_any_magnitude(gpu, kind, by):
    c = _case(gpu, 16, 8, LENS[kind], seed=by)
    _raise_v(c, range(8), by)
    _check(c, _run(c))


@pytest.mark.parametrize("kind", list(LENS))
@pytest.mark.parametrize("heads,kv", [(16, 8), (8, 1), (8, 4), (2, 2)])
def test_some_rows_and_heads_are_large(gpu, kind, heads, kv):
    """Large rows that come late, early or here and there, beside heads that have none."""
    for which in range(3):
        c = _case(gpu, heads, kv, LENS[kind], seed=which)
        at = torch.arange(c["vc"].shape[0] * 64, device=gpu).view(-1, 64)
        rows = [at % 64 >= 60, at % 64 < 3, at % 397 == 5][which]
        _raise_v(c, range(0, kv, 2), 126, rows)
        _check(c, _run(c))


@pytest.mark.parametrize("kind", list(LENS))
def test_large_values_under_scores_that_grow(gpu, kind):
    """References that move by hundreds on the way, before and after the first large row."""
    for scale in (1.0, 4.0):
        c = _case(gpu, 8, 4, LENS[kind], seed=3)
        for i, (_, n) in enumerate(zip(c["q_lens"], c["k_lens"])):
            for j in range(-(-n // 64)):
                c["kc"][int(c["tables"][i, j]), :, 64 * 4:68 * 4] = 124 + min(4, j // 2)
        at = torch.arange(c["vc"].shape[0] * 64, device=gpu).view(-1, 64)
        _raise_v(c, range(4), 126, at % 64 >= 40)
        _check(c, _run(c, softmax_scale=scale), scale)


def test_what_is_not_large_keeps_its_bits(gpu):
    """Heads without large rows, and the other sequences of the call, are computed as they are without them."""
    lens = [(1, 900), (1, 700), (60, 500), (4, 300)]
    c = _case(gpu, 8, 4, lens, seed=5)
    want = _run(c)
    large = torch.zeros(c["vc"].shape[:2], dtype=torch.bool, device=gpu)
    for i in (0, 2):
        large[c["tables"][i, :-(-lens[i][1] // 64)].long()] = True
    _raise_v(c, [1], 126, large)
    got = _run(c)
    _check(c, got)
    same = torch.ones(c["q"].shape[:2], dtype=torch.bool, device=gpu)
    same[0, 2:4] = same[2:62, 2:4] = False
    assert torch.equal(got[same], want[same])


def test_lengths_that_overlap_have_no_more_steps_than_a_call(gpu):
    """Lengths that fall and rise again, so that 656 sequences have the same 6400 rows: their 2^32 + 4194304 steps
    are no small number of steps (2^32 is 0 in 32 bits), and nothing is computed. Without a block no key is read."""
    n, heads, pairs, keys = 6400, 8, 656, 1 << 21
    assert pairs * (n * heads // 256) * (keys // 64) == 2 ** 32 + 4194304
    cache = torch.zeros(1, keys, 80, dtype=torch.uint8, device=gpu)  # one page holds all keys
    q = torch.zeros(n, heads, D, dtype=torch.bfloat16, device=gpu)
    out = torch.full_like(q, 7.0)
    cu_q = torch.tensor([0, n] * pairs + [0], dtype=torch.int32, device=gpu)
    cu_k = torch.tensor([0, keys] * pairs + [0], dtype=torch.int32, device=gpu)
    table = torch.full((2 * pairs, 1), -1, dtype=torch.int32, device=gpu)
    pagedkv.varlen_attention_fp4(q, cache, cache, cu_q, cu_k, n, keys, table, causal=False, out=out)
    torch.cuda.synchronize()
    assert (out == 7).all()
    # one of them alone: its rows see no key
    pagedkv.varlen_attention_fp4(q[:64], cache, cache, cu_q[:2].clamp(max=64), cu_k[:2].clamp(max=640), 64, keys, table[:1],
                                 causal=False, out=out[:64])
    assert (out[:64] == 0).all() and (out[64:] == 7).all()


def test_two_keys_of_which_one_has_all_the_value(gpu):
    """V of one of two keys is 0: the roundings of both weights move what is left of the other."""
    n = 512
    c = _case(gpu, 16, 8, [(1, 2)] * n, seed=8)
    kv = 8
    for i in range(n):
        c["vc"][int(c["tables"][i, 0]), 0, :64 * kv] = 0
    _raise_v(c, range(4), 126)
    _check(c, _run(c))
