"""Infinities and NaN in the inputs of lora_linear and lora_add, in each of their forms: results that such a
value does not reach keep their bits, those that it reaches are NaN, +inf or -inf as the formula in 64 bits
is. The one exception is an infinite element of lora_b, for which NaN may stand where the formula has an
infinity (t is multiplied in two parts of either sign, or with a part of 0): not finite is all that is said."""
import pytest
import torch

import pagedkv
from test_lora_gpu import DOWN, GATE_UP, O, QKV, _add, _case, _exact, _gpu, _linear

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def _set(name, index, value):
    def change(c):
        c[name][index] = value
    return change


# what is changed (row 0 has adapter 2, row 1 none), and whether an operator has it
ROWS = [("x[0] nan", _set("x", 0, NAN)), ("x[0, 5] inf", _set("x", (0, 5), INF)), ("x[1, 5] -inf", _set("x", (1, 5), -INF)),
        ("x[1] nan", _set("x", 1, NAN))]
ADAPTERS = [("a inf", _set("a", (2, 3, 5), INF)), ("a nan", _set("a", (2, 3, 5), NAN)), ("b nan", _set("b", (2, 30, 1), NAN)),
            ("scale inf", _set("scales", 2, INF)), ("scale -inf", _set("scales", 2, -INF)), ("scale nan", _set("scales", 2, NAN)),
            ("unused adapter", _set("b", 4, NAN))]
LINEAR = [("w inf", _set("w", (9, 7), INF)), ("w nan", _set("w", (9, 7), NAN))]
ADD = [("y -inf", _set("y", (0, 9), -INF)), ("y nan", _set("y", (1, 9), NAN))]


def _inputs(rows, k, widths, rank):
    c = _case(rows + rank, rows, k, widths, rank, 5)
    c["ids"][c["ids"] == 4] = 3
    c["ids"][0], c["ids"][1] = 2, -1
    return c


def _kind(t):
    """0 finite, 1 +inf, 2 -inf, 3 NaN"""
    return t.isposinf() + 2 * t.isneginf() + 3 * t.isnan()


def _check(run, base, make, k, changes, gpu, what):
    clean = run(_gpu(make(), gpu)).cpu()
    assert clean.isfinite().all()
    for name, change in changes:
        print(f"[lora] {what} {name}", flush=True)
        c = make()
        change(c)
        got = run(_gpu(c, gpu)).cpu()
        want = _kind(_exact(c, base(c), torch.zeros(1, dtype=torch.float64), k)[0])
        assert torch.equal(_kind(got.double()), want), f"{what} {name}"
        keep = want == 0
        assert torch.equal(got[keep].view(torch.int16), clean[keep].view(torch.int16)), f"{what} {name}"
    for value in (INF, -INF):
        print(f"[lora] {what} b {value}", flush=True)
        c = make()
        c["b"][2, 30, 1] = value
        got = run(_gpu(c, gpu)).cpu()
        reached = torch.zeros_like(got, dtype=torch.bool)
        reached[c["ids"] == 2, 30] = True
        assert not got[reached].isfinite().any()
        assert torch.equal(got[~reached].view(torch.int16), clean[~reached].view(torch.int16))


# scratch: none (one launch), t alone (a shrink before it), or t and partial sums
@pytest.mark.parametrize("rows,proj,rank,scratch", [
    (2, QKV, 16, "none"), (2, GATE_UP, 8, "none"), (40, QKV, 16, "t"), (2, O, 16, "partial"), (40, QKV, 24, "partial"),
    (128, DOWN, 64, "partial"), (17, O, 128, "partial")])
def test_linear(gpu, rows, proj, rank, scratch):
    k, widths = proj
    need = pagedkv.lora_workspace_bytes(rows, sum(widths), k, rank, widths, linear=True)
    t = rows * len(widths) * rank * 4
    assert (need == 0) == (scratch == "none") and (need == t) == (scratch == "t")
    _check(_linear, lambda c: c["x"].double() @ c["w"].double().T, lambda: _inputs(rows, k, widths, rank), k,
           ROWS + ADAPTERS + LINEAR, gpu, f"linear rows={rows} k={k} rank={rank}")


# scratch: none (one launch), t alone (two), or what a sort needs too
@pytest.mark.parametrize("rows,proj,rank,scratch", [
    (40, O, 16, "none"), (33, QKV, 32, "none"), (400, QKV, 16, "t"), (200, QKV, 40, "t"), (2700, (512, (64, 64)), 16, "sort"),
    (2500, (264, (96, 64)), 72, "sort")])
def test_add(gpu, rows, proj, rank, scratch):
    k, widths = proj
    need = pagedkv.lora_workspace_bytes(rows, sum(widths), k, rank, widths, 5)
    t = rows * len(widths) * rank * 4
    assert (need == 0) == (scratch == "none") and (need == t) == (scratch == "t")
    _check(_add, lambda c: c["y"].double(), lambda: _inputs(rows, k, widths, rank), k, ROWS + ADAPTERS + ADD, gpu,
           f"add rows={rows} k={k} rank={rank}")


@pytest.mark.parametrize("op,rows,rank", [
    ("linear", 2, 16), ("linear", 40, 16), ("linear", 40, 24), ("linear", 40, 128), ("add", 40, 16), ("add", 33, 32),
    ("add", 200, 40), ("add", 2700, 16), ("add", 2700, 128)])
def test_t_beyond_the_largest_bf16(gpu, op, rows, rank):
    """t = 3.4e38 fits fp32 but rounds to an infinity in bf16 (largest value 3.39e38): a tiny B brings it back
    to an ordinary number, in every form. Every product but one is 0, so fp32 sums lose nothing:
    half a bf16 step of the output and t's 2^-16."""
    k, widths = 1024, (2048, 1024, 1024)
    c = _case(1, rows, k, widths, rank, 3)
    for name in ("x", "w", "y", "a", "b"):
        c[name].zero_()
    c["ids"].fill_(1)
    c["ids"][1:] = torch.randint(-1, 3, (rows - 1,), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    c["x"][:, 9], c["a"][:, 3, 9] = 1.0, 1.0
    c["x"][rows // 2:, 9] = -1.0
    c["b"][:, :, 3] = 2.0 ** -126
    c["scales"].fill_(3.4e38)
    assert c["scales"].isfinite().all() and c["scales"].to(torch.bfloat16).isinf().all()
    want = _exact(c, torch.zeros(rows, sum(widths), dtype=torch.float64), torch.zeros(1, dtype=torch.float64), k)[0]
    assert want[c["ids"] >= 0, :2048].abs().min() > 3.9
    print(f"[lora] {op} rows={rows} rank={rank} large t", flush=True)
    got = (_linear if op == "linear" else _add)(_gpu(c, gpu)).cpu().double()
    assert ((got - want).abs() <= (2.0 ** -8 + 2.0 ** -16) * want.abs()).all()
