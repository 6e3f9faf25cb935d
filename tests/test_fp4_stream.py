"""CPU check of the built code of the attention over 4-bit caches. Its loads to LDS are inline assembly, of which the
compiler knows neither that they use M0 nor that a scalar base written by a vector instruction (a value read back from a
lane, a spilled one among them) may be used by a vector load 5 wait states later at the earliest."""
import re

import pytest

from test_prefill_stream import _code, kernels  # noqa: F401

BASE_STATES = 5
_SGPR = re.compile(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b|\b(vcc)\b")
_TWO_RESULTS = re.compile(r"_co_|div_scale|mad_[ui]64")


def _sgprs(text):
    out = set()
    for lo, hi, one, vcc in _SGPR.findall(text):
        out |= {vcc} if vcc else {int(one)} if one else set(range(int(lo), int(hi) + 1))
    return out


def _operands(text):
    return [o.strip() for o in re.split(r",(?![^\[]*\])", text.partition(" ")[2])]


def check_m0(code):
    """M0 is set only right before a load to LDS, by the load's own instructions, and used by nothing else."""
    bad = []
    for i, (_, text, _) in enumerate(code):
        if re.search(r"\bm0\b", text) and not text.startswith("s_mov_b32 m0, "):
            bad.append(text)
        loads = i + 2 < len(code) and code[i + 1][1].startswith("s_nop") and code[i + 2][1].startswith("global_load_lds_dword")
        if text.startswith("s_mov_b32 m0, ") and not loads:
            bad.append(text + " without its load")
        if "load_lds" in text and not (i >= 2 and code[i - 2][1].startswith("s_mov_b32 m0, ")):
            bad.append(text + " without its M0")
    return bad


def check_bases(code):
    """The loads to LDS whose scalar base a vector instruction wrote fewer than 5 wait states ago, along any path."""
    at = {a: i for i, (a, _, _) in enumerate(code)}
    come = {}
    for i, (_, _, target) in enumerate(code):
        if target is not None:
            come.setdefault(at[target], []).append(i)
    bad = []
    for i, (_, text, _) in enumerate(code):
        if "load_lds" not in text:
            continue
        base = _sgprs(_operands(text)[1])
        work, seen = [(i, 0)], set()
        while work:
            j, states = work.pop()
            before = list(come.get(j, []))
            if j and not re.match(r"s_branch|s_endpgm|s_setpc", code[j - 1][1]):
                before.append(j - 1)
            for k in before:
                op = code[k][1]
                if op.startswith("v_"):
                    if _sgprs(" ".join(_operands(op)[:2 if _TWO_RESULTS.search(op) else 1])) & base:
                        bad.append(f"{op}, {states} states before {text}")
                n = states + (int(op.split()[1], 0) + 1 if op.startswith("s_nop") else 1)
                if n < BASE_STATES and (k, n) not in seen:
                    seen.add((k, n))
                    work.append((k, n))
    return bad


@pytest.mark.parametrize("wanted,count", [("17attend_few_kernelI", 4), ("19attend_mixed_kernelI", 4)])
def test_loads_to_lds(kernels, wanted, count):  # noqa: F811
    found = kernels(wanted)
    assert len(found) == count
    for name, code in found.items():
        assert sum("load_lds" in t for _, t, _ in code) >= 15, name
        assert not check_m0(code), name
        assert not check_bases(code), name


LOAD = "s_mov_b32 m0, s9\ns_nop 0\nglobal_load_lds_dword v1, s[2:3]\n"


def test_planted_m0_uses_are_found():
    assert not check_m0(_code(LOAD + "s_endpgm"))
    assert check_m0(_code(LOAD + "s_mov_b32 s4, m0\ns_endpgm"))
    assert check_m0(_code("global_load_lds_dwordx4 v1, s[2:3]\ns_endpgm"))
    assert check_m0(_code("s_mov_b32 m0, s9\nglobal_load_lds_dwordx4 v1, s[2:3]\ns_endpgm"))
    assert check_m0(_code("s_mov_b32 m0, -1\nv_nop\nv_nop\ns_endpgm"))


@pytest.mark.parametrize("text,bad", [
    ("v_readlane_b32 s3, v5, 1\n" + LOAD, 1), ("v_readfirstlane_b32 s2, v5\ns_nop 1\n" + LOAD, 1),
    ("v_readfirstlane_b32 s2, v5\ns_nop 2\n" + LOAD, 0), ("v_readlane_b32 s4, v5, 1\n" + LOAD, 0),
    ("v_add_co_u32_e64 v0, s[2:3], v1, v2\n" + LOAD, 1), ("v_cmp_gt_i32_e64 s[2:3], v1, v2\n" + LOAD, 1),
    ("v_mov_b32_e32 v0, s2\n" + LOAD, 0), ("s_mov_b32 s2, s4\n" + LOAD, 0),
    # only along the back edge of a loop
    ("s_nop 0\n" + LOAD + "v_readlane_b32 s2, v5, 1\ns_cbranch_scc1 1 -> 1\n", 1),
    ("s_nop 0\n" + LOAD + "v_readlane_b32 s2, v5, 1\ns_nop 1\ns_cbranch_scc1 1 -> 1\n", 0),
    # not past an end
    ("v_readlane_b32 s2, v5, 1\ns_branch 5 -> 5\n" + LOAD + "s_endpgm\n", 0)])
def test_planted_bases_are_found(text, bad):
    assert len(check_bases(_code(text + "s_endpgm"))) == bad
