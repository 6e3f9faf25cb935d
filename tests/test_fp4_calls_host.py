"""CPU tests of what the 4-bit cache's wrappers hand to the C entry points, and of calls that they have to refuse."""
import pytest
import torch

import fp4_oracle as ref
import pagedkv
from pagedkv import _lib, fp4
from test_fp4_host import SPACE, UNSUPPORTED, _call

KV, HEADS, BS, NB = 8, 16, 64, 4


def _attention(table, num_seqs=4, max_k=150):
    c = torch.zeros(NB, BS, ref.row_bytes(KV), dtype=torch.uint8)
    cu = torch.arange(num_seqs + 1, dtype=torch.int32)
    return pagedkv.varlen_attention_fp4(torch.zeros(num_seqs, HEADS, 128, dtype=torch.bfloat16), c, c.clone(), cu, cu, 1, max_k, table)


def _gather(table, num_seqs=4, max_k=150):
    c = torch.zeros(NB, BS, ref.row_bytes(KV), dtype=torch.uint8)
    return pagedkv.gather_kv_fp4(c, table, torch.arange(num_seqs + 1, dtype=torch.int32), max_k, num_seqs)


@pytest.fixture
def handed(monkeypatch):
    """The arguments that reach the C entry points, by entry point, which are not called."""
    out = {}
    monkeypatch.setattr(fp4, "call", lambda fn, what, device, *args: out.__setitem__(what, args))
    return out


@pytest.mark.parametrize("op", [_attention, _gather])
def test_tables_whose_rows_overlap_are_refused(handed, op):
    """An expanded table has the storage of one row: stepping from row to row by its width would leave it."""
    one = torch.zeros(1, 3, dtype=torch.int32)
    for table in (one.expand(4, 3), one[0].expand(4, 3), torch.zeros(9, dtype=torch.int32).as_strided((4, 3), (2, 1))):
        with pytest.raises(ValueError, match="entries apart"):
            op(table)
    assert not handed


@pytest.mark.parametrize("op,what,at", [(_attention, "pk_varlen_attention_fp4", 9), (_gather, "pk_gather_kv_fp4", 7)])
def test_row_strides_of_tables(handed, op, what, at):
    """The stride that a table has is the one that is handed over, rows that overlap behind max_seqlen_k among them."""
    wide = torch.zeros(4, 9, dtype=torch.int32)
    for table, stride in ((wide, 9), (wide[:, 2:5], 9), (wide[:, :3].contiguous(), 3),
                          (torch.zeros(20, dtype=torch.int32).as_strided((4, 5), (4, 1)), 4)):
        op(table)
        assert handed[what][at - 1] == table.data_ptr() and handed[what][at] == stride
    op(torch.zeros(1, 3, dtype=torch.int32).expand(4, 3), num_seqs=1)  # one sequence steps nowhere
    assert handed[what][at] == 3


@pytest.mark.parametrize("heads,kv,slots", [(16, 8, 8), (8, 4, 4), (3, 3, 4), (2, 2, 2), (4, 1, 1), (22, 11, 1), (24, 12, 8)])
def test_most_steps_of_single_rows(heads, kv, slots):
    """The largest max_seqlen_k for 65535 sequences passes the check of the steps, one step more does not, and the
    message has the numbers."""
    step = 256 // slots
    most = min((2 ** 31 - 1) // 65535 * step, 65535 * 64)
    row = ref.row_bytes(kv)
    kw = dict(num_seqs=65535, rows=65535, heads=heads, kv=kv, q_stride=128 * heads, out_stride=128 * heads, k_block=64 * row,
              v_block=64 * row, table_stride=65535, ws_bytes=0)
    assert _call("pk_varlen_attention_fp4", **kw, max_k=most) == SPACE, _lib.lib().pk_last_error()
    if most < 65535 * 64:
        assert _call("pk_varlen_attention_fp4", **kw, max_k=most + 1) == UNSUPPORTED
        count = 65535 * (most // step + 1)
        assert count >= 2 ** 31 and f"{count} steps of {step} keys".encode() in _lib.lib().pk_last_error()


@pytest.mark.parametrize("group", [2, 8])
def test_most_steps_of_more_rows(group):
    """Steps of 64 keys of one kv head: tiles of 256 columns, and one more for every sequence."""
    kw = dict(num_seqs=100, max_q=1 << 21, heads=group, kv=1, q_stride=128 * group, out_stride=128 * group, k_block=64 * 80,
              v_block=64 * 80, table_stride=65535, max_k=65535 * 64, ws_bytes=0)
    tiles = (2 ** 31 - 1) // 65535
    rows = (tiles - 100 + 1) * 256 // group - 1
    assert _call("pk_varlen_attention_fp4", **kw, rows=rows) == SPACE, _lib.lib().pk_last_error()
    assert _call("pk_varlen_attention_fp4", **kw, rows=rows + 1) == UNSUPPORTED
    assert f"{(tiles + 1) * 65535} steps of 64 keys".encode() in _lib.lib().pk_last_error()


def test_how_far_a_stored_value_is_off():
    """Every finite bf16 value as the largest of its 32, beside values between it and 0: at most a fifth of it, or 2^-128
    where the scale can get no smaller; a quarter where the scale can get no larger. Both ends reach beyond a fifth."""
    every = torch.arange(1, 0x7f80, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    x = (every.double().unsqueeze(1) * torch.linspace(1, -1, 128, dtype=torch.float64)).to(torch.bfloat16)
    # (the four blocks of a row have different largest values)
    off = (ref.values(ref.pack(x.unsqueeze(1)), 1).squeeze(1) - x.double()).abs().view(-1, 4, 32)
    top = x.double().abs().view(-1, 4, 32).amax(-1, keepdim=True)
    end = top > 7 * 2.0 ** 125
    assert (off <= torch.where(end, top / 4, torch.maximum(top / 5, torch.tensor(2.0 ** -128, dtype=torch.float64)))).all()
    assert (off[end.expand_as(off)] > 0.24 * top.expand_as(off)[end.expand_as(off)]).any()
    small = top < 2.0 ** -128
    assert (off == x.double().abs().view(-1, 4, 32))[small.expand_as(off)].all() and small.any()


@pytest.mark.parametrize("n,kv", [(1, 2), (3, 1), (1, 1)])
def test_strides_of_single_rows_and_heads_do_not_count(handed, n, kv):
    """A dimension of size one may have any stride: rows are taken that only differ in it."""
    row = kv * 128
    caches = [torch.zeros(NB, BS, ref.row_bytes(kv), dtype=torch.uint8) for _ in range(2)]
    slots = torch.zeros(n, dtype=torch.int32)
    shape, stride = (n, kv, 128), (row + 132 if n == 1 else 2 * row, 300 if kv == 1 else 128, 1)
    rows = torch.zeros(4096, dtype=torch.bfloat16).as_strided(shape, stride)
    assert rows.stride() == stride
    pagedkv.store_kvcache_fp4(rows, rows, *caches, slots)
    assert handed["pk_store_kvcache_fp4"][1] == handed["pk_store_kvcache_fp4"][3] == (row if n == 1 else 2 * row)
    q = torch.zeros(1 << 26, dtype=torch.bfloat16).as_strided((n, kv, 128), (1 << 25 if n == 1 else 2 * row, stride[1], 1))
    cu = torch.arange(n + 1, dtype=torch.int32)
    pagedkv.varlen_attention_fp4(q, *caches, cu, cu, 1, 10, torch.zeros(n, 1, dtype=torch.int32))
    assert handed["pk_varlen_attention_fp4"][1] == (row if n == 1 else 2 * row)
    if kv > 1:
        with pytest.raises(ValueError, match="contiguous heads"):
            pagedkv.store_kvcache_fp4(rows.as_strided(shape, (row, 136, 1)), rows, *caches, slots)
