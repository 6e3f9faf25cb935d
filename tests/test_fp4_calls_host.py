"""CPU tests of what the 4-bit cache's wrappers hand to the C entry points, and of calls that they have to refuse."""
import pytest
import torch

import fp4_oracle as ref
import pagedkv
from pagedkv import fp4

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
