"""CPU tests of the page operators' refusals: the C entry points return before any GPU work, the
Python wrappers raise before they call them."""
import ctypes

import pytest
import torch

import pagedkv
from pagedkv import _lib
from pool_oracle import Pool, make_pool

BUF = (ctypes.c_char * 4096)()
PTR = (ctypes.addressof(BUF) + 255) // 256 * 256


def _call(name, **kw):
    row = 8 * 128
    cache = dict(k=PTR, v=PTR, kl=0, vl=0, kb=256 * row, vb=256 * row, layers=1, blocks=4, bs=256, row=row)
    pool = dict(tables=PTR, stride=4, rows=2, width=4, lens=PTR, refs=PTR)
    args = {
        "pk_copy_blocks": dict(**cache, src=PTR, dst=PTR, tok=None, pairs=0, stream=None),
        "pk_fork_sequences": dict(**cache, **pool, parents=PTR, children=PTR, n=0, new=PTR, ws=PTR, ws_bytes=4096,
                                  stream=None),
        "pk_extend_sequences": dict(**pool, blocks=4, bs=256, list=PTR, n=0, slots=PTR, stream=None),
        "pk_free_sequences": dict(**pool, blocks=4, bs=256, list=PTR, n=0, stream=None),
        "pk_compact_blocks": dict(**cache, **pool, map=PTR, live=PTR, ws=PTR, ws_bytes=4096, stream=None),
    }[name]
    assert set(kw) <= set(args), kw
    args.update(kw)
    return getattr(_lib.lib(), name)(*args.values())


CACHE = ["pk_copy_blocks", "pk_fork_sequences", "pk_compact_blocks"]
POOL = ["pk_fork_sequences", "pk_extend_sequences", "pk_free_sequences", "pk_compact_blocks"]


@pytest.mark.parametrize("name", CACHE)
@pytest.mark.parametrize("kw,code", [
    (dict(k=None), _lib.PK_ERR_INVALID_ARG), (dict(v=PTR + 2), _lib.PK_ERR_INVALID_ARG),
    (dict(layers=0), _lib.PK_ERR_INVALID_ARG), (dict(blocks=-1), _lib.PK_ERR_INVALID_ARG),
    (dict(bs=0), _lib.PK_ERR_INVALID_ARG), (dict(row=12), _lib.PK_ERR_UNSUPPORTED),
    (dict(kb=256 * 1024 - 8), _lib.PK_ERR_INVALID_ARG), (dict(vb=256 * 1024 + 4), _lib.PK_ERR_INVALID_ARG),
    (dict(layers=2), _lib.PK_ERR_INVALID_ARG),      # layers on top of each other
    (dict(row=2 ** 24, kb=2 ** 40, vb=2 ** 40), _lib.PK_ERR_UNSUPPORTED),
])
def test_cache_refusals(name, kw, code):
    assert _call(name, **kw) == code
    assert name[3:].encode() in _lib.lib().pk_last_error()


@pytest.mark.parametrize("name", POOL)
@pytest.mark.parametrize("kw", [dict(tables=None), dict(stride=3), dict(rows=-1), dict(width=-1), dict(lens=None),
                                dict(refs=None), dict(blocks=0), dict(bs=0)])
def test_pool_refusals(name, kw):
    assert _call(name, **kw) == _lib.PK_ERR_INVALID_ARG


def test_list_refusals():
    assert _call("pk_copy_blocks", pairs=-1) == _lib.PK_ERR_INVALID_ARG
    assert _call("pk_copy_blocks", pairs=1, src=None) == _lib.PK_ERR_INVALID_ARG
    assert _call("pk_copy_blocks", pairs=2 ** 31 - 1) == _lib.PK_ERR_UNSUPPORTED  # pieces past 32 bits
    for name in ("pk_fork_sequences", "pk_extend_sequences"):
        assert _call(name, n=-1) == _lib.PK_ERR_INVALID_ARG
        assert _call(name, n=1025) == _lib.PK_ERR_UNSUPPORTED
    assert _call("pk_free_sequences", n=-1) == _lib.PK_ERR_INVALID_ARG
    assert _call("pk_free_sequences", n=2 ** 24 + 1) == _lib.PK_ERR_UNSUPPORTED
    assert _call("pk_fork_sequences", n=1, parents=None) == _lib.PK_ERR_INVALID_ARG
    assert _call("pk_extend_sequences", n=1, slots=None) == _lib.PK_ERR_INVALID_ARG
    assert _call("pk_extend_sequences", blocks=2 ** 24) == _lib.PK_ERR_UNSUPPORTED  # slots past 31 bits
    for name in ("pk_extend_sequences", "pk_free_sequences"):                       # steps over blocks past 31 bits
        assert _call(name, blocks=2 ** 30 + 1, bs=1) == _lib.PK_ERR_UNSUPPORTED
        assert _call(name, blocks=2 ** 30, bs=1) == _lib.PK_OK
    assert _call("pk_free_sequences", n=1, list=None) == _lib.PK_ERR_INVALID_ARG
    assert _call("pk_compact_blocks", map=None) == _lib.PK_ERR_INVALID_ARG
    need = _lib.lib().pk_fork_workspace_bytes(8)
    assert _call("pk_fork_sequences", n=8, ws_bytes=need - 1) == _lib.PK_ERR_WORKSPACE
    assert _call("pk_fork_sequences", n=8, ws=PTR + 4) == _lib.PK_ERR_WORKSPACE
    assert _call("pk_compact_blocks", ws_bytes=_lib.lib().pk_compact_workspace_bytes(4) - 1) == _lib.PK_ERR_WORKSPACE
    # nothing listed: success without touching a pointer
    for name in ("pk_copy_blocks", "pk_fork_sequences", "pk_extend_sequences", "pk_free_sequences"):
        assert _call(name) == _lib.PK_OK


def test_python_refusals():
    k, v = torch.zeros(2, 4, 8, 1, 8, dtype=torch.bfloat16), torch.zeros(2, 4, 8, 1, 8, dtype=torch.bfloat16)
    t, ln = torch.full((3, 2), -1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    rc = torch.zeros(4, dtype=torch.int32)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="one GPU"):
        pagedkv.copy_blocks(k, v, one, one)
    with pytest.raises(ValueError, match="caches"):
        pagedkv.copy_blocks(k, v[:1], one, one)
    with pytest.raises(TypeError, match="16-bit"):
        pagedkv.copy_blocks(k.float(), v.float(), one, one)
    with pytest.raises(TypeError, match="int32"):
        pagedkv.extend_sequences(t.long(), ln, rc, 8, one)
    with pytest.raises(ValueError, match="one length per row"):
        pagedkv.extend_sequences(t, ln[:2], rc, 8, one)
    with pytest.raises(ValueError, match="contiguous"):
        pagedkv.free_sequences(t, ln, rc, 8, torch.zeros(4, dtype=torch.int32)[::2])
    with pytest.raises(ValueError, match="contiguous rows"):
        pagedkv.free_sequences(t.t(), ln[:2], rc, 8, one)
    with pytest.raises(ValueError, match="on a GPU"):
        pagedkv.extend_sequences(t, ln, rc, 8, one)


def test_oracle_pool_by_hand():
    """The oracle itself: a fork of 5 tokens in pages of 4, its growth, the parent freed, compaction."""
    tables, lens, refs, k, v = make_pool(0, [5, 0], 4, 6, 3)
    p = Pool(tables, lens, refs, k, v, 4)
    a, b = p.tables[0][:2]
    new = p.fork([0], [1])[0]
    assert new == min(set(range(6)) - {a, b}) and p.refs[a] == 2 and p.refs[b] == 1 and p.refs[new] == 1
    assert p.tables[1] == [a, new, -1] and p.lens == [5, 5]
    assert torch.equal(p.k[:, new, 0], p.k[:, b, 0]) and torch.equal(p.k[:, new, 1:], k[:, new, 1:])
    assert p.extend([1]) == [new * 4 + 1] and p.lens == [5, 6]
    p.free([0])
    assert p.refs[a] == 1 and p.refs[b] == 0 and p.tables[0] == [-1, -1, -1]
    kept = p.k[:, a].clone()
    block_map, live = p.compact()
    assert live == 2 and sorted(p.tables[1][:2]) == [0, 1] and p.refs[:3] == [1, 1, 0]
    assert torch.equal(p.k[:, block_map[a]], kept)
