"""CPU tests of the per-row adapters' refusals: the C entry points return before any GPU work, the Python
wrappers raise before they call them."""
import ctypes

import pytest
import torch

import pagedkv
from pagedkv import _lib

BUF = (ctypes.c_char * 65536)()
PTR = (ctypes.addressof(BUF) + 255) // 256 * 256


def _call(name, **kw):
    lora = dict(a=PTR, a_adapter=16 * 256, a_row=256, b=PTR, b_adapter=64 * 16, b_row=16, adapters=4, rank=16,
                ids=PTR, scales=None, slices=None, num_slices=1, out=PTR + 8192, out_stride=64, ws=PTR,
                ws_bytes=1 << 20, stream=None)
    if name == "pk_lora_linear":
        args = dict(x=PTR, x_stride=256, w=PTR, w_stride=256, rows=4, n_out=64, k=256, **lora)
    else:
        args = dict(y=PTR + 8192, y_stride=64, x=PTR, x_stride=256, rows=4, n_out=64, k=256, **lora)
    assert set(kw) <= set(args), kw
    args.update(kw)
    if args["slices"] is not None:
        args["slices"] = (ctypes.c_int32 * len(args["slices"]))(*args["slices"])
    return getattr(_lib.lib(), name)(*args.values())


@pytest.mark.parametrize("name", ["pk_lora_linear", "pk_lora_add"])
@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), _lib.PK_ERR_INVALID_ARG), (dict(n_out=0), _lib.PK_ERR_INVALID_ARG),
    (dict(k=-8), _lib.PK_ERR_INVALID_ARG), (dict(adapters=-1), _lib.PK_ERR_INVALID_ARG),
    (dict(k=252), _lib.PK_ERR_UNSUPPORTED), (dict(rank=0), _lib.PK_ERR_UNSUPPORTED),
    (dict(rank=12), _lib.PK_ERR_UNSUPPORTED), (dict(rank=136), _lib.PK_ERR_UNSUPPORTED),
    (dict(num_slices=0), _lib.PK_ERR_INVALID_ARG), (dict(num_slices=5), _lib.PK_ERR_INVALID_ARG),
    (dict(num_slices=2), _lib.PK_ERR_INVALID_ARG),                          # widths missing
    (dict(num_slices=2, slices=[32, 64]), _lib.PK_ERR_INVALID_ARG),         # too many columns
    (dict(num_slices=2, slices=[32, 0]), _lib.PK_ERR_INVALID_ARG),
    (dict(num_slices=2, slices=[2 ** 31 - 32, 2 ** 31 - 32]), _lib.PK_ERR_INVALID_ARG),
    (dict(num_slices=2, slices=[48, 16]), _lib.PK_ERR_UNSUPPORTED), (dict(x=None), _lib.PK_ERR_INVALID_ARG),
    (dict(ids=None), _lib.PK_ERR_INVALID_ARG), (dict(a=None), _lib.PK_ERR_INVALID_ARG),
    (dict(b=PTR + 8), _lib.PK_ERR_INVALID_ARG), (dict(out=PTR + 8194), _lib.PK_ERR_INVALID_ARG),
    (dict(x_stride=248), _lib.PK_ERR_INVALID_ARG), (dict(out_stride=60), _lib.PK_ERR_INVALID_ARG),
    (dict(a_row=255), _lib.PK_ERR_INVALID_ARG), (dict(b_row=8), _lib.PK_ERR_INVALID_ARG),
    (dict(a_adapter=-8), _lib.PK_ERR_INVALID_ARG), (dict(b_adapter=12), _lib.PK_ERR_INVALID_ARG),
    (dict(ws_bytes=8, rank=64, b_row=64), _lib.PK_ERR_WORKSPACE),  # (rank 64: t is left in the workspace)
    (dict(ws=None, rank=64, b_row=64), _lib.PK_ERR_WORKSPACE),
    (dict(ws=PTR + 4, rank=64, b_row=64), _lib.PK_ERR_WORKSPACE)])
def test_refusals(name, kw, code):
    assert _call(name, **kw) == code, _lib.lib().pk_last_error()
    assert name[3:].encode() in _lib.lib().pk_last_error()


def test_refusals_of_one():
    assert _call("pk_lora_linear", rows=129) == _lib.PK_ERR_UNSUPPORTED
    assert _call("pk_lora_linear", k=264, x_stride=264, w_stride=264, a_row=264) == _lib.PK_ERR_UNSUPPORTED
    assert _call("pk_lora_linear", w=None) == _lib.PK_ERR_INVALID_ARG
    assert _call("pk_lora_linear", out=PTR) == _lib.PK_ERR_INVALID_ARG              # out on x
    assert _call("pk_lora_linear", out=PTR + 1024 + 16) == _lib.PK_ERR_INVALID_ARG  # on x's third row
    assert b"overlaps x" in _lib.lib().pk_last_error()
    assert _call("pk_lora_add", y=None) == _lib.PK_ERR_INVALID_ARG
    assert _call("pk_lora_add", y_stride=56) == _lib.PK_ERR_INVALID_ARG
    assert _call("pk_lora_add", y_stride=72) == _lib.PK_ERR_INVALID_ARG             # out is y, other rows
    # out on x or on part of y; a range of columns beside them is neither (refused for its scratch only)
    assert _call("pk_lora_add", out=PTR, y=PTR + 16384) == _lib.PK_ERR_INVALID_ARG
    assert b"overlaps x" in _lib.lib().pk_last_error()
    assert _call("pk_lora_add", out=PTR + 8192 + 16) == _lib.PK_ERR_INVALID_ARG
    assert b"overlaps y" in _lib.lib().pk_last_error()
    beside = dict(x=PTR, x_stride=512, out=PTR + 512, out_stride=512, y=PTR + 640, y_stride=512, rank=64, b_row=64)
    assert _call("pk_lora_add", **beside, ws_bytes=8) == _lib.PK_ERR_WORKSPACE
    assert _call("pk_lora_add", **{**beside, "y": PTR + 624}, ws_bytes=8) == _lib.PK_ERR_INVALID_ARG
    assert _call("pk_lora_add", **{**beside, "x": PTR + 16}, ws_bytes=8) == _lib.PK_ERR_INVALID_ARG
    # (bytes of out's rows: 512..640, 1536..1664, ...; a row of x from 640 ends at 1152, one from 1040 at 1552)
    at = dict(beside, y=PTR + 256 * 9, ws_bytes=8)
    assert _call("pk_lora_add", **{**at, "x": PTR + 640}) == _lib.PK_ERR_WORKSPACE
    assert _call("pk_lora_add", **{**at, "x": PTR + 1040}) == _lib.PK_ERR_INVALID_ARG
    for name in ("pk_lora_linear", "pk_lora_add"):
        assert _call(name, rows=2 ** 22 + 1) == _lib.PK_ERR_UNSUPPORTED
        wide = dict(n_out=2 ** 20 + 32, out_stride=2 ** 20 + 32)
        assert _call(name, **wide, **(dict(y_stride=2 ** 20 + 32) if name == "pk_lora_add" else {})) == \
            _lib.PK_ERR_UNSUPPORTED
    assert _call("pk_lora_add", rows=2 ** 22, n_out=2 ** 20, out_stride=2 ** 20, y_stride=2 ** 20) == \
        _lib.PK_ERR_UNSUPPORTED
    assert b"too many" in _lib.lib().pk_last_error()
    for name in ("pk_lora_linear", "pk_lora_add"):
        assert _call(name, rows=0, x=None, ids=None, out=None, ws=None, ws_bytes=0) == _lib.PK_OK


def test_workspace_sizes():
    lib = _lib.lib()
    qkv = (ctypes.c_int32 * 3)(2048, 1024, 1024)
    # one launch, no scratch, while all its work-groups are on the GPU at once
    assert lib.pk_lora_add_workspace_bytes(64, 4096, 16, qkv, 3, 8) == 0
    assert lib.pk_lora_add_workspace_bytes(160, 4096, 16, qkv, 3, 8) == 0
    assert lib.pk_lora_add_workspace_bytes(200, 4096, 16, qkv, 3, 8) == 200 * 48 * 4
    # sorted: t, the rows of the tiles, their records, the rows' places
    assert lib.pk_lora_add_workspace_bytes(1000, 4096, 16, qkv, 3, 8) == 1000 * 48 * 4 + (15 + 9) * (256 + 8) + 4000
    assert lib.pk_lora_add_workspace_bytes(1000, 4000, 16, qkv, 3, 8) == 0                # refused
    # t, and the projection's partial sums where it leaves them (K split, or ranks above 16)
    base = lib.pk_linear_workspace_bytes(100, 1024, 2048, 2)
    assert lib.pk_lora_linear_workspace_bytes(100, 1024, 2048, 16, 1) == base + 100 * 16 * 4
    assert lib.pk_lora_linear_workspace_bytes(100, 4096, 1024, 24, 3) == 100 * (4096 + 72) * 4
    assert lib.pk_lora_linear_workspace_bytes(100, 4096, 1024, 16, 3) == 100 * 48 * 4
    assert lib.pk_lora_linear_workspace_bytes(2, 4096, 1024, 16, 3) == 0
    assert lib.pk_lora_linear_workspace_bytes(129, 1024, 1024, 16, 1) == 0
    assert pagedkv.lora_workspace_bytes(200, 4096, 1024, 16, (2048, 1024, 1024), 8) == 200 * 48 * 4


def test_python_refusals():
    bf = dict(dtype=torch.bfloat16)
    x, w, y = torch.zeros(4, 256, **bf), torch.zeros(64, 256, **bf), torch.zeros(4, 64, **bf)
    a, b, ids = torch.zeros(2, 16, 256, **bf), torch.zeros(2, 64, 16, **bf), torch.zeros(4, dtype=torch.int32)
    for call in (lambda **k: pagedkv.lora_add(**{**dict(y=y, x=x, lora_a=a, lora_b=b, adapter_ids=ids), **k}),
                 lambda **k: pagedkv.lora_linear(**{**dict(x=x, weight=w, lora_a=a, lora_b=b, adapter_ids=ids), **k})):
        for kw, match in [(dict(x=x.float()), "bf16"), (dict(lora_a=a[:, :8]), "must be"),
                          (dict(lora_a=a[:1]), "must be"), (dict(lora_b=b[:, :32]), "must be"),
                          (dict(lora_b=b.transpose(1, 2)), "contiguous rows"),
                          (dict(slices=(32, 16)), "add up"), (dict(slices=(32, 32)), "must be"),
                          (dict(adapter_ids=ids[:3]), "adapter_ids"), (dict(scales=torch.ones(3)), "scales"),
                          (dict(scales=torch.ones(2, dtype=torch.float64)), "scales"),
                          (dict(slices=()), "add up"), (dict(out=torch.zeros(4, 32, **bf)), "out must be")]:
            with pytest.raises(ValueError, match=match):
                call(**kw)
        with pytest.raises(TypeError, match="int32"):
            call(adapter_ids=ids.long())
    with pytest.raises(ValueError, match="does not match"):
        pagedkv.lora_add(y[:3], x, a, b, ids)
    with pytest.raises(ValueError, match="does not match"):
        pagedkv.lora_linear(x, w[:, :128], a, b, ids)
    with pytest.raises(ValueError, match="on a GPU"):  # tensors of one device, which is not a GPU
        pagedkv.lora_add(y, x, a, b, ids)
    with pytest.raises(ValueError, match="at most 128"):
        pagedkv.lora_linear(torch.zeros(129, 256, **bf), w, a, b, torch.zeros(129, dtype=torch.int32))


def test_workspace_sizes_take_the_slices_of_the_operators():
    """Any sequence of widths, as lora_linear and lora_add take them."""
    for linear in (False, True):
        want = pagedkv.lora_workspace_bytes(200, 4096, 1024, 24, (2048, 1024, 1024), 8, linear)
        got = [pagedkv.lora_workspace_bytes(200, 4096, 1024, 24, s, 8, linear)
               for s in ([2048, 1024, 1024], torch.Size((2048, 1024, 1024)), iter((2048, 1024, 1024)))]
        assert got == [want] * 3
        assert pagedkv.lora_workspace_bytes(200, 4096, 1024, 24, None, 8, linear) == \
            pagedkv.lora_workspace_bytes(200, 4096, 1024, 24, [4096], 8, linear)
    with pytest.raises(ValueError, match="add up"):
        pagedkv.lora_workspace_bytes(200, 4096, 1024, 24, [2048, 1024], 8)
