"""CPU: what the catalogue head refuses, before anything is launched (C ABI and nncf_amd/catalogue.py)."""
import ctypes

import pytest
import torch

from nncf_amd import _lib, catalogue

P = 1 << 20      # an address that is never read: every call below is refused before a launch


def xent(**kw):
    x = _lib.Xent()
    for f in ("rows", "table", "target", "loss", "lse", "d_rows", "d_table"):
        setattr(x, f, P)
    x.n, x.c, x.dim, x.dtype, x.reduction, x.scale, x.rows_stride, x.table_stride = 8, 100, 20, 0, 1, 1.0, 20, 20
    for k, v in kw.items():
        setattr(x, k, v)
    return x


@pytest.mark.parametrize("change,word", [
    (dict(rows=None), "NULL"), (dict(table=None), "NULL"), (dict(target=None), "NULL"), (dict(loss=None), "NULL"), (dict(lse=None), "NULL"),
    (dict(d_rows=None), "together"), (dict(d_table=None), "together"), (dict(d_bias=P), "bias"), (dict(n=0), "n = 0"), (dict(c=0), "c = 0"),
    (dict(n=128 * 65535 + 1), "out of range"), (dict(c=128 * 65535 + 1), "out of range"), (dict(dim=0), "dim"), (dict(dim=129), "dim"),
    (dict(dtype=3), "dtype"), (dict(reduction=7), "reduction"), (dict(rows_stride=19), "stride"), (dict(table_stride=19), "stride"),
    (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(rows=P + 2), "aligned"), (dict(d_table=P + 1), "aligned"),
])
def test_xent_refuses(change, word):
    L = _lib.lib()
    with pytest.raises(ValueError, match=word):
        _lib.check(L.nncf_softmax_xent(ctypes.byref(xent(**change)), P, 1 << 40, None))


def test_xent_refuses_a_small_or_crooked_workspace():
    L = _lib.lib()
    need = L.nncf_softmax_xent_ws_bytes(8, 100, 20, 0, 1)
    assert need > L.nncf_softmax_xent_ws_bytes(8, 100, 20, 0, 0) > 0
    with pytest.raises(ValueError, match="needed"):
        _lib.check(L.nncf_softmax_xent(ctypes.byref(xent()), P, need - 1, None))
    with pytest.raises(ValueError, match="aligned"):
        _lib.check(L.nncf_softmax_xent(ctypes.byref(xent()), P + 16, need, None))
    with pytest.raises(ValueError, match="NULL"):
        _lib.check(L.nncf_softmax_xent(None, P, need, None))
    assert L.nncf_softmax_xent_ws_bytes(8, 100, 129, 0, 1) == -1 and L.nncf_softmax_xent_ws_bytes(0, 100, 20, 0, 1) == -1


@pytest.mark.parametrize("i,v,word", [(0, None, "NULL"), (1, 9, "stride"), (2, 5, "dtype"), (3, -1, "rows"), (4, 0, "k = 0"), (4, 131073, "k ="),
                                      (6, None, "NULL"), (6, P + 8, "aligned"), (7, None, "NULL"), (0, P + 2, "aligned")])
def test_quantize_refuses(i, v, word):
    args = [P, 10, 0, 4, 10, 0, P, P, None]
    args[i] = v
    with pytest.raises(ValueError, match=word):
        _lib.check(_lib.lib().nncf_quantize_rows(*args))


@pytest.mark.parametrize("i,v,word", [(0, None, "NULL"), (1, None, "NULL"), (2, -1, "out of range"), (3, None, "NULL"), (5, -1, "out of range"),
                                      (6, 0, "k = 0"), (9, None, "NULL"), (10, 99, "stride"), (11, 4, "dtype"), (0, P + 4, "aligned"),
                                      (3, P + 4, "aligned"), (9, P + 2, "aligned")])
def test_scores_refuse(i, v, word):
    args = [P, P, 4, P, P, 100, 10, None, None, P, 100, 0, None]
    args[i] = v
    with pytest.raises(ValueError, match=word):
        _lib.check(_lib.lib().nncf_int8_scores(*args))


@pytest.mark.parametrize("i,v,word", [(0, None, "NULL"), (1, 9, "stride"), (2, 3, "dtype"), (3, 33, "first"), (3, 0, "first"), (4, None, "NULL"),
                                      (5, None, "NULL"), (6, -1, "out of range"), (7, 0, "first"), (7, 4097, "first"), (10, None, "NULL"),
                                      (11, 99, "stride"), (12, 7, "dtype"), (0, P + 2, "aligned"), (4, P + 8, "aligned"), (10, P + 1, "aligned")])
def test_scores_of_float_rows_refuse(i, v, word):
    args = [P, 10, 0, 4, P, P, 100, 10, None, None, P, 100, 0, None]
    args[i] = v
    with pytest.raises(ValueError, match=word):
        _lib.check(_lib.lib().nncf_int8_scores_rows(*args))


def test_dequantize_refuses():
    L = _lib.lib()
    for args in ([None, P, 4, 10, P, 0, None], [P, P, 4, 0, P, 0, None], [P, P, 4, 10, P, 3, None], [P, P, 4, 10, P + 4, 0, None], [P, P, -1, 10, P, 0, None]):
        with pytest.raises(ValueError):
            _lib.check(L.nncf_dequantize_rows(*args))


def test_nothing_to_do_is_no_error():
    L = _lib.lib()
    assert L.nncf_quantize_rows(None, 10, 0, 0, 10, 0, None, None, None) == 0
    assert L.nncf_dequantize_rows(None, None, 0, 10, None, 0, None) == 0
    assert L.nncf_int8_scores(None, None, 0, None, None, 5, 10, None, None, None, 5, 0, None) == 0
    assert [L.nncf_int8_pitch(k) for k in (0, 1, 64, 65, 128, 129, 131072, 131073)] == [-1, 64, 64, 128, 128, 256, 131072, -1]


def test_host_tensors_are_refused():
    x, t = torch.zeros(4, 10), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: catalogue.softmax_xent(x, x, t), lambda: catalogue.quantize_rows(x), lambda: catalogue.int8_scores(x, x),
                 lambda: catalogue.softmax_xent(x.numpy(), x, t)):
        with pytest.raises(TypeError):
            call()


@pytest.mark.parametrize("m,c,k", [(1 << 22, 1 << 31, 100), (1 << 22, 300_000, 60), (1 << 22, 1 << 18, 300)])
def test_more_scores_than_a_launch_holds_are_refused(m, c, k):
    """2^32 work items: refused as an argument, not as a launch that fails (such a matrix has a terabyte)."""
    with pytest.raises(ValueError, match="in one call"):
        _lib.check(_lib.lib().nncf_int8_scores(P, P, m, P, P, c, k, None, None, P, c, 0, None))
