"""CPU: what nncf_gather_rows_bias refuses, before anything is launched."""
import pytest

from nncf_amd import _lib

P = 1 << 20      # an address that is never read


@pytest.mark.parametrize("i,v,word", [(0, None, "NULL"), (1, -1, "rows"), (2, 19, "row shape"), (3, 0, "row shape"), (3, 18, "row shape"), (3, 132, "row shape"),
                                      (5, -1, "biases"), (6, None, "NULL"), (7, 1 << 28, "out of range"), (8, None, "NULL"), (9, None, "NULL")])
def test_gather_refuses(i, v, word):
    args = [P, 100, 20, 20, P, 100, P, 4, P, P, None]
    args[i] = v
    with pytest.raises(ValueError, match=word):
        _lib.check(_lib.lib().nncf_gather_rows_bias(*args))


def test_no_ids_are_no_error():
    assert _lib.lib().nncf_gather_rows_bias(None, 0, 20, 20, None, 0, None, 0, None, None, None) == 0
