"""GPU: codes that were made elsewhere are looked at when Int8Rows takes them over."""
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from nncf_amd import catalogue  # noqa: E402


@pytest.mark.parametrize("n,k", [(1, 1), (9, 70), (300, 64), (5, 300)])
def test_codes_that_the_products_do_not_take(n, k):
    r = catalogue.quantize_rows(torch.randn(n, k, device="cuda"))
    assert torch.equal(catalogue.Int8Rows(r.codes.clone(), r.scale, k).dequantize(), r.dequantize())
    pitch = r.codes.shape[1]
    low = r.codes.clone()
    low[n - 1, k - 1] = -128
    with pytest.raises(ValueError, match="-127"):
        catalogue.Int8Rows(low, r.scale, k)
    if pitch > k:
        for col in (k, pitch - 1):
            behind = r.codes.clone()
            behind[n // 2, col] = 1
            with pytest.raises(ValueError, match="zeros behind"):
                catalogue.Int8Rows(behind, r.scale, k)


def test_no_rows_and_a_capture():
    empty = catalogue.quantize_rows(torch.empty(0, 30, device="cuda"))
    assert len(catalogue.Int8Rows(empty.codes, empty.scale, 30)) == 0
    r = catalogue.quantize_rows(torch.randn(4, 30, device="cuda"))
    g = torch.cuda.CUDAGraph()
    said = []
    with torch.cuda.graph(g):
        try:
            catalogue.Int8Rows(r.codes, r.scale, 30)
        except RuntimeError as e:
            said.append(str(e))
        back = r.dequantize()
    assert said and "capture" in said[0]
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(back, r.dequantize())
        back.zero_()
