"""GPU: more rows than one launch's 2^32 work items hold -- quantised, brought back and scored in pieces."""
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from nncf_amd import catalogue  # noqa: E402

BF16 = torch.bfloat16


@pytest.fixture(autouse=True)
def _memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n,k", [(2 ** 29 + 70, 1), (2 ** 26 + 3, 129)])
def test_rows_to_codes(n, k):
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.empty(n, k, dtype=BF16, device="cuda")
    for i in range(0, n, 2 ** 24):
        x[i:i + 2 ** 24].normal_(generator=g)
    r = catalogue.quantize_rows(x)
    for i in (0, 2 ** 25 - 40, 2 ** 28 - 20, 2 ** 29 - 20, n - 100):      # the first rows, where pieces may meet, the last ones
        i = min(i, n - 100)
        part = catalogue.quantize_rows(x[i:i + 100].clone())
        assert torch.equal(r.codes[i:i + 100], part.codes) and torch.equal(r.scale[i:i + 100], part.scale)
    for i in range(0, n, 2 ** 24):                                       # every row's scale: its largest value / 127
        want = x[i:i + 2 ** 24].float().abs().amax(1) / torch.full((), 127.0, device="cuda")
        assert torch.equal(r.scale[i:i + 2 ** 24], want)


def test_codes_to_rows():
    n, k = 2 ** 26 + 5, 513                                              # 65 groups of 8 columns a row
    codes = torch.zeros(n, 640, dtype=torch.int8, device="cuda")
    scale = torch.rand(n, device="cuda")
    at = [0, 2 ** 25 + 1, (2 ** 31) // 65 - 2, (2 ** 32) // 65 - 2, n - 7]
    for i in at:
        codes[i:i + 7, :k] = torch.randint(-127, 128, (7, k), device="cuda", dtype=torch.int8)
    out = catalogue.Int8Rows(codes, scale, k).dequantize(BF16)
    for i in at:
        part = catalogue.Int8Rows(codes[i:i + 7].clone(), scale[i:i + 7].clone(), k).dequantize(BF16)
        assert torch.equal(out[i:i + 7], part) and part.any()
    for i in range(0, n, 2 ** 22):                                       # every value is written: zeros behind those
        got, want = out[i:i + 2 ** 22], codes[i:i + 2 ** 22, :k]
        assert torch.equal(got.ne(0).sum(1), (want.ne(0) & (scale[i:i + 2 ** 22, None] > 0)).sum(1))


def test_scores_of_very_many_rows():
    m = 2 ** 31
    codes = torch.zeros(m, 64, dtype=torch.int8, device="cuda")
    scale = torch.ones(m, device="cuda")
    rb = torch.zeros(m, device="cuda")
    at = [0, 2 ** 22 - 3, 2 ** 30 - 3, m - 6]
    for i in at:
        codes[i:i + 6, :30] = torch.randint(-127, 128, (6, 30), device="cuda", dtype=torch.int8)
        rb[i:i + 6] = torch.randn(6, device="cuda")
    t = catalogue.quantize_rows(torch.randn(2, 30, device="cuda"))
    s = catalogue.int8_scores(catalogue.Int8Rows(codes, scale, 30), t, row_bias=rb, dtype=BF16)
    for i in at:
        few = catalogue.Int8Rows(codes[i:i + 6].clone(), scale[i:i + 6].clone(), 30)
        assert torch.equal(s[i:i + 6], catalogue.int8_scores(few, t, row_bias=rb[i:i + 6].clone(), dtype=BF16))
    assert int(sum(s[i:i + 2 ** 28].ne(0).sum() for i in range(0, m, 2 ** 28))) <= 12 * len(at)
    assert torch.isfinite(s[::4097]).all()
