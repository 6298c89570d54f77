"""GPU: sums over long catalogues and large batches, with terms that are all alike: the case in which the roundings of a running sum lean
one way and add up instead of cancelling.

Rows (or the table) are zeros, so that every logit is the item's bias b and everything is known in closed form."""
import math

import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from nncf_amd import catalogue  # noqa: E402

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
E = 2.0 ** -24

# lse = b + log c.  In units of E = 2^-24: the exponent b log2(e) - shift - reference is formed of values up to 32 in four roundings, 128 ln 2;
# an exponential 2; a sub-tile's sum of 16 or 32 terms 10, the compensated sum 2, its halves and the splits 16; the logarithm's
# value below 24, three roundings of it, 72 ln 2; the result below 16, two roundings.  201 in all, whatever the number of terms.
LSE = 201 * E
# a coefficient exp(z - lse) is off by lse's error and by its own exponent's: values up to 32, four roundings, and an exponential
COEF = LSE + (128 * math.log(2) + 2) * E


def long_rows(n, c, d, dtype, b, reduction="none", **kw):
    g = torch.Generator(device="cuda").manual_seed(n + c)
    table = torch.rand(c, d, generator=g, device="cuda") + 0.37
    table[:, 0], table[:, 1] = 1 / 3, 0.7              # columns of equal values
    table = table.to(dtype)
    table[:n] = 0                                      # the targets' rows
    target = torch.arange(n, device="cuda").int()
    bias = torch.full((c,), b, device="cuda")
    return table, bias, catalogue.softmax_xent(torch.zeros(n, d, device="cuda", dtype=dtype), table, target, bias=bias, reduction=reduction, **kw)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,c", [(4096, 1_000_000), (8192, 1_000_003), (130, 1_000_000), (4, 2_000_001), (20_000, 300_000)])
@pytest.mark.parametrize("b", [0.123, -3.7])
def test_the_normaliser_of_equal_terms(n, c, b, dtype):
    table, bias, r = long_rows(n, c, 16, dtype, b, grad=False)
    lse = math.log(c) + bias[0].item()
    assert (r.lse.double() - lse).abs().max().item() <= LSE
    assert (r.loss.double() - math.log(c)).abs().max().item() <= LSE + 2 * 16 * E


def many_users(n, c, d, dtype, weight=None):
    g = torch.Generator(device="cuda").manual_seed(n)
    rows = torch.rand(n, d, generator=g, device="cuda") + 0.37
    rows[:, 0], rows[:, 1] = 1 / 3, 0.7
    rows = rows.to(dtype)
    bias = torch.full((c,), 0.123, device="cuda")
    target = torch.zeros(n, device="cuda").int()
    return rows, catalogue.softmax_xent(rows, torch.zeros(c, d, device="cuda", dtype=dtype), target, bias=bias, reduction="none", weight=weight)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,c", [(8192, 40_000), (100_000, 40_000), (70_001, 300)])
@pytest.mark.parametrize("w", [None, 0.7])
def test_the_bias_gradient_of_equal_terms(n, c, w, dtype):
    weight = None if w is None else torch.full((n,), w, device="cuda")
    k = 1.0 if w is None else weight[0].item()
    rows, r = many_users(n, c, 16, dtype, weight)
    # 16 for a sub-tile's sum, the compensated sum and the splits, 2 for the weight and the result
    assert (r.d_bias[1:].double() / (k * n / c) - 1).abs().max().item() <= COEF + 30 * E
    # the target's: 1 - p_t of each user, to 4 roundings, and its sums
    assert abs(r.d_bias[0].item() / (k * n * (1 / c - 1)) - 1) <= LSE / c + 40 * E
