"""GPU: an item that a bias of -inf leaves out has no gradient, whatever the rows hold."""
import math

import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from nncf_amd import catalogue  # noqa: E402


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 2, 4, 5, 40, 300])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_an_item_left_out_of_rows_that_are_no_numbers(n, bad, dtype):
    g = torch.Generator().manual_seed(n)
    rows, table = (0.3 * torch.randn(k, 40, generator=g) for k in (n, 700))
    rows[n - 1] = bad
    bias = torch.randn(700, generator=g)
    out = torch.rand(700, generator=g) < 0.2
    out[:10] = False
    bias[out] = -math.inf
    target = torch.arange(n, dtype=torch.int32) % 10
    r = catalogue.softmax_xent(rows.to(dtype).cuda(), table.to(dtype).cuda(), target.cuda(), bias=bias.cuda(), reduction="none")
    out = out.cuda()
    assert not r.d_table[out].any() and not r.d_bias[out].any()
    assert torch.isnan(r.d_table[~out]).all() and torch.isnan(r.loss[n - 1]) and torch.isfinite(r.loss[:n - 1]).all()
