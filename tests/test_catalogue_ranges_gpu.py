"""GPU: the magnitudes of fp32 rows that softmax_xent is documented for: 2^-80 .. 2^90, rows of one call within 2^100 of each other, zeros."""
import math

import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from nncf_amd import catalogue  # noqa: E402

E = 2.0 ** -24


@pytest.mark.parametrize("n,c", [(40, 700), (300, 5000), (3, 900)])
@pytest.mark.parametrize("low,high,users", [(-50, 50, 0), (-79, 20, 0), (-10, 89, -60), (60, 89, -79), (0, 0, 60)])
def test_rows_of_all_documented_magnitudes(n, c, low, high, users):
    """Logits of +-10 for the largest rows, 0 for the smallest and the rows of zeros: every item counts in the normaliser."""
    d = 24
    g = torch.Generator().manual_seed(n + c + low)
    f = 2.0 ** torch.randint(low, high + 1, (c, 1), generator=g).double()
    f[3], f[4], f[5] = 2.0 ** low, 2.0 ** high, 0.0
    table = (torch.nn.functional.normalize(torch.randn(c, d, generator=g), dim=1).double() * f * 0.9).float()
    rows = (torch.nn.functional.normalize(torch.randn(n, d, generator=g), dim=1).double() * 2.0 ** users * 0.9).float()
    rows[n - 1] = 0
    target = torch.randint(c, (n,), generator=g)
    target[0], target[1] = 3, 5
    scale = 10.0 * 2.0 ** -(high + users)
    r = catalogue.softmax_xent(rows.cuda(), table.cuda(), target.int().cuda(), scale=scale, reduction="none")
    z = scale * (rows.double() @ table.double().t())
    lse = torch.logsumexp(z, 1)
    loss = lse - z.gather(1, target[:, None])[:, 0]
    # planes and d products of a logit below 10; the exponent's additions of values up to 128 beside the rows' powers of two
    z_err = (3 * 2.0 ** -22 + (d + 2) * E) * 10 * math.sqrt(d) + 4 * E * 128
    assert (r.lse.double().cpu() - lse).abs().max().item() <= 2 * z_err
    assert (r.loss.double().cpu() - loss).abs().max().item() <= 4 * z_err
    p = torch.softmax(z, 1)
    p[torch.arange(n), target] -= 1
    want, terms = scale * (p @ table.double()), abs(scale) * (p.abs() @ table.double().abs())
    # 2^-22 of the largest term may be missing in smaller ones: here of the largest row's, 10 (scale times the largest row and user)
    tol = (4 * z_err + 32 * E) * terms + 2.0 ** -22 * 10 / 2.0 ** users
    assert ((r.d_rows.double().cpu() - want).abs() <= tol).all()
    want, terms = scale * (p.t() @ rows.double()), abs(scale) * (p.abs().t() @ rows.double().abs())
    tol = (4 * z_err + 32 * E + 2.0 ** -22) * terms + abs(scale) * 2.0 ** users * 2.0 ** -22
    assert ((r.d_table.double().cpu() - want).abs() <= tol).all()
