"""GPU: the catalogue head (nncf_amd/catalogue.py) against plain implementations in 64 bits.

Tolerances.  u(t) = eps(t) / 2 is the most one rounding to t moves a value, relative to it (2^-24, 2^-11, 2^-8).

softmax_xent.  A logit is a sum of d <= 128 products of values kept to 2^-22 (fp32: two planes) or exactly (16-bit types), summed in
fp32: |dz| <= Z = scale (3 * 2^-22 + (d + 2) 2^-24) max_ij sum_k |u_ik v_jk| + 4 * 2^-24 max|z| -- the last term is what the exponent's own
additions round.  exp(z - lse) is then off by at most P = 2 Z + 16 * 2^-24 relative (z and lse; the exponential, its scale, the sum's
division), a loss by 2 Z + 4 * 2^-24 max|loss|, and a coefficient that is rounded to 16 bits before its product by u(t) more.  A
gradient row is sum_b coef_b x_b, so it is off by at most (P + u_p) sum_b |coef_b x_b| + N 2^-24 sum_b |coef_b x_b| for the fp32 sum of N
terms in 32-term tiles (N / 16 roundings of the running sum at most), plus u(t) of the result for the output's own type."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from nncf_amd import catalogue  # noqa: E402

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = {t: torch.finfo(t).eps / 2 for t in (F32, F16, BF16)}


def make(n, c, d, dtype, seed=0, lean=2.0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    table = torch.randn(c, d, generator=g) / math.sqrt(d) * spread
    target = torch.randint(c, (n,), generator=g)
    rows = lean * torch.rand(n, 1, generator=g) * table[target] + 0.5 * torch.randn(n, d, generator=g) / math.sqrt(d)
    return rows.to(dtype).to(DEV), table.to(dtype).to(DEV), target.int().to(DEV)


def oracle(rows, table, target, bias=None, weight=None, scale=1.0, reduction="mean"):
    """Everything in float64 on the CPU, straight from the definition, and the sums of absolute terms that the tolerances need."""
    u, v, t = rows.double().cpu(), table.double().cpu(), target.long().cpu()
    n, c = u.shape[0], v.shape[0]
    b = bias.double().cpu() if bias is not None else torch.zeros(c, dtype=torch.float64)
    w = weight.double().cpu() if weight is not None else torch.ones(n, dtype=torch.float64)
    has = t >= 0
    out = torch.isneginf(b)
    v = torch.where(out[:, None], 0.0, v)
    u = torch.where(has[:, None], u, 0.0)
    z = scale * (u @ v.t()) + b
    at = t.clamp(min=0)
    lse = torch.logsumexp(z, 1)
    zt = z.gather(1, at[:, None])[:, 0]
    each = torch.where(out[at], torch.full_like(lse, math.inf), lse - zt)
    rest = z.clone()
    rest[torch.arange(n), at] = -math.inf
    apart = torch.logsumexp(rest, 1) - zt
    each = torch.where(out[at], each, torch.nn.functional.softplus(apart))
    w = torch.where(has, w, 0.0)
    count = max(1, int(has.sum()))
    each = torch.where(w == 0, torch.zeros_like(each), w * each)
    g = torch.where(out[at], 0.0, w)
    if reduction == "mean":
        g = g / count
    p = torch.exp(z - torch.where(torch.isinf(lse), 0.0, lse)[:, None])
    p[torch.arange(n), at] = torch.where(out[at], p[torch.arange(n), at], -torch.sigmoid(apart))
    coef = g[:, None] * p
    loss = each if reduction == "none" else each.sum() / (count if reduction == "mean" else 1)
    terms = dict(rows=scale * (coef.abs() @ v.abs()), table=abs(scale) * (coef.abs().t() @ u.abs()), bias=coef.abs().sum(0))
    dots = abs(scale) * (u.abs() @ v.abs().t()).max().item()
    return dict(loss=loss, lse=torch.where(has, lse, 0.0), d_rows=scale * (coef @ v), d_table=scale * (coef.t() @ u), d_bias=coef.sum(0),
                terms=terms, dots=dots, zmax=z[~torch.isinf(z)].abs().max().item() if (~out).any() else 0.0, each=each)


def check(r, want, dtype, d, reduction, n, c):
    e = 2.0 ** -24
    planes = 3 * 2.0 ** -22 if dtype == F32 else 0.0
    zt = (planes + (d + 2) * e) * want["dots"] + 4 * e * (want["zmax"] + 32)    # + 32: rows' own exponents ride in the same addition
    p = 2 * zt + 16 * e
    up = 2.0 ** -22 if dtype == F32 else U[dtype]
    fin = torch.isfinite(want["each"])
    scale_of = want["each"][fin].abs().max().item() if fin.any() else 0.0
    got = r.loss.double().cpu()
    if reduction == "none":
        ok = torch.isfinite(want["loss"])
        assert torch.equal(torch.isfinite(got), ok)
        assert (got - want["loss"])[ok].abs().max().item() <= (2 * zt + 4 * e) * max(1.0, scale_of) if ok.any() else True
    elif torch.isfinite(want["loss"]):
        k = want["each"].abs().sum().item() if reduction == "sum" else scale_of
        rowsn = n if reduction == "sum" else 1
        assert abs(got.item() - want["loss"].item()) <= 2 * zt * rowsn * max(1.0, scale_of) + 4 * e * k
    else:
        assert not math.isfinite(got.item())
    ok = torch.isfinite(want["lse"])
    assert (r.lse.double().cpu() - want["lse"])[ok].abs().max().item() <= 2 * zt + 4 * e * want["zmax"]
    if r.d_rows is None:
        return
    tiny = 1e-30 if dtype != F16 else 2.0 ** -24
    for got, key, N in ((r.d_rows, "rows", c), (r.d_table, "table", n)):
        ref = want["d_" + key]
        tol = (p + up + (N / 16 + 32) * e) * want["terms"][key] + U[dtype] * ref.abs() + tiny
        err = (got.double().cpu() - ref).abs()
        assert got.dtype == dtype and (err <= tol).all(), (key, (err / tol).max().item())
    if r.d_bias is not None:
        err = (r.d_bias.double().cpu() - want["d_bias"]).abs()
        assert (err <= (p + (n / 16 + 32) * e) * want["terms"]["bias"] + tiny).all(), (err / want["terms"]["bias"]).max().item()


SHAPES = [(1, 1, 1), (1, 2, 3), (2, 63, 50), (3, 64, 64), (33, 65, 65), (31, 129, 100), (64, 1000, 128), (127, 517, 99), (128, 128, 4), (129, 2050, 127),
          (300, 77, 36), (5, 20011, 100), (1025, 300, 128), (513, 4099, 50),
          (4, 4100, 128), (2, 300, 33), (6, 131073, 48), (70, 66003, 101), (200, 3000, 96), (200, 3000, 112), (40, 500, 65), (150, 700, 97), (150, 700, 113)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,c,d", SHAPES)
def test_xent_against_the_definition(n, c, d, dtype):
    rows, table, target = make(n, c, d, dtype, seed=n + c)
    for reduction in ("mean", "none"):
        r = catalogue.softmax_xent(rows, table, target, scale=10.0, reduction=reduction)
        check(r, oracle(rows, table, target, scale=10.0, reduction=reduction), dtype, d, reduction, n, c)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,c,d,seed", [(37, 333, 50, 0), (200, 1111, 100, 1), (130, 64, 128, 2), (1, 700, 30, 11), (3, 2000, 100, 4), (4, 65, 128, 5),
                                        (40, 70001, 24, 6), (5, 66000, 65, 7)])
def test_xent_bias_weight_padding(n, c, d, seed, dtype):
    rows, table, target = make(n, c, d, dtype, seed=seed)
    g = torch.Generator().manual_seed(seed)
    bias = torch.randn(c, generator=g)
    bias[torch.rand(c, generator=g) < 0.2] = -math.inf
    weight = torch.randn(n, generator=g)        # either sign
    weight[torch.rand(n, generator=g) < 0.1] = 0.0
    target = target.cpu()
    target[torch.rand(n, generator=g) < 0.2] = -1
    # values that are not to be used
    rows[(target < 0).to(DEV)] = math.nan
    table[torch.isinf(bias).to(DEV)] = math.inf
    keep = torch.isinf(bias)[target.clamp(min=0).long()]
    for drop in (True, False):      # targets that are left out: +inf loss, no gradient
        t = torch.where(keep, torch.full_like(target, -1), target) if drop else target
        args = dict(bias=bias.to(DEV), weight=weight.to(DEV), scale=3.0)
        for reduction in ("sum", "none", "mean"):
            r = catalogue.softmax_xent(rows, table, t.to(DEV), reduction=reduction, **args)
            want = oracle(torch.nan_to_num(rows), torch.nan_to_num(table, posinf=0.0), t, reduction=reduction, **args)
            if not drop and reduction != "none" and (keep & (target >= 0) & (weight != 0)).any():
                assert not math.isfinite(r.loss.item())
                want["loss"] = torch.tensor(r.loss.item())
            check(r, want, dtype, d, reduction, n, c)


def test_xent_rows_that_take_no_part():
    rows, table, _ = make(5, 40, 16, F32)
    none = torch.full((5,), -1, dtype=torch.int32, device=DEV)
    r = catalogue.softmax_xent(rows, table, none)
    assert r.loss.item() == 0 and not r.lse.any() and not r.d_rows.any() and not r.d_table.any()
    out = torch.full((40,), -math.inf, device=DEV)
    t = torch.arange(5, dtype=torch.int32, device=DEV)
    r = catalogue.softmax_xent(rows, table, t, bias=out, reduction="none")
    assert torch.isposinf(r.loss).all() and torch.isneginf(r.lse).all()
    assert not r.d_rows.any() and not r.d_table.any() and not r.d_bias.any()
    bad = t.clone()
    bad[3] = 40
    r = catalogue.softmax_xent(rows, table, bad)
    assert torch.isnan(r.loss) and torch.isnan(r.d_rows[3]).all() and torch.isnan(r.d_table).all()
    assert not torch.isnan(r.d_rows[:3]).any()


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n", [2, 5, 200])
def test_xent_values_that_are_no_numbers_are_not_lost(n, dtype):
    rows, table, target = make(n, 700, 40, dtype)
    for bad in (math.nan, math.inf):
        item = table.clone()
        item[699, 3] = bad                      # an item of the catalogue: every row's logits
        r = catalogue.softmax_xent(rows, item, target.clamp(max=600))
        if math.isnan(bad):
            assert torch.isnan(r.loss) and torch.isnan(r.d_rows).all() and torch.isnan(r.d_table).all()
        else:       # a row with a negative value there has the logit -inf, and only 0 * inf in its gradient
            assert torch.isnan(r.loss) == bool((rows[:, 3] >= 0).any() or dtype == F32 or n > 4) or not torch.isfinite(r.loss)
            assert torch.isnan(r.d_rows[:, 3]).all()
        one = rows.clone()
        one[1] = bad                            # a row: its loss, and every item's gradient
        r = catalogue.softmax_xent(one, table, target, reduction="none")
        assert torch.isnan(r.loss[1]) and torch.isnan(r.d_rows[1]).all() and torch.isnan(r.d_table).all()
        assert torch.isfinite(r.loss[0]) and torch.isfinite(r.d_rows[0]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_xent_a_whole_part_of_nan_is_not_lost(dtype):
    """NaN in every item (user) that one workgroup streams, and in no other."""
    rows, table, target = make(300, 9000, 40, dtype)
    item = table.clone()
    item[4096:4096 + 512] = math.nan
    r = catalogue.softmax_xent(rows, item, target.clamp(max=4000), reduction="none")
    assert torch.isnan(r.loss).all() and torch.isnan(r.d_rows).all() and torch.isnan(r.d_table).all()
    assert torch.isnan(catalogue.softmax_xent(rows[:3], item, target[:3].clamp(max=4000), reduction="none").loss).all()
    user = rows.clone()
    user[64:192] = math.nan
    for sl in (slice(0, 9000), slice(0, 400)):
        r = catalogue.softmax_xent(user, table[sl], target.clamp(max=399), reduction="none")
        assert torch.isnan(r.loss[64:192]).all() and torch.isfinite(r.loss[:64]).all() and torch.isnan(r.d_table).all()


def test_xent_of_tiny_rows():
    """A table of 2^-79: full precision; the sums of its scales stay finite over many items."""
    rows, table, target = make(40, 5000, 32, F32, seed=8)
    table = table * 2.0 ** -76
    kw = dict(scale=10.0 * 2.0 ** 76, reduction="none")
    r = catalogue.softmax_xent(rows, table, target, **kw)
    want = oracle(rows, table, target, **kw)
    check(r._replace(d_rows=None), want, F32, 32, "none", 40, 5000)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_xent_confident_rows_keep_their_gradient(dtype):
    """p_t -> 1: the gradient is (1 - p_t) (mean of the others - v_t), down to 1 - p_t of 1e-13, where 1 - p_t by subtraction is 0."""
    c, d = 300, 64
    g = torch.Generator().manual_seed(5)
    table = torch.nn.functional.normalize(torch.randn(c, d, generator=g), dim=1).to(dtype)
    target = torch.arange(0, 40, dtype=torch.int32)
    rows = (table[:40].float() * torch.linspace(0.1, 3.5, 40)[:, None]).to(dtype)
    rows, table, target = rows.to(DEV), table.to(DEV), target.to(DEV)
    r = catalogue.softmax_xent(rows, table, target, scale=10.0, reduction="none")
    want = oracle(rows, table, target, scale=10.0, reduction="none")
    assert want["loss"].min() < 1e-9
    check(r, want, dtype, d, "none", 40, c)
    # relative to each row's own loss: logits are off by Z absolutely, so is its logarithm
    e = 2.0 ** -24
    z = ((3 * 2.0 ** -22 if dtype == F32 else 0) + (d + 2) * e) * want["dots"] + 4 * e * (want["zmax"] + 32)
    assert ((r.loss.double().cpu() / want["loss"] - 1).abs() <= 2 * z + 8 * e).all()


def test_xent_rows_of_any_magnitude():
    """fp32 rows next to each other over 2^40 in magnitude, zero rows among them: every row has its own scale."""
    rows, table, target = make(70, 500, 40, F32, seed=3)
    f = 2.0 ** torch.randint(-20, 20, (500, 1), generator=torch.Generator().manual_seed(1)).float().to(DEV)
    f[7] = 0
    table = table * f
    rows = rows * 1e-7
    r = catalogue.softmax_xent(rows, table, target, scale=10.0, reduction="none")
    want = oracle(rows, table, target, scale=10.0, reduction="none")
    check(r, want, F32, 40, "none", 70, 500)
    # and for the small rows of the table by themselves
    small = f[:, 0].cpu() <= 1
    tol = 1e-4 * want["terms"]["table"][small] + 1e-30
    assert ((r.d_table.double().cpu() - want["d_table"])[small].abs() <= tol).all()


@pytest.mark.parametrize("dtype,f", [(F16, 2.0 ** -18), (BF16, 2.0 ** -120), (F16, 2.0 ** 9), (F32, 2.0 ** -60)])
@pytest.mark.parametrize("n", [3, 60])
def test_xent_at_the_ends_of_a_type(n, dtype, f):
    """Tables of f16's subnormal values, or near its largest; of bfloat16's and fp32's small ones: the scale brings the logits back."""
    rows, table, target = make(n, 400, 40, F32, seed=2)
    table = (table * f).to(dtype)
    rows = rows.to(dtype)
    scale = 10.0 / f if dtype != BF16 else 2.0 ** 100
    r = catalogue.softmax_xent(rows, table, target, scale=scale, reduction="none")
    want = oracle(rows, table, target, scale=scale, reduction="none")
    assert want["zmax"] > 1 or dtype == BF16      # they are
    fine = dtype == F32 or f > 1        # gradients of the other tables leave the type: held to the fp32 results alone
    if fine:
        check(r, want, dtype, 40, "none", n, 400)
    else:
        check(r._replace(d_rows=None), want, dtype, 40, "none", n, 400)


def test_xent_strides_and_alignment():
    rows, table, target = make(50, 333, 30, F32, seed=9)
    base = catalogue.softmax_xent(rows, table, target, scale=5.0)
    for pad, off in ((2, 1), (3, 0), (2, 2), (98, 5)):
        wide_r = torch.full((50, 30 + pad + off), math.nan, device=DEV)
        wide_t = torch.full((333, 30 + pad + off), math.nan, device=DEV)
        wide_r[:, off:off + 30], wide_t[:, off:off + 30] = rows, table
        r = catalogue.softmax_xent(wide_r[:, off:off + 30], wide_t[:, off:off + 30], target, scale=5.0)
        for a, b in zip(base[:4], r[:4]):
            assert torch.equal(a, b)
    lone = catalogue.softmax_xent(rows[:1].expand(1, 30), table, target[:1], scale=5.0, grad=False)
    assert lone.d_rows is None and torch.isfinite(lone.loss)


def test_xent_is_the_same_every_time_and_in_loss_only_form():
    rows, table, target = make(700, 3001, 100, F32, seed=4)
    a = catalogue.softmax_xent(rows, table, target, scale=10.0)
    b = catalogue.softmax_xent(rows, table, target, scale=10.0)
    for x, y in zip(a[:4], b[:4]):
        assert torch.equal(x, y)
    c = catalogue.softmax_xent(rows, table, target, scale=10.0, grad=False)
    assert torch.equal(a.loss, c.loss) and torch.equal(a.lse, c.lse)


def test_xent_gradient_against_differences():
    """Central differences of the fp32 loss itself: h = 2^-6, so the loss's rounding (2^-24 of it each side) moves the quotient by
    2^-24 * 2 |L| / 2h and the third derivative by h^2 / 6 * scale^3 |v|^3."""
    n, c, d = 6, 90, 20
    rows, table, target = make(n, c, d, F32, seed=11)
    kw = dict(scale=2.0, reduction="sum")
    r = catalogue.softmax_xent(rows, table, target, **kw)
    h = 2.0 ** -6
    for t, grad, other in ((rows, r.d_rows, table), (table, r.d_table, rows)):
        top = other.norm(dim=1).max().item()
        tol = (2 ** -21) * r.loss.item() / h + h * h / 6 * (2.0 * top) ** 3 * n
        for i, k in ((0, 0), (3, 7), (5, 19)):
            keep = t[i, k].item()
            t[i, k] = keep + h
            up, x1 = catalogue.softmax_xent(rows, table, target, grad=False, **kw).loss.item(), t[i, k].item()
            t[i, k] = keep - h
            dn, x0 = catalogue.softmax_xent(rows, table, target, grad=False, **kw).loss.item(), t[i, k].item()
            t[i, k] = keep
            assert abs((up - dn) / (x1 - x0) - grad[i, k].item()) <= tol


def _codes(x):
    x = x.float().cpu().numpy()
    top = np.abs(x).max(1).astype(np.float32)
    inv = np.zeros_like(top)
    np.divide(np.float32(127), top, out=inv, where=top > 0)
    return np.rint(x * inv[:, None]).astype(np.int64), (top / np.float32(127)).astype(np.float32)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 50), (33, 64), (16, 65), (17, 100), (1000, 128), (5, 129), (9, 515), (4, 4096), (2, 20001)])
def test_rows_to_codes_and_back(n, k, dtype):
    x = (torch.randn(n, k, generator=torch.Generator().manual_seed(k)) * 3).to(dtype).to(DEV)
    if n > 2:
        x[1] = 0
    q, s = _codes(x)
    r = catalogue.quantize_rows(x)
    assert np.array_equal(r.codes[:, :k].cpu().numpy(), q) and not r.codes[:, k:].any()
    assert np.array_equal(r.scale.cpu().numpy(), s)
    want = (q * s[:, None].astype(np.float64))
    for t in (F32, F16, BF16):
        got = r.dequantize(t)
        assert torch.equal(got.cpu(), torch.from_numpy(q.astype(np.float32) * s[:, None]).to(t))
    assert np.abs(want - x.double().cpu().numpy()).max() <= 0.5001 * s.max()      # half a step, and the factor's rounding


def test_rows_that_codes_cannot_hold():
    x = torch.ones(5, 40, device=DEV)
    x[0, 3], x[1, 39], x[2, 0] = math.inf, math.nan, -math.inf
    x[3] *= 1e-42      # subnormal
    r = catalogue.quantize_rows(x)
    assert torch.isnan(r.scale[:3]).all() and not r.codes[:3].any()
    assert (r.codes[3, :40] == 127).all() and r.scale[3] > 0 and (r.codes[4, :40] == 127).all()
    s = catalogue.int8_scores(r, catalogue.quantize_rows(torch.ones(7, 40, device=DEV)))
    assert torch.isnan(s[:3]).all() and torch.isfinite(s[3:]).all()


@pytest.mark.parametrize("normalize", [False, True])
def test_rows_strided_and_normalised(normalize):
    wide = torch.randn(21, 130, generator=torch.Generator().manual_seed(2)).to(DEV)
    x = wide[:, 3:103]
    r = catalogue.quantize_rows(x, normalize=normalize)
    q, s = _codes(x)
    assert np.array_equal(r.codes[:, :100].cpu().numpy(), q)
    want = s / np.linalg.norm(x.double().cpu().numpy(), axis=1) if normalize else s
    # the norm: a 100-term fp32 sum, its root and reciprocal (a hardware estimate of 2^-22), one product
    np.testing.assert_allclose(r.scale.cpu().numpy(), want, rtol=(100 / 2 + 8) * 2.0 ** -24 if normalize else 0)


@pytest.mark.parametrize("m,c,k", [(1, 1, 1), (1, 17, 50), (2, 1000, 64), (31, 129, 100), (32, 128, 128), (33, 127, 128), (1, 70001, 128), (65, 130, 36),
                                   (200, 333, 129), (129, 1000, 640), (300, 513, 64), (4, 900, 4096), (130, 260, 4096), (33, 40, 20000)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_scores(m, c, k, dtype):
    g = torch.Generator().manual_seed(m + c + k)
    x, t = torch.randn(m, k, generator=g).to(DEV), torch.randn(c, k, generator=g).to(DEV)
    rb, cb = torch.randn(m, generator=g), torch.randn(c, generator=g)
    (qx, sx), (qt, st) = _codes(x), _codes(t)
    exact = (qx @ qt.T) * sx[:, None].astype(np.float64) * st[None, :].astype(np.float64)
    table = catalogue.quantize_rows(t)
    for biases in (False, True):
        want = exact + (rb.double().numpy()[:, None] + cb.double().numpy()[None, :] if biases else 0)
        kw = dict(row_bias=rb.to(DEV), col_bias=cb.to(DEV)) if biases else {}
        got = catalogue.int8_scores(x, table, dtype=dtype, **kw)
        # the sum's conversion, two products, two additions: 5 fp32 roundings of the parts; one of the output
        tol = 5 * 2.0 ** -24 * (np.abs(exact) + (np.abs(rb.numpy())[:, None] + np.abs(cb.numpy())[None, :] if biases else 0)) + U[dtype] * np.abs(want) + 1e-30
        if dtype == F16:
            tol = tol + 2.0 ** -25
        assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()
    assert torch.equal(got, catalogue.int8_scores(catalogue.quantize_rows(x), table, dtype=dtype, **kw))


@pytest.mark.parametrize("m,c,k,pad,off", [(1000, 8001, 100, 0, 0), (4100, 2000, 50, 0, 0), (2050, 4100, 128, 4, 4), (2000, 3999, 64, 30, 13),
                                           (3000, 2244, 20, 0, 0), (300, 30000, 100, 0, 0), (3000, 2200, 300, 0, 0),
                                           (4200, 4301, 300, 0, 0), (4100, 4356, 200, 4, 0)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_scores_of_many_rows(m, c, k, pad, off, dtype):
    """Launches of many workgroups: rows that start anywhere in a line, in rows of a wider matrix, whose other columns stay."""
    g = torch.Generator(device=DEV).manual_seed(m)
    x, t = catalogue.quantize_rows(torch.randn(m, k, generator=g, device=DEV)), catalogue.quantize_rows(torch.randn(c, k, generator=g, device=DEV))
    rb, cb = torch.randn(m, generator=g, device=DEV), torch.randn(c, generator=g, device=DEV)
    wide = torch.full((m, c + pad + off), 7.0, device=DEV, dtype=dtype)
    out = wide[:, off:off + c]
    catalogue.int8_scores(x, t, row_bias=rb, col_bias=cb, out=out)
    exact = (x.codes[:, :k].double() @ t.codes[:, :k].double().t()) * x.scale[:, None].double() * t.scale[None].double()
    want = exact + rb[:, None].double() + cb[None].double()
    tol = 5 * 2.0 ** -24 * (exact.abs() + rb.abs()[:, None] + cb.abs()[None]) + U[dtype] * want.abs() + (2.0 ** -25 if dtype == F16 else 1e-30)
    assert ((out.double() - want).abs() <= tol).all()
    assert (wide[:, :off] == 7).all() and (wide[:, off + c:] == 7).all()


@pytest.mark.parametrize("m", [3, 40])
def test_scores_write_only_their_columns(m):
    x, t = torch.randn(m, 30, device=DEV), torch.randn(45, 30, device=DEV)
    wide = torch.full((m + 1, 60), 7.0, device=DEV)
    out = wide[:m, 5:50]
    got = catalogue.int8_scores(x, catalogue.quantize_rows(t), out=out)
    assert got is out and torch.equal(out, catalogue.int8_scores(x, catalogue.quantize_rows(t)))
    assert (wide[:, :5] == 7).all() and (wide[:, 50:] == 7).all() and (wide[m] == 7).all()


def test_offsets_past_32_bits():
    """A table of codes of 2.2 GB, scores of 9 GB, and a table whose rows lie 4.8 GB apart from first to last."""
    g = torch.Generator(device=DEV).manual_seed(1)
    c = 17_000_001
    big = catalogue.Int8Rows(torch.randint(-127, 128, (c, 128), generator=g, device=DEV, dtype=torch.int8), torch.rand(c, generator=g, device=DEV), 128)
    x = torch.randn(2, 128, generator=g, device=DEV)
    s = catalogue.int8_scores(x, big)
    last = catalogue.Int8Rows(big.codes[-1000:].clone(), big.scale[-1000:].clone(), 128)
    assert torch.equal(s[:, -1000:], catalogue.int8_scores(x, last))
    back = catalogue.Int8Rows(big.codes[-4:].clone(), big.scale[-4:].clone(), 128).dequantize()
    assert torch.equal(big.dequantize(BF16)[-4:], back.to(BF16))
    del big, s
    m, c = 70_000, 33_001
    x, t = (catalogue.quantize_rows(torch.randn(n, 30, generator=g, device=DEV)) for n in (m, c))
    s = catalogue.int8_scores(x, t)
    few = catalogue.Int8Rows(x.codes[-20:].clone(), x.scale[-20:].clone(), 30)
    assert torch.equal(s[-20:], catalogue.int8_scores(few, t))
    del s
    c = 200_000
    wide = torch.empty(c, 12_000, dtype=BF16, device=DEV)
    table = wide[:, :32]
    table.copy_(torch.randn(c, 32, generator=g, device=DEV) / 6)
    target = torch.tensor([c - 1, 5, c - 3, 7, 9, c // 2], dtype=torch.int32, device=DEV)
    rows = table[target.long()] * 2
    r = catalogue.softmax_xent(rows, table, target, scale=10.0)
    want = catalogue.softmax_xent(rows, table.contiguous(), target, scale=10.0)
    for a, b in zip(r[:4], want[:4]):
        assert torch.equal(a, b)


def test_codes_kept_elsewhere():
    x = torch.randn(9, 70, device=DEV)
    r = catalogue.quantize_rows(x)
    again = catalogue.Int8Rows(r.codes.clone(), r.scale.clone(), 70)
    t = catalogue.quantize_rows(torch.randn(50, 70, device=DEV))
    assert torch.equal(catalogue.int8_scores(again, t), catalogue.int8_scores(r, t))
    for codes, scale, k in ((r.codes[:, :70], r.scale, 70), (r.codes, r.scale, 60), (r.codes, r.scale, 129), (r.codes, r.scale[:8], 70),
                            (r.codes[:, :64], r.scale, 64), (r.codes, r.scale, 0)):
        with pytest.raises(ValueError):
            catalogue.Int8Rows(codes, scale, k)
    for codes, scale, k in ((r.codes.float(), r.scale, 70), (r.codes, r.scale.double(), 70), (r.codes, None, 70), (r.codes.cpu(), r.scale, 70)):
        with pytest.raises(TypeError):
            catalogue.Int8Rows(codes, scale, k)


def test_calls_that_are_refused():
    rows, table, target = make(4, 50, 20, F32)
    f = catalogue.softmax_xent
    for call, error in ((lambda: f(rows, table.half(), target), TypeError), (lambda: f(rows, table[:, :10], target), ValueError),
                        (lambda: f(rows, table, target.long()), TypeError), (lambda: f(rows, table, target[:3]), ValueError),
                        (lambda: f(rows, table, None), TypeError), (lambda: f(rows, table, target, bias=torch.zeros(49, device=DEV)), ValueError),
                        (lambda: f(rows, table, target, weight=torch.zeros(4)), TypeError), (lambda: f(rows, table, target, reduction="max"), ValueError),
                        (lambda: f(rows, table, target, scale=math.inf), ValueError), (lambda: f(rows[:0], table, target[:0]), ValueError),
                        (lambda: f(rows.t(), table, target), ValueError), (lambda: f(rows[:1].expand(4, 20), table, target), ValueError),
                        (lambda: f(torch.zeros(4, 129, device=DEV), torch.zeros(50, 129, device=DEV), target), ValueError),
                        (lambda: f(rows.double(), table.double(), target), TypeError), (lambda: f(rows[0], table, target), ValueError)):
        with pytest.raises(error):
            call()
    t = catalogue.quantize_rows(table)
    g = catalogue.int8_scores
    for call, error in ((lambda: g(rows, table), TypeError), (lambda: g(rows[:, :19].contiguous(), t), ValueError),
                        (lambda: g(rows, t, out=torch.empty(4, 49, device=DEV)), ValueError), (lambda: g(rows, t, dtype=torch.float64), TypeError),
                        (lambda: g(rows, t, row_bias=torch.zeros(5, device=DEV)), ValueError), (lambda: g(rows, t, out=torch.empty(4, 50)), TypeError),
                        (lambda: g(rows.double(), t), TypeError), (lambda: t.dequantize(torch.int8), TypeError)):
        with pytest.raises(error):
            call()


def test_scores_of_rows_that_codes_cannot_hold():
    t = catalogue.quantize_rows(torch.randn(1000, 40, device=DEV))
    for m in (3, 40):       # coded in the launch, and before it
        x = torch.randn(m, 40, device=DEV)
        x[1, 7] = math.nan
        s = catalogue.int8_scores(x, t)
        assert torch.isnan(s[1]).all() and torch.isfinite(s[0]).all() and torch.isfinite(s[2:]).all()


def test_scores_of_no_rows():
    t = catalogue.quantize_rows(torch.randn(45, 30, device=DEV))
    assert catalogue.int8_scores(torch.empty(0, 30, device=DEV), t).shape == (0, 45)


def test_calls_on_two_streams_and_in_graphs():
    """Two calls in flight on two streams, and two captured graphs, replayed with eager work between, give the eager results."""
    sets = [make(300, 2000, 100, F32, seed=s) for s in (1, 2)]

    def work(s):
        r = catalogue.softmax_xent(*s, scale=10.0)
        return [r.loss, r.lse, r.d_rows, r.d_table, catalogue.int8_scores(s[0], catalogue.quantize_rows(s[1]))]

    want = [work(s) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s, st in zip(sets, streams):
        with torch.cuda.stream(st):
            for _ in range(5):
                r = work(s)
            got.append(r)
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    graphs, outs = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(work(s))
        graphs.append(g)
    for _ in range(4):
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, b in zip(want, outs):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
        for o in outs:
            for x in o:
                x.zero_()
        work(sets[0])


def test_train_then_serve():
    """The head as a program uses it: SGD on the whole-catalogue loss, then the table to 8 bits and the items ranked."""
    g = torch.Generator().manual_seed(0)
    users, items, d = 64, 500, 50
    liked = torch.randint(items, (users,), generator=g).int().to(DEV)
    u = (0.1 * torch.randn(users, d, generator=g)).to(DEV)
    v = (0.1 * torch.randn(items, d, generator=g)).to(DEV)
    for _ in range(60):
        r = catalogue.softmax_xent(u, v, liked, scale=10.0, reduction="sum")
        u -= 0.02 * r.d_rows
        v -= 0.02 * r.d_table
    z = 10 * (u.double() @ v.double().t())
    ref = torch.nn.functional.cross_entropy(z, liked.long(), reduction="sum")
    assert abs(catalogue.softmax_xent(u, v, liked, scale=10.0, reduction="sum", grad=False).loss.item() - ref.item()) <= 1e-3 * max(1.0, ref.item())
    s = catalogue.int8_scores(u, catalogue.quantize_rows(v))
    exact = (u.double() @ v.double().t())
    step = (u.abs().amax(1, keepdim=True) / 127 * v.abs().sum(1)[None] + v.abs().amax(1)[None] / 127 * u.abs().sum(1, keepdim=True)).double()
    assert ((s.double() - exact).abs() <= 0.51 * step + 1e-6).all()      # half a step of either side, and both at once
