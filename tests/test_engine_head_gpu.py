"""GPU: the catalogue head on an engine's own tables -- the logits are the engine's own scores, ids that no table holds, refusals."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from nncf_amd.engine import Engine  # noqa: E402


def engine(d=50, loss="skip-gram", gamma=10.0, norm=False, bias=None):
    e = Engine(200, 333, d, 64, 2, loss, gamma, 1.0, 0.0, 0.1, norm, norm, seed=1, init_scale=0.5, interaction_bias=bias)
    g = torch.Generator().manual_seed(3)
    for k in ("ub", "cb"):
        if e.bias is not None and e.bias[k] is not None:
            e.bias[k].copy_(torch.randn(e.bias[k].numel(), generator=g))
    return e


@pytest.mark.parametrize("bias", [None, "user", "item", "both"])
@pytest.mark.parametrize("loss,gamma,scale", [("log-loss", 10.0, None), ("log-loss", 3.5, None), ("max-margin", 0.1, 4.0), ("skip-gram", 10.0, 1.0)])
def test_the_head_learns_the_scores_that_the_engine_ranks_by(loss, gamma, scale, bias):
    """Logits = scale * predict_scores(uid, all items): the user's bias that these hold adds the same to a row's logits and drops out.

    predict_scores is a sum of d = 50 products below 0.25 and two biases in fp32, |error| <= (d + 4) 2^-24 * (d / 4 + |b|); the head's own
    logits are within (3 * 2^-22 + (d + 2) 2^-24) of the same sizes, times the scale."""
    e = engine(loss=loss, gamma=gamma, bias=bias)
    r = np.random.RandomState(0)
    uid, cid = r.randint(200, size=77), r.randint(333, size=77)
    got = e.softmax_xent(uid, cid, reduction="sum", scale=scale)
    k = gamma if scale is None else scale
    d = 50
    scores = e.predict_scores(e.ids(uid), torch.arange(333, dtype=torch.int32, device="cuda")).double().cpu()
    z = (k * scores).requires_grad_()
    loss64 = torch.nn.functional.cross_entropy(z, torch.as_tensor(cid), reduction="sum")
    loss64.backward()
    size = d / 4 + 2 * max([0.0] + [e.bias[n].abs().max().item() for n in ("ub", "cb") if e.bias is not None and e.bias[n] is not None])
    z_err = k * size * (3 * 2.0 ** -22 + 2 * (d + 4) * 2.0 ** -24) + 2.0 ** -22 * 64
    assert abs(got.loss.item() - loss64.item()) <= 77 * 2 * z_err
    U, V = e.U[:, :d].double().cpu(), e.V[:, :d].double().cpu()
    coef = k * z.grad                                    # d loss / d score
    p_err = 2 * z_err + 2.0 ** -20
    assert (got.d_rows.double().cpu() - coef @ V).abs().max().item() <= 2 * k * 0.5 * p_err      # sum_j |p - [t]| <= 2, |v| <= 0.5
    assert (got.d_table.double().cpu() - coef.t() @ U[uid]).abs().max().item() <= 77 * k * 0.5 * p_err
    if bias in ("item", "both"):
        assert (got.d_bias.double().cpu() - coef.sum(0)).abs().max().item() <= 77 * k * p_err
    else:
        assert got.d_bias is None


def test_the_bias_gradient_against_differences_of_the_engine_s_own_loss():
    """h = 2^-5: the loss's rounding moves the quotient by 2^-23 |L| / 2h, the third derivative by h^2 / 6 * scale^3 / 4 a link at most
    (the third cumulant of an indicator is below 1 / 4)."""
    e = engine(loss="log-loss", gamma=2.0, bias="item")
    uid, cid = np.arange(6), np.array([5, 7, 5, 9, 300, 11])
    r = e.softmax_xent(uid, cid, reduction="sum")
    h = 2.0 ** -5
    for j in (5, 11, 40):
        keep = e.bias["cb"][j].item()
        at = []
        for s in (h, -h):
            e.bias["cb"][j] = keep + s
            at.append((e.softmax_xent(uid, cid, reduction="sum", grad=False).loss.item(), e.bias["cb"][j].item()))
        e.bias["cb"][j] = keep
        slope = (at[0][0] - at[1][0]) / (at[0][1] - at[1][1])
        assert abs(slope - r.d_bias[j].item()) <= 2.0 ** -23 * (6 * 10 + r.loss.item()) / (2 * h) + 6 * h * h / 6 * 8 / 4


def test_a_margin_is_no_scale():
    e = engine(loss="max-margin", gamma=0.1)
    with pytest.raises(ValueError, match="margin"):
        e.softmax_xent([1, 2], [3, 4])
    assert torch.isfinite(e.softmax_xent([1, 2], [3, 4], scale=2.0).loss)


@pytest.mark.parametrize("bias", [None, "both"])
@pytest.mark.parametrize("norm", [False, True])
def test_ids_that_the_tables_do_not_hold(norm, bias):
    """Past the tables: NaN, for that user or item alone.  Negative: a row of zeros without a bias.  Nothing is read out of range."""
    e = engine(norm=norm, bias=bias)
    top = 2 ** 31 - 1
    uid, cid = np.array([3, 200, -1, 7, top, -2 ** 31]), np.array([0, 333, 5, -1, top, 332, -2 ** 31])
    known_u, known_c = np.array([0, 3]), np.array([0, 2, 5])         # places of ids that are there
    zero_u, zero_c = np.array([2, 5]), np.array([3, 6])
    want = e.predict_scores_int8(uid[known_u], cid[known_c])
    for items in (None, e.quantize_items(cid)):
        s = e.predict_scores_int8(uid, cid, items=items)
        assert torch.equal(s[known_u][:, known_c], want)
        assert torch.isnan(s[[1, 4]]).all() and torch.isnan(s[:, [1, 4]]).all()
        ub, cb = (torch.zeros(len(i), device="cuda") if bias is None else e.bias[k][torch.as_tensor(i, device="cuda")]
                  for k, i in (("ub", uid[known_u]), ("cb", cid[known_c])))
        assert torch.equal(s[zero_u][:, known_c], cb.expand(2, 3)) and torch.equal(s[known_u][:, zero_c], ub[:, None].expand(2, 2))
        assert not s[zero_u][:, zero_c].any()


def test_links_that_the_tables_do_not_hold():
    e = engine(bias="both")
    uid, cid = np.array([3, 200, 5, 2 ** 31 - 1]), np.array([1, -1, 7, -1])
    r = e.softmax_xent(uid, cid, reduction="none")       # such a user in a link that takes no part
    want = e.softmax_xent(uid[[0, 2]], cid[[0, 2]], reduction="none")
    assert torch.equal(r.loss[[0, 2]], want.loss) and not r.loss[[1, 3]].any() and not r.d_rows[[1, 3]].any()
    assert torch.isfinite(r.d_table).all()
    for n in (3, 40):                                    # few rows, many rows
        u, c = np.arange(n), np.arange(n)
        u[1], c[2] = 200, 333
        r = e.softmax_xent(u, c, reduction="none")
        assert torch.isnan(r.loss[1:3]).all() and torch.isfinite(r.loss[0]) and torch.isfinite(r.loss[3:]).all()
        assert torch.isnan(r.d_rows[1:3]).all() and torch.isfinite(r.d_rows[3:]).all() and torch.isnan(r.d_table).all()


def test_items_in_8_bits_of_another_number_than_the_ids():
    e = engine()
    coded = e.quantize_items(np.arange(20))
    with pytest.raises(ValueError, match="20 items"):
        e.predict_scores_int8([1, 2], np.arange(19), items=coded)
    with pytest.raises(ValueError, match="20 items"):
        e.predict_scores_int8([1, 2], np.arange(333), items=coded)


@pytest.mark.parametrize("d,n", [(50, 1), (100, 33), (128, 1000)])
def test_gathered_rows_and_biases(d, n):
    e = engine(d, bias="both")
    ids = torch.randint(-3, 210, (n,), generator=torch.Generator().manual_seed(n)).int().cuda()
    rows, b = e._rows(e.U, ids, e.bias["ub"])
    there, past = (ids >= 0) & (ids < 200), ids >= 200
    at = torch.where(there, ids, 0).long()
    assert torch.equal(rows[there], e.U[at][there]) and torch.equal(b[there], e.bias["ub"][at][there])
    assert torch.isnan(rows[past]).all() and torch.isnan(b[past]).all()
    assert not rows[ids < 0].any() and not b[ids < 0].any()
    assert e._rows(e.U, ids)[1] is None and e._rows(e.U, ids[:0], e.bias["ub"])[0].shape == (0, e.dim_p)
