"""GPU: the framework's own paths on the catalogue head -- Engine.softmax_xent / predict_scores_int8, the evaluator's 8-bit scores."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

import torch  # noqa: E402

from nncf_amd import _lib, synthetic  # noqa: E402
from nncf_amd.conf import get_conf  # noqa: E402
from nncf_amd.data_utils import get_data  # noqa: E402
from nncf_amd.engine import Engine  # noqa: E402
from nncf_amd.model_framework import get_model  # noqa: E402
from nncf_amd.objectives import Evaluator  # noqa: E402


def engine(d=50, norm=False, bias=None):
    e = Engine(200, 333, d, 64, 2, "skip-gram", 10.0, 1.0, 0.0, 0.1, norm, norm, seed=1, init_scale=0.5, interaction_bias=bias)
    g = torch.Generator().manual_seed(3)
    if bias:
        for k in ("ub", "cb"):
            if e.bias[k] is not None:
                e.bias[k].copy_(torch.randn(e.bias[k].numel(), generator=g))
    return e


@pytest.mark.parametrize("d", [50, 100])
@pytest.mark.parametrize("bias", [None, "both"])
def test_engine_softmax_xent(d, bias):
    e = engine(d, bias=bias)
    r = np.random.RandomState(0)
    uid, cid = r.randint(200, size=77), r.randint(333, size=77)
    got = e.softmax_xent(uid, cid, reduction="sum")
    U, V = e.U[:, :d].double().cpu().requires_grad_(), e.V[:, :d].double().cpu().requires_grad_()
    u = U[uid]
    u.retain_grad()
    cb = torch.zeros(333, dtype=torch.float64) if bias is None else e.bias["cb"].double().cpu()
    cb.requires_grad_()
    z = e.cfg.loss_gamma * (u @ V.t()) + cb
    loss = torch.nn.functional.cross_entropy(z, torch.as_tensor(cid), reduction="sum")
    loss.backward()
    # logits to 2^-20 of sum |u v| (two planes of 22 bits, d sums): their size here is below 10 * 100 * 0.25
    z_err = 10 * d * 0.25 * (3 * 2.0 ** -22 + (d + 2) * 2.0 ** -24) + 2.0 ** -22 * 64
    assert abs(got.loss.item() - loss.item()) <= 77 * 2 * z_err
    for a, b in ((got.d_rows, u.grad), (got.d_table, V.grad)):
        assert (a.double().cpu() - b).abs().max().item() <= 10 * 77 * 0.5 * (2 * z_err + 2.0 ** -20)
    if bias:
        assert (got.d_bias.double().cpu() - cb.grad).abs().max().item() <= 77 * (2 * z_err + 2.0 ** -20)
    before = e.U.clone(), e.V.clone()
    assert e.softmax_xent(uid, cid, grad=False).d_rows is None
    assert torch.equal(before[0], e.U) and torch.equal(before[1], e.V)


def test_engine_refuses_rows_it_would_normalise():
    with pytest.raises(ValueError, match="normalises"):
        engine(norm=True).softmax_xent([1, 2], [3, 4])
    with pytest.raises(ValueError, match="users"):
        engine().softmax_xent([1, 2], [3])


@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("bias", [None, "both"])
@pytest.mark.parametrize("users", [3, 150])
def test_engine_scores_in_8_bits(norm, bias, users):
    e = engine(50, norm=norm, bias=bias)
    uid, cid = torch.arange(users).int().cuda(), torch.arange(332, -1, -1).int().cuda()
    full, got = e.predict_scores(uid, cid), e.predict_scores_int8(uid, cid)
    u, v = e.U[uid.long(), :50].double(), e.V[cid.long(), :50].double()
    if norm:
        u, v = (x / x.norm(dim=1, keepdim=True) for x in (u, v))
    # half a step of either side against the other's values, and of both at once
    a, b = u.abs().amax(1, keepdim=True) / 254, v.abs().amax(1)[None] / 254
    tol = a * v.abs().sum(1)[None] + b * u.abs().sum(1, keepdim=True) + 50 * a * b + 1e-5
    assert ((full.double() - got.double()).abs() <= tol).all()
    coded = e.quantize_items(cid)
    assert torch.equal(got, e.predict_scores_int8(uid, cid, items=coded))


@pytest.mark.parametrize("model,norm", [("mf", False), ("mf", True), ("basic_embedding", False)])
def test_evaluator_ranks_by_8_bit_scores(model, norm):
    """eval_scores = 'int8' ranks exactly the matrix that predict_scores_int8 gives, chunk by chunk."""
    data = synthetic.make_citeulike_like(users=90, items=120, train_links=1500, seed=3, content_len=12, vocab=80)
    pd = {"reset_after_getconf": True, "max_epoch": 1, "loss": "skip-gram", "num_negatives": 0, "neg_loss_weight": 16, "loss_gamma": 10,
          "learn_rate": 0.1, "neg_dist": "unigram", "neg_sampling_power": 1, "batch_size_p": 64, "user_dim": 24, "item_dim": 24, "word_dim": 24,
          "chop_size": 4, "u_reg": 0., "eval_topk": 7, "optimizer": "sgd", "eval_scores": "int8"}
    conf = get_conf("synthetic", "best", pd, model_choice=model)
    conf.emb_normalization = norm
    helper = get_data(dict(data), conf, rand_seed=5)
    head = get_model(conf, helper, model, seed=2)["model_neg_shared"]
    ev = Evaluator(helper, helper.data_spec, conf)
    got = ev._whole(head, "train", 7, user_chunk=32)
    metrics, valid = ev._dev["metrics"].clone(), ev._dev["valid"].clone()
    items, ptr, idx = ev._dev["train"]
    e = head.predict_engine()
    scores = e.predict_scores_int8(ev._dev["users"], items)
    m2, v2 = torch.zeros_like(metrics), torch.zeros_like(valid)
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    _lib.check(_lib.lib().nncf_eval_topk(p(scores), 90, items.numel(), items.numel(), p(ptr), p(idx), 7, p(m2), p(v2), _lib.stream_ptr()))
    assert torch.equal(valid, v2) and torch.equal(metrics.view(-1, 3)[v2.bool()], m2.view(-1, 3)[v2.bool()])
    assert got["users"] == int(v2.sum())
    ev.eval_scores = "f32"
    assert abs(ev._whole(head, "train", 7)["recall@7"] - got["recall@7"]) <= 0.2      # 8 bits order near ties differently, not the list


def test_unknown_scores_are_refused():
    conf = get_conf("synthetic", "best", {"reset_after_getconf": True, "user_dim": 8, "item_dim": 8, "eval_scores": "int4"}, model_choice="mf")
    helper = get_data(dict(synthetic.make_citeulike_like(users=30, items=30, train_links=200, seed=1, content_len=5, vocab=20)), conf, rand_seed=5)
    with pytest.raises(AssertionError, match="eval_scores"):
        Evaluator(helper, helper.data_spec, conf)
