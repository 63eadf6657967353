"""Losses of a language model head without its logits (train/head_loss.py): the CPU statement and the kernels against 64 bits, refusals, left-out rows."""
import math

import pytest
import torch

import head_loss_plain as P
from volta_engine_b200.train import head_loss as L


def make(rows, hidden, vocab, topk=0, x="bf16", head="bf16", seed=0, left_out=0.0, device="cpu", spread=2.5):
    """-> (x, head, targets, dloss): a label's logit raised by up to 15; a teacher close to the states; some rows left out."""
    g = torch.Generator().manual_seed(seed)
    dt = {"bf16": torch.bfloat16, "fp32": torch.float32, "fp64": torch.float64}
    w = (torch.randn(vocab, hidden, generator=g) * spread / math.sqrt(hidden)).to(dt[head])
    labels = torch.randint(0, vocab, (rows,), generator=g)
    xs = torch.randn(rows, hidden, generator=g) + 6 * torch.rand(rows, 1, generator=g) * torch.nn.functional.normalize(w[labels].float(), dim=1)
    out = torch.randperm(rows, generator=g)[: int(rows * left_out)]
    dloss = torch.rand(rows, generator=g) + 0.5
    if not topk:
        labels[out] = -100
        targets = (labels,)
    else:
        lp = torch.log_softmax((xs + 0.9 * torch.randn(rows, hidden, generator=g)) @ w.float().t(), 1)
        logp, ids = lp.topk(topk, 1)
        tail = (1 - logp.exp().sum(1)).clamp(min=1e-9).log()
        ids = ids.int()
        ids[out] = -1
        if topk > 2:
            ids[1::5, 1:3] = -1
        targets = (ids, logp, tail)
    return xs.to(dt[x]).to(device), w.to(device), tuple(t.to(device) for t in targets), dloss.to(device)


def run(x, head, targets, dloss, softcap=0.0, want_dx=True, want_dhead=True):
    f, b = (L.head_cross_entropy, L.head_cross_entropy_backward) if len(targets) == 1 else (L.head_kl, L.head_kl_backward)
    loss, stats = f(x, head, *targets, softcap=softcap)
    dx, dhead = b(x, head, *targets, stats, dloss.to(stats.dtype), softcap=softcap, want_dx=want_dx, want_dhead=want_dhead)
    return {"loss": loss, "stats": stats, "dx": dx, "dhead": dhead}


def hold(got, x, head, targets, dloss, softcap, only=("loss", "stats", "dx", "dhead")):
    w = P.wanted(x, head, targets, dloss, softcap)
    mass = 1.0 if len(targets) == 1 else float(torch.logaddexp(targets[1].double().logsumexp(1), targets[2].double()).exp().max()) * (
        1 + float((targets[1].double().exp() * targets[1].double().abs()).sum(1).max()))
    tol = P.allowed(w, x, head, dloss, mass)
    for k in only:
        a, b = got[k].double(), w[k]
        assert a.shape == b.shape, k
        same = a == b                               # (infinities among the statistics)
        over = ((a - b).abs() > tol[k]) & ~same
        assert not bool(over.any()) and not bool(torch.isnan(a).any()), (k, float(((a - b).abs() / tol[k])[~same].max()), int(over.sum()))
    return w


# ------------------------------------------------------------------------------------------------ CPU
@pytest.mark.parametrize("topk", [0, 1, 5])
@pytest.mark.parametrize("softcap", [0.0, 4.0])
def test_statement_is_the_formula_and_its_derivative(topk, softcap):
    x, head, targets, dloss = make(7, 12, 33, topk, "fp64", "fp64", seed=topk, left_out=0.3)
    if topk:
        targets = (targets[0], targets[1].double(), targets[2].double())
    got = run(x, head, targets, dloss.double(), softcap)
    w = P.wanted(x, head, targets, dloss, softcap)
    for k in ("loss", "stats", "dx", "dhead"):
        assert torch.allclose(got[k], w[k], rtol=1e-9, atol=1e-12), k
    # and by differences, through the differentiable call
    fn = L.head_cross_entropy_loss if not topk else L.head_kl_loss
    assert torch.autograd.gradcheck(lambda a, b: fn(a, b, *targets, softcap), (x.clone().requires_grad_(), head.clone().requires_grad_()))


def test_statement_agrees_with_the_tools_divergence():
    from volta_engine_b200.tools.ppl import kl_topk, topk_teacher
    g = torch.Generator().manual_seed(3)
    x, head = torch.randn(9, 16, generator=g), torch.randn(50, 16, generator=g)
    ids, logp, tail = topk_teacher((x + 0.5 * torch.randn(9, 16, generator=g)) @ head.t(), 6)
    assert torch.allclose(L.head_kl(x, head, ids, logp, tail)[0], kl_topk(x @ head.t(), ids, logp, tail), rtol=1e-4, atol=1e-5)


def test_statement_edges():
    x, head = torch.randn(3, 4, generator=torch.Generator().manual_seed(0)), torch.randn(5, 4, generator=torch.Generator().manual_seed(1))
    # left-out rows: zeros, and what stands in them does not matter
    y = x.clone()
    y[1] = math.nan
    lab = torch.tensor([2, -1, 4])
    a, b = run(x, head, (lab,), torch.ones(3)), run(y, head, (lab,), torch.ones(3))
    for k in a:
        assert torch.equal(a[k], b[k]) and not torch.isnan(a[k]).any()
    assert a["loss"][1] == 0 and a["dx"][1].abs().sum() == 0 and a["stats"][:, 1].abs().sum() == 0
    # a label behind the vocabulary is not passed over
    c = run(x, head, (torch.tensor([2, 5, 4]),), torch.ones(3))
    assert torch.isnan(c["loss"][1]) and torch.isnan(c["dx"][1]).all() and torch.isnan(c["dhead"]).all() and not torch.isnan(c["dx"][0]).any()
    # a vocabulary of one token, no rows at all, every row left out
    d = run(x, head[:1], (torch.zeros(3, dtype=torch.int64),), torch.ones(3))
    assert float(d["loss"].abs().max()) == 0 and float(d["dx"].abs().max()) == 0
    e = run(x[:0], head, (lab[:0],), torch.ones(0))
    assert e["loss"].shape == (0,) and e["dx"].shape == (0, 4) and float(e["dhead"].abs().max()) == 0
    f = run(x, head, (torch.full((3,), -100),), torch.ones(3))
    assert all(float(f[k].abs().max()) == 0 for k in f)
    # every token a teacher's: the rest is at its floor and pulls on nothing
    ids = torch.arange(5, dtype=torch.int32)[None].expand(3, 5).contiguous()
    lp = torch.log_softmax(torch.randn(3, 5, generator=torch.Generator().manual_seed(2)), 1)
    k = run(x, head, (ids, lp, torch.full((3,), math.log(1e-12))), torch.ones(3))
    want = (lp.exp() * (lp - torch.log_softmax(x @ head.t(), 1))).sum(1)
    assert torch.allclose(k["loss"], want, atol=1e-6) and torch.isinf(k["stats"][1]).all() and not torch.isnan(k["dx"]).any()
    # a token listed twice is one token whose mass is the sum
    two = (torch.tensor([[1, 1, 3]] * 3, dtype=torch.int32), torch.log(torch.tensor([[0.1, 0.2, 0.4]] * 3)), torch.log(torch.full((3,), 0.3)))
    one = (torch.tensor([[1, 3]] * 3, dtype=torch.int32), torch.log(torch.tensor([[0.3, 0.4]] * 3)), two[2])
    p, q = run(x, head, two, torch.ones(3)), run(x, head, one, torch.ones(3))
    assert torch.allclose(p["dx"], q["dx"], atol=1e-6) and torch.allclose(p["stats"], q["stats"])


def test_refusals():
    x, head, lab = torch.randn(3, 8), torch.randn(11, 8), torch.zeros(3, dtype=torch.int64)
    t = (torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2), torch.zeros(3))
    with pytest.raises(ValueError, match="hidden"):
        L.head_cross_entropy(x, head[:, :7], lab)
    with pytest.raises(ValueError, match="labels of shape"):
        L.head_cross_entropy(x, head, lab[:2])
    with pytest.raises(TypeError, match="labels of type"):
        L.head_cross_entropy(x, head, lab.float())
    with pytest.raises(TypeError, match="states of type"):
        L.head_cross_entropy(x.half(), head, lab)
    with pytest.raises(TypeError, match="head of type"):
        L.head_cross_entropy(x, head.half(), lab)
    for cap in (-1.0, math.nan, math.inf):
        with pytest.raises(ValueError, match="softcap"):
            L.head_cross_entropy(x, head, lab, softcap=cap)
    with pytest.raises(ValueError, match="no logits"):
        L.head_cross_entropy(x, head[:0], lab)
    with pytest.raises(TypeError, match="ids of type"):
        L.head_kl(x, head, t[0].long(), *t[1:])
    with pytest.raises(ValueError, match="logp of shape"):
        L.head_kl(x, head, t[0], t[1][:, :1], t[2])
    with pytest.raises(ValueError, match="K of 1 to"):
        L.head_kl(x, head, torch.zeros(3, 1025, dtype=torch.int32), torch.zeros(3, 1025), t[2])
    with pytest.raises(ValueError, match="K of 1 to"):
        L.head_kl(x, head, t[0][:, :0], t[1][:, :0], t[2])
    nll, stats = L.head_cross_entropy(x, head, lab)
    with pytest.raises(ValueError, match="dloss of shape"):
        L.head_cross_entropy_backward(x, head, lab, stats, torch.ones(4))
    with pytest.raises(ValueError, match="stats of shape"):
        L.head_cross_entropy_backward(x, head, lab, stats[:1], torch.ones(3))
    with pytest.raises(ValueError, match="on meta"):
        L.head_cross_entropy(x, head.to("meta"), lab)
    assert L.head_cross_entropy_backward(x, head, lab, stats, nll, want_dx=False, want_dhead=False) == (None, None)


# ------------------------------------------------------------------------------------------------ GPU
SIZES = [(1, 64, 300), (1, 2048, 1000), (5, 72, 1), (3, 8, 127), (130, 136, 513), (257, 320, 1025), (300, 1001, 2050), (64, 515, 4099), (700, 256, 5000)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden,vocab", SIZES)
@pytest.mark.parametrize("types", ["bf16 bf16", "fp32 bf16", "fp32 fp32", "bf16 fp32"])
def test_cross_entropy(rows, hidden, vocab, types):
    xt, ht = types.split()
    a = make(rows, hidden, vocab, 0, xt, ht, seed=rows, left_out=0.25 if rows > 4 else 0.0, device="cuda")
    hold(run(*a, 0.0), *a, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden,vocab,topk", [(1, 64, 300, 1), (2, 128, 40, 40), (130, 136, 513, 7), (257, 320, 1025, 64), (77, 515, 5003, 17), (9, 256, 3000, 1024)])
@pytest.mark.parametrize("types", ["bf16 bf16", "fp32 bf16", "fp32 fp32"])
def test_divergence(rows, hidden, vocab, topk, types):
    xt, ht = types.split()
    a = make(rows, hidden, vocab, topk, xt, ht, seed=rows, left_out=0.25 if rows > 4 else 0.0, device="cuda")
    hold(run(*a, 0.0), *a, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("topk", [0, 9])
@pytest.mark.parametrize("types", ["bf16 bf16", "fp32 fp32"])
def test_soft_cap(topk, types):
    xt, ht = types.split()
    a = make(150, 200, 777, topk, xt, ht, seed=4, left_out=0.2, device="cuda", spread=8.0)
    hold(run(*a, 20.0), *a, 20.0, only=("loss", "stats"))
    # the gradients beside those of the CPU statement in 64 bits of the same inputs: the cap takes no more from dz than it gives
    got, w = run(*a, 20.0), P.wanted(*a, 20.0)
    for k, limit in (("dx", 2.0 ** -8), ("dhead", 2.0 ** -8)) if xt == "bf16" else (("dx", 2.0 ** -16), ("dhead", 2.0 ** -16)):
        assert float((got[k].double() - w[k]).norm() / w[k].norm()) < limit, k
