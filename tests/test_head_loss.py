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
    for cap in (-1.0, 1e-50, math.nan, math.inf):
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
SIZES = [(1, 64, 300), (1, 2048, 1000), (5, 72, 1), (3, 8, 127), (130, 136, 513), (257, 320, 1025), (300, 1001, 2050), (64, 515, 4099), (700, 256, 5000), (12, 196, 2889), (300, 200, 20001)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden,vocab", SIZES)
@pytest.mark.parametrize("types", ["bf16 bf16", "fp32 bf16", "fp32 fp32", "bf16 fp32"])
def test_cross_entropy(rows, hidden, vocab, types):
    xt, ht = types.split()
    a = make(rows, hidden, vocab, 0, xt, ht, seed=rows, left_out=0.25 if rows > 4 else 0.0, device="cuda")
    hold(run(*a, 0.0), *a, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden,vocab,topk", [(1, 64, 300, 1), (2, 128, 40, 40), (130, 136, 513, 7), (257, 320, 1025, 64), (77, 515, 5003, 17), (9, 256, 3000, 1024), (8, 132, 1877, 62), (260, 136, 19500, 33)])
@pytest.mark.parametrize("types", ["bf16 bf16", "fp32 bf16", "fp32 fp32"])
def test_divergence(rows, hidden, vocab, topk, types):
    xt, ht = types.split()
    a = make(rows, hidden, vocab, topk, xt, ht, seed=rows, left_out=0.25 if rows > 4 else 0.0, device="cuda")
    hold(run(*a, 0.0), *a, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("topk", [0, 9])
@pytest.mark.parametrize("types", ["bf16 bf16", "fp32 fp32"])
@pytest.mark.parametrize("vocab", [777, 20100])                       # tiles of 64 columns, and of 256
def test_soft_cap(topk, types, vocab):
    xt, ht = types.split()
    a = make(300 if vocab > 777 else 150, 200, vocab, topk, xt, ht, seed=4, left_out=0.2, device="cuda", spread=8.0)
    hold(run(*a, 20.0), *a, 20.0, only=("loss", "stats"))
    # the gradients beside those of the CPU statement in 64 bits of the same inputs: the cap takes no more from dz than it gives
    got, w = run(*a, 20.0), P.wanted(*a, 20.0)
    for k, limit in (("dx", 2.0 ** -8), ("dhead", 2.0 ** -8)) if xt == "bf16" else (("dx", 2.0 ** -16), ("dhead", 2.0 ** -16)):
        assert float((got[k].double() - w[k]).norm() / w[k].norm()) < limit, k


@pytest.mark.gpu
@pytest.mark.parametrize("topk", [0, 6])
def test_left_out_rows_and_what_stands_in_them(topk):
    a = make(290, 136, 700, topk, seed=9, left_out=0.6, device="cuda")
    live = (a[2][0] >= 0) if not topk else (a[2][0] >= 0).any(1)
    want = run(*a)
    x = a[0].clone()
    x[~live] = math.nan
    targets = a[2]
    if topk:
        targets = (targets[0], targets[1].clone(), targets[2].clone())
        targets[1][~live], targets[2][~live] = math.nan, math.inf
    dloss = a[3].clone()
    dloss[~live] = math.inf
    got = run(x, a[1], targets, dloss)
    for k in want:
        assert torch.equal(got[k], want[k]), k
    assert float(got["dx"][~live].abs().max()) == 0 and float(got["loss"][~live].abs().max()) == 0 and float(got["stats"][:, ~live].abs().max()) == 0
    # every row left out, and no rows
    none = tuple(torch.full_like(t, -1) if i == 0 else t for i, t in enumerate(targets))
    got = run(x, a[1], none, dloss)
    assert all(float(got[k].abs().max()) == 0 for k in got)
    got = run(x[:0], a[1], tuple(t[:0] for t in targets), dloss[:0])
    assert got["loss"].shape == (0,) and got["dx"].shape == (0, 136) and float(got["dhead"].abs().max()) == 0


@pytest.mark.gpu
def test_labels_behind_the_vocabulary_make_nan():
    for types in ("bf16", "fp32"):
        x, head, (lab,), dl = make(20, 72, 300, 0, types, types, seed=2, device="cuda")
        for v in (300, 383, 384, 1 << 20, (1 << 40) + 1):
            lab2 = lab.clone()
            lab2[3] = v
            got = run(x, head, (lab2,), dl)
            assert torch.isnan(got["loss"][3]) and torch.isnan(got["dx"][3]).all() and torch.isnan(got["dhead"]).all()
            assert int(torch.isnan(got["loss"]).sum()) == 1 and int(torch.isnan(got["dx"]).any(1).sum()) == 1
    x, head, t, dl = make(20, 72, 300, 4, seed=2, device="cuda")
    t[0][5, 2] = 300
    got = run(x, head, t, dl)
    assert torch.isnan(got["loss"][5]) and int(torch.isnan(got["loss"]).sum()) == 1 and torch.isnan(got["dx"][5]).all()


@pytest.mark.gpu
def test_teachers_of_odd_forms():
    x, head, (ids, logp, tail), dl = make(40, 136, 500, 8, seed=12, device="cuda")
    # a token listed twice is one whose mass is the sum; the order of the tokens does not matter
    perm = torch.randperm(8, generator=torch.Generator().manual_seed(0)).cuda()
    p, q = run(x, head, (ids[:, perm].contiguous(), logp[:, perm].contiguous(), tail), dl), run(x, head, (ids, logp, tail), dl)
    for k in p:
        assert torch.allclose(p[k], q[k], rtol=2.0 ** -7, atol=1e-6), k
    half = (torch.cat([ids, ids[:, :1]], 1), torch.cat([logp, logp[:, :1] - math.log(2)], 1), tail)
    half[1][:, 0] -= math.log(2)
    two = run(x, head, half, dl)
    assert torch.equal(two["stats"], q["stats"]) and torch.allclose(two["dx"].float(), q["dx"].float(), rtol=2.0 ** -7, atol=1e-5)
    # no mass outside, tokens without mass
    t = (ids, logp.clone(), torch.full_like(tail, -math.inf))
    t[1][:, 3] = -math.inf
    got = run(x, head, t, dl)
    w = P.wanted(x, head, t, dl, 0.0)
    assert torch.allclose(got["loss"].double(), w["loss"], rtol=1e-4, atol=1e-5) and not torch.isnan(got["dx"]).any()
    assert float((got["dx"].double() - w["dx"]).norm() / w["dx"].norm()) < 2.0 ** -8
    # the model gives the rest less than the floor: it is held at the floor and pulls on nothing
    big = (x * 0 + 60 * head[ids[:, 0].long()]).to(torch.bfloat16)
    got = run(big, head, (ids, logp, tail), dl)
    hold(got, big, head, (ids, logp, tail), dl, 0.0, only=("loss", "stats"))


@pytest.mark.gpu
@pytest.mark.parametrize("types", ["bf16 bf16", "fp32 fp32"])
def test_strides_and_starts(types):
    xt, ht = types.split()
    x, head, t, dl = make(70, 128, 333, 0, xt, ht, seed=6, device="cuda")
    want = run(x, head, t, dl)

    def placed(m, left, right, step=1):
        big = torch.full((m.shape[0] * step, left + m.shape[1] + right), math.nan, dtype=m.dtype, device="cuda")
        v = big[::step, left:left + m.shape[1]]
        v.copy_(m)
        return v
    for xs, hs in ((placed(x, 8, 8), placed(head, 8, 16)), (placed(x, 3, 2), placed(head, 1, 0)), (placed(x, 0, 0, 2), placed(head, 0, 8, 3)),
                   (x.t().contiguous().t(), head.t().contiguous().t())):
        got = run(xs, hs, t, dl)
        for k in got:
            assert torch.equal(got[k], want[k]), k
    # a single row of an expanded matrix, for either side
    one = run(x[:1].expand(2, -1)[:1], head[:1].expand(3, -1)[:1], (torch.zeros(1, dtype=torch.int64, device="cuda"),), dl[:1])
    assert float(one["loss"]) == 0 and float(one["dx"].abs().max()) == 0
    # labels of 32 bits, strided
    lab = torch.stack([t[0].int(), t[0].int() * 0], 1)[:, 0]
    got = run(x, head, (lab,), dl)
    assert all(torch.equal(got[k], want[k]) for k in got)


@pytest.mark.gpu
def test_one_gradient_alone_and_the_same_bits_again():
    for topk, vocab in ((0, 3000), (5, 3000), (5, 38000)):
        x, head, t, dl = make(300, 264, vocab, topk, seed=8, left_out=0.1, device="cuda")
        a, b = run(x, head, t, dl), run(x, head, t, dl)
        assert all(torch.equal(a[k], b[k]) for k in a)
        c, d = run(x, head, t, dl, want_dhead=False), run(x, head, t, dl, want_dx=False)
        assert c["dhead"] is None and d["dx"] is None and torch.equal(c["dx"], a["dx"]) and torch.equal(d["dhead"], a["dhead"])
        # a row does not depend on the rows beside it (while the tiles are of one width)
        e = run(x[40:120], head, tuple(v[40:120] for v in t), dl[40:120])
        assert torch.equal(e["loss"], a["loss"][40:120]) and torch.equal(e["stats"], a["stats"][:, 40:120])


@pytest.mark.gpu
def test_streams_and_graphs():
    x, head, t, dl = make(64, 256, 2000, 7, seed=1, device="cuda")
    want = run(x, head, t, dl)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, head, t, dl)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[k], want[k]) for k in got)
    # two captured calls replayed in turn, and on two streams at once: each has its own workspace
    x2 = x.roll(1, 0).contiguous()
    want2 = run(x2, head, t, dl)
    graphs = []
    for v in (x, x2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(v, head, t, dl)
        graphs.append((g, out))
    for _ in range(3):
        for (g, out), w in zip(graphs, (want, want2)):
            g.replay()
            assert all(torch.equal(out[k], w[k]) for k in out)
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(side):
            graphs[0][0].replay()
        with torch.cuda.stream(other):
            graphs[1][0].replay()
    torch.cuda.synchronize()
    for (_, out), w in zip(graphs, (want, want2)):
        assert all(torch.equal(out[k], w[k]) for k in out)
    # the differentiable call gives the pair's gradients, and is not captured
    xs, hs = x.clone().requires_grad_(), head.clone().requires_grad_()
    L.head_kl_loss(xs, hs, *t).backward(dl)
    assert torch.equal(xs.grad, want["dx"]) and torch.equal(hs.grad, want["dhead"])
    with pytest.raises(RuntimeError, match="not captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            L.head_kl_loss(xs, hs, *t)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_gradients_by_differences():
    """Directional differences of the kernel's own losses in fp32: a step of 2^-6 in a direction of norm one changes the loss by its gradient, up to the
    cube of the step (third derivatives of these losses are below 30 here) and the losses' rounding (2^-20) over the step."""
    for topk in (0, 5):
        x, head, t, dl = make(24, 40, 120, topk, "fp32", "fp32", seed=3, device="cuda", spread=1.0)
        got = run(x, head, t, dl, 10.0)
        f = L.head_cross_entropy if not topk else L.head_kl
        g = torch.Generator(device="cuda").manual_seed(4)
        for which in (0, 1):
            d = torch.randn((x, head)[which].shape, generator=g, device="cuda")
            d /= d.norm()
            h = 2.0 ** -6
            up, dn = (f(*((x + s * d, head) if which == 0 else (x, head + s * d)), *t, softcap=10.0)[0] for s in (h, -h))
            num = float(((up - dn).double() * dl.double()).sum()) / (2 * h)
            ana = float(((got["dx"], got["dhead"])[which].double() * d.double()).sum())
            assert abs(num - ana) < 30 * h * h * float(dl.sum()) / 6 + float(dl.sum()) * 2.0 ** -20 * 8 / h, (topk, which, num, ana)


@pytest.mark.gpu
def test_pieces_of_the_vocabulary():
    """dz of more than one piece (256 MB: 100 000 columns of 1300 rows), and packed fp32 rows of a head of more than one piece (512 MB)."""
    x, head, t, dl = make(1300, 64, 100500, 0, seed=5, left_out=0.01, device="cuda")
    w = hold(run(x, head, t, dl), x, head, t, dl, 0.0)
    del w
    x, head, t, dl = make(40, 1000, 90000, 5, "fp32", "fp32", seed=5, device="cuda")
    hold(run(x, head, t, dl), x, head, t, dl, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("topk", [0, 3])
def test_many_rows(topk):
    """More rows (or ids) than one block looks through for those that count."""
    a = make(9001, 32, 300, topk, seed=5, left_out=0.3, device="cuda")
    hold(run(*a), *a, 0.0)
    if topk:
        a = make(400, 32, 700, 200, seed=6, left_out=0.7, device="cuda")
        hold(run(*a), *a, 0.0)


@pytest.mark.gpu
def test_offsets_that_pass_32_bits():
    """A head of 2.2 G values; the last rows' labels stand at its end."""
    vocab, hidden = 540000, 4096
    head = torch.empty(vocab, hidden, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    for lo in range(0, vocab, 60000):
        head[lo:lo + 60000] = (torch.randn(60000, hidden, generator=g, device="cuda") * (2.0 / 64)).to(torch.bfloat16)
    x = torch.randn(3, hidden, generator=g, device="cuda").to(torch.bfloat16)
    labels = torch.tensor([vocab - 1, 5, vocab - 70000], device="cuda")
    dl = torch.ones(3, device="cuda")
    got = run(x, head, (labels,), dl)
    z = torch.cat([x.double() @ head[lo:lo + 60000].double().t() for lo in range(0, vocab, 60000)], 1)
    lse = torch.logsumexp(z, 1)
    assert torch.allclose(got["loss"].double(), lse - z.gather(1, labels[:, None])[:, 0], atol=1e-3)
    s = torch.exp(z - lse[:, None]).scatter_add_(1, labels[:, None], torch.full((3, 1), -1.0, dtype=torch.float64, device="cuda"))
    dx = sum(s[:, lo:lo + 60000] @ head[lo:lo + 60000].double() for lo in range(0, vocab, 60000))
    assert float((got["dx"].double() - dx).norm() / dx.norm()) < 2.0 ** -8
    tail = s[:, -100:].t() @ x.double()
    assert float((got["dhead"][-100:].double() - tail).norm() / tail.norm()) < 2.0 ** -8


def near(rows, hidden, vocab, topk, noise, common, device, seed=0, spread=2.5):
    """bf16 inputs whose head rows have a part in common (``common`` times their spread), as the rows of trained heads do; a teacher of the same states
    but for ``noise``."""
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(vocab, hidden, generator=g) + common * torch.randn(1, hidden, generator=g)
    w = (w * spread / math.sqrt(hidden)).bfloat16()
    labels = torch.randint(0, vocab, (rows,), generator=g)
    x = torch.randn(rows, hidden, generator=g) + 6 * torch.rand(rows, 1, generator=g) * torch.nn.functional.normalize(w[labels].float(), dim=1)
    x, dloss = x.bfloat16(), torch.rand(rows, generator=g) + 0.5
    targets = (labels,)
    if topk:
        lp = torch.log_softmax((x.double() + noise * torch.randn(rows, hidden, generator=g).double()) @ w.double().t(), 1)
        logp, ids = lp.topk(topk, 1)
        targets = (ids.int(), logp.float(), (1 - logp.exp().sum(1)).clamp(min=1e-9).log().float())
    return x.to(device), w.to(device), tuple(t.to(device) for t in targets), dloss.to(device)


def beside_rounding(got, want):
    """Errors of a bf16 result's rows over what rounding the 64-bit result to bf16 would be off by."""
    return (got.double() - want).norm(dim=1) / (want.to(torch.bfloat16).double() - want).norm(dim=1)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden,vocab,topk,softcap", [(40, 256, 3000, 0, 0.0), (300, 264, 20100, 0, 20.0), (1300, 64, 50000, 0, 0.0), (40, 256, 3000, 8, 0.0),
                                                            (300, 264, 20100, 16, 0.0)])
def test_bf16_gradients_are_off_by_their_rounding(rows, hidden, vocab, topk, softcap):
    """Rows of dx and dhead (those of nobody's label too) in 47 to 682 blocks of 64 columns, in ranges of the vocabulary, in two pieces of it, with a cap:
    what stands in front of the last rounding adds less than a tenth to it. dz comes in two slabs, 2^-16 of a value, where the result's rounding is 2^-8
    of its own, and a common part of three times the spread makes 2^-16 of dz about 2^-14 of dx; the logits' share is below 2^-14 of s, 2^-12 beside
    that part, an eighth of the rounding (2^-9 as a root mean square): sqrt(1 + 1/64). Near a teacher (noise 0.1) a row's dz is a difference of two nearly equal shares, in some
    rows to the logits' own error: the middle row is looked at."""
    a = near(rows, hidden, vocab, topk, 0.1, 3.0, "cuda")
    got, want = run(*a, softcap), P.wanted(*a, softcap)
    for k in ("dx", "dhead"):
        r = beside_rounding(got[k], want[k])
        assert float(r.median() if topk else r.max()) < 1.1, (k, float(r.median()), float(r.max()))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden,vocab,common", [(60, 4096, 5000, 0.0), (500, 1024, 20100, 0.0), (60, 4096, 5000, 3.0), (300, 264, 20100, 0.0)])
def test_logits_of_gradients_are_those_of_the_loss(rows, hidden, vocab, common):
    """Every row of the gradients beside an ordinary teacher, those of a confident model among them, whose dz is 2^-7 and less of what it is the difference
    of: logits to 2^-21 of theirs, as the loss takes them, are some 2^-12 of such rows, an eighth of the rounding; 2^-19 would be half of it and more."""
    a = near(rows, hidden, vocab, 16, 0.9, common, "cuda")
    got, want = run(*a), P.wanted(*a, 0.0)
    for k in ("dx", "dhead"):
        r = beside_rounding(got[k], want[k])
        assert float(r.max()) < 1.1, (k, float(r.max()))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("vocab,gone", [(257, (256, 257)), (300, (32, 64)), (700, (128, 256)), (3000, (384, 512)), (20100, (20096, 20100))])
@pytest.mark.parametrize("topk", [0, 3])
def test_nan_in_the_head(vocab, gone, topk, device):
    """NaN logits of tokens that are no targets, alone in a block of columns: every loss is NaN, as its gradients are."""
    x, head, targets, dl = make(300 if vocab > 20000 else 6, 72, vocab, topk, seed=1, device=device)
    if topk:
        targets = (torch.arange(topk, dtype=torch.int32, device=device).expand(x.shape[0], topk).contiguous(), *targets[1:])
    else:
        targets = (targets[0].clamp(max=gone[0] - 1),)
    head[gone[0]:gone[1]] = math.nan
    got = run(x, head, targets, dl)
    assert torch.isnan(got["loss"]).all() and torch.isnan(got["stats"]).all() and torch.isnan(got["dx"]).all()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_the_largest_id_is_behind_the_vocabulary(device):
    x, head, t, dl = make(20, 72, 300, 4, seed=2, device=device)
    t[0][5, 2] = 2 ** 31 - 1
    got = run(x, head, t, dl)
    assert torch.isnan(got["loss"][5]) and int(torch.isnan(got["loss"]).sum()) == 1
    assert torch.isnan(got["dx"][5]).all() and int(torch.isnan(got["dx"]).any(1).sum()) == 1


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_a_token_listed_twice_is_one_in_the_loss_too(device):
    """Each result as of the teacher whose masses are added first. fp32 sums of the same numbers in another order: 2^-20, and bf16 gradients one step of theirs."""
    x, head, _, dl = make(3, 72, 300, 0, seed=3, device=device)
    two = (torch.tensor([[1, 1, 3, -1, 1], [9, 7, 9, 7, 8], [2, 2, 2, 2, 2]], dtype=torch.int32),
           torch.log(torch.tensor([[0.1, 0.2, 0.4, 0.9, 0.1], [0.1, 0.1, 0.1, 0.1, 0.0], [0.1, 0.2, 0.0, 0.3, 0.1]])), torch.log(torch.tensor([0.2, 0.6, 0.3])))
    one = (torch.tensor([[1, 3, -1], [9, 7, 8], [2, -1, -1]], dtype=torch.int32),
           torch.log(torch.tensor([[0.4, 0.4, 1.0], [0.2, 0.2, 0.0], [0.7, 1.0, 1.0]])), two[2])
    a, b = (run(x, head, tuple(v.to(device) for v in t), dl) for t in (two, one))
    for k in a:
        assert torch.allclose(a[k].float(), b[k].float(), rtol=2.0 ** -7 if k in ("dx", "dhead") else 2.0 ** -20, atol=1e-6), k
    w = P.wanted(x, head, tuple(v.to(device) for v in one), dl, 0.0)
    assert torch.allclose(a["loss"].double(), w["loss"], rtol=1e-5, atol=1e-6)


@pytest.mark.gpu
def test_a_piece_of_more_than_2_31_values():
    """dhead of 256000 x 8448 in one piece, its pitch in bytes beyond 32 bits."""
    vocab, hidden = 256000, 8448
    g = torch.Generator(device="cuda").manual_seed(0)
    head = torch.empty(vocab, hidden, dtype=torch.bfloat16, device="cuda")
    for lo in range(0, vocab, 32000):
        head[lo:lo + 32000] = torch.randn(32000, hidden, generator=g, device="cuda") * (2.0 / math.sqrt(hidden))
    x = torch.randn(3, hidden, generator=g, device="cuda").to(torch.bfloat16)
    labels = torch.tensor([vocab - 1, 5, vocab - 1700], device="cuda")
    got = run(x, head, (labels,), torch.ones(3, device="cuda"))
    z = torch.cat([x.double() @ head[lo:lo + 32000].double().t() for lo in range(0, vocab, 32000)], 1)
    dz = torch.softmax(z, 1).scatter_add_(1, labels[:, None], torch.full((3, 1), -1.0, dtype=torch.float64, device="cuda"))
    for lo in (0, vocab - 1750, vocab - 100):                    # (and labels among them)
        assert float(beside_rounding(got["dhead"][lo:lo + 100], dz[:, lo:lo + 100].t() @ x.double()).max()) < 1.1


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_nan_of_a_teacher(device):
    """A log-probability or a rest of NaN in a row that counts is its loss; beside a padded id it is nothing."""
    x, head, (ids, logp, tail), dl = make(6, 72, 300, 4, seed=5, device=device)
    logp[2, 1], tail[4] = math.nan, math.nan
    ids[5, 3], logp[5, 3] = -1, math.nan
    got = run(x, head, (ids, logp, tail), dl)
    bad = torch.tensor([False, False, True, False, True, False], device=device)
    assert torch.equal(torch.isnan(got["loss"]), bad) and torch.equal(torch.isnan(got["dx"]).all(1), bad) and torch.equal(torch.isnan(got["dx"]).any(1), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [900, 20100])
@pytest.mark.parametrize("topk", [0, 3])
def test_sums_beside_large_logits(vocab, topk):
    """Logits of 60 to 140 that 32 bits hold (quarters times quarters, and a column that adds a hundred): the log-sums are off by the exponentials, 2^-22 of
    their terms, the rounding of their arguments, 2^-22, and their own rounding, 2^-18 at most; the loss, a difference of a few units, by 2^-20 in all and
    a rounding of its own."""
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randint(-8, 9, (200, 16), generator=g) / 4).to(torch.bfloat16)
    head = (torch.randint(-8, 9, (vocab, 16), generator=g) / 4).to(torch.bfloat16)
    x[:, 0], head[:, 0] = 100.0, 1.0
    z = x.double() @ head.double().t()
    labels = (z + 3 * torch.randn(z.shape, generator=g).double()).argmax(1)
    targets = (labels,) if not topk else (z.topk(topk, 1)[1].int(), torch.full((200, topk), math.log(0.9 / topk)), torch.full((200,), math.log(0.1)))
    targets = tuple(t.cuda() for t in targets)
    x, head = x.cuda(), head.cuda()
    w = P.wanted(x, head, targets, torch.ones(200, device="cuda"), 0.0)
    loss, stats = (L.head_cross_entropy if not topk else L.head_kl)(x, head, *targets)
    assert bool(((loss.double() - w["loss"]).abs() <= 2.0 ** -20 + w["loss"].abs() * 2.0 ** -24).all()), float((loss.double() - w["loss"]).abs().max()) * 2 ** 20
    assert bool(((stats.double() - w["stats"]).abs() <= 2.0 ** -20 + w["stats"].abs() * 2.0 ** -24).all())


@pytest.mark.parametrize("topk", [0, 5])
def test_fine_statistics_on_the_cpu(topk):
    x, head, t, dl = make(7, 12, 33, topk, "fp32", "fp32", seed=1, left_out=0.3)
    f, b = (L.head_cross_entropy, L.head_cross_entropy_backward) if not topk else (L.head_kl, L.head_kl_backward)
    (l1, s1), (l2, s2) = f(x, head, *t), f(x, head, *t, fine=True)
    assert s2.shape == (4, 7) and torch.equal(l1, l2) and torch.equal(s1, s2[:2]) and not s2[2:].any()
    assert all(torch.equal(u, v) for u, v in zip(b(x, head, *t, s1, dl), b(x, head, *t, s2, dl)))
    s2[2:] = 0.25                                          # and they are added
    s1 = s1 + 0.25
    assert all(torch.equal(u, v) for u, v in zip(b(x, head, *t, s1, dl), b(x, head, *t, s2, dl)))
    for bad in (s2[:3], s2[:, :5], s2[0]):
        with pytest.raises(ValueError, match="stats of shape"):
            b(x, head, *t, bad, dl)


@pytest.mark.gpu
@pytest.mark.parametrize("topk", [0, 6])
@pytest.mark.parametrize("vocab", [900, 20100])
def test_fine_statistics_keep_what_sums_lose(topk, vocab):
    """Column 0 of the head is one and that column of the states a hundred, so that log-sums lie in 64 to 128, where 32 bits round by up to 2^-18, and column 0
    of dx is the sum of the row's dz: zero. Exponentials are off by 2^-22 here and in the sums, their arguments' rounding by as much, and the sum
    of a row's |dz| (two dloss at most) by 2^-23 of it: 1.25 * 2^-20 dloss with the lower parts; without them some row is off by twice that."""
    x, head, t, dl = make(200, 72, vocab, topk, "fp32", "fp32", seed=2, left_out=0.1, device="cuda")
    x[:, 0], head[:, 0] = 100.0, 1.0
    f, b = (L.head_cross_entropy, L.head_cross_entropy_backward) if not topk else (L.head_kl, L.head_kl_backward)
    (l1, s1), (l2, s2) = f(x, head, *t), f(x, head, *t, fine=True)
    assert torch.equal(l1, l2) and torch.equal(s1, s2[:2])
    assert bool((s2[2:].abs() <= s2[:2].abs() * 2.0 ** -24).all()) and bool(s2[2:].any())
    off = [(b(x, head, *t, s, dl, want_dhead=False)[0][:, 0].abs() / dl) for s in (s1, s2)]
    assert float(off[1].max()) < 1.25 * 2.0 ** -20 < float(off[0].max()) / 2, [float(v.max()) * 2 ** 20 for v in off]
    # the differentiable call with them
    xs = x.clone().requires_grad_()
    (L.head_cross_entropy_loss if not topk else L.head_kl_loss)(xs, head, *t, fine=True).backward(dl)
    assert torch.equal(xs.grad, b(x, head, *t, s2, dl, want_dhead=False)[0])


def test_sizes_that_tiles_do_not_count_are_refused():
    for rows, vocab in (((1 << 24) - 255, 2), (2, 1 << 24)):
        x, head = torch.zeros(1, 8).expand(rows, 8), torch.zeros(1, 8).expand(vocab, 8)
        with pytest.raises(ValueError, match="below 2"):
            L.head_cross_entropy(x, head, torch.zeros(1, dtype=torch.int64).expand(rows))
