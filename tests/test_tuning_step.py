"""The tuner's step and the perplexity tool through the head losses and the computed dropout (tools/e2e.py, tools/ppl.py)."""
import json
import os
import socket
import subprocess
import sys

import pytest
import torch

from volta_engine_b200.models.dense import DenseConfig, DenseModel
from volta_engine_b200.tools import e2e as E
from volta_engine_b200.tools.ppl import topk_teacher

HERE = os.path.dirname(os.path.abspath(__file__))


def _setup(seed=0, **kw):
    cfg = DenseConfig(n_layers=2, hidden=64, n_q=4, n_kv=2, head_dim=16, ffn=128, vocab=200, quant="bf16", **kw)
    model = DenseModel(cfg, "cpu").init_random(seed=seed, std=0.08, search=False)
    g = torch.Generator().manual_seed(seed + 1)
    ids = torch.randint(0, cfg.vocab, (40,), generator=g)
    return model, ids, topk_teacher(2 * torch.randn(40, cfg.vocab, generator=g), 9)


def _grads(m, ids, teacher, head, p=0.0, seed=0):
    m.zero_grad(set_to_none=True)
    m.train()
    E.set_dropout(m, p, seed, ids.shape[0])
    loss = E.objective(m, ids, teacher, head)
    loss.backward()
    return loss.detach(), {n: q.grad.clone() for n, q in m.named_parameters()}


def _close(a, b, rel):
    for n in a:
        assert float((a[n] - b[n]).norm()) <= rel * float(b[n].norm()) + 1e-9, n


def test_divergence_without_logits_is_the_divergence():
    model, ids, teacher = _setup()
    m = E.build_from_engine_model(model)
    head = E.scoring_head(m)
    assert head.dtype == torch.bfloat16                    # the head of a bf16 model: its rows hold every value
    a, ga = _grads(m, ids, teacher, None)
    b, gb = _grads(m, ids, teacher, head)
    # both are fp32 sums over 200 logits: some 2^-24 * sqrt(200) each, through two layers
    assert torch.allclose(a, b, rtol=1e-5)
    _close(gb, ga, 1e-4)
    m.head[0, 0] += 2.0 ** -20                             # one value that bf16 does not hold: fp32 rows
    assert E.scoring_head(m).dtype == torch.float32


def test_labels_are_the_next_tokens():
    model, ids, _ = _setup(1)
    m = E.build_from_engine_model(model)
    got, g1 = _grads(m, ids, None, E.scoring_head(m))
    m.zero_grad(set_to_none=True)
    want = torch.nn.functional.cross_entropy(m(ids)[:-1], ids[1:])
    want.backward()
    assert torch.allclose(got, want.detach(), rtol=1e-5)
    _close(g1, {n: p.grad for n, p in m.named_parameters()}, 1e-4)


def test_dropout_masks_are_those_of_the_seed_and_survive_checkpointing():
    model, ids, teacher = _setup(2)
    m = E.build_from_engine_model(model)
    head = E.scoring_head(m)
    a, ga = _grads(m, ids, teacher, head, 0.3, 5)
    b, gb = _grads(m, ids, teacher, head, 0.3, 5)
    c, _ = _grads(m, ids, teacher, head, 0.3, 6)
    assert torch.equal(a, b) and not torch.equal(a, c)
    assert all(torch.equal(ga[n], gb[n]) for n in ga)
    # without checkpoints the same gradients: the layers that ran again dropped the same elements
    m.zero_grad(set_to_none=True)
    E.set_dropout(m, 0.3, 5, ids.shape[0])
    h = m.embed[ids] * m.cfg.embed_scale
    for L in m.layers:
        h = L(h)
    d = E.head_kl_loss(m.final_norm(h), head, *teacher).mean()
    d.backward()
    assert torch.allclose(d.detach(), a, rtol=1e-6)
    _close({n: p.grad for n, p in m.named_parameters()}, ga, 1e-5)
    m.eval()
    with torch.no_grad():
        assert torch.equal(E.objective(m, ids, teacher, head), E.objective(m, ids, teacher, head))
    assert not torch.equal(E.objective(m, ids, teacher, head).detach(), a)      # no masks while evaluating


def test_tuning_runs_with_each_objective():
    model, ids, teacher = _setup(3)
    for teachers, kw in (([teacher] * 3, {"no_logits": True, "dropout": 0.1}), ([None] * 3, {"dropout": 0.1})):
        m = E.build_from_engine_model(model)
        lines = []
        hist = E.tune(m, [ids] * 3, teachers, E.E2EOptions(steps=2, batch=2, eval_every=1, **kw), log=lines.append)
        assert len(hist["train"]) == 2 and all(torch.isfinite(torch.tensor(v)) for v in hist["train"])
        assert ("cross entropy" if teachers[0] is None else "KL") in lines[0]
    with pytest.raises(ValueError, match="top-K teachers"):
        E.tune(E.build_from_engine_model(model), [ids] * 2, [torch.randn(40, 200)] * 2, E.E2EOptions(no_logits=True), log=lambda s: None)


def test_ranks_of_a_row_sharded_model_take_the_same_step():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    procs = []
    for rank in range(2):
        env = dict(os.environ, RANK=str(rank), WORLD_SIZE="2", MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), OMP_NUM_THREADS="1")
        procs.append(subprocess.Popen([sys.executable, os.path.join(HERE, "e2e_step_worker.py")], env=env, stdout=subprocess.PIPE, stderr=subprocess.STDOUT,
                                      text=True))
    outs = [p.communicate(timeout=240)[0] for p in procs]
    assert all(p.returncode == 0 for p in procs) and "E2E_STEP_OK" in outs[0], outs


def _ppl(args, capsys):
    from volta_engine_b200.tools import ppl
    assert ppl.main(args) == 0
    return json.loads(capsys.readouterr().out.strip().splitlines()[-1])


def _scores(tmp_path, capsys, device, softcap):
    from volta_engine_b200.models.factory import save_dense_checkpoint
    cfg = DenseConfig(n_layers=2, hidden=128, n_q=2, n_kv=1, head_dim=64, ffn=256, vocab=300)
    src = tmp_path / f"src{softcap}"
    save_dense_checkpoint(src, cfg, seed=5, fmt="bf16", std=0.08)
    if softcap:
        c = json.loads((src / "config.json").read_text())
        c["final_logit_softcapping"] = softcap
        (src / "config.json").write_text(json.dumps(c))
    g = torch.Generator().manual_seed(2)
    # 70 = 32 + 32 + 6 and 45 = 32 + 13: portions of rows that score from states, and short ones
    torch.save([torch.randint(0, 300, (n,), generator=g, dtype=torch.int32) for n in (70, 45)], tmp_path / "tok.pt")
    base = ["--model", str(src), "--tokens-file", str(tmp_path / "tok.pt"), "--chunk", "32", "--device", device]
    teacher = str(tmp_path / "t.pt")
    _ppl(base + ["--topk-out", teacher, "--topk", "8"], capsys)
    t = torch.load(teacher, weights_only=True)
    t["logp"] = [torch.log_softmax(x + 0.5 * torch.randn(x.shape, generator=g), 1) + torch.log1p(-u.exp())[:, None] for x, u in zip(t["logp"], t["tail"])]
    torch.save(t, teacher)
    a = _ppl(base + ["--kl-teacher", teacher], capsys)
    b = _ppl(base + ["--kl-teacher", teacher, "--no-logits"], capsys)
    assert a["tokens"] == b["tokens"] == 113
    # sums of 113 fp32 losses around 6, of logits whose last bits differ by the order of summation
    assert abs(a["nll"] - b["nll"]) < 1e-4 and abs(a["kl"] - b["kl"]) < 1e-4 and a["kl"] > 0.01


@pytest.mark.parametrize("softcap", [0.0, 3.0])
def test_ppl_without_logits(tmp_path, capsys, softcap):
    _scores(tmp_path, capsys, "cpu", softcap)


def test_ppl_refusals(tmp_path):
    from volta_engine_b200.tools import ppl
    with pytest.raises(SystemExit):
        ppl.main(["--model", "x", "--file", "y", "--no-logits", "--topk-out", "z"])


# ------------------------------------------------------------------------------------------------ GPU
@pytest.mark.gpu
@pytest.mark.parametrize("softcap", [0.0, 3.0])
def test_ppl_without_logits_gpu(tmp_path, capsys, softcap):
    _scores(tmp_path, capsys, "cuda:0", softcap)


@pytest.mark.gpu
def test_tuning_step_gpu():
    """Dropout, layers, loss and all gradients together on the GPU against the CPU's step of the same masks."""
    model, ids, teacher = _setup(4)
    for t in (teacher, None):
        m = E.build_from_engine_model(model)
        a, ga = _grads(m, ids, t, E.scoring_head(m), 0.3, 9)
        mc = E.build_from_engine_model(model, ("cuda:0",))
        dt = tuple(x.cuda() for x in t) if t is not None else None
        b, gb = _grads(mc, ids.cuda(), dt, E.scoring_head(mc), 0.3, 9)
        b2, gb2 = _grads(mc, ids.cuda(), dt, E.scoring_head(mc), 0.3, 9)
        assert torch.allclose(a, b.cpu(), rtol=1e-5)
        _close({n: g.cpu() for n, g in gb.items()}, ga, 1e-3)
        assert torch.equal(b, b2)
        # and the loss that goes through the logits, where there is one
        if t is not None:
            c, gc = _grads(mc, ids.cuda(), dt, None, 0.3, 9)
            assert torch.allclose(b, c, rtol=1e-5)
            _close(gb, gc, 1e-3)


def _capped_objectives(device):
    """A model whose logits are soft-capped: the tuner's objectives are those of the engine's logits, in fp32 sums over 200 of them."""
    from volta_engine_b200.runtime.batch import BatchRows
    from volta_engine_b200.runtime.kv_cache import PagedKVCache
    model, ids, teacher = _setup(5, logit_softcap=3.0)
    model.lm_head.weight.mul_(8)                           # logits that reach the cap
    kv = PagedKVCache(2, 2, 16, 4, 1, 64, "cpu")
    kv.reserve(0, 41)
    logits = model.forward(BatchRows.make(ids.tolist(), list(range(40)), [0] * 40, "cpu", G=2, prefill=True), kv)[:, :200].float()
    assert 2.9 < float(logits.abs().max()) <= 3.0
    m = E.build_from_engine_model(model, (device,)).eval()
    head, dev = E.scoring_head(m), torch.device(device)
    t = tuple(v.to(dev) for v in teacher)
    ce, kl = torch.nn.functional.cross_entropy(logits[:-1], ids[1:]), E.kl_teacher(logits, teacher)
    with torch.no_grad():
        # (the engine's layers are bf16: logits in front of the cap, 5 to 10 here, off by some 2^-8 of theirs, the means of 40 losses by less)
        assert abs(float(E.objective(m, ids.to(dev), None, head)) - float(ce)) < 0.04
        assert abs(float(E.objective(m, ids.to(dev), t, head)) - float(kl)) < 0.04
    a, ga = _grads(m, ids.to(dev), t, head)
    b, gb = _grads(m, ids.to(dev), t, None)
    assert torch.allclose(a, b, rtol=1e-5)
    _close(ga, gb, 1e-3)


def test_soft_caps_are_part_of_the_objective():
    _capped_objectives("cpu")


@pytest.mark.gpu
def test_soft_caps_are_part_of_the_objective_gpu():
    _capped_objectives("cuda:0")


def test_a_teacher_file_called_labels_is_a_teacher(tmp_path, monkeypatch, capsys):
    from volta_engine_b200.models.factory import save_dense_checkpoint
    cfg = DenseConfig(n_layers=1, hidden=64, n_q=2, n_kv=1, head_dim=32, ffn=64, vocab=50)
    save_dense_checkpoint(tmp_path / "src", cfg, seed=5, fmt="bf16", std=0.08)
    g = torch.Generator().manual_seed(2)
    seqs = [torch.randint(0, 50, (8,), generator=g, dtype=torch.int32) for _ in range(2)]
    torch.save(seqs, tmp_path / "seqs.pt")
    monkeypatch.chdir(tmp_path)
    args = ["--model", "src", "--inputs", "seqs.pt", "--teacher", "labels", "--out", "out", "--steps", "1", "--batch", "1"]
    assert E.main(args) == 0 and "held-out cross entropy" in capsys.readouterr().out
    torch.save([torch.randn(8, 50, generator=g) for _ in seqs], tmp_path / "labels")
    assert E.main(args) == 0 and "held-out KL" in capsys.readouterr().out


def test_ppl_without_logits_takes_the_teachers_that_it_takes_with_them(tmp_path, capsys):
    """Ids of 64 bits and log-probabilities of 16 and 64, as other programs write them."""
    from volta_engine_b200.models.factory import save_dense_checkpoint
    cfg = DenseConfig(n_layers=1, hidden=64, n_q=2, n_kv=1, head_dim=32, ffn=64, vocab=50)
    save_dense_checkpoint(tmp_path / "src", cfg, seed=5, fmt="bf16", std=0.08)
    g = torch.Generator().manual_seed(2)
    torch.save([torch.randint(0, 50, (24,), generator=g, dtype=torch.int32)], tmp_path / "tok.pt")
    base = ["--model", str(tmp_path / "src"), "--tokens-file", str(tmp_path / "tok.pt"), "--device", "cpu"]
    for it, ft in ((torch.int64, torch.float64), (torch.int32, torch.float16)):
        ids, logp, tail = topk_teacher(2 * torch.randn(24, 50, generator=g), 4)
        torch.save({"k": 4, "ids": [ids.to(it)], "logp": [logp.to(ft)], "tail": [tail.to(ft)]}, tmp_path / "t.pt")
        a, b = (_ppl(base + ["--kl-teacher", str(tmp_path / "t.pt")] + more, capsys) for more in ([], ["--no-logits"]))
        # (what float16 loses of its log-probabilities both read alike; their sums are in its 2^-11 where logits are held)
        assert abs(a["kl"] - b["kl"]) < (1e-4 if ft == torch.float64 else 2.0 ** -8 * a["kl"])
