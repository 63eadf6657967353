"""Child process of tests/test_tuning_step.py: one CPU rank of a gloo world; the sequence-parallel tuning step with dropout and losses without logits
against the single-rank one."""
import datetime
import os
import sys

import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from volta_engine_b200.models.dense import DenseConfig, DenseModel  # noqa: E402
from volta_engine_b200.tools import e2e as E  # noqa: E402
from volta_engine_b200.tools.ppl import topk_teacher  # noqa: E402


def main():
    dist.init_process_group("gloo", timeout=datetime.timedelta(seconds=120))
    rank, world = dist.get_rank(), dist.get_world_size()
    cfg = DenseConfig(n_layers=2, hidden=64, n_q=4, n_kv=2, head_dim=16, ffn=128, vocab=96, quant="bf16")
    model = DenseModel(cfg, "cpu").init_random(seed=3, std=0.08, search=False)
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, cfg.vocab, (24,), generator=g)
    teacher = topk_teacher(torch.randn(24, cfg.vocab, generator=g), 7)
    hd, nq = cfg.head_dim, cfg.n_q // world
    q = slice(rank * nq * hd, (rank + 1) * nq * hd)
    for t in (teacher, None):
        one, sp = E.build_from_engine_model(model), E.TunedModelSP(E.build_from_engine_model(model), rank, world)
        for m in (one, sp):
            m.train()
            E.set_dropout(m, 0.3, 41, 24)
        loss1 = E.objective(one, ids, t, E.scoring_head(one))
        loss1.backward()
        mine = tuple(x[sp.rows(24)] for x in t) if t is not None else None
        loss = E.objective(sp, ids, mine, E.scoring_head(sp)) / world
        loss.backward()
        sp.sync_grads()
        total = loss.detach().clone()
        dist.all_reduce(total)
        assert torch.allclose(total, loss1.detach(), rtol=1e-5), (float(total), float(loss1))
        a, b = one.layers[0], sp.layers[0]
        assert torch.allclose(b.n1.delta.grad, a.n1.delta.grad, rtol=1e-3, atol=1e-7)
        assert torch.allclose(b.qkv.a_v.grad[: nq * hd], a.qkv.a_v.grad[q], rtol=1e-3, atol=1e-7)
        assert torch.allclose(b.dn.a_v.grad, a.dn.a_v.grad, rtol=1e-3, atol=1e-7)
    dist.barrier()
    if rank == 0:
        print("E2E_STEP_OK", flush=True)
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
