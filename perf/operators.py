"""The operators of a tuning step behind the decoder layers: what they compute, in plain torch operations, and the cases their speed is measured on.

``ce``       softmax cross entropy of next-token labels against a language model head, ``nll_r = lse_r - z_ry`` with
             ``z = cap(x head^T)`` (``cap(z) = c tanh(z / c)`` where a soft cap c is given), and its gradients. Rows whose label
             is negative are left out: no loss, no gradient.
``kl``       KL(teacher || model) against a teacher that is known by its K most likely tokens and the mass of the rest,
             ``kl_r = sum_k a_k (log a_k - log s_k) + t (log t - log max(r, 1e-12))`` with the model's probabilities ``s`` and
             their rest ``r``, and its gradients. Entries with a negative id are padding; a row of padding alone is left out.
``dropout``  ``y = residual + x m / (1 - p)`` and ``dx = dy m / (1 - p)`` with a mask m that is computed from (seed, site, row,
             column) wherever it is needed and never stored: Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011), 16 bits an element.

``stats`` are the rows' ``log sum_v exp z_v`` and the same sum without the label or the teacher's tokens.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
FLOOR = 1e-12                      # least probability of "any other token" (kl)


# ------------------------------------------------------------------------------------------------ cases
def _ce(name, rows, hidden, vocab, x="bf16", head="bf16", left_out=0.0, softcap=0.0, dx=False, dhead=False):
    return {"name": name, "op": "ce", "rows": rows, "hidden": hidden, "vocab": vocab, "x": x, "head": head, "left_out": left_out, "softcap": softcap,
            "dx": dx, "dhead": dhead}


def _kl(name, rows, hidden, vocab, topk, x="bf16", head="bf16", left_out=0.0, softcap=0.0, dx=False, dhead=False):
    return {"name": name, "op": "kl", "rows": rows, "hidden": hidden, "vocab": vocab, "topk": topk, "x": x, "head": head, "left_out": left_out,
            "softcap": softcap, "dx": dx, "dhead": dhead}


def _dropout(name, rows, cols, x="bf16", p=0.1, residual=True):
    return {"name": name, "op": "dropout", "rows": rows, "cols": cols, "x": x, "p": p, "residual": residual}


def listed():
    return [
        # one position scored against its label: the smallest call of a perplexity run (the last row of a text)
        _ce("ce_score_row", 1, 2048, 32000),
        # a prompt portion of a perplexity run over the 27B-class decoder's head
        _ce("ce_score_portion", 512, 5120, 151936),
        # soft-capped head of odd sizes, a third of the positions not scored
        _ce("ce_score_ragged", 333, 1001, 50003, left_out=0.33, softcap=30.0),
        # a small head trained throughout in 32 bits
        _ce("ce_train_small_fp32", 96, 512, 4099, x="fp32", head="fp32", dx=True, dhead=True),
        # one training batch: both gradients
        _ce("ce_train_batch", 4096, 4096, 131072, dx=True, dhead=True),
        # tuning on replies: the prompts' positions carry no label
        _ce("ce_train_replies", 2048, 2048, 151936, left_out=0.6, dx=True, dhead=True),
        # divergence from a saved teacher, forward only (quality of a quantised model)
        _kl("kl_score_portion", 512, 2048, 151936, 64),
        # the scale tuner's step: fp32 states, frozen bf16 head, top-64 teacher
        _kl("kl_tune", 2048, 2048, 151936, 64, x="fp32", dx=True),
        # odd sizes, padded teacher rows, soft cap, both gradients
        _kl("kl_train_ragged", 77, 515, 5003, 17, left_out=0.2, softcap=20.0, dx=True, dhead=True),
        # a short sequence's sublayer result
        _dropout("dropout_short", 24, 2048, x="fp32"),
        # the scale tuner's sublayer results: fp32 rows of the 27B-class width
        _dropout("dropout_tune", 2048, 5120, x="fp32", p=0.05),
        # a training batch in bf16
        _dropout("dropout_batch", 16384, 5120),
    ]


MOST_FLOPS = 6.0 * 4096 * 4096 * 131072
MOST_BYTES = 5 * 2.0 * 16384 * 5120


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ce", "ce", "ce", "kl", "kl", "dropout"])
    if op == "dropout":
        x = rng.choice(["bf16", "fp32"])
        rows, cols = _log(rng, 1, 16384), _log(rng, 64, 8192)
        if rng.random() < 0.5:
            cols = (cols + 7) // 8 * 8
        while rows * cols * 5 * (2 if x == "bf16" else 4) > MOST_BYTES:
            rows = max(1, rows // 2)
        return {"op": op, "rows": rows, "cols": cols, "x": x, "p": round(rng.uniform(0.01, 0.6), 3), "residual": rng.random() < 0.7}
    x, head = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("fp32", "bf16"), ("fp32", "fp32")])
    rows, hidden, vocab = _log(rng, 1, 8192), _log(rng, 64, 5120), _log(rng, 256, 160000)
    if rng.random() < 0.5:
        hidden = (hidden + 63) // 64 * 64
    grads = rng.choice([(False, False), (True, False), (True, True)])
    while 2.0 * rows * hidden * vocab * (1 + sum(grads)) > MOST_FLOPS / (1 if x == "bf16" else 4):
        rows = max(1, rows // 2)
    c = {"op": op, "rows": rows, "hidden": hidden, "vocab": vocab, "x": x, "head": head, "left_out": rng.choice([0.0, 0.0, round(rng.uniform(0.05, 0.9), 2)]),
         "softcap": rng.choice([0.0, 0.0, 20.0, 30.0]), "dx": grads[0], "dhead": grads[1]}
    if op == "kl":
        c["topk"] = min(vocab // 2, _log(rng, 1, 128))
    return c


def _n_left_out(case):
    return min(case["rows"] - 1, int(case["rows"] * case["left_out"]))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")
    rows, dt = case["rows"], DTYPES[case["x"]]
    s = {"case": case}
    if case["op"] == "dropout":
        s["x"], s["dy"] = randn(rows, case["cols"]).to(dt), randn(rows, case["cols"]).to(dt)
        s["residual"] = (4 * randn(rows, case["cols"])).to(dt) if case["residual"] else None
        s["seed"], s["row0"], s["site"] = 0x9E3779B97F4A7C15 * (seed + 1) & 0x7FFFFFFFFFFFFFFF, 1000 * (seed % 7), seed % 61
        return s
    hidden, vocab = case["hidden"], case["vocab"]
    # states behind a final norm and a head whose logits spread by about 2.5; a label's logit is raised by 0 to 15, as behind layers that
    # know something: losses from nearly nothing to that of a guess
    head = (randn(vocab, hidden) * (2.5 / math.sqrt(hidden))).to(DTYPES[case["head"]])
    labels = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    x = randn(rows, hidden) + 6 * torch.rand(rows, 1, generator=g, device="cuda") * torch.nn.functional.normalize(head[labels].float(), dim=1)
    out = torch.randperm(rows, generator=g, device="cuda")[: _n_left_out(case)]
    s["x"], s["head"] = x.to(dt), head
    s["dloss"] = (0.5 + torch.rand(rows, generator=g, device="cuda")) / max(1, rows - out.numel())
    if case["op"] == "ce":
        labels[out] = -100
        s["labels"] = labels
        return s
    # the teacher: another state through the same head, its K most likely tokens
    k = case["topk"]
    t = (x + 0.9 * randn(rows, hidden)).to(torch.bfloat16)
    ids, logp, tail = [], [], []
    for lo in range(0, rows, 1024):
        lp = torch.log_softmax((t[lo:lo + 1024] @ head.to(torch.bfloat16).t()).float(), dim=-1)
        v, i = lp.topk(k, dim=-1)
        ids.append(i.int())
        logp.append(v)
        tail.append((1 - v.exp().sum(-1)).clamp(min=1e-6).log())
    s["ids"], s["logp"], s["tail"] = torch.cat(ids), torch.cat(logp), torch.cat(tail)
    if out.numel():
        s["ids"][out] = -1
        if k > 2:                                  # and rows that know fewer tokens
            s["ids"][::5, k - 2:] = -1
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _capped_logits(x, head, softcap):
    z = x.float() @ head.float().t()
    if not softcap:
        return z, None
    t = torch.tanh(z / softcap)
    return softcap * t, 1 - t * t


def _head_grads(s, dz, slope):
    """Gradients of the states and the head from those of the logits."""
    case = s["case"]
    if slope is not None:
        dz = dz * slope
    dx = (dz @ s["head"].float()).to(s["x"].dtype) if case["dx"] else None
    dhead = (dz.t() @ s["x"].float()).to(s["head"].dtype) if case["dhead"] else None
    return {k: v for k, v in (("dx", dx), ("dhead", dhead)) if v is not None}


def _plain_ce(s):
    case, labels = s["case"], s["labels"]
    z, slope = _capped_logits(s["x"], s["head"], case["softcap"])
    live = labels >= 0
    y = labels.clamp(min=0)[:, None]
    m = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - m)
    ey, zy = e.gather(1, y), z.gather(1, y)
    rest = e.scatter(1, y, 0.0).sum(dim=1, keepdim=True)
    total = rest + ey
    zero = torch.zeros_like(m)
    nll = torch.where(live[:, None], m - zy + torch.log(total), zero)
    lse, lrest = (torch.where(live[:, None], m + torch.log(v), zero) for v in (total, rest))
    out = {"loss": nll[:, 0], "stats": torch.cat([lse, lrest], dim=1).t()}
    if case["dx"] or case["dhead"]:
        dz = (e / total).scatter(1, y, -rest / total) * torch.where(live, s["dloss"], zero[:, 0])[:, None]
        out.update(_head_grads(s, dz, slope))
    return out


def _plain_kl(s):
    case, ids = s["case"], s["ids"].long()
    z, slope = _capped_logits(s["x"], s["head"], case["softcap"])
    known = ids >= 0
    live = known.any(dim=1, keepdim=True)
    at = ids.clamp(min=0)
    vocab = z.shape[1]
    # 1 at the teacher's tokens (padding goes to a column behind the vocabulary)
    listed_ = torch.zeros(z.shape[0], vocab + 1, device=z.device).scatter(1, torch.where(known, ids, vocab), 1.0)[:, :vocab]
    m = z.amax(dim=1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(dim=1, keepdim=True)
    rest = (e * (1 - listed_)).sum(dim=1, keepdim=True)
    lse = m + torch.log(total)
    a = torch.where(known, torch.exp(s["logp"]), torch.zeros_like(s["logp"]))
    mass, t = a.sum(dim=1, keepdim=True), torch.where(live, torch.exp(s["tail"])[:, None], torch.zeros_like(m))
    r = (rest / total).clamp(min=FLOOR)
    terms = torch.where(a > 0, a * (s["logp"] - (z.gather(1, at) - lse)), torch.zeros_like(a))
    kl = terms.sum(dim=1, keepdim=True) + torch.where(t > 0, t * (s["tail"][:, None] - torch.log(r)), torch.zeros_like(t))
    zero = torch.zeros_like(m)
    out = {"loss": torch.where(live, kl, zero)[:, 0],
           "stats": torch.cat([torch.where(live, lse, zero), torch.where(live, m + torch.log(rest), zero)], dim=1).t()}
    if case["dx"] or case["dhead"]:
        p = e / total
        above = (rest / total >= FLOOR).float()
        dz = p * (mass + t * above) - p * (1 - listed_) * (t * above / r)
        dz = dz.scatter_add(1, at, -a)
        dz = dz * torch.where(live, s["dloss"][:, None], zero)
        out.update(_head_grads(s, dz, slope))
    return out


def _philox(counter, key):
    """Philox4x32-10 on int64 tensors (values below 2^32): four words for each counter of four."""
    c0, c1, c2, c3 = counter
    k0, k1 = key
    low = 0xFFFFFFFF
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57              # (64-bit products: the words are read from their bits)
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return c0, c1, c2, c3


def _plain_dropout(s):
    case, x = s["case"], s["x"]
    rows, cols = x.shape
    groups = (cols + 7) // 8
    row = (torch.arange(rows, device=x.device) + s["row0"])[:, None].expand(rows, groups)
    group = torch.arange(groups, device=x.device)[None].expand(rows, groups)
    words = _philox((group, row & 0xFFFFFFFF, row >> 32, torch.full_like(row, s["site"])), (s["seed"] & 0xFFFFFFFF, s["seed"] >> 32))
    halves = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], dim=-1).reshape(rows, groups * 8)[:, :cols]
    threshold = int(round(case["p"] * 65536))
    keep, scale = halves >= threshold, 65536.0 / (65536 - threshold)
    zero = torch.zeros((), device=x.device)
    y = torch.where(keep, x.float() * scale, zero)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(x.dtype), "dx": torch.where(keep, s["dy"].float() * scale, zero).to(x.dtype)}


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    op, grads = case["op"], case["dx"] or case["dhead"] if case["op"] != "dropout" else True
    if not own:
        return _plain_ce(s) if op == "ce" else _plain_kl(s) if op == "kl" else _plain_dropout(s)
    if op == "dropout":
        from volta_engine_b200.train import dropout as D
        y = D.dropout_add(s["x"], case["p"], s["seed"], residual=s["residual"], row0=s["row0"], site=s["site"])
        return {"y": y, "dx": D.dropout_backward(s["dy"], case["p"], s["seed"], row0=s["row0"], site=s["site"])}
    from volta_engine_b200.train import head_loss as L
    kw = {"softcap": case["softcap"]}
    if op == "ce":
        loss, stats = L.head_cross_entropy(s["x"], s["head"], s["labels"], **kw)
    else:
        loss, stats = L.head_kl(s["x"], s["head"], s["ids"], s["logp"], s["tail"], **kw)
    out = {"loss": loss, "stats": stats}
    if grads:
        kw.update(want_dx=case["dx"], want_dhead=case["dhead"])
        if op == "ce":
            dx, dhead = L.head_cross_entropy_backward(s["x"], s["head"], s["labels"], stats, s["dloss"], **kw)
        else:
            dx, dhead = L.head_kl_backward(s["x"], s["head"], s["ids"], s["logp"], s["tail"], stats, s["dloss"], **kw)
        out.update({k: v for k, v in (("dx", dx), ("dhead", dhead)) if v is not None})
    return out


def work(case):
    size = {"bf16": 2, "fp32": 4}
    rows = case["rows"]
    if case["op"] == "dropout":
        n = rows * case["cols"]
        # two rows of the mask's generator (forward and backward) are counted as the products that make them: 20 for 8 elements
        return {"bytes": n * size[case["x"]] * (5 if case["residual"] else 4), "flops": 2 * n * (2 + 20 / 8)}
    live, hidden, vocab = rows - _n_left_out(case), case["hidden"], case["vocab"]
    xs, ws = rows * hidden * size[case["x"]], vocab * hidden * size[case["head"]]
    teacher = rows * (8 * case["topk"] + 4) if case["op"] == "kl" else rows * 8
    grads = case["dx"] + case["dhead"]
    return {"bytes": xs + ws + teacher + 12 * rows + (xs if case["dx"] else 0) + (ws if case["dhead"] else 0) + (4 * rows if grads else 0),
            "flops": 2.0 * live * hidden * vocab * (1 + grads)}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """From the definitions, in 64 bits: log_softmax and automatic differentiation for the losses, a counter at a time for the masks."""
    s = prepare(case, seed)
    if case["op"] == "dropout":
        rows, cols = case["rows"], case["cols"]
        n = (cols + 7) // 8
        c = [np.tile(np.arange(n, dtype=np.uint64), rows), np.repeat(np.arange(s["row0"], s["row0"] + rows, dtype=np.uint64), n),
             np.zeros(rows * n, np.uint64), np.full(rows * n, s["site"], np.uint64)]
        k = [s["seed"] % 2 ** 32, s["seed"] // 2 ** 32]
        mask32, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
        for i in range(10):
            key = [np.uint64((k[0] + i * 0x9E3779B9) % 2 ** 32), np.uint64((k[1] + i * 0xBB67AE85) % 2 ** 32)]
            a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
            c = [(b >> shift) ^ c[1] ^ key[0], b & mask32, (a >> shift) ^ c[3] ^ key[1], a & mask32]
        u = np.stack(c, axis=1).astype("<u4").view("<u2").reshape(rows, n * 8)[:, :cols]
        t = int(round(case["p"] * 65536))
        keep = torch.from_numpy((u >= t).astype(np.float64)).cuda() * (65536.0 / (65536 - t))
        y = s["x"].double() * keep
        return {"y": y if s["residual"] is None else y + s["residual"].double(), "dx": s["dy"].double() * keep}
    x, head = s["x"].double().requires_grad_(case["dx"]), s["head"].double().requires_grad_(case["dhead"])
    with torch.enable_grad():
        z = torch.matmul(x, head.transpose(0, 1))
        if case["softcap"]:
            z = torch.tanh(z / case["softcap"]) * case["softcap"]
        logs = torch.log_softmax(z, dim=1)
        if case["op"] == "ce":
            live = s["labels"] >= 0
            ids = s["labels"].clamp(min=0)[:, None]
            gone = torch.zeros_like(logs, dtype=torch.bool).scatter_(1, ids, True)
            loss = -logs.gather(1, ids)[:, 0]
        else:
            known = s["ids"] >= 0
            live = known.any(1)
            ids = s["ids"].clamp(min=0).long()
            gone = torch.zeros_like(logs, dtype=torch.int32).scatter_add_(1, ids, known.int()) > 0
            lp, tail = s["logp"].double(), s["tail"].double()
            rest = logs.exp().masked_fill(gone, 0.0).sum(1).clamp(min=FLOOR)
            loss = ((lp - logs.gather(1, ids)) * lp.exp()).masked_fill(~known, 0.0).sum(1) + tail.exp() * (tail - rest.log())
        loss = loss.masked_fill(~live, 0.0)
        wanted = [v for v, w in ((x, case["dx"]), (head, case["dhead"])) if w]
        grads = iter(torch.autograd.grad(loss, wanted, s["dloss"].double()) if wanted else ())
    with torch.no_grad():
        stats = torch.stack([torch.logsumexp(z, 1), torch.logsumexp(z.masked_fill(gone, -math.inf), 1)]).masked_fill(~live[None], 0.0)
        out = {"loss": loss.detach(), "stats": stats}
        for name, w in (("dx", case["dx"]), ("dhead", case["dhead"])):
            if w:
                out[name] = next(grads)
    return out
