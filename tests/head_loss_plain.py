"""The head losses in 64 bits, by automatic differentiation, and how far a 32-bit computation of them may be off (test_head_loss.py)."""
import math

import torch


def logits(x, head, softcap):
    z = x @ head.t()
    return softcap * torch.tanh(z / softcap) if softcap else z


def cross_entropy(z, labels):
    live = labels >= 0
    nll = -torch.log_softmax(z, 1).gather(1, labels.long().clamp(min=0)[:, None])[:, 0]
    hit = torch.zeros_like(z, dtype=torch.bool).scatter_(1, labels.long().clamp(min=0)[:, None], True)
    return nll.masked_fill(~live, 0.0), hit, live


def divergence(z, ids, logp, tail):
    known = ids >= 0
    live = known.any(1)
    logs = torch.log_softmax(z, 1)
    hit = torch.zeros(z.shape[0], z.shape[1], dtype=torch.int32, device=z.device).scatter_add_(1, ids.long().clamp(min=0), known.int()) > 0
    lp = logp.double().masked_fill(~known, -math.inf)
    a = lp.exp()
    terms = torch.where(a > 0, a * (lp - logs.gather(1, ids.long().clamp(min=0))), torch.zeros_like(a)).sum(1)
    rest = logs.exp().masked_fill(hit, 0.0).sum(1).clamp(min=1e-12)
    t = tail.double().exp()
    kl = terms + torch.where(t > 0, t * (tail.double() - rest.log()), torch.zeros_like(t))
    return kl.masked_fill(~live, 0.0), hit, live


def wanted(x, head, targets, dloss, softcap):
    """-> dict of 64-bit results; "dz": gradient of the logits in front of the cap (per row of x)."""
    xd, hd = x.double(), head.double()
    z0 = (xd @ hd.t()).requires_grad_()
    z = softcap * torch.tanh(z0 / softcap) if softcap else z0
    loss, hit, live = (cross_entropy if len(targets) == 1 else divergence)(z, *targets)
    (dz,) = torch.autograd.grad(loss, z0, dloss.double())
    z = z.detach()
    stats = torch.stack([torch.logsumexp(z, 1), torch.logsumexp(z.masked_fill(hit, -math.inf), 1)]).masked_fill(~live[None], 0.0)
    return {"loss": loss.detach(), "stats": stats, "dz": dz, "dx": dz @ hd, "dhead": dz.t() @ xd, "z0": z0.detach(), "live": live}


def allowed(w, x, head, dloss, teacher_mass=1.0):
    """Bounds on |computed - 64 bits|, elementwise, from the arithmetic of the kernels:

    a logit     one MMA adds 16 products to the sum and may lose 2^-22 of the magnitudes added (each addend is cut off to the accumulator's
                bits); 16 of them stand in a piece of 256, and the pieces are added with ordinary rounding, 2^-24 each:
                e_z = |x| |W| (16 * 2^-22 + pieces * 2^-24)
    a loss      the difference of sums and logits: 2 e_z; the sums' exponentials 2^-21 each; the result's own rounding 2^-24, that of the
                statistics 2^-24 of lse
    dz          s carries e_z of its logit, e_z of lse, the rounding of lse (2^-24 |lse|) and 2^-21 of the exponential; what is added to it
                (the teacher's mass) 2^-22; rounded to its slabs: 2^-8 of its value in bf16, 2^-22 in three slabs
    dx, dhead   sums of |dz error| times the other operand, cut off as above (16 * 2^-22 a piece of 256, or 64 * 2^-22 a piece of 1024), an fp32
                addition a piece, and the rounding to the type."""
    bits = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
    xd, hd = x.double().abs(), head.double().abs()
    xd = xd * w["live"][:, None]
    h, v, r = x.shape[1], head.shape[0], x.shape[0]
    e_z = (xd @ hd.t()).amax(1) * (16 * 2.0 ** -22 + math.ceil(h / 256) * 2.0 ** -24) * (1 if x.dtype == head.dtype == torch.bfloat16 else 3)
    lse = w["stats"].abs().amax(0).nan_to_num(posinf=0.0)
    stat = e_z + 2.0 ** -21 + lse * 2.0 ** -23
    loss = teacher_mass * (2 * e_z + 2.0 ** -20) + (lse + w["loss"].abs()) * 2.0 ** -23
    exact = x.dtype == torch.float32 or head.dtype == torch.float32
    slab = 2.0 ** -22 if exact else 2.0 ** -8
    g = dloss.double().abs() * w["live"]
    s = torch.exp(w["z0"] - w["stats"][0][:, None]).clamp(max=1.0)        # (with a cap this is an upper bound only where the cap lowers z)
    rel = (2 * e_z + 2.0 ** -20 + lse * 2.0 ** -23)[:, None]
    dz = w["dz"].abs() * slab + (s + w["dz"].abs() / g.clamp(min=1e-30)[:, None]) * g[:, None] * (rel + 2.0 ** -21) * (1 + teacher_mass)

    def product(err, val, other, k, out):
        cut = 16 * 2.0 ** -22 if out == torch.float32 else 64 * 2.0 ** -22
        return err @ other + (val @ other) * (cut + math.ceil(k / 256) * 2.0 ** -24 + (2.0 ** -15 if exact and out == torch.bfloat16 else 0.0))
    dx = product(dz, w["dz"].abs(), hd, v, x.dtype) + w["dx"].abs() * bits[x.dtype]
    dhead = product(dz.t(), w["dz"].abs().t(), xd, r, head.dtype) + w["dhead"].abs() * bits[head.dtype]
    return {"loss": loss, "stats": stat, "dx": dx * 1.01 + 1e-38, "dhead": dhead * 1.01 + 1e-38}
