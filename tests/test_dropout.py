"""Dropout with a computed mask (train/dropout.py): the generator, the mask's independence of rows' places, gradients, refusals, the kernel."""
import math

import pytest
import torch

from volta_engine_b200.train import dropout as D


def test_generator_known_answers():
    """The published vectors of Philox4x32-10."""
    for counter, key, want in ((((0,) * 4), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                               (((0xFFFFFFFF,) * 4), (0xFFFFFFFF,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                               ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(w) for w in D.philox4x32([torch.tensor([c]) for c in counter], key)) == want


def test_mask_counts_and_places():
    m = D.keep_mask(400, 1000, 0.25, 7)
    # 400 000 draws: three standard deviations of the share are 0.0021
    assert abs(float(m.double().mean()) - 0.75) < 0.0021
    assert torch.equal(D.keep_mask(100, 1000, 0.25, 7, row0=300), m[300:])                 # rows know their place
    assert torch.equal(D.keep_mask(400, 37, 0.25, 7), m[:, :37])                           # and columns theirs
    for other in (D.keep_mask(400, 1000, 0.25, 8), D.keep_mask(400, 1000, 0.25, 7, site=1), D.keep_mask(400, 1000, 0.25, 7 + (1 << 40))):
        # two independent masks agree where both keep or both drop: 0.75^2 + 0.25^2, three deviations 0.0023
        assert abs(float((other == m).double().mean()) - 0.625) < 0.0023
    assert bool(D.keep_mask(5, 9, 0.0, 1).all()) and not bool(D.keep_mask(5, 9, 1.0, 1).any())


def test_gradients_by_differences():
    g = torch.Generator().manual_seed(0)
    x, r = (torch.randn(5, 11, generator=g, dtype=torch.float64).requires_grad_() for _ in range(2))
    assert torch.autograd.gradcheck(lambda a, b: D.dropout_residual(a, 0.4, 99, b, 3, 2), (x, r))
    y = D.dropout_residual(x, 0.4, 99, r, 3, 2)
    t = D.threshold_of(0.4)
    assert torch.allclose(y, r + x * D.keep_mask(5, 11, 0.4, 99, 3, 2) * 65536 / (65536 - t))
    seed = torch.tensor([99])
    y2 = D.dropout_residual(x, 0.4, seed, r, 3, 2)
    assert torch.equal(y, y2)
    seed += 1                                              # the seed has to stay until the backward pass
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y2.sum().backward()


def test_refusals_and_edges():
    x = torch.randn(3, 8)
    for p in (-0.1, 1.1, math.nan):
        with pytest.raises(ValueError, match="probability"):
            D.dropout_add(x, p, 1)
    with pytest.raises(TypeError, match="rows of type"):
        D.dropout_add(x.half(), 0.1, 1)
    with pytest.raises(ValueError, match="rows, cols"):
        D.dropout_add(x[0], 0.1, 1)
    with pytest.raises(ValueError, match="residual"):
        D.dropout_add(x, 0.1, 1, residual=x[:, :7])
    with pytest.raises(ValueError, match="residual"):
        D.dropout_add(x, 0.1, 1, residual=x.double())
    for seed in (-1, 1 << 64):
        with pytest.raises(ValueError, match="seed"):
            D.dropout_add(x, 0.1, seed)
    with pytest.raises(ValueError, match="seed tensor"):
        D.dropout_add(x, 0.1, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="row0"):
        D.dropout_add(x, 0.1, 1, row0=-1)
    with pytest.raises(ValueError, match="site"):
        D.dropout_add(x, 0.1, 1, site=1 << 32)
    assert D.dropout_add(x[:0], 0.5, 1).shape == (0, 8) and D.dropout_add(x[:, :0], 0.5, 1).shape == (3, 0)
    assert torch.equal(D.dropout_add(x, 1.0, 1, residual=x), x) and torch.equal(D.dropout_add(x, 0.0, 1), x)
    keep = D.keep_mask(3, 8, 0.5, 1)
    bad = torch.where(keep, x, torch.full_like(x, math.nan))
    assert torch.equal(D.dropout_add(bad, 0.5, 1), D.dropout_add(x, 0.5, 1))               # dropped places are not read as numbers


# ------------------------------------------------------------------------------------------------ GPU
def _near(got, x, residual, p, seed, row0, site):
    """The kernel's rows against 64 bits: one rounding of the product-and-sum to the type (2^-24 or 2^-8 of the value, half a step), and 2^-24 of both
    addends in front of it for bf16."""
    t = D.threshold_of(p)
    keep = D.keep_mask(*x.shape, p, seed, row0, site).to(x.device)
    xs = torch.where(keep, x.double() * D._scale_of(t), torch.zeros((), dtype=torch.float64, device=x.device))
    want = xs + (residual.double() if residual is not None else 0.0)
    # (the scale itself is rounded to fp32: 2^-24 of the product)
    tol = want.abs() * (2.0 ** -24 if x.dtype == torch.float32 else 2.0 ** -8) + xs.abs() * 2.0 ** -23 + want.abs() * 2.0 ** -23
    assert got.dtype == x.dtype and got.shape == x.shape
    assert bool(((got.double() - want).abs() <= tol).all())
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 7), (17, 513), (64, 2048), (129, 1000), (2, 70001)])
def test_kernel(rows, cols, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, r = (torch.randn(rows, cols, generator=g, device="cuda").to(dtype) for _ in range(2))
    for p, seed, row0, site in ((0.1, 5, 0, 0), (0.5, (1 << 63) + 12345, (1 << 33) + 7, 4000000000), (0.0, 1, 2, 3), (1.0, 1, 2, 3)):
        _near(D.dropout_add(x, p, seed, residual=r, row0=row0, site=site), x, r, p, seed, row0, site)
        _near(D.dropout_backward(x, p, seed, row0=row0, site=site), x, None, p, seed, row0, site)
    seed = torch.tensor([77], device="cuda")
    assert torch.equal(D.dropout_add(x, 0.3, seed, residual=r), D.dropout_add(x, 0.3, 77, residual=r))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_kernel_on_strided_rows_and_odd_starts(dtype):
    g = torch.Generator(device="cuda").manual_seed(1)
    base = torch.randn(40, 700, generator=g, device="cuda").to(dtype)
    for x in (base[:, 8:264], base[:, 3:259], base[::3, :256], base.t()[:256, :40]):
        _near(D.dropout_add(x, 0.2, 3, residual=base[:x.shape[0], :x.shape[1]] if x.shape[0] <= 40 else x), x,
              base[:x.shape[0], :x.shape[1]] if x.shape[0] <= 40 else x, 0.2, 3, 0, 0)


@pytest.mark.gpu
def test_kernel_gradient_and_graph():
    g = torch.Generator(device="cuda").manual_seed(2)
    x, r = (torch.randn(33, 136, generator=g, device="cuda").requires_grad_() for _ in range(2))
    dy = torch.randn(33, 136, generator=g, device="cuda")
    D.dropout_residual(x, 0.3, 11, r, 5, 1).backward(dy)
    t = D.threshold_of(0.3)
    keep = D.keep_mask(33, 136, 0.3, 11, 5, 1).cuda()
    assert torch.allclose(x.grad, dy * keep * (65536 / (65536 - t)), rtol=2.0 ** -22, atol=0) and torch.equal(r.grad, dy)
    # a captured step draws a new mask at every replay from the seed on the device; two graphs share nothing
    seed = torch.zeros(1, dtype=torch.int64, device="cuda")
    xs, rs = x.detach(), r.detach()
    D.dropout_add(xs, 0.3, seed, residual=rs)
    torch.cuda.synchronize()
    graphs = []
    for site in (0, 9):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = D.dropout_add(xs, 0.3, seed, residual=rs, site=site)
            dx = D.dropout_backward(dy, 0.3, seed, site=site)
            seed += 1
        graphs.append((gr, y, dx, site))
    seed.zero_()
    for step in range(4):
        gr, y, dx, site = graphs[step % 2]
        gr.replay()
        assert torch.equal(y, D.dropout_add(xs, 0.3, step, residual=rs, site=site)) and torch.equal(dx, D.dropout_backward(dy, 0.3, step, site=site))
    with pytest.raises(RuntimeError, match="not captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            D.dropout_residual(x, 0.3, 1, r)
    torch.cuda.synchronize()
