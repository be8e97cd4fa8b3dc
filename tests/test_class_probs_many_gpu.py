"""Rows and pixels past the first turn of every grid, and the forms that many of them choose (semseg_amd.distill): the same rows over and
over, compared with the definition in 64 bits once and with each other everywhere."""
import pytest
import torch

import class_probs_ref as ref
from class_probs_check import HALF, TINY, close
from semseg_amd import distill as D

pytestmark = pytest.mark.gpu
DEV = "cuda"


def repeated(base, n, dim):
    """[n, ...] of one [1, ...] or [p, C]: the same memory read n times."""
    return base.expand((n,) + base.shape) if dim == -1 else base.expand((n,) + base.shape[1:])


def alike(t, first, bound, what, tiny=1e-37):
    """Every one of t's first dimension is t[0], and that is `first` within its bound."""
    same = t == t[:1]
    assert bool(same.all()), "%s: %d of %d differ between equal rows" % (what, int((~same).sum()), same.numel())
    if bound is None:
        assert torch.equal(t[0].long().cpu(), first), what
    else:
        close(t[0], first, bound, what, tiny)


MANY = [  # (shape of what is repeated, class_dim, repetitions, type, alternatives)
    ((67, 5), -1, 15700, torch.float32, 3), ((67, 5), -1, 31400, torch.bfloat16, 0), ((67, 200), -1, 7900, torch.bfloat16, 9), ((67, 300), -1, 4000, torch.float32, 2),
    ((97, 2049), -1, 86500, torch.bfloat16, 2), ((97, 2053), -1, 800, torch.float32, 33),
    ((1, 17, 33, 41), 1, 360, torch.float32, 3), ((1, 24, 33, 41), 1, 360, torch.bfloat16, 8), ((1, 41, 33, 41), 1, 360, torch.float16, 1), ((1, 41, 33, 41), 1, 360, torch.float32, 16),
    ((1, 41, 33, 41), 1, 360, torch.bfloat16, 32), ((1, 150, 33, 41), 1, 200, torch.float32, 8), ((1, 19, 33, 41), 1, 360, torch.float16, 4), ((1, 19, 33, 41), 1, 360, torch.bfloat16, 2),
    ((1, 3, 1, 3), 1, 8400000, torch.float32, 1), ((1, 70, 33, 41), 1, 3, torch.float32, 40),
]


@pytest.mark.parametrize("shape,dim,n,dt,k", MANY)
def test_many_equal_rows(shape, dim, n, dt, k):
    gen = torch.Generator().manual_seed(33)
    base = (torch.randn(shape, generator=gen) * 2).to(dt).to(DEV)
    z = repeated(base, n, dim)
    rows = z.movedim(dim, -1).shape[1:-1]
    C = shape[-1] if dim == -1 else shape[1]
    y = torch.randint(0, C, rows, generator=gen)
    y = torch.where(torch.rand(rows, generator=gen) < 0.2, torch.full_like(y, -1), y)
    o = D.class_logprobs(z, y.to(DEV).expand((n,) + rows), topk=k, temperature=0.8, ignore_index=-1, class_dim=dim)
    zl = z[0].double().cpu().movedim(0 if dim == 1 else -1, -1)
    want = ref.logprobs(zl, y, 0.8, k, -1)
    for name, (v, b) in want.items():
        t = getattr(o, name)
        alike(t.movedim(dim, -1) if name.startswith("top") else t, v, b, name)


@pytest.mark.parametrize("shape,dim,n,dt", [
    ((67, 5), -1, 31400, torch.float32), ((67, 300), -1, 4000, torch.float32), ((97, 2100), -1, 680, torch.bfloat16), ((97, 1100), -1, 680, torch.float32),
    ((1, 24, 33, 41), 1, 360, torch.bfloat16), ((1, 41, 33, 41), 1, 360, torch.float32), ((1, 3, 1, 3), 1, 8400000, torch.float32)])
def test_gradients_of_many_equal_rows(shape, dim, n, dt):
    gen = torch.Generator().manual_seed(34)
    z = repeated((torch.randn(shape, generator=gen) * 2).to(dt).to(DEV), n, dim).requires_grad_()
    rows = z.movedim(dim, -1).shape[1:-1]
    C = shape[-1] if dim == -1 else shape[1]
    y, g1, g2 = torch.randint(0, C, rows, generator=gen), torch.randn(rows, generator=gen), torch.randn(rows, generator=gen)
    many = lambda t: t.to(DEV).expand((n,) + rows)  # noqa: E731
    o = D.class_logprobs(z, many(y), ignore_index=-1, class_dim=dim)
    grad, = torch.autograd.grad((o.logprob, o.entropy), z, (many(g1), many(g2)))
    zl = z[0].detach().double().cpu().movedim(0 if dim == 1 else -1, -1)
    v, b = ref.logprobs_grad(zl, y, 1.0, -1, g1.double(), g2.double(), None, HALF[dt])
    alike(grad.movedim(dim, -1), v, b, "gradient", TINY[dt])


@pytest.mark.parametrize("shape,dim,n,dt,k,tail", [
    ((67, 21), -1, 7900, torch.float32, 4, False), ((67, 21), -1, 7900, torch.bfloat16, 12, True), ((67, 300), -1, 1000, torch.float32, 20, True),
    ((97, 2100), -1, 680, torch.bfloat16, 8, True), ((1, 70, 33, 41), 1, 360, torch.float32, 4, True), ((1, 70, 33, 41), 1, 360, torch.bfloat16, 8, False),
    ((1, 70, 33, 41), 1, 360, torch.float32, 20, True), ((1, 70, 33, 41), 1, 360, torch.float16, 8, True), ((1, 70, 33, 41), 1, 800, torch.float32, 8, False),
    ((1, 70, 33, 41), 1, 1500, torch.bfloat16, 4, True), ((1, 19, 33, 41), 1, 800, torch.float32, 17, False), ((1, 3, 1, 3), 1, 8400000, torch.float32, 2, False)])
@pytest.mark.parametrize("how", ["autograd", "fused"])
def test_distillation_of_many_equal_rows(shape, dim, n, dt, k, tail, how):
    gen = torch.Generator().manual_seed(35)
    z = repeated((torch.randn(shape, generator=gen) * 2).to(dt).to(DEV), n, dim)
    rows = z.movedim(dim, -1).shape[1:-1]
    C = shape[-1] if dim == -1 else shape[1]
    t = torch.randn(rows + (C,), generator=gen) * 2
    top, ids = (t.log_softmax(-1) if tail else t).topk(k, -1)
    w = torch.rand(rows, generator=gen)
    w = torch.where(w < 0.2, torch.zeros_like(w), w)
    at = lambda t: t.movedim(-1, 0 if dim == 1 else -1).to(DEV)  # noqa: E731
    many = lambda t: t.to(DEV).expand((n,) + t.shape)  # noqa: E731
    args = (many(at(ids.int())), many(at(top)))
    zl = z[0].double().cpu().movedim(0 if dim == 1 else -1, -1)
    one = torch.ones((), dtype=torch.float64)
    (lv, lb), (gv, gb) = ref.distill(zl, ids, top.double(), 1.0, tail, w.double(), "mean", HALF[dt], one / n)
    if how == "autograd":
        zz = z.detach().requires_grad_()
        loss = D.distill_loss(zz, *args, tail=tail, weight=many(w), class_dim=dim)
        grad, = torch.autograd.grad(loss, zz)
        (rv, rb), _ = ref.distill(zl, ids, top.double(), 1.0, tail, w.double(), "none", HALF[dt], torch.ones(rows, dtype=torch.float64))
        alike(D.distill_loss(z, *args, tail=tail, weight=many(w), class_dim=dim, reduction="none"), rv, rb, "rows", 1e-30)
    else:
        loss, grad = D.distill_loss_grad(z, *args, tail=tail, weight=many(w), class_dim=dim)
    close(loss, lv, lb, "loss")
    alike(grad.movedim(dim, -1), gv, gb, "gradient", TINY[dt])
