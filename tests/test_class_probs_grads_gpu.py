"""Gradients of semseg_amd.distill's operators that are added to what is there, and beside rows that have none."""
import pytest
import torch

import class_probs_ref as ref
from class_probs_check import HALF, TINY, close
from semseg_amd import distill as D
from semseg_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def test_rows_beside_one_whose_id_is_no_class_keep_their_gradient():
    gen = torch.Generator().manual_seed(36)
    for shape, dim in (((5, 30), -1), ((5, 700), -1), ((5, 4000), -1), ((1, 30, 1, 5), 1)):
        z = torch.randn(shape, generator=gen)
        top, ids = z.topk(3, dim)
        ids[(2, 1) if dim == -1 else (0, 1, 0, 2)] = 10 ** 6 if dim == -1 else 30
        zz = z.to(DEV).requires_grad_()
        rows = zz.movedim(dim, -1).shape[:-1]
        loss = D.distill_loss(zz, ids.to(DEV), top.to(DEV), class_dim=dim, reduction="none")
        grad, = torch.autograd.grad(loss, zz, torch.ones(rows, device=DEV))
        one = torch.ones(rows, dtype=torch.float64)
        (lv, lb), (gv, gb) = ref.distill(*[t.movedim(dim, -1) for t in (z.double(), ids, top.double())], 1.0, False, None, "none", HALF[torch.float32], one)
        close(loss, lv, lb, "loss")
        close(grad.movedim(dim, -1), gv, gb, "gradient")
        assert (grad.movedim(dim, -1).reshape(5, -1).abs().amax(1) > 1e-3).tolist() == [True, True, False, True, True]


ADD = [((33, 19), -1), ((33, 150), -1), ((9, 300), -1), ((9, 2000), -1), ((5, 5000), -1), ((2, 21, 5, 7), 1), ((2, 150, 5, 7), 1), ((3, 2, 1, 1), 1)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape,dim", ADD)
@pytest.mark.parametrize("tail", [False, True])
def test_distillation_adds_to_a_gradient(shape, dim, dt, tail):
    """What is there plus the gradient, rounded once (16 bits: half a step of the sum)."""
    gen = torch.Generator().manual_seed(37)
    z = (torch.randn(shape, generator=gen) * 2).to(dt)
    C, k = shape[dim], 2 if shape[dim] < 12 else 12
    top, ids = torch.randn(shape, generator=gen).log_softmax(dim).topk(k, dim)
    ids.movedim(dim, -1)[0, ..., 1] = ids.movedim(dim, -1)[0, ..., 0]        # the same class twice
    rows = z.movedim(dim, -1).shape[:-1]
    w = torch.rand(rows, generator=gen)
    w = torch.where(w < 0.3, torch.zeros_like(w), w)
    old = (torch.randn(shape, generator=gen) * 0.05).to(dt)
    out = old.to(DEV)
    loss, got = D.distill_loss_grad(z.to(DEV), ids.to(DEV), top.to(DEV), temperature=2.0, tail=tail, weight=w.to(DEV), class_dim=dim, reduction="sum", grad_scale=0.5,
                                    out=out, accumulate=True)
    assert got is out
    last = lambda t: t.movedim(dim, -1)  # noqa: E731
    half = torch.tensor(0.5, dtype=torch.float64)
    (lv, lb), (gv, gb) = ref.distill(last(z.double()), last(ids), last(top.double()), 2.0, tail, w.double(), "sum", 0.0, half)
    close(loss, lv, lb, "loss")
    want = last(old.double()) + gv
    close(last(out), want, gb + want.abs() * HALF[dt] * 1.01 + ref.H24 * (gv.abs() + want.abs()), "gradient", TINY[dt])
    assert torch.equal(last(out)[w.to(DEV) == 0], last(old.to(DEV))[w.to(DEV) == 0])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape,dim", ADD)
def test_class_logprobs_adds_to_a_gradient(shape, dim, dt):
    """semseg_class_logprobs_bwd with accumulate, as a training loop that keeps its own gradients calls it."""
    gen = torch.Generator().manual_seed(38)
    z = (torch.randn(shape, generator=gen) * 2).to(dt)
    C = shape[dim]
    rows = z.movedim(dim, -1).shape[:-1]
    y, g1, g2, g3 = torch.randint(0, C, rows, generator=gen), *(torch.randn(rows, generator=gen) for _ in range(3))
    y.view(-1)[1] = -1
    old = (torch.randn(shape, generator=gen) * 0.05).to(dt)
    zd, out, yd = z.to(DEV), old.to(DEV), y.to(DEV)
    g = D.Geom(zd, D._dim(zd, dim))
    logprob, entropy, lse = (torch.empty(rows, device=DEV) for _ in range(3))
    stats = torch.empty((2,) + rows, device=DEV)
    need = ops.class_logprobs_scratch_bytes(dt, *g.geom, g.strides[2], 0)
    scratch = torch.empty(need, dtype=torch.uint8, device=DEV) if need else None
    ops.class_logprobs_fwd(zd, g.geom, g.strides, yd, -1, 1.5, 0, logprob, entropy, lse, stats, scratch=scratch)
    ops.class_logprobs_bwd(zd, g.geom, g.strides, yd, -1, 1.5, stats, entropy, *(t.to(DEV) for t in (g1, g2, g3)), out, g.strides_of(out), accumulate=True)
    last = lambda t: t.movedim(dim, -1)  # noqa: E731
    v, b = ref.logprobs_grad(last(z.double()), y, 1.5, -1, g1.double(), g2.double(), g3.double(), 0.0)
    want = last(old.double()) + v
    close(last(out), want, b + want.abs() * HALF[dt] * 1.01 + ref.H24 * (v.abs() + want.abs()), "gradient", TINY[dt])
