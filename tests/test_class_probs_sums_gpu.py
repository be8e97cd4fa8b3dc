"""Sums over many classes (semseg_amd.distill) against their exact values; bounds as class_probs_ref.py counts them."""
import math

import pytest
import torch

import class_probs_ref as ref
from class_probs_check import close
from semseg_amd import distill as D

pytestmark = pytest.mark.gpu
DEV = "cuda"

# Roundings (half steps of fp32) that a sum over a row may collect, whatever the number of classes.  Short rows: at most 40 values of a lane
# one by one, then 6 levels of lanes.  Long rows: 32 values one by one into a compensated sum (2), which is moved to another base only when
# that at least halves it (4 a move, 8 in all), then moved to the wave's, the block's and the row's maximum (4 each) and added over 6 levels
# of lanes, 4 waves and 6 levels of slices: 32 + 2 + 8 + 12 + 16 = 70.  Planes: 16 into a compensated sum, four parts: fewer.
LONGEST = 72


FLAT = [  # shape of the logits, class_dim, type, alternatives
    ((1, 1024, 512, 520), 1, torch.float32, 0), ((1, 4099, 260, 512), 1, torch.bfloat16, 1), ((2, 8192, 256, 514), 1, torch.float16, 0),
    ((1, 65536, 2, 3), 1, torch.float32, 3), ((1, 65536, 3, 3), 1, torch.bfloat16, 0), ((2, 8000, 1, 5), 1, torch.float16, 20),
    ((1, 140001, 1, 3), 1, torch.float32, 2), ((1, 30000, 2, 2), 1, torch.bfloat16, 40),
    ((300, 160), -1, torch.float32, 8), ((9, 2048), -1, torch.float32, 0), ((9, 2048), -1, torch.bfloat16, 3),
    ((600, 131072), -1, torch.float32, 4), ((520, 262145), -1, torch.bfloat16, 0), ((1, 1 << 26), -1, torch.float32, 2),
]


def flat(shape, dim, dt, low):
    """Logits of 0 at every fourth class (2, 6, ...) and `low` at the others; the exact S, sum of e d, and d."""
    C = shape[dim]
    z = torch.full(shape, low, dtype=dt, device=DEV)
    d = float(z.reshape(-1)[0])
    z.movedim(dim, -1)[..., 2::4] = 0
    top, e = len(range(2, C, 4)), math.exp(d)
    return z, top + (C - top) * e, (C - top) * e * d, d


@pytest.mark.parametrize("shape,dim,dt,k", FLAT)
def test_sums_of_equal_terms(shape, dim, dt, k):
    z, S, U, d = flat(shape, dim, dt, math.log(0.55))
    rows, h = shape[:1] + shape[2:], ref.H24
    ls, H, Ed = math.log(S), math.log(S) - U / S, -U / S
    o = D.class_logprobs(z, torch.full(rows, 2, device=DEV), topk=k, ignore_index=-1, class_dim=dim)
    err = h * (5 * Ed + LONGEST + 10 + ls)
    err_H = err + h * (5 * Ed * Ed + (2 * LONGEST + 22) * Ed + 5 * Ed * Ed + H)
    full = lambda v: torch.full(rows, v, dtype=torch.float64)  # noqa: E731
    close(o.lse, full(ls), err + h * ls, "lse")
    close(o.logprob, full(-ls), err + 2 * h * ls, "logprob")
    close(o.entropy, full(H), err_H, "entropy")
    for j in range(k):
        assert bool((o.top_ids.movedim(dim, -1)[..., j] == 2 + 4 * j).all())


@pytest.mark.parametrize("shape,dim,dt,k", [c for c in FLAT if c[1] == 1 or c[0][0] in (9, 520)])
def test_distillation_over_sums_of_equal_terms(shape, dim, dt, k):
    z, S, _, d = flat(shape, dim, dt, math.log(0.55))
    rows, h = shape[:1] + shape[2:], ref.H24
    ids = torch.full(rows + (1,), 2, dtype=torch.int32, device=DEV).movedim(-1, dim)
    ls = math.log(S)
    err = h * (5 * abs(d) + LONGEST + 10 + ls)
    full = lambda v: torch.full(rows, v, dtype=torch.float64)  # noqa: E731
    loss = D.distill_loss(z, ids, torch.zeros(ids.shape, device=DEV), class_dim=dim, reduction="none")
    close(loss, full(ls), err + 10 * h * (1 + ls), "loss")
    # half of the teacher's mass on that class, half on the rest
    half = torch.full(ids.shape, 0.5, device=DEV).log()
    q = math.exp(float(half.reshape(-1)[0]))
    loss = D.distill_loss(z, ids, half, tail=True, class_dim=dim, reduction="none")
    want = q * (math.log(q) + ls) + (1 - q) * (math.log(1 - q) - math.log((S - 1) / S))
    close(loss, full(want), 2 * err + 40 * h * (1 + ls), "loss with a tail")


@pytest.mark.parametrize("up", [1.0, -1.0])
@pytest.mark.parametrize("case", [("planes", 60000), ("planes", 70001), ("planes", 300), ("rows", 60000), ("rows", 2000)])
def test_logits_that_rise_or_fall_slowly(case, up, monkeypatch):
    """The running maximum moves with every piece of a row."""
    monkeypatch.setattr(ref, "chain", lambda C: LONGEST)
    C = case[1]
    ramp = (torch.arange(C, dtype=torch.float32) * (9.0 / C) * up).expand(4, C)
    dim = 1 if case[0] == "planes" else -1
    z = (ramp.reshape(1, 2, 2, C).permute(0, 3, 1, 2) if dim == 1 else ramp).contiguous().to(DEV)
    rows = (1, 2, 2) if dim == 1 else (4,)
    y = torch.full(rows, C // 2)
    o = D.class_logprobs(z, y.to(DEV), topk=2, ignore_index=-1, class_dim=dim)
    zl = z.movedim(dim, -1).double().cpu()
    want = ref.logprobs(zl, y, 1.0, 2, -1)
    for name in ("lse", "entropy", "logprob"):
        close(getattr(o, name), *want[name], name)
    assert torch.equal(o.top_ids.movedim(dim, -1).long().cpu(), want["top_ids"][0])
    ids = torch.tensor([0, C // 3, C - 1]).expand(rows + (3,))
    top = torch.tensor([0.3, 0.2, 0.25]).log().expand(rows + (3,))
    for tail in (False, True):
        (lv, lb), _ = ref.distill(zl, ids, top.double(), 1.0, tail, None, "none", 0.0, torch.ones(rows, dtype=torch.float64))
        loss = D.distill_loss(z, ids.movedim(-1, dim).to(DEV), top.movedim(-1, dim).to(DEV), tail=tail, class_dim=dim, reduction="none")
        close(loss, lv, lb, "loss")


def test_no_probability_above_one():
    """However the sums round: no log probability above 0, no entropy below."""
    gen = torch.Generator().manual_seed(31)
    for rows, C, dim in (((3000,), 17, -1), ((500,), 700, -1), ((600,), 5000, -1), ((3,), 40000, -1), ((2, 33, 35), 21, 1), ((1, 5, 7), 900, 1)):
        z = torch.randn(rows + (C,), generator=gen) * torch.tensor([0.01, 1.0, 30.0])[torch.randint(0, 3, rows, generator=gen)].unsqueeze(-1)
        z = z.movedim(-1, dim).contiguous().to(DEV)
        o = D.class_logprobs(z, topk=2, class_dim=dim)
        assert float(o.top_logprobs.max()) <= 0 and float(o.entropy.min()) >= 0
