"""semseg_amd.distill on the device against plain forms in 64 bits (class_probs_ref.py, where the bounds are derived)."""
import math

import pytest
import torch

import class_probs_ref as ref
from semseg_amd import distill as D
from semseg_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# the smallest normal value of fp16 is 6.1e-5: below it a gradient's step is 2^-24, half of it the rounding; flush of fp32 below 1e-38
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}

# (layout, shape of the rows, classes, values between rows beyond the classes)
ROWS = [
    ("rows", (1,), 1, 0), ("rows", (1,), 2, 0), ("rows", (5,), 3, 0), ("rows", (130,), 19, 0), ("rows", (67,), 21, 3), ("rows", (2, 9, 7), 150, 106),
    ("rows", (33,), 64, 0), ("rows", (9,), 65, 0), ("rows", (300,), 150, 0), ("rows", (40,), 151, 5), ("rows", (17,), 257, 0), ("rows", (11,), 513, 1),
    ("rows", (6,), 1000, 24), ("rows", (7,), 1025, 0), ("rows", (3,), 2049, 0), ("rows", (5,), 4099, 2), ("rows", (2,), 32000, 0),
    ("rows", (3,), 50001, 0), ("rows", (1,), 131072, 0), ("rows", (1,), 262147, 0),
]
PLANES = [
    ("planes", (1, 1, 1), 2, 0), ("planes", (2, 3, 5), 1, 0), ("planes", (2, 9, 7), 2, 0), ("planes", (1, 13, 11), 19, 0), ("planes", (3, 8, 8), 21, 0),
    ("planes", (2, 65, 65), 19, 0), ("planes", (1, 33, 31), 150, 0), ("planes", (2, 17, 15), 150, 0), ("planes", (2, 3, 5), 257, 0), ("planes", (1, 1, 3), 1000, 0),
    ("planes", (1, 5, 1), 5000, 0), ("planes", (2, 8, 16), 40, 0), ("planes", (1, 2, 3), 9000, 0), ("planes", (1, 1, 2), 70001, 0),
]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(case, dt, gen, scale=2.0):
    """(logits, class_dim) on the device."""
    layout, rows, C, pad = case
    if layout == "rows":
        z = (torch.randn(rows + (C + pad,), generator=gen) * scale).to(dt).to(DEV)[..., :C]
        return z, -1
    n = rows[0]
    return (torch.randn((n, C) + rows[1:], generator=gen) * scale).to(dt).to(DEV), 1


def close(got, want, bound, what, tiny=1e-37):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ": NaN elsewhere"
    rest = ~fin & ~torch.isnan(want)
    assert torch.equal(got[rest], want[rest]), what + ": infinities"
    bound = torch.broadcast_to(bound, want.shape)[fin]
    off = (got[fin] - want[fin]).abs()
    over = off - bound.nan_to_num(0, 0, 0) - tiny
    if over.numel():
        i = int(over.argmax())
        assert float(over[i]) <= 0, "%s: off %.3g, allowed %.3g, value %.6g" % (what, off[i], bound[i], want[fin][i])


def last(t, dim):
    return ref.rows_last(t, dim)


def check_logprobs(z, dim, label, T, k, ignore=255):
    o = D.class_logprobs(z, label, topk=k, temperature=T, ignore_index=ignore, class_dim=dim)
    want = ref.logprobs(last(z, dim), None if label is None else label.cpu(), T, k, ignore)
    assert (o.logprob is None) == (label is None) and (o.top_ids is None) == (k == 0)
    for name, (v, b) in want.items():
        got = getattr(o, name)
        if name == "top_ids":
            assert got.dtype == torch.int32
            assert torch.equal(last(got, dim), v), name
        else:
            assert got.dtype == torch.float32
            close(last(got, dim) if name == "top_logprobs" else got, v, b, name)
    return o


def labels(rows, C, gen, void=0.15, ignore=255):
    y = torch.randint(0, C, rows, generator=gen)
    return torch.where(torch.rand(rows, generator=gen) < void, torch.full_like(y, ignore), y).to(DEV)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", ROWS + PLANES)
def test_logprobs(case, dt):
    gen = torch.Generator().manual_seed(case[2])
    z, dim = make(case, dt, gen)
    C = case[2]
    y = labels(case[1], C, gen, ignore=-1)
    for T, k in ((1.0, min(C, 3)), (0.7, min(C, 20)), (3.0, 0), (1.0, min(C, 8))):
        check_logprobs(z, dim, y, T, k, ignore=-1)
    check_logprobs(z, dim, None, 1.0, min(C, 64))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", [("rows", (40,), 19, 0), ("rows", (12,), 150, 2), ("rows", (4,), 5000, 0), ("planes", (2, 7, 5), 150, 0), ("planes", (1, 5, 3), 900, 0)])
def test_alternatives_of_equal_logits_come_by_rising_class(case, dt):
    gen = torch.Generator().manual_seed(5)
    z, dim = make(case, dt, gen)
    C, k = case[2], min(case[2], 33)
    v = (torch.randint(0, 4, z.shape, generator=gen).to(z.dtype).to(DEV) - 1.0)
    v = torch.where(v == 0, torch.where(torch.rand(z.shape, generator=gen).to(DEV) < 0.5, v, -v), v)       # -0 and +0 are equal
    check_logprobs(v.contiguous(), dim, None, 1.0, k)
    check_logprobs(torch.zeros_like(z).contiguous(), dim, None, 1.0, k)
    for up in (1.0, -1.0):                                                                               # sorted either way
        ramp = torch.arange(C, dtype=torch.float32).div(C / 8.0).mul(up)
        ramp = ramp.view((1,) * (z.dim() - 1) + (C,)) if dim == -1 else ramp.view((1, C) + (1,) * (z.dim() - 2))
        check_logprobs(ramp.expand(z.shape).to(dt).to(DEV).contiguous(), dim, None, 1.0, k)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", [("rows", (24,), 19, 0), ("rows", (24,), 150, 106), ("rows", (24,), 3000, 0), ("planes", (2, 4, 3), 21, 0), ("planes", (2, 4, 3), 150, 0)])
def test_masked_classes_and_rows(case, dt):
    """-inf, the type's lowest value and void rows that hold NaN and infinities."""
    gen = torch.Generator().manual_seed(6)
    z, dim = make(case, dt, gen)
    zl = z.movedim(dim, -1)
    flat = zl.reshape(24, -1).clone()
    C, low = case[2], torch.finfo(dt).min
    flat[0] = -math.inf
    flat[1] = low
    flat[2, : C // 2] = -math.inf
    flat[3, 1:] = low
    flat[4, 1:] = -math.inf
    flat[5, : C - 1] = low
    flat[6] = math.nan
    flat[7] = math.inf
    flat[8, 0] = math.nan
    flat[9] = torch.where(torch.rand(C, generator=gen).to(DEV) < 0.5, flat[9], torch.full_like(flat[9], -math.inf))
    y = torch.randint(0, C, (24,), generator=gen)
    y[6:9] = 255 if C <= 255 else -1
    y[2] = 0                      # a label that is masked
    ig = 255 if C <= 255 else -1
    z2 = flat.view(zl.shape).movedim(-1, dim).contiguous()
    y2 = y.view(zl.shape[:-1]).to(DEV)
    assert torch.isnan(z2).any()
    o = D.class_logprobs(z2.requires_grad_(), y2, topk=min(C, 5), ignore_index=ig, class_dim=dim)
    clean = torch.where(torch.isnan(z2.detach()) | (z2.detach() == math.inf), torch.zeros_like(z2), z2.detach())      # void rows: any value
    want = ref.logprobs(last(clean, dim), y2.cpu(), 1.0, min(C, 5), ig)
    for name, (v, b) in want.items():
        got = getattr(o, name)
        if name == "top_ids":
            assert torch.equal(last(got, dim), v)
        else:
            close(last(got, dim) if name == "top_logprobs" else got, v, b, name)
    assert float(o.lse.detach().reshape(-1)[0]) == -math.inf and float(o.entropy.detach().reshape(-1)[0]) == 0
    g1, g2 = torch.randn(zl.shape[:-1], generator=gen), torch.randn(zl.shape[:-1], generator=gen)
    g1v, g2v = g1.clone().view(-1), g2.clone().view(-1)
    g1v[6:9] = math.nan           # what reaches a void row is not used
    grad, = torch.autograd.grad((o.logprob, o.entropy), z2, (g1v.view(g1.shape).to(DEV), g2v.view(g2.shape).to(DEV)))
    v, b = ref.logprobs_grad(last(clean, dim), y2.cpu(), 1.0, ig, g1.double(), g2.double(), None, HALF[dt])
    close(last(grad, dim), v, b, "grad", TINY[dt])


def test_nan_and_infinity_stay_in_their_row():
    for case in (("rows", (6,), 150, 0), ("rows", (6,), 9000, 0), ("planes", (1, 2, 3), 150, 0)):
        gen = torch.Generator().manual_seed(7)
        z, dim = make(case, torch.float32, gen)
        zl = z.movedim(dim, -1).reshape(6, -1)
        zl[1, 7], zl[3, 2], zl[4, 0] = math.nan, math.inf, -math.inf
        z2 = zl.view(z.movedim(dim, -1).shape).movedim(-1, dim).contiguous()
        y = torch.randint(0, case[2], (6,), generator=gen).view(z.movedim(dim, -1).shape[:-1]).to(DEV)
        o = D.class_logprobs(z2, y, topk=4, class_dim=dim, ignore_index=-1)
        for t in (o.logprob, o.entropy, o.lse):
            assert torch.isnan(t.reshape(-1)).tolist() == [False, True, False, True, False, False]
        ids = last(o.top_ids, dim).view(6, 4)
        assert bool(((ids >= 0) & (ids < case[2])).all()) and int(ids[1, 0]) == 7 and int(ids[3, 0]) == 2


def test_labels_that_are_no_class():
    z = torch.randn(4, 9, device=DEV).requires_grad_()
    y = torch.tensor([3, 9, -7, 255], device=DEV)
    o = D.class_logprobs(z, y)
    assert torch.isnan(o.logprob).tolist() == [False, True, True, False]
    assert bool(torch.isfinite(o.entropy).all()) and float(o.entropy.detach()[3]) == 0
    g, = torch.autograd.grad(o.logprob, z, torch.ones(4, device=DEV))
    assert bool(torch.isfinite(g).all()) and float(g[1:].abs().max()) == 0


def test_the_default_void_label_is_no_class():
    y = torch.tensor([255, -100, 3], device=DEV)
    few, many = (D.class_logprobs(torch.zeros(3, C, device=DEV), y) for C in (255, 256))
    assert torch.isnan(few.logprob).tolist() == [False, True, False] and few.entropy[0] == 0
    assert torch.isnan(many.logprob).tolist() == [False, False, False] and many.entropy[0] > 0 and many.entropy[1] == 0


@pytest.mark.parametrize("scale", [1000.0, 1e-3])
def test_far_and_near_logits(scale):
    gen = torch.Generator().manual_seed(8)
    for case in (("rows", (50,), 150, 0), ("rows", (5,), 5000, 0), ("planes", (1, 7, 9), 150, 0)):
        z, dim = make(case, torch.float32, gen, scale)
        z = z + (5000.0 if scale < 1 else 0.0)
        check_logprobs(z, dim, labels(case[1], case[2], gen), 1.0, 3)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", [c for c in ROWS + PLANES if c[2] < 60000])
def test_logprobs_gradient(case, dt):
    gen = torch.Generator().manual_seed(9)
    z, dim = make(case, dt, gen)
    z = z.requires_grad_()
    rows = case[1]
    y = labels(rows, case[2], gen, ignore=-1)
    g1, g2, g3 = (torch.randn(rows, generator=gen) for _ in range(3))
    for T, use in ((1.0, (1, 1, 0)), (2.0, (1, 0, 0)), (0.5, (0, 1, 1))):
        o = D.class_logprobs(z, y, temperature=T, ignore_index=-1, class_dim=dim)
        outs = [t for t, u in zip((o.logprob, o.entropy, o.lse), use) if u]
        grad, = torch.autograd.grad(outs, z, [g.to(DEV) for g, u in zip((g1, g2, g3), use) if u])
        assert grad.dtype == dt and grad.shape == z.shape
        v, b = ref.logprobs_grad(last(z, dim), y.cpu(), T, -1, *[g.double() if u else None for g, u in zip((g1, g2, g3), use)], HALF[dt])
        close(last(grad, dim), v, b, "grad %s" % (use,), TINY[dt])


def teacher(case, z, dim, k, T, tail, gen, dt=torch.float32):
    t = torch.randn(z.shape, generator=gen) * 2 + z.detach().float().cpu() * 0.5
    tl = t.movedim(dim, -1)
    if tail:
        tl = (tl.double() / T).log_softmax(-1).float()
    top, ids = tl.topk(k, -1)
    ids = ids.int()
    if ids.numel() > 6 and k > 1:
        ids.view(-1, k)[0, 1] = -1                      # an absent entry
        ids.view(-1, k)[-1, -1] = ids.view(-1, k)[-1, 0]      # the same class twice
    return ids.movedim(-1, dim).to(DEV), top.movedim(-1, dim).to(dt).to(DEV)


def check_distill(z, dim, ids, top, T, tail, w, reduction, how="autograd", dt=None):
    dt = z.dtype
    gen = torch.Generator().manual_seed(1)
    rows = z.movedim(dim, -1).shape[:-1]
    gl = torch.randn(rows, generator=gen) if reduction == "none" else torch.tensor(0.37)
    zz = z.detach().requires_grad_()
    if how == "autograd":
        loss = D.distill_loss(zz, ids, top, temperature=T, tail=tail, weight=w, class_dim=dim, reduction=reduction)
        grad, = torch.autograd.grad(loss, zz, gl.to(DEV))
    else:
        loss, grad = D.distill_loss_grad(z.detach(), ids, top, temperature=T, tail=tail, weight=w, class_dim=dim, reduction=reduction,
                                         grad_scale=0.37)
    assert grad.dtype == dt and grad.shape == z.shape and loss.dtype == torch.float32
    (lv, lb), (gv, gb) = ref.distill(last(z, dim), last(ids, dim), last(top, dim), T, tail, None if w is None else w.double().cpu(), reduction,
                                     HALF[dt], gl.double())
    close(loss, lv, lb, "loss", 1e-30)
    close(last(grad, dim), gv, gb, "grad", TINY[dt])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", [c for c in ROWS + PLANES if c[2] < 140000])
def test_distill(case, dt):
    gen = torch.Generator().manual_seed(11)
    z, dim = make(case, dt, gen)
    C, rows = case[2], case[1]
    w = torch.rand(rows, generator=gen)
    w = torch.where(w < 0.2, torch.zeros_like(w), w).to(DEV)
    w.view(-1)[0] = 1.0
    for T, k, tail, red, weight, how, tdt in (
            (1.0, min(C, 4), False, "mean", None, "autograd", torch.float32), (4.0, min(C, 8), False, "mean", w, "fused", torch.bfloat16),
            (2.0, min(C, 16), True, "mean", w, "autograd", torch.float32), (1.0, min(C, 5), True, "sum", None, "fused", torch.float32),
            (0.5, min(C, 33), True, "none", w, "autograd", torch.float32), (1.0, min(C, 64), False, "sum", None, "autograd", torch.float16)):
        ids, top = teacher(case, z, dim, k, T, tail, gen, tdt)
        check_distill(z, dim, ids, top, T, tail, weight, red, how)


@pytest.mark.parametrize("k", [9, 15, 16, 17, 40])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("how", ["autograd", "fused"])
def test_distill_entries_drawn_with_repeats(k, tail, how):
    """Entries sampled with repetition, some absent: every class collects what all its entries hold, however many a lane has."""
    gen = torch.Generator().manual_seed(13)
    for case, dt in ((("rows", (45,), 150, 256), torch.float32), (("rows", (45,), 21, 0), torch.bfloat16), (("rows", (5,), 700, 0), torch.float32),
                     (("rows", (3,), 2500, 0), torch.bfloat16), (("planes", (1, 7, 5), 21, 0), torch.float32)):
        z, dim = make(case, dt, gen)
        ids = torch.randint(0, case[2] // 3, case[1] + (k,), generator=gen).int()
        ids[torch.rand(ids.shape, generator=gen) < 0.1] = -1
        top = torch.randn(ids.shape, generator=gen).double().log_softmax(-1).float() - 0.5
        check_distill(z, dim, ids.movedim(-1, dim).to(DEV), top.movedim(-1, dim).to(DEV), 1.5, tail, None, "mean", how)


@pytest.mark.parametrize("case", [("rows", (12,), 19, 0), ("rows", (12,), 150, 106), ("rows", (12,), 4000, 0), ("planes", (1, 4, 3), 21, 0), ("planes", (1, 4, 3), 150, 0)])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("how", ["autograd", "fused"])
def test_distill_masks(case, tail, how):
    """Weight-0 rows with NaN, rows without entries, -inf students, entries of no mass, ids as int64, all entries absent."""
    gen = torch.Generator().manual_seed(12)
    z, dim = make(case, torch.float32, gen)
    zl = z.movedim(dim, -1).reshape(12, -1).clone()
    ids, top = teacher(case, z, dim, 3, 1.0, tail, gen)
    il, tl = ids.movedim(dim, -1).reshape(12, 3).clone(), top.movedim(dim, -1).reshape(12, 3).clone()
    w = torch.ones(12)
    w[1], w[5] = 0.0, 0.25
    zl[1] = math.nan
    il[1] = 10 ** 6               # not read
    il[2] = -1
    tl[3] = -math.inf             # entries present, none with mass
    il[4, 1:] = -1
    zl[6, (int(il[6, 0]) + 1) % case[2]] = -math.inf
    if int((il[6] == (int(il[6, 0]) + 1) % case[2]).sum()):
        il[6, 1:] = -1
    zl[7] = torch.finfo(torch.float32).min
    shape = z.movedim(dim, -1).shape
    z2 = zl.view(shape).movedim(-1, dim).contiguous()
    back = lambda t: t.view(shape[:-1] + (3,)).movedim(-1, dim).contiguous()  # noqa: E731
    clean = zl.clone()
    clean[1] = 0
    i2, t2, w2 = back(il.long()), back(tl), w.view(shape[:-1]).to(DEV)
    if how == "autograd":
        zz = z2.requires_grad_()
        loss = D.distill_loss(zz, i2, t2, tail=tail, weight=w2, class_dim=dim)
        grad, = torch.autograd.grad(loss, zz)
    else:
        loss, grad = D.distill_loss_grad(z2, i2, t2, tail=tail, weight=w2, class_dim=dim)
    il[1] = 0
    (lv, lb), (gv, gb) = ref.distill(clean.double().cpu(), il.long().cpu(), tl.double().cpu(), 1.0, tail, w.double(), "mean", HALF[torch.float32])
    close(loss, lv, lb, "loss")
    close(last(grad, dim).reshape(12, -1), gv, gb, "grad")
    assert bool((last(grad, dim).reshape(12, -1)[[1, 2]] == 0).all())


def test_distill_of_nothing_and_of_ids_that_are_no_class():
    z = torch.randn(5, 30, device=DEV).requires_grad_()
    top, ids = z.detach().topk(3, 1)
    loss = D.distill_loss(z, ids, top, weight=torch.zeros(5, device=DEV))
    grad, = torch.autograd.grad(loss, z)
    assert math.isnan(float(loss.detach())) and float(grad.abs().max()) == 0
    ids = ids.clone()
    ids[2, 1] = 30
    rows = D.distill_loss(z, ids, top, reduction="none")
    grad, = torch.autograd.grad(rows, z, torch.ones(5, device=DEV))
    assert torch.isnan(rows).tolist() == [False, False, True, False, False]
    assert float(grad[2].abs().max()) == 0 and bool(torch.isfinite(grad).all()) and float(grad[0].abs().max()) >= 0
    zn = torch.full((2, 30), -math.inf, device=DEV).requires_grad_()
    loss = D.distill_loss(zn, ids[:2], top[:2])
    grad, = torch.autograd.grad(loss, zn)
    assert float(loss.detach()) == math.inf and float(grad.abs().max()) == 0


def test_a_student_equal_to_its_teacher_has_no_loss_and_no_gradient_on_the_entries():
    z = torch.randn(64, 8, device=DEV)
    top, ids = z.topk(8, 1)
    loss, grad = D.distill_loss_grad(z, ids, top, temperature=2.0)
    assert abs(float(loss)) < 4 * 40 * 2.0 ** -24 and float(grad.abs().max()) < 2 * 40 * 2.0 ** -24


# ---------------------------------------------------------------------------------------------
# layouts, accumulation, streams, graphs
# ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("order", [(0, 1, 2, 3), (0, 2, 3, 1), (1, 0, 2, 3)])
@pytest.mark.parametrize("class_dim", [1, -1])
def test_every_order_of_memory(order, class_dim, dt):
    """Logits in each order of memory, the classes named as dimension 1 or the last, a teacher in every other order."""
    gen = torch.Generator().manual_seed(14)
    z = (torch.randn(3, 21, 5, 7, generator=gen) * 2).to(dt)
    inverse = tuple(sorted(range(4), key=lambda i: order[i]))
    v = z.to(DEV).permute(order).contiguous().permute(inverse)
    assert torch.equal(v.cpu(), z)
    seen = lambda t: t if class_dim == 1 else t.movedim(1, -1)  # noqa: E731
    v = seen(v)
    top, ids = torch.randn(3, 21, 5, 7, generator=gen).topk(4, 1)
    for o in ((0, 1, 2, 3), (0, 2, 3, 1), (1, 0, 2, 3), (2, 0, 1, 3)):
        back = tuple(sorted(range(4), key=lambda i: o[i]))
        t_ids, t_top = (seen(t.to(DEV).permute(o).contiguous().permute(back)) for t in (ids, top))
        for how in ("autograd", "fused"):
            check_distill(v, class_dim, t_ids, t_top, 2.0, False, None, "mean", how)
    y = labels((3, 5, 7), 21, gen, ignore=-1)
    check_logprobs(v, class_dim, y, 1.0, 6, -1)
    x, g1 = v.detach().requires_grad_(), torch.randn(3, 5, 7, generator=gen)
    o = D.class_logprobs(x, y, ignore_index=-1, class_dim=class_dim)
    grad, = torch.autograd.grad(o.logprob, x, g1.to(DEV))
    want, b = ref.logprobs_grad(last(v, class_dim), y.cpu(), 1.0, -1, g1.double(), None, None, HALF[dt])
    close(last(grad, class_dim), want, b, "gradient", TINY[dt])


def test_layouts_agree_and_gradients_reach_views():
    """The same logits as planes, channels_last, pixel-major with padding, and broadcast over a batch."""
    gen = torch.Generator().manual_seed(13)
    z = torch.randn(2, 150, 9, 11, generator=gen).to(DEV)
    y = labels((2, 9, 11), 150, gen)
    wide = torch.zeros(2, 9, 11, 256, device=DEV)
    wide[..., :150] = z.movedim(1, -1)
    views = [z, z.contiguous(memory_format=torch.channels_last), wide[..., :150].movedim(-1, 1)]
    ids, top = teacher(("planes", None, 150, 0), z, 1, 4, 1.0, False, gen)
    first = None
    for v in views:
        v = v.detach().requires_grad_()
        o = D.class_logprobs(v, y, topk=5)
        loss = D.distill_loss(v, ids, top, temperature=2.0)
        grad, = torch.autograd.grad(loss + o.logprob.mean(), v)
        got = (o.top_ids.contiguous(), o.entropy, o.top_logprobs, loss, grad)
        first = first or got
        assert torch.equal(got[0], first[0])
        for a, b in zip(got[1:], first[1:]):
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
    # the same teacher kept pixel-major
    loss = D.distill_loss(z, ids.contiguous(memory_format=torch.channels_last), top.contiguous(memory_format=torch.channels_last), temperature=2.0)
    assert torch.allclose(loss, first[3], rtol=1e-6)
    # one row for many: the gradient of a broadcast input is the sum
    one = torch.randn(1, 30, generator=gen).to(DEV).requires_grad_()
    o = D.class_logprobs(one.expand(50, 30), torch.arange(50, device=DEV) % 30, ignore_index=-1)
    g, = torch.autograd.grad(o.logprob.sum(), one)
    p = one.detach().double().softmax(-1)
    want = torch.bincount(torch.arange(50, device=DEV) % 30, minlength=30).double() - 50 * p
    assert float((g.double() - want).abs().max()) < 50 * 64 * 2.0 ** -24


@pytest.mark.parametrize("case", [("rows", (3, 5, 7), 150, 106), ("rows", (9,), 3001, 0), ("planes", (2, 5, 7), 150, 0)])
def test_gradient_into_a_given_buffer(case):
    gen = torch.Generator().manual_seed(14)
    z, dim = make(case, torch.float32, gen)
    ids, top = teacher(case, z, dim, 4, 1.0, False, gen)
    loss, grad = D.distill_loss_grad(z, ids, top, class_dim=dim, grad_scale=0.5)
    base = torch.randn(z.movedim(dim, -1).shape[:-1] + (case[2] + 6,), generator=gen).to(DEV)
    buf = base.clone()[..., :case[2]] if dim == -1 else torch.randn(z.shape, generator=gen).to(DEV)
    before, pad = buf.clone(), None
    if dim == -1:
        whole = base.clone()
        buf = whole[..., :case[2]]
        before = buf.clone()
    loss2, out = D.distill_loss_grad(z, ids, top, class_dim=dim, grad_scale=0.5, out=buf, accumulate=True)
    assert out is buf and torch.equal(loss, loss2)
    assert torch.allclose(buf, before + grad, rtol=0, atol=2.0 ** -24 * 8)
    if dim == -1:
        assert torch.equal(whole[..., case[2]:], base[..., case[2]:])      # what lies between the rows is left as it was
    loss3, _ = D.distill_loss_grad(z, ids, top, class_dim=dim, grad_scale=0.5, out=buf)
    assert torch.equal(buf, grad)
    for bad in (z, buf[..., 1:], buf.double()):
        with pytest.raises(ValueError):
            D.distill_loss_grad(z, ids, top, class_dim=dim, out=bad)
    with pytest.raises(ValueError):
        D.distill_loss_grad(z, ids, top, class_dim=dim, accumulate=True)


def test_outputs_repeat_exactly_and_streams_do_not_mix():
    gen = torch.Generator().manual_seed(15)
    cases = [("rows", (500,), 150, 106), ("rows", (3,), 50001, 0), ("planes", (2, 33, 35), 150, 0)]
    sets = []
    for c in cases:
        z, dim = make(c, torch.float32, gen)
        ids, top = teacher(c, z, dim, 4, 1.0, True, gen)
        sets.append((z, dim, ids, top, labels(c[1], c[2], gen, ignore=-1)))

    def once(s):
        z, dim, ids, top, y = s
        o = D.class_logprobs(z, y, topk=4, class_dim=dim, ignore_index=-1)
        return list(o) + list(D.distill_loss_grad(z, ids, top, tail=True, class_dim=dim))
    first = [once(s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(4):
        outs = []
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                outs.append(once(s))
        torch.cuda.synchronize()
        for a, b in zip(first, outs):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_captured_graphs_replay_with_new_inputs():
    """Two graphs captured from the same calls, replayed in turn with eager work between them: no workspace is shared, nothing is kept."""
    gen = torch.Generator().manual_seed(16)
    cases = [("rows", (200,), 150, 106), ("rows", (2,), 40000, 0), ("planes", (1, 21, 23), 21, 0)]
    for c in cases:
        z, dim = make(c, torch.float32, gen)
        ids, top = teacher(c, z, dim, 4, 1.0, False, gen)
        y = labels(c[1], c[2], gen, ignore=-1)
        w = (torch.rand(c[1], generator=gen) + 0.5).to(DEV)

        def once():
            zz = z.detach().requires_grad_()
            o = D.class_logprobs(zz, y, topk=4, class_dim=dim, ignore_index=-1)
            loss = D.distill_loss(zz, ids, top, temperature=2.0, weight=w, class_dim=dim)
            g, = torch.autograd.grad(loss + o.entropy.mean(), zz)
            l2, g2 = D.distill_loss_grad(z, ids, top, temperature=2.0, weight=w, class_dim=dim)
            return [o.logprob.detach(), o.top_ids, loss.detach(), g, l2, g2]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                once()
        torch.cuda.current_stream().wait_stream(side)
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = once()
            graphs.append((g, out))
        for i in range(4):
            z.copy_(torch.randn(z.shape, generator=gen).to(DEV))
            want = once()
            for g, out in graphs:
                g.replay()
            torch.cuda.synchronize()
            for _, out in graphs:
                for k, (a, b) in enumerate(zip(out, want)):
                    assert torch.equal(a, b), (c, i, k)


@pytest.mark.parametrize("C", [21, 150, 300, 4000])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_rows_that_two_strides_walk(C, dt):
    """Cropped maps: rows of images that do not follow each other; alternatives, entries and gradients into such maps."""
    gen = torch.Generator().manual_seed(20)
    whole = torch.randn(3, 6, 5, C + 3, generator=gen).to(dt).to(DEV)
    z = whole[:, 1:5, :, :C]
    assert D.Geom(z, 3).geom == (3, 20, C)
    y = labels((3, 4, 5), C, gen, ignore=-1)
    o = check_logprobs(z, -1, y, 1.0, 6, ignore=-1)
    zz = z.detach().requires_grad_()
    o = D.class_logprobs(zz, y, ignore_index=-1, class_dim=-1)
    g1 = torch.randn(3, 4, 5, generator=gen)
    grad, = torch.autograd.grad(o.logprob, zz, g1.to(DEV))
    v, b = ref.logprobs_grad(last(z, -1), y.cpu(), 1.0, -1, g1.double(), None, None, HALF[dt])
    close(last(grad, -1), v, b, "grad", TINY[dt])
    ids, top = teacher(("rows", (3, 4, 5), C, 3), z, -1, 5, 1.0, False, gen)
    wide = torch.zeros(3, 9, 5, 5, dtype=torch.int32, device=DEV)
    wide[:, 2:6] = ids
    wtop = torch.zeros(3, 9, 5, 5, device=DEV)
    wtop[:, 2:6] = top
    for how in ("autograd", "fused"):
        check_distill(z, -1, wide[:, 2:6], wtop[:, 2:6], 2.0, False, None, "mean", how)
    out = torch.zeros_like(whole)
    loss, _ = D.distill_loss_grad(z, ids, top, class_dim=-1, out=out[:, 1:5, :, :C])
    loss2, g2 = D.distill_loss_grad(z, ids, top, class_dim=-1)
    assert torch.equal(out[:, 1:5, :, :C], g2) and torch.equal(loss, loss2)
    assert float(out[:, 0].abs().max()) == float(out[:, 5].abs().max()) == float(out[..., C:].abs().max()) == 0


@pytest.mark.parametrize("case", [("rows", (6,), 21, 0), ("rows", (6,), 150, 0), ("rows", (6,), 1500, 0), ("rows", (6,), 9000, 0),
                                  ("planes", (1, 2, 3), 21, 0), ("planes", (1, 2, 3), 150, 0)])
@pytest.mark.parametrize("how", ["autograd", "fused"])
def test_a_rest_far_below_the_entries(case, how):
    """A student sure of the teacher's classes: what is outside them has a mass that fp32 does not hold, but a finite logarithm."""
    gen = torch.Generator().manual_seed(21)
    z, dim = make(case, torch.float32, gen)
    zl = z.movedim(dim, -1).reshape(6, -1).clone()
    ids = torch.stack([torch.randperm(case[2], generator=gen)[:3] for _ in range(6)]).to(DEV)
    up = torch.tensor([[60.0], [120.0], [200.0], [400.0], [0.0], [1000.0]], device=DEV)
    zl.scatter_add_(1, ids, up.expand(6, 3).contiguous())
    top = torch.tensor([0.5, 0.2, 0.1], device=DEV).log().expand(6, 3).contiguous()
    shape = z.movedim(dim, -1).shape
    back = lambda t: t.view(shape[:-1] + (t.shape[-1],)).movedim(-1, dim).contiguous()  # noqa: E731
    check_distill(back(zl), dim, back(ids), back(top), 1.0, True, None, "mean", how)
    rows = D.distill_loss(back(zl), back(ids), back(top), tail=True, class_dim=dim, reduction="none").reshape(-1)
    assert bool(torch.isfinite(rows).all()) and float(rows[5]) > 150


@pytest.mark.parametrize("dt,C", [(torch.float32, 70001), (torch.bfloat16, 140003), (torch.float32, 150001)])
def test_many_long_rows_as_few(dt, C):
    """520 rows take a block each, 8 are sliced over many: the same rows either way (the latter are checked against the definition above);
    long enough that a block turns to its map of the entries more than once, and that lines share a maximum."""
    gen = torch.Generator().manual_seed(22)
    z = (torch.randn(8, C, generator=gen) * 2).to(dt).to(DEV)
    ids = torch.stack([torch.randperm(C, generator=gen)[:30] for _ in range(8)])
    ids[:, 0], ids[:, 1] = C - 1, 0
    top = torch.randn(8, 30, generator=gen).log_softmax(-1) - 0.3
    ids, top, y = ids.to(DEV), top.to(DEV), torch.randint(0, C, (8,), generator=gen).to(DEV)
    many = lambda t: t.repeat(65, *[1] * (t.dim() - 1))  # noqa: E731
    few, all_ = (D.class_logprobs(a, b, topk=12, temperature=0.9, ignore_index=-1) for a, b in ((z, y), (many(z), many(y))))
    assert torch.equal(many(few.top_ids), all_.top_ids)
    for a, b in zip(few, all_):
        assert torch.allclose(many(a), b, rtol=1e-5, atol=1e-5)
    for tail in (True, False):
        a = D.distill_loss(z, ids, top, tail=tail, reduction="none")
        b = D.distill_loss(many(z), many(ids), many(top), tail=tail, reduction="none")
        assert torch.allclose(many(a), b, rtol=1e-5, atol=1e-5) and bool((a > 0).all())


def test_second_differentiation_is_refused():
    z = torch.randn(4, 9, device=DEV).requires_grad_()
    o = D.class_logprobs(z, torch.zeros(4, dtype=torch.int64, device=DEV))
    g, = torch.autograd.grad(o.logprob.sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    with pytest.raises(RuntimeError):
        o2 = D.class_logprobs(z, None, topk=3)
        o2.top_logprobs.sum().backward()


def test_offsets_past_32_bits():
    """Rows and planes that start beyond 2^32 elements of their storage's start (bf16: 8.6 GB)."""
    far = (1 << 32) + 8
    store = torch.zeros(far + 4096, dtype=torch.bfloat16, device=DEV)
    gen = torch.Generator().manual_seed(17)
    small = torch.randn(2, 19, generator=gen).to(torch.bfloat16).to(DEV)
    z = torch.as_strided(store, (2, 19), (far, 1))
    z.copy_(small)
    ids, top = teacher(None, small, -1, 3, 1.0, False, gen)
    a, b = D.class_logprobs(z, None, topk=3), D.class_logprobs(small, None, topk=3)
    assert all(torch.equal(x, y) for x, y in zip(a[1:], b[1:]))
    la, lb = D.distill_loss(z, ids, top), D.distill_loss(small, ids, top)
    assert torch.equal(la, lb)
    store.zero_()
    planes = torch.as_strided(store, (1, 2, 1, 40), (1, far, 40, 1))      # the second class is far away
    sp = torch.randn(1, 2, 1, 40, generator=gen).to(torch.bfloat16).to(DEV)
    planes.copy_(sp)
    a, b = D.class_logprobs(planes, None, topk=2), D.class_logprobs(sp, None, topk=2)
    assert all(torch.equal(x, y) for x, y in zip(a[1:], b[1:]))


def test_a_teacher_and_its_student():
    """The operators as they are used together: the teacher's answers feed the student's loss; a few steps of descent run, and the
    gradient of every step agrees with the definition."""
    gen = torch.Generator().manual_seed(18)
    t = (torch.randn(2, 21, 13, 13, generator=gen) * 3).to(DEV)
    top = D.class_logprobs(t, topk=6, temperature=2.0)
    z = torch.randn(2, 21, 13, 13, generator=gen).to(DEV).requires_grad_()
    for _ in range(3):
        z.grad = None
        loss = D.distill_loss(z, top.top_ids, top.top_logprobs, temperature=2.0, tail=True)
        loss.backward()
        (lv, lb), (gv, gb) = ref.distill(last(z, 1), last(top.top_ids, 1), last(top.top_logprobs, 1), 2.0, True, None, "mean", HALF[torch.float32])
        close(loss, lv, lb, "loss")
        close(last(z.grad, 1), gv, gb, "grad")
        with torch.no_grad():
            z -= 50 * z.grad


# ---------------------------------------------------------------------------------------------
# the training path
# ---------------------------------------------------------------------------------------------
def _net(seed, classes=21, dropout=0.0):
    from model.pspnet import PSPNet
    from oracle import segnet
    torch.manual_seed(5)
    m = PSPNet(layers=50, classes=classes, zoom_factor=8, dropout=dropout, pretrained=False)
    m.load_state_dict(segnet.recipe_state_dict({k: tuple(v.shape) for k, v in m.state_dict().items()}, seed=seed))
    return m.cuda()


def test_top_logits_are_the_score_map_s():
    m = _net(1234).eval()
    x = torch.randn(2, 3, 73, 73, generator=torch.Generator().manual_seed(1)).cuda()
    o = m.top_logits(x, 4, temperature=2.0)
    assert o.top_ids.shape == o.top_logprobs.shape == (2, 4, 10, 10) and o.logprob is None
    logits = m(x)                                        # align_corners=True: every 8th pixel (but for the grid's last) is a point of the map
    eng = m._engine(x, False)
    s = eng.scores_eval(x)
    z = s.data[..., :21].movedim(-1, 1)
    assert torch.allclose(logits[:, :, 0, 0], z[:, :, 0, 0], rtol=1e-5, atol=1e-5)
    want = ref.logprobs(last(z, 1), None, 2.0, 4, 255)
    assert torch.equal(last(o.top_ids, 1), want["top_ids"][0])
    close(last(o.top_logprobs, 1), *want["top_logprobs"], "top_logprobs")
    close(o.entropy, *want["entropy"], "entropy")
    kept = o.top_ids.clone()
    m.top_logits(x + 1, 4)
    assert torch.equal(o.top_ids, kept)                  # new tensors, not the engine's buffers


@pytest.mark.parametrize("tail", [False, True])
def test_trainer_distils_the_score_map(tail):
    """The loss is the definition's on the step's own scores, and the scores' gradient is the cross entropy's plus distill_weight times the
    definition's."""
    from semseg_amd.trainer import Trainer
    T, alpha = 2.0, 0.3
    t, m = _net(77).eval(), _net(1234).train()
    tr = Trainer(m, sync_bn=False, distill_weight=alpha, distill_temperature=T, distill_tail=tail)
    tr.use_plan = False
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(2, 3, 73, 73, generator=gen).cuda()
    y = torch.randint(0, 21, (2, 73, 73), generator=gen).cuda()
    o = t.top_logits(x, 5, temperature=T if tail else 1.0)
    w = (torch.rand(2, 10, 10, generator=gen) > 0.2).float().cuda()
    assert len(tr.step(x, y, 0.0)) == 3                  # learning rate 0: the weights stay
    e = tr.engine(x)
    plain = e.grad_of(e._rec_main["scores"])[..., :21].double().cpu().clone()
    before = e._rec_main["scores"].data[..., :21].double().cpu().clone()
    pred, main, aux, kd = tr.step(x, y, 0.0, top=(o.top_ids, o.top_logprobs, w))
    s = e._rec_main["scores"]
    z = s.data[..., :21].double().cpu()
    (lv, lb), (gv, gb) = ref.distill(z, last(o.top_ids, 1), last(o.top_logprobs, 1), T, tail, w.double().cpu(), "mean", HALF[torch.float32],
                                     torch.tensor(alpha, dtype=torch.float64))
    close(kd[0], lv, lb, "loss")
    both = e.grad_of(s)[..., :21].double().cpu()
    # the two steps' scores agree up to the merging order of the normalisations' statistics; so do the cross entropy's gradients
    drift = float((z - before).abs().max())
    assert drift < 1e-4
    tol = gb + both.abs() * 2.0 ** -23 + plain.abs() * 2.0 ** -23 + 4 * drift * float(plain.abs().max()) + 1e-12
    off = (both - plain - gv).abs()
    assert bool((off <= tol).all()), float((off - tol).max())
    assert float(e.grad_of(s)[..., 21:].abs().max()) == 0
    for bad in ((o.top_ids[:1], o.top_logprobs[:1]), (o.top_ids, o.top_logprobs[:, :2]), (o.top_ids.float(), o.top_logprobs),
                (o.top_ids, o.top_logprobs, w[:1])):
        with pytest.raises((ValueError, TypeError)):
            tr.step(x, y, 0.0, top=bad)
    assert len(tr.step(x, y, 0.0)) == 3


def test_replayed_distillation_steps_equal_eager_ones(report):
    """Eight steps with a new batch, teacher's answer and learning rate each: replayed from the recorded step as launch by launch, inside 4x
    the noise between two eager runs; a step without a teacher in between is not replayed from the record with one."""
    from semseg_amd.trainer import Trainer

    def run(plan):
        t, m = _net(77).eval(), _net(1234, dropout=0.1).train()
        tr = Trainer(m, sync_bn=False, distill_weight=0.5, distill_temperature=2.0)
        tr.use_plan = plan
        gen = torch.Generator().manual_seed(3)
        losses = []
        for it in range(8):
            x = torch.randn(2, 3, 73, 73, generator=gen).cuda()
            y = torch.randint(0, 21, (2, 73, 73), generator=gen).cuda()
            o = t.top_logits(x, 4)
            _, ml, al, kd = tr.step(x, y, 0.01 / (it + 1), top=(o.top_ids, o.top_logprobs))
            losses.append((float(ml), float(al), float(kd)))
        e = tr.engine(x)
        return torch.tensor(losses), tr.flat_w.detach().cpu().clone(), tr, e, (x, y, o)
    la, wa, _, _, _ = run(False)
    lb, wb, _, _, _ = run(False)
    lp, wp, tr, e, (x, y, o) = run(True)
    assert e._plan is not None and e._plan_replays == 4, tr.plan_log
    noise_l, noise_w = float((la - lb).abs().max()), float((wa - wb).abs().max())
    off_l, off_w = float((lp - la).abs().max()), float((wp - wa).abs().max())
    report("distillation steps replayed: losses off %.1e (eager twice %.1e), weights %.1e (%.1e)" % (off_l, noise_l, off_w, noise_w))
    assert off_l <= 4 * noise_l + 1e-6 * float(la.abs().max()) and off_w <= 4 * noise_w + 1e-6 * float(wa.abs().max())
    assert len(tr.step(x, y, 0.01)) == 3 and e._plan is None            # recorded again without the teacher
    for _ in range(3):
        out = tr.step(x, y, 0.01)
    assert e._plan is not None and len(out) == 3
    assert len(tr.step(x, y, 0.01, top=(o.top_ids, o.top_logprobs))) == 4 and e._plan is None


def test_a_record_with_a_teacher_ends_with_its_buffers():
    """A step without a teacher that is not replayed itself ends the record of the steps with one: the next of those reads its own entries."""
    from semseg_amd.trainer import Trainer
    t, m = _net(77).eval(), _net(1234, dropout=0.0).train()
    tr = Trainer(m, sync_bn=False, distill_temperature=2.0)
    gen = torch.Generator().manual_seed(4)
    x, y = torch.randn(2, 3, 73, 73, generator=gen).cuda(), torch.randint(0, 21, (2, 73, 73), generator=gen).cuda()
    o = t.top_logits(x, 4)
    for _ in range(7):
        tr.step(x, y, 0.0, top=(o.top_ids, o.top_logprobs))
    e = tr.engine(x)
    assert e._plan is not None, tr.plan_log
    tr.use_plan = False
    tr.step(x, y, 0.0)
    assert e._plan is None
    tr.use_plan = True
    for it in range(6):                  # launch by launch, recorded, replayed: the teacher's answer changes every time
        top = (o.top_ids.roll(it, 0), o.top_logprobs.roll(it, 0) - 0.1 * it)
        kd = tr.step(x, y, 0.0, top=top)[3]
        s = e._rec_main["scores"]
        want = D.distill_loss(s.data[..., :s.C].movedim(-1, 1), *top, temperature=2.0)
        assert abs(float(kd) - float(want)) <= 1e-5 * abs(float(want)), (it, float(kd), float(want))
    assert e._plan is not None, tr.plan_log
