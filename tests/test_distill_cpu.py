"""semseg_amd.distill without a GPU: how logits are walked, what is refused, the definitions behind the GPU tests against differences."""
import math

import pytest
import torch

import class_probs_ref as ref
from semseg_amd import distill as D


@pytest.mark.parametrize("make,dim,geom,strides,by_rows", [
    (lambda: torch.zeros(2, 5, 4, 3), 1, (2, 12, 5), (60, 1, 12), False),
    (lambda: torch.zeros(2, 5, 4, 3).contiguous(memory_format=torch.channels_last), 1, (1, 24, 5), (0, 5, 1), True),
    (lambda: torch.zeros(2, 4, 3, 8)[..., :5], -1, (1, 24, 5), (0, 8, 1), True),
    (lambda: torch.zeros(2, 4, 3, 8)[:, 1:, :, :5], -1, (2, 9, 5), (96, 8, 1), True),
    (lambda: torch.zeros(7, 5), 1, (1, 7, 5), (0, 5, 1), True),
    (lambda: torch.zeros(5, 7).t(), 1, (1, 7, 5), (0, 1, 7), False),
    (lambda: torch.zeros(1, 5).expand(7, 5), 1, (1, 7, 5), (0, 0, 1), True),
    (lambda: torch.zeros(2, 5, 6, 7)[:, :, 1:], 1, (2, 35, 5), (210, 1, 42), False),
    (lambda: torch.zeros(3, 5, 1, 1), 1, (1, 3, 5), (0, 5, 1), True),
    (lambda: torch.zeros(3, 1, 4, 4), 1, (1, 48, 1), (0, 1, 1), True),
])
def test_rows_of_a_tensor(make, dim, geom, strides, by_rows):
    z = make()
    g = D.Geom(z, D._dim(z, dim))
    assert (g.geom, g.strides, g.by_rows) == (geom, strides, by_rows)
    # every element is reached exactly where the strides say
    src = torch.arange(z.untyped_storage().nbytes() // 4)
    zi = torch.as_strided(src, z.shape, z.stride(), z.storage_offset()).movedim(g.dim, -1).reshape(-1, g.C)
    i, j, c = torch.meshgrid(torch.arange(g.n), torch.arange(g.p), torch.arange(g.C), indexing="ij")
    want = z.storage_offset() + i * g.strides[0] + j * g.strides[1] + c * g.strides[2]
    assert torch.equal(src[want.reshape(-1, g.C)], zi)
    # a new tensor beside it has the same rows
    e = g.empty(3, torch.float32, "cpu")
    assert e.shape == z.shape[:g.dim] + (3,) + z.shape[g.dim + 1:]
    s = g.strides_of(e)
    ei = torch.as_strided(torch.arange(e.numel()), e.shape, e.stride()).movedim(g.dim, -1).reshape(-1, 3)
    i, j, c = torch.meshgrid(torch.arange(g.n), torch.arange(g.p), torch.arange(3), indexing="ij")
    assert torch.equal((i * s[0] + j * s[1] + c * s[2]).reshape(-1, 3), ei)


LAYOUTS = {
    "planes": lambda: (torch.zeros(2, 5, 3, 4), 1),
    "channels_last": lambda: (torch.zeros(2, 3, 4, 5).movedim(-1, 1), 1),
    "planes, classes named last": lambda: (torch.zeros(2, 5, 3, 4).movedim(1, -1), -1),
    "a plane per class over the batch": lambda: (torch.zeros(5, 2, 3, 4).transpose(0, 1), 1),
    "the same, classes named last": lambda: (torch.zeros(5, 2, 3, 4).movedim(0, -1), -1),
    "transposed rows": lambda: (torch.zeros(5, 7).t(), 1),
    "transposed rows of a batch": lambda: (torch.zeros(2, 5, 7).transpose(1, 2), -1),
    "images of a larger channels_last batch": lambda: (torch.zeros(4, 3, 4, 5)[::2].movedim(-1, 1), 1),
    "one class": lambda: (torch.zeros(2, 1, 3, 4), 1),
    "three dimensions of pixels": lambda: (torch.zeros(2, 5, 2, 3, 4), 1),
    "one pixel": lambda: (torch.zeros(2, 5, 1, 1), 1),
}


@pytest.mark.parametrize("layout", LAYOUTS)
def test_new_tensors_lie_as_the_kernels_are_told(layout):
    """Outputs, gradients (empty with the strides of dense) and a teacher's entries in any order of memory: row r, entry j of the tensor
    is where the strides handed to the kernels say."""
    z, dim = LAYOUTS[layout]()
    dim = D._dim(z, dim)
    g = D.Geom(z, dim)
    rows, j = torch.arange(g.n * g.p)[:, None], torch.arange(3)

    def where(s):
        return rows // g.p * s[0] + rows % g.p * s[1] + j * s[2]
    e = g.empty(3, torch.float32, "cpu")
    assert e.shape == z.shape[:dim] + (3,) + z.shape[dim + 1:]
    flat = torch.arange(e.numel())
    assert torch.equal(where(g.dense(3)), flat.as_strided(e.shape, e.stride()).movedim(dim, -1).reshape(-1, 3))
    d = g.dense(3)
    assert d[2] == 1 if g.by_rows else d[1] == 1          # a gradient in the form of its logits
    ids = torch.arange(e.numel()).view(e.shape)                # contiguous, and in two other orders
    for t in (ids, ids.movedim(dim, -1).contiguous().movedim(-1, dim), ids.movedim(0, -1).contiguous().movedim(-1, 0)):
        got, s, top, s2, k, _ = D.check_top(g, z.device, t, t.float(), None)
        assert k == 3 and torch.equal(got, ids)
        for u, us in ((got, s), (top.long(), s2)):
            mem = torch.empty(u.numel(), dtype=torch.long)
            mem.as_strided(u.shape, got.stride()).copy_(u)
            assert us == s and torch.equal(mem[where(us)], ids.movedim(dim, -1).reshape(-1, 3))



def test_refusals():
    z = torch.zeros(2, 5, 4, 3)
    y = torch.zeros(2, 4, 3, dtype=torch.int64)
    ids, top = torch.zeros(2, 2, 4, 3, dtype=torch.int32), torch.zeros(2, 2, 4, 3)
    for bad, err in [
        (lambda: D.class_logprobs(z.double(), y), TypeError),
        (lambda: D.class_logprobs(z.long(), y), TypeError),
        (lambda: D.class_logprobs(z[0, 0, 0], None), ValueError),
        (lambda: D.class_logprobs(z[:0], None), ValueError),
        (lambda: D.class_logprobs(z, y.int()), TypeError),
        (lambda: D.class_logprobs(z, y[:1]), ValueError),
        (lambda: D.class_logprobs(z, y, class_dim=2), ValueError),
        (lambda: D.class_logprobs(z, y, topk=6), ValueError),
        (lambda: D.class_logprobs(z, y, topk=-1), ValueError),
        (lambda: D.class_logprobs(z, y, topk=1.0), ValueError),
        (lambda: D.class_logprobs(torch.zeros(2, 100), None, topk=65), ValueError),
        (lambda: D.class_logprobs(z, y, temperature=0.0), ValueError),
        (lambda: D.class_logprobs(z, y, temperature=math.inf), ValueError),
        (lambda: D.class_logprobs(z, y, temperature=1e-16), ValueError),
        (lambda: D.distill_loss(z, ids, top.detach(), temperature=1e16), ValueError),
        (lambda: D.class_logprobs(z, y, temperature=math.nan), ValueError),
        (lambda: D.class_logprobs(z[..., ::2], None), ValueError),
        (lambda: D.class_logprobs(torch.zeros(4, 10)[:, ::2], None), ValueError),
        (lambda: D.distill_loss(z, ids.float(), top), TypeError),
        (lambda: D.distill_loss(z, ids, top.double()), TypeError),
        (lambda: D.distill_loss(z, ids[:, :1], top), ValueError),
        (lambda: D.distill_loss(z, ids[0], top[0]), ValueError),
        (lambda: D.distill_loss(z, ids[:, :0], top[:, :0]), ValueError),
        (lambda: D.distill_loss(z, ids.expand(2, 2, 4, 3).repeat(1, 33, 1, 1), top.repeat(1, 33, 1, 1)), ValueError),
        (lambda: D.distill_loss(z, ids, top.requires_grad_()), ValueError),
        (lambda: D.distill_loss(z, ids, top.detach(), weight=torch.zeros(2, 4, 3).double()), TypeError),
        (lambda: D.distill_loss(z, ids, top.detach(), weight=torch.zeros(2, 4)), ValueError),
        (lambda: D.distill_loss(z, ids, top.detach(), reduction="batchmean"), ValueError),
        (lambda: D.distill_loss_grad(z, ids, top.detach(), reduction="none"), ValueError),
        # and nothing runs on the CPU
        (lambda: D.class_logprobs(z, y), RuntimeError),
        (lambda: D.distill_loss(z, ids, top.detach()), RuntimeError),
        (lambda: D.distill_loss_grad(z, ids, top.detach()), RuntimeError),
    ]:
        with pytest.raises(err):
            bad()


def test_the_c_entries_refuse_bad_arguments_without_a_gpu():
    from semseg_amd._lib import lib
    p = 4096      # never read: every call below is refused on the host
    none3, s3 = (0, 0, 0), (0, 8, 1)
    fwd = lambda z=p, t=0, n=1, pp=4, C=8, T=1.0, k=0, lp=None, ids=None, lab=None: lib.semseg_class_logprobs_fwd(  # noqa: E731
        z, t, n, pp, C, *s3, lab, 255, T, k, lp, None, None, None, ids, ids, *none3, None, 0, None)
    for kw in (dict(z=None), dict(t=3), dict(t=-1), dict(n=0), dict(pp=0), dict(C=0), dict(T=0.0), dict(T=-1.0), dict(T=math.nan),
               dict(T=math.inf), dict(T=1e-16), dict(T=1e16), dict(k=-1), dict(k=1), dict(k=9, ids=p), dict(C=100, k=65, ids=p), dict(lp=p), dict(n=1 << 30, pp=1 << 30)):
        assert fwd(**kw) == -1, kw
    assert fwd(C=100000) == -1                  # one row in several slices needs scratch
    assert lib.semseg_class_logprobs_scratch_bytes(0, 1, 4, 8, 1, 5) == 0 < lib.semseg_class_logprobs_scratch_bytes(0, 1, 1, 100000, 1, 5)
    assert lib.semseg_class_logprobs_bwd(p, 0, 1, 4, 8, *s3, None, 255, 1.0, None, None, None, None, None, p, *s3, 0, None) == -1
    assert lib.semseg_class_logprobs_bwd(p, 0, 1, 4, 8, *s3, None, 255, 1.0, p, None, p, None, None, p, *s3, 0, None) == -1
    assert lib.semseg_class_logprobs_bwd(p, 0, 1, 4, 8, *s3, None, 255, 1.0, p, None, None, p, None, p, *s3, 0, None) == -1
    need = lib.semseg_distill_scratch_bytes(0, 1, 4, 8, 1)
    assert need > 0 and lib.semseg_distill_scratch_bytes(0, 0, 4, 8, 1) == 0
    assert lib.semseg_distill_scratch_bytes(1, 1, 4, 100000, 1) > need
    head = (p, 0, 1, 4, 8, *s3)
    dist = lambda ids=p, i64=0, top=p, tt=0, k=2, T=1.0, red=1, rows=None, stats=p, acc=p, loss=p, scr=p, nb=need: lib.semseg_distill_fwd(  # noqa: E731
        *head, ids, i64, top, tt, k, 0, 2, 1, 0, 2, 1, None, T, 0, red, rows, stats, acc, loss, scr, nb, None)
    for kw in (dict(ids=None), dict(i64=2), dict(top=None), dict(tt=3), dict(k=0), dict(k=65), dict(T=0.0), dict(red=3), dict(red=-1),
               dict(red=0), dict(stats=None), dict(acc=None), dict(loss=None), dict(scr=None), dict(nb=need - 1)):
        assert dist(**kw) == -1, kw
    assert lib.semseg_distill_bwd(*head, p, 0, p, 0, 2, 0, 2, 1, 0, 2, 1, None, 1.0, 0, 1, p, None, None, 1.0, p, *s3, 0, None) == -1
    assert lib.semseg_distill_bwd(*head, p, 0, p, 0, 2, 0, 2, 1, 0, 2, 1, None, 1.0, 0, 1, p, p, None, 1.0, None, *s3, 0, None) == -1
    assert lib.semseg_distill_fwd_bwd(*head, p, 0, p, 0, 2, 0, 2, 1, 0, 2, 1, None, 1.0, 0, 0, p, p, p, 1.0, p, *s3, 0, p, need, None) == -1


def _differences(f, z, h=1e-6):
    g = torch.zeros_like(z)
    for i in range(z.numel()):
        for s in (1, -1):
            zz = z.clone()
            zz.view(-1)[i] += s * h
            g.view(-1)[i] += s * f(zz) / (2 * h)
    return g


@pytest.mark.parametrize("T", [1.0, 2.5])
def test_logprob_gradient_formula_against_differences(T):
    gen = torch.Generator().manual_seed(3)
    z = torch.randn(4, 6, generator=gen, dtype=torch.float64) * 2
    z[1, 2] = -math.inf
    y = torch.tensor([0, 3, 255, 5])
    g1, g2, g3 = (torch.randn(4, generator=gen, dtype=torch.float64) for _ in range(3))

    def f(zz):
        o = ref.logprobs(zz, y, T, 0, 255)
        keep = y != 255
        return float((g1 * o["logprob"][0] + g2 * o["entropy"][0] + g3 * o["lse"][0])[keep].sum())
    want = _differences(f, z)
    got, _ = ref.logprobs_grad(z, y, T, 255, g1, g2, g3, 0.0)
    fin = torch.isfinite(z)
    assert float((got - want)[fin].abs().max()) < 1e-7 and bool((got[~fin] == 0).all())


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_distill_gradient_formula_against_differences(tail, reduction):
    gen = torch.Generator().manual_seed(4)
    z = torch.randn(5, 7, generator=gen, dtype=torch.float64) * 2
    t = torch.randn(5, 7, generator=gen, dtype=torch.float64) * 2
    T = 2.0
    top, ids = (t / T).log_softmax(-1).topk(3, -1) if tail else t.topk(3, -1)
    ids = ids.clone()
    ids[1, 2] = -1
    ids[2, 1] = ids[2, 0]          # the same class twice
    ids[3] = -1
    w = torch.tensor([1.0, 0.5, 2.0, 1.0, 0.0], dtype=torch.float64)
    f = lambda zz: float(ref.distill(zz, ids, top, T, tail, w, reduction, 0.0)[0][0])  # noqa: E731
    got = ref.distill(z, ids, top, T, tail, w, reduction, 0.0)[1][0]
    want = _differences(f, z)
    assert float((got - want).abs().max()) < 1e-6


def test_a_teacher_answers_in_eval_mode_on_the_gpu_only():
    from model.pspnet import PSPNet
    m = PSPNet(layers=50, classes=5, pretrained=False)
    with pytest.raises(RuntimeError, match="eval"):
        m.train().top_logits(torch.zeros(1, 3, 9, 9), 2)
    with pytest.raises(RuntimeError, match="MI355X"):
        m.eval().top_logits(torch.zeros(1, 3, 9, 9), 2)
