"""Measured cases of the class-probability operators: log probabilities of given classes with entropy and top alternatives, and
distillation from a teacher's top logits, each with its gradient.

A case names its operator (`op`), the type and layout of the logits and their sizes:
  layout "rows"   [rows, C], classes contiguous, `ld` >= C values from one row to the next (the engine's score buffers, [tokens, classes])
  layout "planes" [N, C, H, W], one contiguous plane per class (what a model returns in eval mode)
With `own` false, `run` computes the operators in their plain form; with `own` true through semseg_amd.distill."""
import math

import torch

own = False

IGNORE = 255
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
MAX_VALUES = 40_000_000      # values of a drawn case's logits


def listed():
    return [
        # what a teacher hands to its student: the eight best classes of every point of a batch's 60 x 60 score map (473 x 473 images,
        # 150 classes, rows padded to 256 values as the engine keeps them)
        dict(name="top8 of a score map", op="logprobs", layout="rows", dtype="fp32", rows=57600, C=150, ld=256, k=8, T=1.0, labels=False),
        # maps of uncertainty, label probability and three alternatives of full-resolution logits, a batch of eight images
        dict(name="maps of 473x473 logits", op="logprobs", layout="planes", dtype="fp32", N=8, C=150, H=473, W=473, k=3, T=1.0, labels=True),
        # the same of two large street scenes with few classes, 16-bit logits
        dict(name="maps of 713x713 logits", op="logprobs", layout="planes", dtype="bf16", N=2, C=19, H=713, W=713, k=3, T=1.0, labels=True),
        # one row of a large vocabulary, as a server asks for it at every token: latency
        dict(name="one row of 131072", op="logprobs", layout="rows", dtype="bf16", rows=1, C=131072, ld=131072, k=20, T=1.0, labels=True),
        # a batch of rows of an odd vocabulary, scored at a temperature
        dict(name="4096 rows of 50001", op="logprobs", layout="rows", dtype="bf16", rows=4096, C=50001, ld=50001, k=16, T=0.7, labels=True),
        # training on label probability and entropy together (entropy minimisation on unlabelled images): forward and backward
        dict(name="entropy step, 21 classes", op="logprobs_grad", layout="planes", dtype="fp32", N=4, C=21, H=473, W=473, T=1.0),
        # the same on rows of a large vocabulary
        dict(name="entropy step, 32000 classes", op="logprobs_grad", layout="rows", dtype="bf16", rows=4096, C=32000, ld=32000, T=1.0),
        # the distillation part of a training step on the score map: loss and gradient at once
        dict(name="distil a score map", op="distill_grad", layout="rows", dtype="fp32", rows=57600, C=150, ld=256, k=8, T=4.0, tail=False, weights=False),
        # distillation at full resolution, border and void pixels masked
        dict(name="distil 473x473 logits", op="distill", layout="planes", dtype="fp32", N=4, C=150, H=473, W=473, k=4, T=2.0, tail=False, weights=True),
        # a small validation crop, 16-bit
        dict(name="distil 65x65 logits", op="distill", layout="planes", dtype="fp16", N=2, C=19, H=65, W=65, k=3, T=1.0, tail=True, weights=True),
        # a long vocabulary, 32 stored logits to a row and the rest of the teacher's mass as one class
        dict(name="distil 2048 rows of 131072", op="distill", layout="rows", dtype="bf16", rows=2048, C=131072, ld=131072, k=32, T=1.0, tail=True, weights=True),
        # a short tail of a batch: few rows, odd sizes
        dict(name="distil 7 rows of 50001", op="distill", layout="rows", dtype="fp32", rows=7, C=50001, ld=50001, k=16, T=2.0, tail=False, weights=False),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("logprobs", "logprobs", "logprobs_grad", "distill", "distill", "distill_grad"))
    case = dict(op=op, layout=rng.choice(("rows", "planes")), dtype=rng.choice(("fp32", "bf16", "fp16")))
    if case["layout"] == "rows":
        C = _spread(rng, 2, 131072)
        case.update(C=C, rows=_spread(rng, 1, max(1, min(100_000, MAX_VALUES // C))), ld=C + rng.choice((0, 0, 1, 6, 64)))
    else:
        C, N = _spread(rng, 2, 1024), rng.randint(1, 4)
        side = max(3, min(713, int(math.sqrt(MAX_VALUES / (C * N)))))
        case.update(C=C, N=N, H=_spread(rng, 1, side), W=_spread(rng, 1, side))
    case["T"] = rng.choice((0.5, 1.0, 1.0, 2.0, 4.0))
    most = min(32, case["C"])
    if op == "logprobs":
        case.update(k=rng.choice((0, 1, _spread(rng, 1, most), _spread(rng, 1, most))), labels=rng.random() < 0.7)
        case["k"] = min(case["k"], case["C"])
    elif op != "logprobs_grad":
        case.update(k=_spread(rng, 1, most), tail=rng.random() < 0.4, weights=rng.random() < 0.5)
    return case


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _logits(case, gen, also=None):
    """Logits as a network gives them: noise of a few units and one favoured class to a row (that of `also` where it is given)."""
    C, dt = case["C"], TYPES[case["dtype"]]
    if case["layout"] == "rows":
        store = torch.randn(case["rows"], case["ld"], device="cuda", generator=gen).mul_(2.0)
        z = store[:, :C]
    else:
        store = z = torch.randn(case["N"], C, case["H"], case["W"], device="cuda", generator=gen).mul_(2.0)
    hit = torch.randint(0, C, (z.shape[0], 1) + tuple(z.shape[2:]), device="cuda", generator=gen) if also is None else also
    z.scatter_add_(1, hit, torch.rand(hit.shape, device="cuda", generator=gen).mul_(8.0))
    return store.to(dt)[:, :C], hit


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    z, hit = _logits(case, gen)
    state = dict(op=case["op"], logits=z, T=case["T"], class_dim=1)
    rows = (z.shape[0],) + tuple(z.shape[2:])
    if case["op"] in ("logprobs", "logprobs_grad"):
        label = None
        if case.get("labels", True):
            label = torch.randint(0, case["C"], rows, device="cuda", generator=gen)
            label = torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.6, hit[:, 0], label)
            if case["C"] <= IGNORE:       # about a tenth of a labelled image is void
                label = torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.1, torch.full_like(label, IGNORE), label)
            else:                         # with more classes than that the void label is a negative one
                label = torch.where(torch.rand(rows, device="cuda", generator=gen) < 0.1, torch.full_like(label, -1), label)
        if label is not None:             # never nothing but void
            label.view(-1)[0] = hit.view(-1)[0]
        state.update(label=label, ignore=IGNORE if case["C"] <= IGNORE else -1, k=case.get("k", 0))
        if case["op"] == "logprobs_grad":
            state.update(g_logprob=torch.randn(rows, device="cuda", generator=gen), g_entropy=torch.randn(rows, device="cuda", generator=gen))
        return state
    # the teacher: the same scene seen by another network, its best k classes
    teacher, _ = _logits(case, gen, hit)
    top, ids = torch.topk(teacher.float() if case["layout"] == "planes" else teacher.float().contiguous(), case["k"], dim=1)
    if case["tail"]:      # log-probabilities at the temperature: what is left of the mass is the tail's
        top = top / case["T"] - torch.logsumexp(teacher.float() / case["T"], 1, keepdim=True)
    del teacher
    state.update(ids=ids.int().contiguous(), top=top.contiguous(), tail=case["tail"], weight=None)
    if case["weights"]:
        state["weight"] = (torch.rand(rows, device="cuda", generator=gen) >= 0.1).float()
        state["weight"].view(-1)[0] = 1.0     # never nothing but masked rows
    return state


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "logprobs":
        return _plain_logprobs(state)
    if state["op"] == "logprobs_grad":
        return _plain_logprobs_grad(state)
    return _plain_distill(state)


def _run_own(s):
    from semseg_amd import distill as D
    if s["op"] == "logprobs":
        o = D.class_logprobs(s["logits"], s["label"], topk=s["k"], temperature=s["T"], ignore_index=s["ignore"], class_dim=s["class_dim"])
        return {k: v for k, v in o._asdict().items() if v is not None}
    if s["op"] == "logprobs_grad":
        z = s["logits"].detach().requires_grad_()
        o = D.class_logprobs(z, s["label"], temperature=s["T"], ignore_index=s["ignore"], class_dim=s["class_dim"])
        grad, = torch.autograd.grad((o.logprob, o.entropy), z, (s["g_logprob"], s["g_entropy"]))
        return dict(logprob=o.logprob.detach(), entropy=o.entropy.detach(), grad=grad)
    if s["op"] == "distill_grad":
        loss, grad = D.distill_loss_grad(s["logits"], s["ids"], s["top"], temperature=s["T"], tail=s["tail"], weight=s["weight"],
                                         class_dim=s["class_dim"])
        return dict(loss=loss, grad=grad)
    z = s["logits"].detach().requires_grad_()
    loss = D.distill_loss(z, s["ids"], s["top"], temperature=s["T"], tail=s["tail"], weight=s["weight"], class_dim=s["class_dim"])
    grad, = torch.autograd.grad(loss, z)
    return dict(loss=loss.detach(), grad=grad)


def _shifted(s):
    """(z - max) / T, the largest logit, log sum exp of the former, of 32-bit logits with the classes in dimension 1."""
    x = s["logits"].float()
    top = x.amax(1, keepdim=True)
    d = (x - top) / s["T"]
    return x, d, top, d.exp().sum(1, keepdim=True).log()


def _at_label(s, d, logsum):
    """Log probability of the labels, which rows have one, and the labels with 0 in the others' place."""
    keep = s["label"] != s["ignore"]
    y = torch.where(keep, s["label"], torch.zeros_like(s["label"])).unsqueeze(1)
    return (d.gather(1, y) - logsum).squeeze(1), keep, y


def _plain_logprobs(s):
    x, d, top, logsum = _shifted(s)
    out = dict(entropy=(logsum - (d.exp() * d).sum(1, keepdim=True) / logsum.exp()).squeeze(1), lse=(top / s["T"] + logsum).squeeze(1))
    keep = None
    if s["label"] is not None:
        lp, keep, _ = _at_label(s, d, logsum)
        out["logprob"] = torch.where(keep, lp, torch.zeros_like(lp))
        out["entropy"] = torch.where(keep, out["entropy"], torch.zeros_like(lp))
        out["lse"] = torch.where(keep, out["lse"], torch.zeros_like(lp))
    if s["k"]:
        ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :s["k"]]      # equal values: the lowest class first
        values = d.gather(1, ids) - logsum
        if keep is not None:
            ids = torch.where(keep.unsqueeze(1), ids, torch.full_like(ids, -1))
            values = torch.where(keep.unsqueeze(1), values, torch.full_like(values, -math.inf))
        out.update(top_ids=ids.int(), top_logprobs=values)
    return {n: out[n] for n in ("logprob", "entropy", "lse", "top_ids", "top_logprobs") if n in out}


def _plain_logprobs_grad(s):
    x, d, _, logsum = _shifted(s)
    lp, keep, y = _at_label(s, d, logsum)
    logp = d - logsum
    p = logp.exp()
    h = -(p * logp).sum(1)
    g1, g2 = (torch.where(keep, s[g], torch.zeros_like(lp)).unsqueeze(1) for g in ("g_logprob", "g_entropy"))
    grad = (-g1 * p - g2 * p * (logp + h.unsqueeze(1))).scatter_add_(1, y, g1) / s["T"]
    zero = torch.zeros_like(lp)
    return dict(logprob=torch.where(keep, lp, zero), entropy=torch.where(keep, h, zero), grad=grad.to(s["logits"].dtype))


def _plain_distill(s):
    """T^2 * mean over rows of KL(teacher || student), the teacher's distribution renormalised over its k classes, or (tail) with
    everything else as one more class on both sides."""
    T, ids = s["T"], s["ids"].long()
    x, d, _, logsum = _shifted(s)
    logp = d - logsum
    p = logp.exp()
    top = s["top"].float()
    if s["tail"]:
        logq = top
        q = logq.exp()
    else:
        t = top / T
        t = t - t.amax(1, keepdim=True)
        logq = t - t.exp().sum(1, keepdim=True).log()
        q = logq.exp()
    rows = (q * (logq - logp.gather(1, ids))).sum(1)
    dz = (p * q.sum(1, keepdim=True)).scatter_add_(1, ids, -q)
    if s["tail"]:
        qt = (1.0 - q.sum(1, keepdim=True)).clamp_min(0.0)
        inside = torch.zeros_like(p, dtype=torch.bool).scatter_(1, ids, torch.ones_like(ids, dtype=torch.bool))
        out = d.masked_fill(inside, -math.inf)
        big = out.amax(1, keepdim=True)
        some = big > -math.inf
        big = torch.where(some, big, torch.zeros_like(big))
        lt = (out - big).exp().sum(1, keepdim=True).log() + big       # log sum exp of the classes outside
        qt = torch.where(some, qt, torch.zeros_like(qt))
        lt = torch.where(some, lt, torch.zeros_like(lt))
        rows = rows + torch.where(qt > 0, qt * (qt.clamp_min(1e-45).log() - (lt - logsum)), torch.zeros_like(qt)).squeeze(1)
        dz = dz + qt * p - qt * (out - lt).exp()
    w = torch.ones_like(rows) if s["weight"] is None else s["weight"]
    total = w.double().sum()
    loss = T * T * ((w * rows).double().sum() / total)
    return dict(loss=loss.float(), grad=(dz * (T * w / total.float()).unsqueeze(1)).to(s["logits"].dtype))


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    rows = case["rows"] if case["layout"] == "rows" else case["N"] * case["H"] * case["W"]
    values, size = rows * case["C"], 4 if case["dtype"] == "fp32" else 2
    b = values * size
    if case["op"] == "logprobs":       # read: logits, labels; written: entropy, log-sum-exp, log-probability, k ids and values
        b += rows * (8 + (12 if case["labels"] else 0) + 8 * case["k"])
        return {"bytes": b, "flops": 6 * values}
    if case["op"] == "logprobs_grad":  # read: logits, labels, two gradients; written: two maps, the logits' gradient
        return {"bytes": 2 * b + rows * (8 + 8 + 8), "flops": 12 * values}
    # read: logits, k ids and values, weights; written: the gradient
    return {"bytes": 2 * b + rows * (8 * case["k"] + (4 if case["weights"] else 0)) + 4, "flops": 9 * values}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _log_softmax64(x, T):
    x = x.to(torch.float64) / T
    x -= torch.logsumexp(x, dim=1, keepdim=True)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    n = s["logits"].shape[0]
    step = max(1, min(n, (1 << 26) // max(1, s["logits"][0].numel())))      # rows or images at a time
    if s["op"] == "logprobs":
        return _join([_exact_logprobs(s, slice(i, i + step)) for i in range(0, n, step)])
    if s["op"] == "logprobs_grad":
        return _join([_exact_logprobs_grad(s, slice(i, i + step)) for i in range(0, n, step)])
    weight = s["weight"].double() if s["weight"] is not None else torch.ones(s["ids"][:, 0].shape, dtype=torch.float64, device="cuda")
    parts = [_exact_distill(s, slice(i, i + step), weight) for i in range(0, n, step)]
    return dict(loss=torch.stack([p[0] for p in parts]).sum(), grad=torch.cat([p[1] for p in parts]))


def _join(parts):
    return {k: None if parts[0][k] is None else torch.cat([p[k] for p in parts]) for k in parts[0]}


def _exact_logprobs(s, at):
    L = _log_softmax64(s["logits"][at], s["T"])
    label = None if s["label"] is None else s["label"][at]
    void = torch.zeros(L[:, 0].shape, dtype=torch.bool, device="cuda") if label is None else label == s["ignore"]
    out = {}
    if label is not None:
        out["logprob"] = L.gather(1, label.masked_fill(void, 0)[:, None])[:, 0].masked_fill(void, 0.0)
    out["entropy"] = -torch.special.xlogy(L.exp(), L.exp()).sum(1).masked_fill(void, 0.0)
    out["lse"] = torch.logsumexp(s["logits"][at].double() / s["T"], 1).masked_fill(void, 0.0)
    if s["k"]:
        out["top_ids"] = None
        out["top_logprobs"] = torch.topk(L, s["k"], dim=1)[0].masked_fill(void[:, None], -math.inf)
    return out


def _exact_logprobs_grad(s, at):
    label = s["label"][at]
    void = label == s["ignore"]
    L = _log_softmax64(s["logits"][at], s["T"])
    P = L.exp()
    H = -torch.special.xlogy(P, P).sum(1)
    a, b = s["g_logprob"][at].double().masked_fill(void, 0.0), s["g_entropy"][at].double().masked_fill(void, 0.0)
    y = label.masked_fill(void, 0)[:, None]
    lp = L.gather(1, y)[:, 0].masked_fill(void, 0.0)
    L += H[:, None]
    L *= -b[:, None]
    L -= a[:, None]
    L *= P
    L.scatter_add_(1, y, a[:, None])
    return dict(logprob=lp, entropy=H.masked_fill(void, 0.0), grad=L / s["T"])


def _exact_distill(s, at, weight):
    """The gradient by the chain rule through the classes' log-probabilities: d(sum_c a_c log p_c) = a - p * sum(a)."""
    L = _log_softmax64(s["logits"][at], s["T"])
    ids, top, T = s["ids"][at].long(), s["top"][at].double(), s["T"]
    q = top.exp() if s["tail"] else torch.softmax(top / T, 1)
    kl = (torch.special.xlogy(q, q) - q * L.gather(1, ids)).sum(1)
    a = torch.zeros_like(L).scatter_add_(1, ids, q)
    if s["tail"]:
        rest = (1.0 - q.sum(1, keepdim=True)).clamp_min(0.0)
        outside = L.scatter(1, ids, torch.full_like(q, -math.inf))
        lr = torch.logsumexp(outside, 1, keepdim=True)
        none = lr == -math.inf
        rest, lr = rest.masked_fill(none, 0.0), lr.masked_fill(none, 0.0)
        kl = kl + (torch.special.xlogy(rest, rest) - rest * lr)[:, 0]
        a += rest * (outside - lr).exp()
    w = weight[at]
    scale = T * T / weight.sum()
    grad = (L.exp() * a.sum(1, keepdim=True) - a) * (w * scale / T)[:, None]
    return (w * kl).sum() * scale, grad
