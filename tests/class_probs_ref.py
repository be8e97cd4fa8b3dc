"""Plain forms in 64 bits of the class-probability operators (semseg_amd.distill) and the error their 32-bit kernels may make.

The bounds count roundings, h = 2^-24 (half a step of fp32, relative).  With d = (z - m) / T and L the longest chain of additions:
  d:      the difference, 1/T and the product round once each:             |d| * 3h
  e^d:    the argument's error, log2(e)'s and its product's (2h |d|), and 4h for the exponential itself: (5 |d| + 4) h, relative
  S:      the mean of the terms' relative errors under p, and (L + 2) h:   (5 E|d| + L + 6) h
  log S:  that, and 4h + h |log S| for the logarithm
  log p:  |d| 3h + err(log S) + h |log p|
E|d| <= log(C) + H in any distribution, but it is computed rather than bounded."""
import math

import torch

H24 = 2.0 ** -24
NEG = -math.inf


def rows_last(t, class_dim):
    """[..., classes] in 64 bits."""
    t = t.detach().movedim(class_dim, -1)
    return t.double().cpu() if t.is_floating_point() else t.long().cpu()


class Rows:
    """log softmax of logits [..., C] at temperature T with its error bounds."""

    def __init__(self, z, T, chain):
        self.z, self.T = z, T
        m = z.amax(-1, keepdim=True)
        self.none = (m == NEG).squeeze(-1)
        m = torch.where(m == NEG, torch.zeros_like(m), m)
        self.d = (z - m) / T
        self.e = self.d.exp()
        S = self.e.sum(-1, keepdim=True)
        self.logS = S.log()
        self.lse = (m / T + self.logS).squeeze(-1)
        self.logp = torch.where(self.none.unsqueeze(-1), torch.full_like(z, NEG), self.d - self.logS)
        self.p = self.logp.exp()
        absd = torch.where(self.p > 0, self.d.abs(), torch.zeros_like(z))
        self.Ed, self.Ed2 = (self.p * absd).sum(-1, keepdim=True), (self.p * absd * absd).sum(-1, keepdim=True)
        self.entropy = -torch.special.xlogy(self.p, self.p).sum(-1)
        self.L = chain
        fin = torch.where(torch.isfinite(self.logS), self.logS, torch.zeros_like(self.logS)).abs()
        self.err_logS = H24 * (5 * self.Ed + chain + 10 + fin)
        absd_all = torch.where(torch.isfinite(self.d), self.d.abs(), torch.zeros_like(z))
        self.err_logp = H24 * (4 * absd_all + fin) + self.err_logS
        self.err_lse = self.err_logS.squeeze(-1) + H24 * (3 * (m / T).abs().squeeze(-1) + self.lse.abs().nan_to_num(0, 0, 0))
        # entropy = log S - U / S: U's terms carry the relative error of e^d and of d (3h) and one product; the quotient that of S and 3h
        U = self.Ed.squeeze(-1)
        self.err_entropy = (self.err_logS.squeeze(-1) + H24 * (5 * self.Ed2.squeeze(-1) + (2 * chain + 22) * U + 5 * U * U
                                                                + self.entropy.abs()))

    def at(self, ids):
        return self.logp.gather(-1, ids)

    def err_at(self, ids):
        return self.err_logp.gather(-1, ids)


def chain(C):
    """Longest chain of additions over a row in any of the kernels: a lane's share of the classes, then joins; never more than C + 16."""
    return min(C, 2048) + 16


def logprobs(z, label, T, k, ignore):
    """dict of (value, bound) with the classes last."""
    r = Rows(z, T, chain(z.shape[-1]))
    void = torch.zeros(z.shape[:-1], dtype=torch.bool) if label is None else label == ignore
    zero = lambda t: torch.where(void, torch.zeros_like(t), t)  # noqa: E731
    out = dict(entropy=(zero(torch.where(r.none, torch.zeros_like(r.entropy), r.entropy)), r.err_entropy), lse=(zero(r.lse), r.err_lse))
    if label is not None:
        ok = (label >= 0) & (label < z.shape[-1])
        y = torch.where(ok, label, torch.zeros_like(label)).unsqueeze(-1)
        lp = torch.where(ok, r.at(y).squeeze(-1), torch.full_like(r.lse, math.nan))
        out["logprob"] = (zero(lp), r.err_at(y).squeeze(-1))
    if k:
        ids = torch.sort(z, dim=-1, descending=True, stable=True)[1][..., :k]
        out["top_ids"] = (torch.where(void.unsqueeze(-1), torch.full_like(ids, -1), ids), None)
        out["top_logprobs"] = (torch.where(void.unsqueeze(-1), torch.full(ids.shape, NEG, dtype=torch.float64), r.at(ids)), r.err_at(ids))
    return out


def logprobs_grad(z, label, T, ignore, g_logprob, g_entropy, g_lse, eps_half):
    """(gradient, bound): dz = p (A + B log p) + [c = y] G."""
    C = z.shape[-1]
    r = Rows(z, T, chain(C))
    void = r.none if label is None else (label == ignore) | r.none
    ok = torch.zeros_like(void) if label is None else (label >= 0) & (label < C)
    zero = torch.zeros(z.shape[:-1], dtype=torch.float64)
    g1 = zero if g_logprob is None else torch.where(ok, g_logprob, zero)
    g2 = zero if g_entropy is None else g_entropy
    g3 = zero if g_lse is None else g_lse
    G, B = g1 / T, -g2 / T
    A = g3 / T - G + B * r.entropy
    lp = r.logp.clamp_min(-200.0)
    A_, B_ = A.unsqueeze(-1), B.unsqueeze(-1)
    hot = torch.zeros_like(z)
    if label is not None:
        hot.scatter_(-1, torch.where(ok, label, torch.zeros_like(label)).unsqueeze(-1), G.unsqueeze(-1))
    v = r.p * (A_ + B_ * lp) + hot
    rel_p = (r.err_logp.nan_to_num(0, 0, 0) + H24 * (2 * lp.abs() + 4))          # of exp(log p)
    err_A = H24 * 3 * (g3.abs() / T + G.abs() + 2 * (B * r.entropy).abs()) + B.abs() * r.err_entropy.nan_to_num(0, 0, 0)
    err = r.p * ((A_.abs() + B_.abs() * lp.abs()) * (rel_p + 4 * H24) + err_A.unsqueeze(-1) + B_.abs() * r.err_logp.nan_to_num(0, 0, 0))
    err = err + (hot.abs() + v.abs()) * 2 * H24 + v.abs() * eps_half
    dead = void.unsqueeze(-1)
    return torch.where(dead, torch.zeros_like(v), v), torch.where(dead, torch.zeros_like(err), err)


def distill(z, ids, top, T, tail, weight, reduction, eps_half, g=None):
    """loss (or losses of the rows) and gradient with their bounds; g: the loss's gradient (one, or one per row for "none")."""
    C, k = z.shape[-1], ids.shape[-1]
    r = Rows(z, T, chain(C))
    bad = (ids >= C).any(-1)
    there = (ids >= 0) & (ids < C)
    at = torch.where(there, ids, torch.zeros_like(ids))
    v = torch.where(there, top, torch.full_like(top, NEG))
    if tail:
        lq = v
        err_lq = torch.zeros_like(v)
    else:
        m = v.amax(-1, keepdim=True)
        m = torch.where(m == NEG, torch.zeros_like(m), m)
        d = (v - m) / T
        lq = d - d.exp().sum(-1, keepdim=True).log()
        err_lq = H24 * (8 * d.abs().nan_to_num(0, 0, 0) + k + 16)
    q = lq.exp().nan_to_num(0.0)
    rel_q = err_lq + H24 * (2 * lq.abs().nan_to_num(0, 0, 0) + 6)
    lp = r.at(at)
    err_lp = r.err_at(at).nan_to_num(0, 0, 0)
    term = torch.where(q > 0, q * (lq - lp), torch.zeros_like(q))
    kl = term.sum(-1)
    diff = torch.where(q > 0, (lq - lp).abs(), torch.zeros_like(q)).nan_to_num(0, 0, 0)
    err_kl = (q * (diff * (rel_q + (k + 3) * H24) + err_lq.nan_to_num(0, 0, 0) + err_lp)).sum(-1)
    Q = q.sum(-1)
    a = torch.zeros_like(z).scatter_add_(-1, at, q)
    err_a = torch.zeros_like(z).scatter_add_(-1, at, q * (rel_q + (k + 1) * H24))
    if tail:
        rest = (1 - Q).clamp_min(0)
        err_rest = (q * rel_q).sum(-1) + (k + 2) * H24 * Q.clamp_min(1)
        inside = torch.zeros(z.shape, dtype=torch.long).scatter_add_(-1, at, there.long()) > 0
        out = torch.where(inside, torch.full_like(z, NEG), r.d)
        some = (out > NEG).any(-1)
        rest = torch.where(some, rest, torch.zeros_like(rest))
        lr = torch.where(some, torch.logsumexp(out, -1) - r.logS.squeeze(-1), torch.zeros_like(rest))
        # the outside sum has an error like S's, about its own maximum
        po = torch.where(some.unsqueeze(-1), torch.softmax(out, -1), torch.zeros_like(out))
        mo = out.amax(-1, keepdim=True)
        do = torch.where(inside | ~torch.isfinite(out), torch.zeros_like(out), (out - mo).abs())
        err_lr = H24 * (5 * (po * do).sum(-1) + chain(C) + 10 + 4 * torch.where(some, mo.squeeze(-1).abs(), torch.zeros_like(lr))
                        + 2 * lr.abs() + 2 * r.logS.squeeze(-1).abs().nan_to_num(0, 0, 0)) + r.err_logS.squeeze(-1).nan_to_num(0, 0, 0)
        kl = kl + torch.where(rest > 0, torch.special.xlogy(rest, rest) - rest * lr, torch.zeros_like(rest))
        # rest log rest changes by at most err (1 + |log err|) where rest itself is of the error's size
        grow = (1 + err_rest.clamp_min(1e-30).log().abs() + lr.abs())
        err_kl = err_kl + torch.where(some, err_rest * grow + rest * err_lr + rest * H24 * 8 * (1 + lr.abs()), torch.zeros_like(rest))
        Q = Q + rest
        a = a + rest.unsqueeze(-1) * po
        err_a = err_a + po * (torch.where(some, err_rest, torch.zeros_like(rest)) + rest * (err_lr + H24 * 8)).unsqueeze(-1) \
            + po * rest.unsqueeze(-1) * H24 * 8 * do
    w = torch.ones_like(kl) if weight is None else weight
    on = (w != 0)
    kl = torch.where(there.any(-1), kl, torch.zeros_like(kl))
    kl = torch.where(bad, torch.full_like(kl, math.nan), kl)
    rows = torch.where(on, T * T * w * kl, torch.zeros_like(kl))
    err_rows = torch.where(on, T * T * w.abs() * (err_kl + 6 * H24 * kl.abs().nan_to_num(0, 0, 0)), torch.zeros_like(kl))
    den = w.sum() if reduction == "mean" else torch.tensor(1.0, dtype=torch.float64)
    if reduction == "none":
        loss = (rows, err_rows)
    else:
        loss = (rows.sum() / den, err_rows.sum() / den.abs() + 3 * H24 * (rows.sum() / den).abs())
    g = torch.ones((), dtype=torch.float64) if g is None else g
    coef = g * T * w / (den if den != 0 else 1.0) * (0.0 if den == 0 else 1.0)
    dead = ~on | bad | r.none | ~there.any(-1)
    coef = torch.where(dead, torch.zeros_like(coef), coef).unsqueeze(-1)
    rel_p = r.err_logp.nan_to_num(0, 0, 0) + H24 * (2 * r.logp.clamp_min(-200).abs() + 6)
    Q_ = Q.unsqueeze(-1)
    grad = coef * (r.p * Q_ - a)
    err_Q = (q * rel_q).sum(-1, keepdim=True) + (k + 2) * H24
    err = coef.abs() * (r.p * (Q_ * rel_p + err_Q) + err_a + 4 * H24 * (r.p * Q_ + a)) + grad.abs() * (6 * H24 + eps_half)
    return loss, (torch.where(dead.unsqueeze(-1), torch.zeros_like(grad), grad), err)
