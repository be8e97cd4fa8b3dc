"""Class probabilities of logits on tensors: log probabilities of given classes with entropy and top alternatives, and distillation from
a teacher's stored top logits.  The kernels are csrc/class_logprobs.hip and csrc/distill.hip (include/semseg_hip.h); nothing here computes.

    top = class_logprobs(teacher_logits, topk=8)                          # what a teacher answers: keep top.top_ids, top.top_logprobs
    loss = distill_loss(student_logits, top.top_ids, top.top_logprobs, temperature=4.0)
    loss.backward()

Logits are fp32, bf16 or fp16 with the classes in dimension `class_dim`: 1 as nn.CrossEntropyLoss takes them ([N, C, H, W], [rows, C]) or
-1 ([N, h, w, C]).  They are read in place through their strides: either the classes are contiguous (pixel-major score buffers with any
row stride, channels_last maps, [tokens, vocabulary]) or the pixels are (an eval model's output, one plane per class); a tensor in
neither form is refused.  Every gradient is a new tensor in the logits' type; double differentiation is refused.

Work is launched on the current stream of the logits' device and never waits for it; workspaces come from torch's allocator call by
call, so calls on several streams and captured graphs share none.  Outputs do not depend on scheduling (no atomics)."""
import contextlib
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import ops

TOP_MAX = 64          # SEMSEG_CLASS_TOP_MAX


class ClassLogprobs(NamedTuple):
    logprob: Optional[torch.Tensor]         # log p of the label; 0 for void rows, NaN for a label that is no class
    entropy: torch.Tensor                   # -sum p log p
    lse: torch.Tensor                       # log sum exp(logits / temperature)
    top_ids: Optional[torch.Tensor]         # int32, k in the place of the classes; -1 for void rows
    top_logprobs: Optional[torch.Tensor]    # fp32; -inf for void rows; not differentiable


# ---------------------------------------------------------------------------------------------
# shapes and strides
# ---------------------------------------------------------------------------------------------
def _dim(x, class_dim):
    if class_dim not in (1, -1):
        raise ValueError("class_dim must be 1 or -1, got %r" % (class_dim,))
    if x.dim() < 2:
        raise ValueError("expected at least two dimensions (rows and classes), got %s" % (tuple(x.shape),))
    return 1 if class_dim == 1 else x.dim() - 1


def _groups(sizes, strides):
    """Runs of dimensions that one stride walks: [(size, stride, number of dimensions)] with sizes of 1 folded in."""
    out = []
    for n, s in zip(sizes, strides):
        if out and (n == 1 or out[-1][0] == 1 or out[-1][1] == n * s):
            pn, ps, pd = out[-1]
            out[-1] = (pn * n, s if n != 1 else ps, pd + 1)
        else:
            out.append((n, s, 1))
    return out


class Geom:
    """Rows of a logits tensor: (n, p, C), element strides and the number of row dimensions that make up n."""

    def __init__(self, z, dim):
        sizes, strides = list(z.shape), list(z.stride())
        self.C, sc = sizes.pop(dim), strides.pop(dim)
        if self.C > 1 << 30:
            raise ValueError("at most 2^30 classes, got %d" % self.C)
        self.dim, self.shape = dim, tuple(sizes)
        g = _groups(sizes, strides)
        if len(g) > 2:
            raise ValueError("logits of shape %s and strides %s: their rows cannot be walked by two strides; pass a contiguous tensor"
                             % (tuple(z.shape), tuple(z.stride())))
        (self.n, sn, self.outer), (self.p, sp, _) = ((1, 0, 0), g[0]) if len(g) == 1 else g
        self.by_rows = sc == 1 or self.C == 1
        if not self.by_rows and not (sp == 1 or self.p == 1):
            raise ValueError("logits of shape %s and strides %s: neither the classes nor the pixels are contiguous; pass a contiguous "
                             "tensor" % (tuple(z.shape), tuple(z.stride())))
        self.strides = (sn, 1 if self.p == 1 and not self.by_rows else sp, 1 if self.C == 1 else sc)
        self.geom = (self.n, self.p, self.C)

    def empty(self, size, dtype, device):
        """A dense tensor with `size` in the place of the classes; in memory that dimension stands behind the rows, or (planes) between
        the n and the p of them, wherever `dim` has it."""
        at = len(self.shape) if self.by_rows else self.outer
        t = torch.empty(self.shape[:at] + (size,) + self.shape[at:], dtype=dtype, device=device)
        return t if at == self.dim else t.movedim(at, self.dim)

    def dense(self, size):
        """Strides (sn, sp, s of `dim`) of what empty(size) gives."""
        return (self.p * size, size, 1) if self.by_rows else (size * self.p, 1, self.p)

    def strides_of(self, t):
        """(sn, sp, s of `dim`) of a tensor with these rows; None where its rows do not split the same way."""
        sizes, strides = list(t.shape), list(t.stride())
        sizes.pop(self.dim)
        s = strides.pop(self.dim)
        a, b = _groups(sizes[:self.outer], strides[:self.outer]), _groups(sizes[self.outer:], strides[self.outer:])
        if len(a) > 1 or len(b) > 1:
            return None
        return (a[0][1] if a else 0, b[0][1] if b and self.p > 1 else 1, s)


def check_temperature(temperature):
    if not 1e-15 <= temperature <= 1e15:
        raise ValueError("temperature must lie in [1e-15, 1e15], got %r" % (temperature,))


def _check_logits(z, class_dim, temperature):
    if not isinstance(z, torch.Tensor) or z.dtype not in ops.TYPES:
        raise TypeError("logits must be an fp32, bf16 or fp16 tensor, got %s" % (z.dtype if isinstance(z, torch.Tensor) else type(z)))
    dim = _dim(z, class_dim)
    if z.numel() == 0:
        raise ValueError("logits of shape %s hold no value" % (tuple(z.shape),))
    check_temperature(temperature)
    return Geom(z, dim)


def _check_rows(t, what, g, dtype, device):
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise TypeError("%s must be a %s tensor" % (what, dtype))
    if tuple(t.shape) != g.shape:
        raise ValueError("%s has shape %s, the logits' rows %s" % (what, tuple(t.shape), g.shape))
    if t.device != device:
        raise ValueError("%s is on %s, the logits on %s" % (what, t.device, device))


def _overlap(a, b):
    """Whether the spans of memory that two tensors reach into meet."""
    span = lambda t: t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))  # noqa: E731
    return a.device == b.device and a.numel() and b.numel() and a.data_ptr() < span(b) and b.data_ptr() < span(a)


def _once(t):
    """Whether no two values of a tensor share memory: every stride passes over all that the smaller ones reach."""
    reach = 0
    for st, n in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n > 1):
        if st <= reach:
            return False
        reach += st * (n - 1)
    return True


def _check_out(out, logits, g, inputs):
    """Strides of the tensor that a gradient is written to."""
    if out.shape != logits.shape or out.dtype != logits.dtype or out.device != logits.device:
        raise ValueError("out must have the logits' shape, type and device")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError("out must not require a gradient")
    if any(_overlap(out, t) for t in inputs if t is not None):
        raise ValueError("out shares memory with an input")
    ds = g.strides_of(out)
    if ds is None or not (ds[2] == 1 if g.by_rows and g.C > 1 else g.C == 1 or ds[1] == 1) or not _once(out):
        raise ValueError("out of strides %s does not have the logits' layout, each value in a place of its own" % (tuple(out.stride()),))
    return ds


def _on_gpu(z):
    if not z.is_cuda:
        raise RuntimeError("semseg_amd runs on the MI355X only: move the logits to cuda (there is no CPU fallback)")


def _on_device(z):
    """The logits' device as the current one (nothing to do where it is: entering a device costs as much as a launch)."""
    return contextlib.nullcontext() if z.device.index == torch.cuda.current_device() else torch.cuda.device(z.device)


# ---------------------------------------------------------------------------------------------
# log probabilities, entropy, top alternatives
# ---------------------------------------------------------------------------------------------
def _logprobs(z, g, label, ignore_index, temperature, k, stats):
    dev, ids, tlp, ts = z.device, None, None, (0, 0, 0)
    logprob = None if label is None else torch.empty(g.shape, dtype=torch.float32, device=dev)
    entropy, lse = (torch.empty(g.shape, dtype=torch.float32, device=dev) for _ in range(2))
    if k:
        ids, tlp, ts = g.empty(k, torch.int32, dev), g.empty(k, torch.float32, dev), g.dense(k)
    need = ops.class_logprobs_scratch_bytes(z.dtype, *g.geom, g.strides[2], k)
    scratch = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    ops.class_logprobs_fwd(z, g.geom, g.strides, label, ignore_index, temperature, k, logprob, entropy, lse, stats, ids, tlp, ts, scratch)
    return logprob, entropy, lse, ids, tlp


class _Logprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, g, label, ignore_index, temperature, k):
        with _on_device(z):
            stats = torch.empty((2,) + g.shape, dtype=torch.float32, device=z.device)
            logprob, entropy, lse, ids, tlp = _logprobs(z, g, label, ignore_index, temperature, k, stats)
        ctx.save_for_backward(z, label, stats, entropy)
        ctx.g, ctx.ignore_index, ctx.temperature = g, ignore_index, temperature
        if k:
            ctx.mark_non_differentiable(ids, tlp)
        ctx.set_materialize_grads(False)
        return logprob, entropy, lse, ids, tlp

    @staticmethod
    @once_differentiable
    def backward(ctx, g_logprob, g_entropy, g_lse, *_):
        z, label, stats, entropy = ctx.saved_tensors
        g = ctx.g
        with _on_device(z):
            dz = g.empty(g.C, z.dtype, z.device)
            if g_logprob is None and g_entropy is None and g_lse is None:
                return dz.zero_(), None, None, None, None, None
            gs = [None if t is None else t.contiguous() for t in (g_logprob, g_entropy, g_lse)]
            ops.class_logprobs_bwd(z, g.geom, g.strides, label, ctx.ignore_index, ctx.temperature, stats, entropy, *gs, dz,
                                   g.dense(g.C))
        return dz, None, None, None, None, None


def class_logprobs(logits, label=None, topk=0, temperature=1.0, ignore_index=None, class_dim=1):
    """Log softmax(logits / temperature) at the rows' labels, its entropy and log-sum-exp, and the `topk` best classes of every row
    with their log probabilities (falling, equal logits by rising class).  logprob, entropy and lse carry gradients.

    label: int64, the logits' shape without the classes.  Rows labelled ignore_index (default: 255, as in the segmentation losses, where
    that is no class, otherwise -100) are void, whatever they hold: zero outputs, no alternatives (ids -1, log probabilities -inf), zero
    gradient.
    A label that is neither gives log probability NaN (ops.label_check counts them).
    A row of -inf logits has log probabilities -inf, entropy 0 and no gradient.  A row with a NaN or +inf has NaN in everything but its
    alternatives: NaN first, then +inf, each by rising class."""
    g = _check_logits(logits, class_dim, temperature)
    if label is not None:
        _check_rows(label, "label", g, torch.int64, logits.device)
        label = label.contiguous()
    if isinstance(topk, bool) or not isinstance(topk, int) or not 0 <= topk <= min(TOP_MAX, g.C):
        raise ValueError("topk must be a whole number of [0, min(%d, classes = %d)], got %r" % (TOP_MAX, g.C, topk))
    if ignore_index is None:
        ignore_index = 255 if g.C <= 255 else -100
    _on_gpu(logits)
    if logits.requires_grad and torch.is_grad_enabled():
        return ClassLogprobs(*_Logprobs.apply(logits, g, label, int(ignore_index), float(temperature), topk))
    with _on_device(logits):
        return ClassLogprobs(*_logprobs(logits, g, label, int(ignore_index), float(temperature), topk, None))


# ---------------------------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------------------------
def check_top(g, device, top_ids, top_values, weight):
    """The teacher's entries of rows `g` on `device`, as the kernels take them."""
    if not isinstance(top_ids, torch.Tensor) or top_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError("top_ids must be an int32 or int64 tensor")
    if not isinstance(top_values, torch.Tensor) or top_values.dtype not in ops.TYPES:
        raise TypeError("top_logits must be an fp32, bf16 or fp16 tensor")
    k = top_ids.shape[g.dim] if top_ids.dim() == len(g.shape) + 1 else -1
    want = g.shape[:g.dim] + (k,) + g.shape[g.dim:]
    if k < 1 or tuple(top_ids.shape) != want or tuple(top_values.shape) != want:
        raise ValueError("top_ids %s and top_logits %s must have the logits' shape %s with the teacher's entries in the place of the "
                         "classes" % (tuple(top_ids.shape), tuple(top_values.shape), g.shape[:g.dim] + (g.C,) + g.shape[g.dim:]))
    if k > TOP_MAX:
        raise ValueError("at most %d entries a row, got %d" % (TOP_MAX, k))
    if top_ids.device != device or top_values.device != device:
        raise ValueError("top_ids and top_logits must be on the logits' device %s" % (device,))
    if top_values.requires_grad and torch.is_grad_enabled():
        raise ValueError("no gradient flows into the teacher: detach top_logits")
    if weight is not None:
        _check_rows(weight, "weight", g, torch.float32, device)
        if weight.requires_grad and torch.is_grad_enabled():
            raise ValueError("no gradient flows into the weights: detach them")
        weight = weight.contiguous()
    out = []
    for t in (top_ids, top_values):
        s = g.strides_of(t)
        if s is None:
            t = g.empty(k, t.dtype, device).copy_(t)
            s = g.strides_of(t)
        out += [t, s]
    return (*out, k, weight)


def _check_distill(logits, top_ids, top_values, temperature, weight, class_dim, reduction, reductions):
    g = _check_logits(logits, class_dim, temperature)
    teacher = check_top(g, logits.device, top_ids, top_values, weight)
    if reduction not in reductions:
        raise ValueError("reduction must be one of %s, got %r" % (", ".join(reductions), reduction))
    _on_gpu(logits)
    return g, teacher


def _distill(z, g, teacher, temperature, tail, reduction):
    """(loss or losses of the rows, workspace, its offsets)"""
    nbytes, at = ops.distill_workspace(z.dtype, *g.geom, g.strides[2])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=z.device)
    out = torch.empty(g.shape if reduction == "none" else (), dtype=torch.float32, device=z.device)
    rows, loss = (out, None) if reduction == "none" else (None, out)
    ops.distill_fwd(z, g.geom, g.strides, *teacher, temperature, tail, reduction, rows, loss, ws, at)
    return out, ws, at


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, g, teacher, temperature, tail, reduction):
        with _on_device(z):
            loss, ws, at = _distill(z, g, teacher, temperature, tail, reduction)
        ids, ids_s, top, top_s, k, weight = teacher
        ctx.save_for_backward(z, ids, top, weight, ws)
        ctx.how = g, ids_s, top_s, k, temperature, tail, reduction, at
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        z, ids, top, weight, ws = ctx.saved_tensors
        g, ids_s, top_s, k, temperature, tail, reduction, at = ctx.how
        with _on_device(z):
            dz = g.empty(g.C, z.dtype, z.device)
            ops.distill_bwd(z, g.geom, g.strides, ids, ids_s, top, top_s, k, weight, temperature, tail, reduction, ws, at, grad.contiguous(),
                            1.0, dz, g.dense(g.C))
        return dz, None, None, None, None, None


def distill_loss(logits, top_ids, top_logits, temperature=1.0, tail=False, weight=None, class_dim=1, reduction="mean"):
    """temperature^2 * mean over rows of KL(teacher || student), the teacher given by its top entries: ids (int32 / int64) and values
    (fp32 / bf16 / fp16) in the logits' shape with k <= 64 entries in the place of the classes.

    tail=False: top_logits are logits (or log probabilities at temperature 1: a row's shift does not matter); the teacher's distribution is
    softmax(top_logits / temperature) over its entries.  tail=True: top_logits are log probabilities AT `temperature` (class_logprobs(...,
    temperature=temperature)); what they leave of 1 is one more class, against the student's mass outside the entries.
    A negative id is an absent entry, a row without entries counts with loss 0; an id that is no class makes the loss NaN.
    weight: fp32 per row; rows of weight 0 are void, whatever they hold.  reduction: "mean" (over the weights' sum; NaN where that is 0), "sum", "none"."""
    g, teacher = _check_distill(logits, top_ids, top_logits, temperature, weight, class_dim, reduction, ("mean", "sum", "none"))
    if logits.requires_grad and torch.is_grad_enabled():
        return _Distill.apply(logits, g, teacher, float(temperature), bool(tail), reduction)
    with _on_device(logits):
        return _distill(logits, g, teacher, float(temperature), bool(tail), reduction)[0]


def distill_loss_grad(logits, top_ids, top_logits, temperature=1.0, tail=False, weight=None, class_dim=1, reduction="mean",
                      grad_scale=1.0, out=None, accumulate=False):
    """(loss, grad_scale * gradient of the loss) in one call, outside autograd: what a training step that writes its own gradients uses.
    out: the tensor the gradient is written to (logits' shape and type; classes or pixels contiguous as in the logits), added to with
    accumulate=True; the default is a new one.  Its values may share memory neither with an input nor with each other.  The loss itself
    is not scaled."""
    g, teacher = _check_distill(logits, top_ids, top_logits, temperature, weight, class_dim, reduction, ("mean", "sum"))
    dev = logits.device
    if out is None:
        if accumulate:
            raise ValueError("accumulate=True needs out")
        out, ds = g.empty(g.C, logits.dtype, dev), g.dense(g.C)
    else:
        ds = _check_out(out, logits, g, (logits, top_ids, top_logits, weight))
    with _on_device(logits):
        # rows that fit registers need no statistics kept for a second pass
        nbytes, at = ops.distill_workspace(logits.dtype, *g.geom, g.strides[2], stats=not (g.by_rows and g.C <= ops.ROW_CLASSES))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev)
        ops.distill_fwd_bwd(logits, g.geom, g.strides, *teacher, temperature, tail, reduction, loss, grad_scale, out, ds, accumulate, ws, at)
    return loss, out
