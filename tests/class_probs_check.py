"""What the device tests of semseg_amd.distill compare with: half a step of each type, its smallest gradient, and values within their bounds
(class_probs_ref.py)."""
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}


def close(got, want, bound, what, tiny=1e-37):
    got, want = got.detach().double().cpu(), torch.as_tensor(want, dtype=torch.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), what + ": infinities or NaN elsewhere"
    fin = torch.isfinite(want)
    off = (got - want).abs()[fin] - torch.broadcast_to(torch.as_tensor(bound, dtype=torch.float64), want.shape)[fin].nan_to_num(0, 0, 0) - tiny
    if off.numel():
        i = int(off.argmax())
        assert float(off[i]) <= 0, "%s: off %.3g over what is allowed, value %.6g" % (what, off[i], want[fin][i])
