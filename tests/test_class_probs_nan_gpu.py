"""Alternatives of rows with NaN and +inf (semseg_amd.distill) on the device."""
import math

import pytest
import torch

from semseg_amd import distill as D

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("shape,dim,k", [
    ((5, 21), -1, 8), ((5, 150), -1, 8), ((5, 200), -1, 12), ((5, 300), -1, 8), ((5, 1500), -1, 20), ((600, 2500), -1, 8), ((5, 9000), -1, 8),
    ((2, 70000), -1, 30), ((1, 21, 2, 3), 1, 4), ((1, 21, 2, 3), 1, 8), ((1, 150, 2, 3), 1, 20), ((1, 150, 1, 1), 1, 8), ((1, 150, 2, 3), 1, 40)])
def test_alternatives_of_a_row_with_nan_and_infinity(shape, dim, k, dt):
    """NaN first, then +inf, each by rising class, then the others as ever; every log probability of the row is NaN."""
    gen = torch.Generator().manual_seed(32)
    z = torch.randn(shape, generator=gen).to(dt)
    zl = z.movedim(dim, -1)
    C = zl.shape[-1]
    zl[..., 2], zl[..., C - 4], zl[..., 5], zl[..., C - 1] = math.inf, math.inf, math.nan, -math.nan
    zl[..., 7] = -math.inf
    o = D.class_logprobs(z.to(DEV), topk=k, class_dim=dim)
    ids = o.top_ids.movedim(dim, -1).long().cpu()
    assert ids[..., :4].reshape(-1, 4).unique(dim=0).tolist() == [[5, C - 1, 2, C - 4]]
    assert torch.equal(ids, torch.sort(zl.double(), dim=-1, descending=True, stable=True)[1][..., :k])
    assert bool(torch.isnan(o.top_logprobs).all()) and bool(torch.isnan(o.lse).all()) and bool(torch.isnan(o.entropy).all())
