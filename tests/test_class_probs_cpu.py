"""semseg_amd.distill without a GPU: where a gradient may be written."""
import pytest
import torch

from semseg_amd import distill as D

STORE = torch.zeros(4096)


def view(shape, strides):
    return torch.as_strided(STORE, shape, strides)


@pytest.mark.parametrize("logits,dim,shape,strides,ok", [
    ((7, 5), -1, (7, 5), (5, 1), True), ((7, 5), -1, (7, 5), (9, 1), True), ((1, 5), -1, (1, 5), (0, 1), True), ((7, 1), -1, (7, 1), (3, 0), True),
    ((7, 5), -1, (7, 5), (4, 1), False),            # rows that run into each other
    ((7, 5), -1, (7, 5), (0, 1), False), ((7, 5), -1, (7, 5), (1, 7), False), ((7, 1), -1, (7, 1), (0, 1), False),
    ((2, 5, 3, 4), 1, (2, 5, 3, 4), (60, 12, 4, 1), True), ((2, 5, 3, 4), 1, (2, 5, 3, 4), (12, 24, 4, 1), True), ((2, 5, 3, 4), 1, (2, 5, 3, 4), (70, 14, 4, 1), True),
    ((2, 5, 3, 4), 1, (2, 5, 3, 4), (60, 11, 4, 1), False), ((2, 5, 3, 4), 1, (2, 5, 3, 4), (59, 12, 4, 1), False), ((2, 5, 3, 4), 1, (2, 5, 3, 4), (30, 12, 4, 1), False),
    ((2, 5, 3, 4), 1, (2, 5, 3, 4), (60, 1, 20, 5), False),
])
def test_a_gradient_goes_where_each_value_has_a_place_of_its_own(logits, dim, shape, strides, ok):
    z = torch.zeros(logits)
    g = D.Geom(z, D._dim(z, dim))
    out = view(shape, strides)
    if ok:
        s = D._check_out(out, z, g, (z,))
        assert s == g.strides_of(out)
    else:
        with pytest.raises(ValueError):
            D._check_out(out, z, g, (z,))


def test_a_gradient_goes_to_no_input():
    z = torch.zeros(7, 9)[:, :5]
    g = D.Geom(z, 1)
    for bad, err in ((z, "shares"), (torch.zeros(7, 5).requires_grad_(), "require"), (torch.zeros(7, 4), "shape"), (torch.zeros(7, 5).double(), "type")):
        with pytest.raises(ValueError, match=err):
            D._check_out(bad, z, g, (z, None))
