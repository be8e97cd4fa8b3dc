"""Distillation in the training path: what a step leaves behind."""
import gc
import weakref

import pytest
import torch

pytestmark = pytest.mark.gpu


def _net(seed, classes=21):
    from model.pspnet import PSPNet
    from oracle import segnet
    torch.manual_seed(5)
    m = PSPNet(layers=50, classes=classes, zoom_factor=8, dropout=0.0, pretrained=False)
    m.load_state_dict(segnet.recipe_state_dict({k: tuple(v.shape) for k, v in m.state_dict().items()}, seed=seed))
    return m.cuda()


@pytest.mark.parametrize("plan", [False, True])
def test_a_step_leaves_no_teacher_behind(plan):
    """A backward pass of the trainer's engine after a step with a teacher is the cross entropy's alone, and the entries are released."""
    from semseg_amd.trainer import Trainer
    t, m = _net(77).eval(), _net(1234).train()
    tr = Trainer(m, sync_bn=False)
    tr.use_plan = plan
    gen = torch.Generator().manual_seed(39)
    x, y = torch.randn(2, 3, 73, 73, generator=gen).cuda(), torch.randint(0, 21, (2, 73, 73), generator=gen).cuda()
    o = t.top_logits(x, 4)
    top = [o.top_ids, o.top_logprobs]
    del o
    for _ in range(6):
        assert len(tr.step(x, y, 0.0, top=tuple(top))) == 4
    e = tr.engine(x)

    def scores_grad():
        e.forward_train(x, y, 255)
        e.backward(tr.g_main, tr.g_aux)
        return e.grad_of(e._rec_main["scores"])[..., :21].clone()
    after = scores_grad()
    kept = weakref.ref(top[0])
    del top[:]
    gc.collect()
    assert kept() is None
    tr.use_plan = False
    tr.step(x, y, 0.0)
    plain = e.grad_of(e._rec_main["scores"])[..., :21]
    # equal up to the merging order of the normalisations' statistics; the distillation's part would be as large as the gradient
    assert float((after - plain).abs().max()) < 1e-2 * float(plain.abs().max())
