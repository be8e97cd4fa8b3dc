"""Distillation in the training path: what a step leaves behind, and several ranks."""
import gc
import os
import socket
import subprocess
import sys
import tempfile
import weakref

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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


def _free_port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


def test_two_ranks_distil_each_its_own_rows(report):
    """The distillation's mean is each rank's own (over its weights), and the ranks' gradients are averaged like the cross entropy's: with
    equal sums of weights two ranks take the step of one process with the whole batch."""
    tmp = tempfile.mkdtemp(prefix="semseg_distill_")
    env = dict(os.environ, HSA_ENABLE_IPC_MODE_LEGACY="0")
    worker = os.path.join(ROOT, "tests", "distill_worker.py")
    subprocess.check_call([sys.executable, worker, tmp], env=env, timeout=110)
    subprocess.check_call([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1", "--master-port",
                           str(_free_port()), worker, tmp], env=env, timeout=110)
    one, r0, r1 = (np.load(os.path.join(tmp, n)) for n in ("rank0_of1.npz", "rank0_of2.npz", "rank1_of2.npz"))
    assert np.array_equal(r0["w"], r1["w"])
    for r in (one, r0, r1):
        assert np.abs(r["kd"] - r["want"]).max() <= 1e-5 * np.abs(r["want"]).max()
    e_kd = np.abs(0.5 * (r0["kd"] + r1["kd"]) - one["kd"])[0] / one["kd"][0]
    e_w = np.abs(r0["w1"] - one["w1"]).max() / np.abs(one["w1"]).max()
    report("2-rank distillation step vs single process: loss %.2e, weights after 1 step %.2e" % (e_kd, e_w))
    assert e_kd < 1e-5 and e_w < 2e-4
