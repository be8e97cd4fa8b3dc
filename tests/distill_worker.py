"""Worker of test_class_probs_gpu.py: one rank of a data-parallel run of Trainer.step with a teacher (gloo, so that both ranks can share
one GPU; every exchange goes through host memory)."""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.join(ROOT, "tests"))

import numpy as np  # noqa: E402
import torch  # noqa: E402
import torch.distributed as dist  # noqa: E402

from dist_worker import data, make_model  # noqa: E402


class _Done:
    def wait(self):
        return True


def through_the_host():
    """torch.distributed.all_reduce of device tensors by way of host memory, with synchronous copies."""
    plain = dist.all_reduce

    def all_reduce(t, op=dist.ReduceOp.SUM, group=None, async_op=False):
        h = t.cpu()
        plain(h, op=op, group=group)
        t.copy_(h)
        return _Done() if async_op else None
    dist.all_reduce = all_reduce


def run(world, rank, steps=2):
    from semseg_amd.distill import distill_loss
    from semseg_amd.trainer import Trainer
    dev = torch.device("cuda", 0)
    tr = Trainer(make_model().to(dev).train(), sync_bn=True, bucket_mb=8, distill_weight=0.7, distill_temperature=2.0)
    x, y = data(4)
    gen = torch.Generator().manual_seed(8)
    top, ids = (torch.randn(4, 7, 8, 8, generator=gen) * 2).topk(3, 1)
    w = (torch.rand(1, 8, 8, generator=gen) > 0.2).float().expand(4, 8, 8).contiguous()      # the same sum in every image
    per = 4 // world
    x, y, top, ids, w = (t[rank * per:(rank + 1) * per].contiguous().to(dev) for t in (x, y, top, ids, w))
    kd, want, w1 = [], [], None
    for it in range(steps):
        out = tr.step(x, y, lr=0.01, top=(ids, top, w))
        s = tr.engine(x)._rec_main["scores"]
        kd.append(float(out[3]))
        want.append(float(distill_loss(s.data[..., :s.C].movedim(-1, 1), ids, top, temperature=2.0, weight=w)))
        w1 = tr.flat_w.cpu().numpy() if it == 0 else w1
    return np.array(kd), np.array(want), w1, tr.flat_w.cpu().numpy()


if __name__ == "__main__":
    out = sys.argv[1]
    world, rank = int(os.environ.get("WORLD_SIZE", "1")), int(os.environ.get("RANK", "0"))
    if world > 1:
        dist.init_process_group("gloo", rank=rank, world_size=world)
        through_the_host()
    kd, want, w1, w = run(world, rank)
    np.savez(os.path.join(out, "rank%d_of%d.npz" % (rank, world)), kd=kd, want=want, w1=w1, w=w)
    if world > 1:
        dist.barrier()
        dist.destroy_process_group()
