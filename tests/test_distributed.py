"""Multi-process logic on CPU ranks (gloo, world_size 2): the batch shards without a
data-path collective, and the weight-gradient exchange is one flat all-reduce whose result
equals the single-process gradient.  The arithmetic on each rank is the CPU oracle (this
test exercises the sharding and reduction plumbing, not the kernels)."""
import os
import sys

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _worker(rank, world, port, out_dir):
    sys.path.insert(0, ROOT)
    from oracle.oracle import Oracle, module_backward, module_forward, round_robin_angles
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        rng = np.random.default_rng(0)                # same global batch on every rank
        N, C, H, W, K = 4, 16, 12, 12, 15
        x = rng.standard_normal((N, H, W, C)).astype(np.float32)
        dy = rng.standard_normal((N, H, W, C)).astype(np.float32)
        w = (0.02 * rng.standard_normal((C, 1, 1, K))).astype(np.float32)
        bias = rng.standard_normal(C).astype(np.float32)
        th = round_robin_angles(C)
        oracle = Oracle()
        lo, hi = rank * N // world, (rank + 1) * N // world          # batch shard of this rank
        y = module_forward(oracle, x[lo:hi], w, th, bias, 1, True, False)
        dx, dw, db = module_backward(oracle, x[lo:hi], w, th, dy[lo:hi], bias, 1, True, False)
        flat = torch.from_numpy(np.concatenate([dw.reshape(-1), db]))  # one flat gradient buffer
        dist.all_reduce(flat)
        np.savez(os.path.join(out_dir, f"rank{rank}.npz"), y=y, dx=dx, flat=flat.numpy(), lo=lo, hi=hi)
    finally:
        dist.destroy_process_group()


def test_batch_sharding_and_gradient_allreduce(tmp_path):
    from oracle.oracle import Oracle, module_backward, module_forward, round_robin_angles
    world, port = 2, 29611 + os.getpid() % 500
    mp.start_processes(_worker, args=(world, port, str(tmp_path)), nprocs=world, join=True, start_method="spawn")
    rng = np.random.default_rng(0)
    N, C, H, W, K = 4, 16, 12, 12, 15
    x = rng.standard_normal((N, H, W, C)).astype(np.float32)
    dy = rng.standard_normal((N, H, W, C)).astype(np.float32)
    w = (0.02 * rng.standard_normal((C, 1, 1, K))).astype(np.float32)
    bias = rng.standard_normal(C).astype(np.float32)
    th = round_robin_angles(C)
    oracle = Oracle()
    y = module_forward(oracle, x, w, th, bias, 1, True, False)
    dx, dw, db = module_backward(oracle, x, w, th, dy, bias, 1, True, False)
    ref_flat = np.concatenate([dw.reshape(-1), db])
    for rank in range(world):
        r = np.load(os.path.join(str(tmp_path), f"rank{rank}.npz"))
        lo, hi = int(r["lo"]), int(r["hi"])
        assert np.array_equal(r["y"], y[lo:hi]) and np.array_equal(r["dx"], dx[lo:hi])   # no exchange needed
        err = np.abs(r["flat"] - ref_flat).max() / np.abs(ref_flat).max()
        assert err <= 1e-4, err                                                           # sum over ranks


class _Classifier:
    """A ConvNeXt1D whose features come from one library conv and whose head's loss is torch's, so that it runs on a CPU rank."""

    def __new__(cls):
        from oriented1d_b200 import convnext1d

        class Model(convnext1d.ConvNeXt1D):
            def forward_features(self, x, all_stages=False):
                return self.features(x)

        torch.manual_seed(0)
        m = Model(depths=(1, 1, 1, 1), dims=(8, 8, 8, 8), num_classes=5, stem_dim1=8)
        del m.downsample_layers, m.stages
        m.features = torch.nn.Conv2d(3, 8, 4, stride=4)
        convnext1d.ops.linear_cross_entropy = lambda x, w, t, b, **kw: torch.nn.functional.cross_entropy(x @ w.t() + b, t, **kw)
        return m


def _batch():
    g = torch.Generator().manual_seed(1)
    return torch.randn(6, 3, 16, 16, generator=g), torch.tensor([0, 1, 2, 3, 4, 0])


def _loss_worker(rank, world, port, out_dir):
    sys.path.insert(0, ROOT)
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        img, t = _batch()
        lo, hi = rank * 6 // world, (rank + 1) * 6 // world
        m = _Classifier()
        ddp = torch.nn.parallel.DistributedDataParallel(m)
        loss = ddp(img[lo:hi], t[lo:hi], label_smoothing=0.1)
        loss.backward()
        torch.save({k: p.grad for k, p in m.named_parameters()}, os.path.join(out_dir, f"grads{rank}.pt"))
    finally:
        dist.destroy_process_group()


def test_the_loss_through_a_data_parallel_wrapper(tmp_path, monkeypatch):
    """The gradients on every rank are those of the whole batch: the wrapper sees the loss as a forward pass."""
    from oriented1d_b200 import ops
    monkeypatch.setattr(ops, "linear_cross_entropy", ops.linear_cross_entropy)            # put back what _Classifier replaces
    world, port = 2, 30111 + os.getpid() % 500
    mp.start_processes(_loss_worker, args=(world, port, str(tmp_path)), nprocs=world, join=True, start_method="spawn")
    m = _Classifier()
    img, t = _batch()
    m(img, t, label_smoothing=0.1).backward()
    assert torch.equal(m(img, t, 0.1), m.loss(img, t, 0.1)) and m(img).shape == (6, 5)
    for rank in range(world):
        got = torch.load(os.path.join(str(tmp_path), f"grads{rank}.pt"))
        for k, p in m.named_parameters():                                                  # (equal shards: the mean of means is the mean)
            assert float((got[k] - p.grad).norm()) <= 1e-5 * float(p.grad.norm()) + 1e-8, k
