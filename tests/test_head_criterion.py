"""The training loop with a criterion that holds the model's head (losses.LinearCrossEntropy), and with one that merely has parameters.  On the CPU the
operators are torch stand-ins; what is tested there is the loop: what is clipped, averaged over ranks, captured, evaluated and saved."""
import os
import socket
import sys
from pathlib import Path

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = Path(__file__).resolve().parent.parent


class Features(torch.nn.Module):
    """a model whose gradients end in one flat buffer that a GradReducer averages when the backward pass reports it"""

    def __init__(self, n=6, d=8, reducer=False):
        super().__init__()
        self.w = torch.nn.Parameter(torch.randn(d, n))
        if reducer:
            from vision_transformers_torch_xla_amd.dp import GradReducer
            flat = torch.zeros(d * n)
            self.reducer = GradReducer(lambda: flat, bucket_bytes=64)

            def done(p):
                flat.copy_(p.grad.reshape(-1))
                p.grad = flat.view_as(p)
                self.reducer.ready(flat.numel(), True)
            self.w.register_post_accumulate_grad_hook(done)

    def forward(self, x):
        return x @ self.w.t()


class Head(torch.nn.Module):
    """LinearCrossEntropy's part in the loop, in torch"""
    takes_features = True
    ignore_index = -100

    def __init__(self, classes=5, d=8):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.randn(classes, d))
        self.bias = torch.nn.Parameter(torch.zeros(classes))

    def logits(self, x):
        return x @ self.weight.t() + self.bias

    def forward(self, x, target):
        return torch.nn.functional.cross_entropy(self.logits(x), target)


class WithTemperature(torch.nn.Module):
    """a criterion with a parameter that is no head; gradients of any type are its own affair"""

    def __init__(self, dtype=torch.float64):
        super().__init__()
        self.t = torch.nn.Parameter(torch.tensor([1.0, 3.0], dtype=dtype))

    def forward(self, x, target):
        return torch.nn.functional.cross_entropy(x * self.t.sum().to(x.dtype), target)


def torch_clip(tensors, max_norm, out=None):
    assert out is None
    norm = torch.sqrt(sum(t.double().square().sum() for t in tensors))
    for t in tensors:
        t.mul_(torch.clamp(max_norm / (norm + 1e-6), max=1.0))
    return norm.float()


def batches(n, rows=8, d=6, classes=5, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(rows, d, generator=g), torch.randint(0, classes, (rows,), generator=g)) for _ in range(n)]


def test_only_a_head_is_clipped_with_the_model(monkeypatch):
    from vision_transformers_torch_xla_amd import engine
    clipped = []
    monkeypatch.setattr(engine, "clip_grad_norm_", lambda what, max_norm: clipped.append(what))
    same = lambda x, t: (x, t)          # noqa: E731   (a mixup that does nothing: accuracy is not measured)
    for criterion in (WithTemperature(), Head()):
        torch.manual_seed(0)
        model = Features()
        opt = torch.optim.SGD([*model.parameters(), *criterion.parameters()], lr=0.1)
        engine.train_one_epoch(model, criterion, batches(2, classes=5), opt, torch.device("cpu"), 0, max_norm=0.5, mixup_fn=same)
    assert len(clipped) == 4 and all(isinstance(c, Features) for c in clipped[:2])
    for c in clipped[2:]:
        assert c[0] is model and [p is q for p, q in zip(c[1], criterion.parameters())] == [True, True]
    for p in criterion.parameters():                                     # a head that is frozen: the model alone
        p.requires_grad_(False)
    clipped.clear()
    engine.train_one_epoch(model, criterion, batches(1), torch.optim.SGD(model.parameters(), lr=0.1), torch.device("cpu"), 0, max_norm=0.5, mixup_fn=same)
    assert clipped == [model]


# ------------------------------------------------------------------------------------------- several ranks (gloo)
def _train(model, criterion, data, max_norm, update_freq=1):
    from vision_transformers_torch_xla_amd import engine
    engine.ops.clip_grads = torch_clip                                   # (a process of its own)
    opt = torch.optim.SGD([*model.parameters(), *criterion.parameters()], lr=0.5)
    engine.train_one_epoch(model, criterion, data, opt, torch.device("cpu"), 0, max_norm=max_norm, update_freq=update_freq)
    return torch.cat([p.detach().reshape(-1) for p in (*model.parameters(), *criterion.parameters())])


def _worker(rank, world, port, tmp):
    sys.path.insert(0, str(ROOT))
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank))
    torch.set_num_threads(1)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        for case, (max_norm, update_freq) in enumerate(((0.3, 1), (0.0, 1), (0.3, 2))):
            torch.manual_seed(5)
            model, criterion = Features(reducer=True), Head()
            torch.manual_seed(50 + rank)                                 # a head of its own on every rank: rank 0's is the one that counts
            with torch.no_grad():
                criterion.weight.add_(torch.randn(criterion.weight.shape) * (rank + 0.5))
                start = [p.detach().clone() for p in criterion.parameters()]
            data = batches(6)
            mine = [(x[4 * rank:4 * rank + 4], t[4 * rank:4 * rank + 4]) for x, t in data]
            got = _train(model, criterion, mine, max_norm, update_freq)
            other = got.clone()
            dist.broadcast(other, src=0)
            assert torch.equal(got, other), f"case {case}: the ranks differ by {float((got - other).abs().max())}"
            if rank == 0:
                torch.save((start, got), Path(tmp) / f"case{case}.pt")
    finally:
        dist.destroy_process_group()


def _alone(tmp):
    """one process, the whole batches, from rank 0's head"""
    sys.path.insert(0, str(ROOT))
    torch.set_num_threads(1)
    for case, (max_norm, update_freq) in enumerate(((0.3, 1), (0.0, 1), (0.3, 2))):
        start, got = torch.load(Path(tmp) / f"case{case}.pt", weights_only=True)
        torch.manual_seed(5)
        model, criterion = Features(), Head()
        with torch.no_grad():
            for p, v in zip(criterion.parameters(), start):
                p.copy_(v)
        want = _train(model, criterion, batches(6), max_norm, update_freq)
        # the same sums of fp32 numbers in another order: 6 steps of a few dozen terms
        assert torch.all((got - want).abs() <= 6 * 64 * 2.0 ** -24 * (1 + want.abs())), float((got - want).abs().max())


def test_a_head_in_the_criterion_trains_alike_on_two_ranks(tmp_path):
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    mp.spawn(_worker, args=(2, port, str(tmp_path)), nprocs=2, join=True)
    p = mp.get_context("spawn").Process(target=_alone, args=(str(tmp_path),))
    p.start()
    p.join()
    assert p.exitcode == 0
