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


CASES = ((0.3, 1, False), (0.0, 1, False), (0.3, 2, False), (0.3, 1, True))          # max_norm, micro-steps to a step, a frozen weight


def _worker(rank, world, port, tmp):
    sys.path.insert(0, str(ROOT))
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank))
    torch.set_num_threads(1)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        for case, (max_norm, update_freq, frozen) in enumerate(CASES):
            torch.manual_seed(5)
            model, criterion = Features(reducer=True), Head()
            criterion.weight.requires_grad_(not frozen)
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
    for case, (max_norm, update_freq, frozen) in enumerate(CASES):
        start, got = torch.load(Path(tmp) / f"case{case}.pt", weights_only=True)
        torch.manual_seed(5)
        model, criterion = Features(), Head()
        criterion.weight.requires_grad_(not frozen)
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


# --------------------------------------------------------------------------------------------- the captured step
def test_a_step_with_parameters_in_the_criterion_is_not_captured(monkeypatch):
    from vision_transformers_torch_xla_amd import engine
    monkeypatch.setenv("VITK_GRAPH_STEP", "1")
    model = Features()
    model.begin_static_droppath = lambda *a: None
    head = Head()
    wanted = lambda c: engine.GraphedStep.wanted(model, 1, c)          # noqa: E731
    assert engine.GraphedStep.wanted(model, 1) and wanted(torch.nn.CrossEntropyLoss()) and wanted(torch.nn.functional.cross_entropy)
    assert not wanted(head) and not wanted(WithTemperature())
    for p in head.parameters():
        p.requires_grad_(False)
    assert wanted(head)


@pytest.mark.gpu
def test_vit_and_head_train_alike_with_and_without_the_graph_switch(device, monkeypatch):
    """a ViT whose outputs are the features, LinearCrossEntropy on them, clipping by the common norm, one fused AdamW over both: the same weights
    with VITK_GRAPH_STEP=1, after five steps; the head learns in every one of them"""
    from vision_transformers_torch_xla_amd import engine, optim_factory
    from vision_transformers_torch_xla_amd.losses import LinearCrossEntropy
    from vision_transformers_torch_xla_amd.vit import create_model
    monkeypatch.setenv("VITK_DROPPATH_COMPACT", "0")
    g = torch.Generator().manual_seed(2)
    data = [(torch.randn(8, 3, 224, 224, generator=g), torch.randint(0, 300, (8,), generator=g)) for _ in range(5)]

    class Args:
        opt, lr, weight_decay, opt_eps, opt_betas = "adamw", 1e-3, 0.05, 1e-8, None

    def run(flag):
        monkeypatch.setenv("VITK_GRAPH_STEP", flag)
        torch.manual_seed(5)
        model = create_model("vit_tiny_patch16_224", num_classes=64, global_pool="avg", drop_path_rate=0.1, depth=2).to(device)
        criterion = LinearCrossEntropy(64, 300, smoothing=0.1).to(device)
        opt = optim_factory.create_optimizer(Args, model)
        opt.add_param_group({"params": list(criterion.parameters()), "weight_decay": 0.0})
        seen, norms = [], []
        step, clip = opt.step, engine.clip_grad_norm_
        monkeypatch.setattr(opt, "step", lambda: (step(), seen.append(criterion.weight.detach().clone())))
        with monkeypatch.context() as m:
            m.setattr(engine, "clip_grad_norm_", lambda what, max_norm: norms.append(clip(what, max_norm)))
            engine.train_one_epoch(model, criterion, data, opt, device, 0, max_norm=0.05, update_freq=1, log_freq=1)
        torch.cuda.synchronize()
        return model._flat["p"].detach().clone(), seen, torch.stack(norms)

    before = engine.GraphedStep.total_replays
    with_flag, without = run("1"), run("0")
    assert engine.GraphedStep.total_replays == before
    assert torch.equal(with_flag[0], without[0]) and torch.equal(with_flag[2], without[2])
    assert all(torch.equal(a, b) for a, b in zip(with_flag[1], without[1]))
    assert len(without[1]) == 5 and all(not torch.equal(a, b) for a, b in zip(without[1], without[1][1:]))


@pytest.mark.gpu
def test_vit_features_and_head_gradients(device):
    """the gradients that the joined pair computes, against the formula on the features that the model gave"""
    from tests.test_vocab_ops import half_ulp, plain_linear_xent
    from vision_transformers_torch_xla_amd.losses import LinearCrossEntropy
    from vision_transformers_torch_xla_amd.vit import create_model
    torch.manual_seed(6)
    model = create_model("vit_tiny_patch16_224", num_classes=64, global_pool="avg", drop_path_rate=0.0, depth=2).to(device)
    criterion = LinearCrossEntropy(64, 211).to(device)
    with torch.no_grad():
        criterion.weight.mul_(20)
    x, t = torch.randn(8, 3, 224, 224, device=device), torch.randint(0, 211, (8,), device=device)
    t[2] = -100
    out = model(x)
    out.retain_grad()
    loss = criterion(out, t)
    loss.backward()
    (want, _, dx, dw, db), (lt, _, dxt, dwt, dbt) = plain_linear_xent(out.detach().to(torch.bfloat16), criterion.weight.detach().to(torch.bfloat16), t,
                                                                      criterion.bias.detach(), 0.0, -100, True)
    assert abs(loss.item() - want.item()) <= lt + 2.0 ** -24 * abs(want)
    for got, v, tol in ((out.grad, dx, dxt), (criterion.weight.grad, dw, dwt), (criterion.bias.grad, db, dbt)):
        # dx is rounded to bf16 on the way (the features are products' factors), whatever the features' type
        assert torch.all((got.double() - v).abs() <= tol + 1.01 * half_ulp(torch.bfloat16) * (v.abs() + tol) + 2.0 ** -133)
    flat = model._flat["g"].detach().clone()
    again = model(x)                                                     # the same gradient by hand through the model alone
    model.zero_grad()
    again.backward(out.grad)
    assert torch.equal(model._flat["g"], flat) and flat.abs().max() > 0


def _rccl_worker(rank, port, tmp):
    sys.path.insert(0, str(ROOT))
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK="0", WORLD_SIZE="1", LOCAL_RANK="0")
    torch.cuda.set_device(0)
    dev = torch.device("cuda", 0)
    from vision_transformers_torch_xla_amd.dp import GradReducer
    dist.init_process_group("nccl", rank=0, world_size=1, device_id=dev)
    try:
        red = GradReducer(lambda: None, single_rank_collectives=True)
        params = [torch.nn.Parameter(torch.randn(300, 64, device=dev)), torch.nn.Parameter(torch.randn(33, device=dev, dtype=torch.bfloat16)),
                  torch.nn.Parameter(torch.randn(5, device=dev))]
        for p in params[:2]:
            p.grad = torch.randn_like(p)
        keep = [(p.detach().clone(), None if p.grad is None else p.grad.clone()) for p in params]
        red.share(params)
        red.average(params)
        torch.cuda.synchronize()
        for p, (v, g) in zip(params, keep):                              # one rank: the average is the identity
            assert torch.equal(p, v) and (torch.equal(p.grad, g) if g is not None else torch.all(p.grad == 0))
        (Path(tmp) / "ok").write_text("ok")
    finally:
        dist.destroy_process_group()


@pytest.mark.gpu
def test_head_collectives_over_rccl(device, tmp_path):
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    port = s.getsockname()[1]
    s.close()
    mp.spawn(_rccl_worker, args=(port, str(tmp_path)), nprocs=1, join=True)
    assert (tmp_path / "ok").exists()


# -------------------------------------------------------------------------------------------- evaluation, checkpoints
@pytest.mark.gpu
@pytest.mark.parametrize("classes", [211, 300])
def test_evaluate_with_the_head_of_the_criterion(device, classes, monkeypatch):
    from vision_transformers_torch_xla_amd import engine
    from vision_transformers_torch_xla_amd.losses import LinearCrossEntropy
    from vision_transformers_torch_xla_amd.vit import create_model
    torch.manual_seed(7)
    model = create_model("vit_tiny_patch16_224", num_classes=64, global_pool="avg", drop_path_rate=0.0, depth=1).to(device).eval()
    head = LinearCrossEntropy(64, classes, smoothing=0.1).to(device)
    with torch.no_grad():
        head.weight.mul_(30), head.bias.normal_()
    data = [(torch.randn(n, 3, 224, 224), torch.randint(0, classes, (n,))) for n in (7, 8, 3)]
    data[1][1][2:5] = -100
    data[2][1][:] = -100                                                  # nothing counts in the last batch
    loss, top1, top5, n = 0.0, 0, 0, 0
    for x, t in data:
        with torch.no_grad():
            f = model(x.to(device)).to(torch.bfloat16).double()
        z = f @ head.weight.detach().to(torch.bfloat16).double().t() + head.bias.detach().double()
        keep = t != -100
        z, t = z.cpu()[keep], t[keep]
        if len(t):
            # fp32 sums of 64 products and the bias
            assert torch.all((head.logits(f.float()).cpu().double()[keep] - z).abs() <= 66 * 2.0 ** -24 * 64 * float(z.abs().max()))
            order = z.topk(5, 1).indices == t[:, None]
            loss += float(torch.nn.functional.cross_entropy(z, t, reduction="sum"))
            top1, top5, n = top1 + int(order[:, 0].sum()), top5 + int(order.sum()), n + len(t)
    for most in (1 << 28, 2 * classes):                                   # whole batches, two rows at a time
        with monkeypatch.context() as m:
            m.setattr(engine._by_head, "__defaults__", (most,))
            got = engine.evaluate(data, model, device, criterion=head)
        assert abs(got["loss"] - loss / n) <= 1e-4 * loss / n
        assert abs(got["acc1"] - 100.0 * top1 / n) < 1e-3 and abs(got["acc5"] - 100.0 * top5 / n) < 1e-3
    assert head.logits(torch.zeros(0, 64, device=device)).shape == (0, classes)
    from vision_transformers_torch_xla_amd._lib import VitkError
    with pytest.raises(VitkError, match="no target counts"):
        engine.evaluate(data[2:], model, device, criterion=head)
    with pytest.raises(VitkError):
        head.logits(torch.zeros(4, 32, device=device))


def test_the_head_of_the_criterion_is_saved_and_restored(tmp_path):
    import argparse

    from vision_transformers_torch_xla_amd import utils
    from vision_transformers_torch_xla_amd._lib import VitkError
    from vision_transformers_torch_xla_amd.losses import CrossEntropyLoss, LinearCrossEntropy
    args = lambda: argparse.Namespace(output_dir=str(tmp_path), auto_resume=True, resume="", start_epoch=0)          # noqa: E731

    def fresh(seed):
        torch.manual_seed(seed)
        model, head = torch.nn.Linear(8, 8), LinearCrossEntropy(8, 33)
        opt = torch.optim.AdamW([*model.parameters(), *head.parameters()], lr=0.1)
        for p in (*model.parameters(), *head.parameters()):
            p.grad = torch.randn_like(p)
        opt.step()
        return model, head, opt
    model, head, opt = fresh(0)
    utils.save_model(args(), 4, model, model, opt, None, criterion=head)
    assert set(torch.load(tmp_path / "checkpoint-4.pth", weights_only=True)["criterion"]) == {"weight", "bias"}
    model2, head2, opt2 = fresh(1)
    a = args()
    utils.auto_load_model(a, model2, model2, opt2, None, criterion=head2)
    assert a.start_epoch == 5 and torch.equal(head.weight, head2.weight) and torch.equal(head.bias, head2.bias) and torch.equal(model.weight, model2.weight)
    assert torch.equal(opt.state[head.weight]["exp_avg"], opt2.state[head2.weight]["exp_avg"])
    # a criterion without parameters: as before; a file without the head is refused before anything is changed
    utils.save_model(args(), 5, model, model, opt, None, criterion=CrossEntropyLoss())
    assert "criterion" not in torch.load(tmp_path / "checkpoint-5.pth", weights_only=True)
    model3, head3, opt3 = fresh(2)
    keep = model3.weight.detach().clone()
    with pytest.raises(VitkError, match="criterion"):
        utils.auto_load_model(args(), model3, model3, opt3, None, criterion=head3)
    assert torch.equal(model3.weight, keep)
    utils.auto_load_model(args(), model3, model3, opt3, None)
    assert torch.equal(model3.weight, model.weight)


@pytest.mark.gpu
def test_a_model_without_a_gradient_stays_out_of_the_common_norm(device):
    """zero_grad only marks the flat buffer; where the next step trains the head alone, the values of the step before are no part of its norm"""
    from vision_transformers_torch_xla_amd import engine
    from vision_transformers_torch_xla_amd.losses import LinearCrossEntropy
    from vision_transformers_torch_xla_amd.vit import create_model
    torch.manual_seed(8)
    model = create_model("vit_tiny_patch16_224", num_classes=64, global_pool="avg", drop_path_rate=0.0, depth=1).to(device)
    head = LinearCrossEntropy(64, 50).to(device)
    x, t = torch.randn(4, 3, 224, 224, device=device), torch.randint(0, 50, (4,), device=device)
    of = lambda *ts: float(torch.sqrt(sum(v.double().square().sum() for v in ts)))          # noqa: E731
    for set_to_none in (True, False):
        head.zero_grad()
        head(model(x), t).backward()
        flat = model._flat["g"].clone()
        own = [p.grad.clone() for p in head.parameters()]
        assert abs(engine.clip_grad_norm_([model, head], 1e9).item() / of(flat, *own) - 1) < 1e-6
        model.zero_grad(set_to_none)
        head.zero_grad()
        with torch.no_grad():
            f = model(x)
        head(f, t).backward()                                            # linear probing
        own = [p.grad.clone() for p in head.parameters()]
        norm = engine.clip_grad_norm_([model, head], 0.5 * of(*own))
        assert abs(norm.item() / of(*own) - 1) < 1e-6 and abs(of(*(p.grad for p in head.parameters())) / (0.5 * of(*own)) - 1) < 1e-5
        assert torch.equal(model._flat["g"], flat)
    for p in model.parameters():                                         # a foreign optimizer's zero_grad
        p.grad = None
    assert abs(engine.clip_grad_norm_([model, head], 1e9).item() / of(*(p.grad for p in head.parameters())) - 1) < 1e-6
