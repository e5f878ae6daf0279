"""Operators around a vocabulary, and clipping over many tensors: against plain forms in 64 bits on the CPU.

Tolerances count roundings: a value rounded to a type is off by at most finfo(type).eps / 2 of itself, an fp32 sum of n terms in any
order by at most n * 2^-24 of the sum of the terms' magnitudes."""
import math

import pytest
import torch

bf16, f16, f32, f64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
U32 = 2.0 ** -24


def _ops():
    from vision_transformers_torch_xla_amd import ops
    return ops


def _error():
    from vision_transformers_torch_xla_amd._lib import VitkError
    return VitkError


def half_ulp(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------------- clipping
def plain_clip(grads, max_norm):
    norm = math.sqrt(sum(float(g.double().pow(2).sum()) for g in grads))
    coef = max_norm / (norm + 1e-6)
    coef = 1.0 if coef > 1.0 else coef
    return norm, [g.double() * coef for g in grads]


def check_clipped(got, want):
    for g, w in zip(got, want):
        # fp32: the norm, norm + 1e-6, the quotient and the product are rounded (the quotient to an ulp), then the result's type
        assert torch.all((g.cpu().double() - w).abs() <= (6 * U32 + (half_ulp(g.dtype) if g.dtype != f32 else 0.0)) * w.abs() + (2.0 ** -25 if g.dtype == f16 else 2.0 ** -133 if g.dtype == bf16 else 1e-45))


@pytest.mark.gpu
@pytest.mark.parametrize("dtypes", [(f32,), (bf16,), (f16,), (f32, bf16, f16)])
@pytest.mark.parametrize("sizes", [(1,), (7, 0, 1, 8191, 8192, 8193), (64, 100000, 3), tuple(1 + 37 * i % 300 for i in range(300))])
@pytest.mark.parametrize("factor", [0.3, 3.0])
def test_clip_grads(device, dtypes, sizes, factor):
    ops = _ops()
    g = torch.Generator().manual_seed(len(sizes) * 10 + len(dtypes))
    grads = [torch.randn(n, generator=g).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]
    norm, _ = plain_clip(grads, 1.0)
    norm_, want = plain_clip(grads, factor * norm)
    dev = [t.to(device) for t in grads]
    got = ops.clip_grads(dev, None)
    assert got.shape == () and got.dtype == f32 and abs(got.item() - norm) <= 2 * U32 * norm
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, grads))
    out = [torch.full_like(t, 77.0) for t in dev]
    assert torch.equal(ops.clip_grads(dev, factor * norm, out=out), got)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, grads))
    check_clipped(out, want)
    assert torch.equal(ops.clip_grads(dev, factor * norm), got)
    assert all(torch.equal(a, b) for a, b in zip(dev, out))
    if factor > 1:
        assert all(torch.equal(a.cpu(), b) for a, b in zip(dev, grads))


@pytest.mark.gpu
def test_clip_grads_views_order_and_extremes(device):
    ops = _ops()
    flat = torch.randn(40000, generator=torch.Generator().manual_seed(1)).to(device)
    before = flat.clone()
    # a view that starts between 16-byte lines, a transposed (dense) one, a four-dimensional one with its dimensions in another order
    views = [flat[1:9001], flat[10000:22000].view(100, 120).t(), flat[22004:22004 + 3 * 4 * 5 * 6].view(3, 4, 5, 6).permute(0, 3, 1, 2)]
    norm, want = plain_clip([v.cpu() for v in views], 1.0)
    got = ops.clip_grads(views, 1.0)
    assert abs(got.item() - norm) <= 2 * U32 * norm
    check_clipped(views, want)
    for lo, hi in ((0, 1), (9001, 10000), (22000, 22004), (22364, 40000)):          # what lies between the views stays
        assert torch.equal(flat[lo:hi], before[lo:hi])
    # squares beyond the range of fp32, and far below it
    for scale in (3e30, 2e-30):
        t = torch.full((1000,), scale, device=device)
        assert abs(ops.clip_grads([t], None).item() / (scale * math.sqrt(1000)) - 1) <= 4 * U32
    t = torch.full((1000,), 3e30, device=device)
    ops.clip_grads([t], 1.0)
    assert torch.all((t * math.sqrt(1000) - 1).abs() <= 1e-6)
    # zeros; infinities and NaN spread as in torch
    z = torch.zeros(10, device=device)
    assert ops.clip_grads([z], 1.0).item() == 0.0 and torch.all(z == 0)
    a, b = torch.tensor([1.0, math.inf], device=device), torch.ones(3, device=device)
    assert ops.clip_grads([a, b], 1.0).item() == math.inf
    assert a[0] == 0 and torch.isnan(a[1]) and torch.all(b == 0)
    a, b = torch.tensor([1.0, math.nan], device=device), torch.ones(3, device=device)
    assert math.isnan(ops.clip_grads([a, b], 1.0).item()) and torch.isnan(a).all() and torch.isnan(b).all()
    b = torch.ones(3, device=device)
    ops.clip_grads([b], 0.0)
    assert torch.all(b == 0)
    e = torch.empty(0, device=device)
    assert ops.clip_grads([e], 1.0).item() == 0.0


@pytest.mark.gpu
def test_clip_grads_in_a_graph_on_another_stream(device):
    ops = _ops()
    grads = [torch.randn(n, device=device).to(dt) for n, dt in ((5000, f32), (777, bf16))]
    out = [torch.empty_like(t) for t in grads]
    ops.clip_grads(grads, 2.0, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grads(grads, 2.0, out=out)
    for k in range(3):
        for t in grads:
            t.copy_(torch.randn(t.shape, device=device) * (k + 1))
        graph.replay()
        want = [torch.empty_like(t) for t in grads]
        eager = ops.clip_grads(grads, 2.0, out=want)
        torch.cuda.synchronize()
        assert torch.equal(norm, eager) and all(torch.equal(a, b) for a, b in zip(out, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [torch.empty_like(t) for t in grads]
        n2 = ops.clip_grads(grads, 2.0, out=other)
    torch.cuda.synchronize()
    assert torch.equal(n2, eager) and all(torch.equal(a, b) for a, b in zip(other, want))


@pytest.mark.gpu
def test_clip_grads_offsets_past_32_bits(device):
    ops = _ops()
    n = (1 << 32) + 12345
    big, small = torch.full((n,), 0.5, dtype=bf16, device=device), torch.randn(1000, device=device)
    big[-5:] = 3.0
    before = small.clone()
    norm = ops.clip_grads([small, big], 100.0)
    want = math.sqrt(0.25 * (n - 5) + 45.0 + float(before.double().square().sum()))
    assert abs(norm.item() - want) <= 2 * U32 * want
    c = 100.0 / want
    assert torch.all((small.double() - before.double() * c).abs() <= 8 * U32 * before.double().abs() * c)
    for part, v in ((big[:1000], 0.5), (big[-1005:-5], 0.5), (big[-5:], 3.0)):
        assert torch.all((part.double() - v * c).abs() <= v * c * (half_ulp(bf16) + 8 * U32))


@pytest.mark.gpu
def test_clip_grads_of_lazy_clones(device):
    """a lazy clone that is written gets memory of its own: the original keeps its values"""
    ops = _ops()
    a, b = torch.randn(300, device=device), torch.randn(70, device=device)
    keep = [a.clone(), b.clone()]
    lazy = [torch._lazy_clone(a), torch._lazy_clone(b)]
    _, want = plain_clip([t.cpu() for t in keep], 1.0)
    ops.clip_grads(lazy, 1.0)                                                        # in place
    assert torch.equal(a, keep[0]) and torch.equal(b, keep[1])
    check_clipped(lazy, want)
    out = [torch._lazy_clone(a), torch._lazy_clone(b)]                               # outputs that share the gradients' own memory so far
    ops.clip_grads([a, b], 1.0, out=out)
    assert torch.equal(a, keep[0]) and torch.equal(b, keep[1])
    check_clipped(out, want)
    half = torch._lazy_clone(a)
    ops.clip_grads([half, b], 1.0, out=[half, out[1]])
    assert torch.equal(a, keep[0])
    check_clipped([half, out[1]], want)
    with pytest.raises(_error()):
        ops.clip_grads([a, a.view(300)], 1.0)
    assert torch.equal(a, keep[0])


@pytest.mark.gpu
def test_clip_grads_refuses(device):
    ops, err = _ops(), _error()
    a = torch.randn(64, device=device)
    for call in (lambda: ops.clip_grads([], 1.0),
                 lambda: ops.clip_grads([a, a], 1.0),                                    # scaled twice
                 lambda: ops.clip_grads([a[:40], a[30:]], 1.0),
                 lambda: ops.clip_grads([a], 1.0, out=[a[1:]]),
                 lambda: ops.clip_grads([a[:32], a[32:]], 1.0, out=[a[32:], a[:32]]),     # an output on another gradient
                 lambda: ops.clip_grads([a], 1.0, out=[]),
                 lambda: ops.clip_grads([a], 1.0, out=[torch.empty(64, device=device, dtype=bf16)]),
                 lambda: ops.clip_grads([a], None, out=[torch.empty_like(a)]),
                 lambda: ops.clip_grads([a], -1.0),
                 lambda: ops.clip_grads([a], math.nan),
                 lambda: ops.clip_grads([a.double()], 1.0),
                 lambda: ops.clip_grads([a[::2]], 1.0),
                 lambda: ops.clip_grads([a[:1].expand(8)], 1.0),
                 lambda: ops.clip_grads([a, torch.zeros(4)], 1.0),
                 lambda: ops.clip_grads(a, 1.0),
                 lambda: ops.clip_grads([a, 3.0], 1.0)):
        keep = a.clone()
        with pytest.raises(err):
            call()
        assert torch.equal(a, keep)


# ----------------------------------------------------------------------------------------------- embeddings
@pytest.mark.gpu
@pytest.mark.parametrize("T,V,D", [(1, 1, 8), (1, 1000, 768), (7, 33, 200), (1000, 50, 1024), (513, 100003, 64), (3, 5, 8200)])
@pytest.mark.parametrize("tt,ot", [(bf16, bf16), (f32, f32), (f32, bf16), (bf16, f32)])
@pytest.mark.parametrize("it", [torch.int64, torch.int32])
def test_embedding_fwd(device, T, V, D, tt, ot, it):
    ops = _ops()
    g = torch.Generator().manual_seed(T + V + D)
    table = torch.randn(V, D, generator=g).to(tt)
    ids = torch.randint(0, V, (T,), generator=g)
    scale = 0.37
    want = (table[ids].float() * torch.tensor(scale, dtype=f32)).to(ot)          # the kernel's own roundings: product in fp32, then the type
    got = ops.embedding_fwd(ids.to(device, it), table.to(device), scale=scale, out_dtype=ot)
    assert got.dtype == ot and torch.equal(got.cpu(), want)
    exact = table[ids].double() * scale
    assert torch.all((got.cpu().double() - exact).abs() <= (half_ulp(ot) + 2 * U32) * exact.abs())


@pytest.mark.gpu
def test_embedding_fwd_shapes_strides_and_bad_ids(device):
    ops = _ops()
    big = torch.randn(40, 64, device=device)
    table = big[:, 8:40]                                                           # rows with a stride, first column on a 16-byte line
    ids = torch.tensor([[3, 39, 0], [40, -1, 7]], device=device)
    got = ops.embedding_fwd(ids, table)
    assert got.shape == (2, 3, 32)
    assert torch.equal(got[0], table[ids[0]]) and torch.equal(got[1, 2], table[7]) and torch.isnan(got[1, :2]).all()
    assert torch.isnan(ops.embedding_fwd(torch.tensor([2 ** 40], device=device), table)).all()
    assert ops.embedding_fwd(torch.empty(0, 4, dtype=torch.int64, device=device), table).shape == (0, 4, 32)
    assert torch.equal(ops.embedding_fwd(ids.t(), table)[2, 1], table[7])          # ids in another order of dimensions
    assert ops.embedding_fwd(ids[0, 0], table).shape == (32,)


def plain_embedding_grad(dout, ids, V, scale, padding):
    ids = ids.reshape(-1).long()
    rows = dout.reshape(ids.numel(), -1).double()
    keep = (ids >= 0) & (ids < V) & (ids != (-1 if padding is None else padding))
    out, mag, count = (torch.zeros(V, rows.shape[1], dtype=f64), torch.zeros(V, rows.shape[1], dtype=f64), torch.zeros(V, 1, dtype=f64))
    out.index_add_(0, ids[keep], rows[keep])
    mag.index_add_(0, ids[keep], rows[keep].abs())
    count.index_add_(0, ids[keep], torch.ones(int(keep.sum()), 1, dtype=f64))
    return out * scale, mag * abs(scale), count


def check_embedding_grad(got, dout, ids, V, scale, padding, base=None):
    want, mag, count = plain_embedding_grad(dout, ids, V, scale, padding)
    if base is not None:
        want, mag = want + base.double(), mag + base.double().abs()
    # the fp32 sum of `count` terms, times the scale, plus what was there, then the type
    tol = (count + 3) * U32 * mag + (half_ulp(got.dtype) * 1.01 * want.abs() if got.dtype != f32 else 0.0)
    assert torch.all((got.cpu().double() - want).abs() <= tol)


EMB_IDS = {
    "uniform": lambda T, V, g: torch.randint(0, V, (T,), generator=g),
    "one": lambda T, V, g: torch.full((T,), V - 1),
    "hot": lambda T, V, g: torch.where(torch.rand(T, generator=g) < 0.5, torch.zeros(T, dtype=torch.int64), torch.randint(0, V, (T,), generator=g)),
    "bad": lambda T, V, g: torch.randint(-2, V + 2, (T,), generator=g),
}


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,D", [(1, 1, 8), (1, 1000, 768), (63, 2, 8), (65, 511, 72), (1025, 512, 64), (2049, 513, 200), (16384, 20000, 64), (16385, 700, 64),
                                   (5000, 262143, 16), (5000, 262144, 16), (5000, 262145, 16), (40000, 300, 2064), (50000, 4131, 24), (3000, 60, 256), (300000, 5000, 8)])
@pytest.mark.parametrize("kind", list(EMB_IDS))
def test_embedding_bwd(device, T, V, D, kind):
    ops = _ops()
    g = torch.Generator().manual_seed(T + V + D)
    ids = EMB_IDS[kind](T, V, g)
    dt = bf16 if kind in ("uniform", "hot") else f32
    dout = torch.randn(T, D, generator=g).to(dt)
    scale, padding = 1.7, (None if kind == "uniform" else V // 2)
    got = ops.embedding_bwd(dout.to(device), ids.to(device), V, scale=scale, padding_idx=padding)
    assert got.dtype == dt and got.shape == (V, D)
    check_embedding_grad(got, dout, ids, V, scale, padding)
    again = ops.embedding_bwd(dout.to(device), ids.to(device, torch.int32), V, scale=scale, padding_idx=padding)
    assert torch.equal(got, again)                                                  # no order of the hardware's in it


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,D", [(28672, 700, 40), (28673, 700, 40), (262144, 511, 8), (262145, 70000, 16), (1000003, 300001, 8)])       # on both sides of the borders: one launch, sort, sort with a scan; one pass and more
def test_embedding_bwd_of_very_many_tokens(device, T, V, D):
    ops = _ops()
    g = torch.Generator().manual_seed(T)
    ids = EMB_IDS["hot"](T, V, g)
    dout = torch.randn(T, D, generator=g)
    check_embedding_grad(ops.embedding_bwd(dout.to(device), ids.to(device), V, scale=-0.3, padding_idx=1), dout, ids, V, -0.3, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 9, 256, 257, 511, 512, 513, 682, 683, 1024, 1025])       # on both sides of the form for few tokens
@pytest.mark.parametrize("V,D", [(3, 8), (4099, 24), (40, 256), (700, 264), (90, 768), (100, 1032), (1, 16384), (300001, 8)])
def test_embedding_bwd_of_few_tokens(device, T, V, D):
    ops = _ops()
    g = torch.Generator().manual_seed(T * V)
    for kind, dt, ot in (("bad", f32, f32), ("hot", bf16, f32), ("one", f32, bf16), ("hot", bf16, bf16)):
        ids = EMB_IDS[kind](T, V, g)
        dout = torch.randn(T, D, generator=g).to(dt)
        out = torch.full((V, D), math.nan, dtype=ot, device=device)
        got = ops.embedding_bwd(dout.to(device), ids.to(device), V, scale=0.7, padding_idx=0 if kind == "hot" else None, out=out)
        check_embedding_grad(got, dout, ids, V, 0.7, 0 if kind == "hot" else None)
    base = torch.randn(V, D, generator=g)
    wide = torch.zeros(V, D + 8, device=device)
    wide[:, :D] = base.to(device)
    ops.embedding_bwd(dout.to(device), ids.to(device, torch.int32), V, out=wide[:, :D], accumulate=True)
    check_embedding_grad(wide[:, :D], dout, ids, V, 1.0, None, base=base)
    assert torch.all(wide[:, D:] == 0)


@pytest.mark.gpu
def test_embedding_bwd_without_tokens(device):
    ops = _ops()
    none = torch.empty(0, 8, device=device), torch.empty(0, dtype=torch.int64, device=device)
    for V in (1, 300000, 5000000):
        assert torch.all(ops.embedding_bwd(*none, V, out=torch.full((V, 8), 7.0, device=device)) == 0)
        assert torch.all(ops.embedding_bwd(*none, V, out=torch.full((V, 8), 7.0, device=device), accumulate=True) == 7.0)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [500, 20000])
def test_embedding_bwd_accumulates_into_a_part_of_a_buffer(device, T):
    ops = _ops()
    g = torch.Generator().manual_seed(T)
    V, D = 700, 40
    ids = torch.randint(0, 300, (T // 4, 4), generator=g) * 2
    dout = torch.randn(T // 4, 4, D + 8, generator=g).to(bf16)[..., :D]             # rows with a stride
    buf = torch.randn(V, D + 16, generator=g).to(device)
    before = buf.clone()
    out = buf[:, 8:8 + D]
    got = ops.embedding_bwd(dout.to(device), ids.to(device), V, scale=0.5, out=out, accumulate=True)
    assert got is out
    check_embedding_grad(out, dout, ids, V, 0.5, None, base=before[:, 8:8 + D].cpu())
    assert torch.equal(buf[:, :8], before[:, :8]) and torch.equal(buf[:, 8 + D:], before[:, 8 + D:])
    missed = torch.ones(V, dtype=torch.bool)
    missed[ids.reshape(-1)] = False
    assert torch.equal(out.cpu()[missed], before[:, 8:8 + D].cpu()[missed])
    whole = torch.full((V, D), 9.0, device=device)                                   # without accumulate everything is written
    ops.embedding_bwd(dout.to(device), ids.to(device), V, scale=0.5, out=whole)
    check_embedding_grad(whole, dout, ids, V, 0.5, None)
    none = ops.embedding_bwd(dout[:0].to(device), ids[:0].to(device), V)
    assert none.shape == (V, D) and torch.all(none == 0)
    assert torch.all(ops.embedding_bwd(dout[:0].to(device), ids[:0].to(device), 300000) == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("T,V", [(3000, 400), (30000, 400), (300, 400), (300000, 400)])
def test_embedding_bwd_in_a_graph(device, T, V):
    ops = _ops()
    ids = torch.randint(0, V, (T,), device=device)
    dout = torch.randn(T, 64, device=device, dtype=bf16)
    ops.embedding_bwd(dout, ids, V)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.embedding_bwd(dout, ids, V)
        out = ops.embedding_fwd(ids, got)
    for k in range(3):
        ids.copy_(torch.randint(0, V, (T,), device=device))
        dout.copy_(torch.randn(T, 64, device=device))
        graph.replay()
        want = ops.embedding_bwd(dout, ids, V)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(out, ops.embedding_fwd(ids, want))


@pytest.mark.gpu
def test_embedding_offsets_past_32_bits(device):
    ops = _ops()
    V, D, T = 3000001, 768, 3000                                                         # 4.6 GB of table, of its gradient
    table = torch.randn(V, D, device=device, dtype=bf16)
    ids = torch.randint(0, V, (T,), device=device)
    ids[:50] = V - 1
    assert torch.equal(ops.embedding_fwd(ids, table), table[ids])
    dout = torch.randn(T, D, device=device)
    got = ops.embedding_bwd(dout, ids, V, out_dtype=bf16)
    rows, where = torch.unique(ids, return_inverse=True)
    check_embedding_grad(got[rows], dout.cpu(), where.cpu(), len(rows), 1.0, None)
    assert torch.count_nonzero(got.abs().amax(1)) == len(rows)
    del got, dout
    dout = table                                                                         # as many tokens, into a small table
    ids = torch.randint(0, 500, (V,), device=device)
    got = ops.embedding_bwd(dout, ids, 500, out_dtype=f32)
    want, mag = (torch.zeros(500, D, dtype=f64, device=device) for _ in range(2))
    for i in range(0, V, 1 << 18):
        want.index_add_(0, ids[i:i + (1 << 18)], dout[i:i + (1 << 18)].double())
        mag.index_add_(0, ids[i:i + (1 << 18)], dout[i:i + (1 << 18)].double().abs())
    count = torch.bincount(ids, minlength=500).double()[:, None]
    assert torch.all((got.double() - want).abs() <= (count + 3) * U32 * mag)


@pytest.mark.gpu
def test_embedding_refuses(device):
    ops, err = _ops(), _error()
    table, ids, dout = torch.randn(10, 16, device=device), torch.zeros(4, dtype=torch.int64, device=device), torch.randn(4, 16, device=device)
    for call in (lambda: ops.embedding_fwd(ids.float(), table),
                 lambda: ops.embedding_fwd(ids.cpu(), table),
                 lambda: ops.embedding_fwd(ids, table.half()),
                 lambda: ops.embedding_fwd(ids, table, out_dtype=f16),
                 lambda: ops.embedding_fwd(ids, table[:, :12]),                       # D % 8
                 lambda: ops.embedding_fwd(ids, table[:, ::2]),
                 lambda: ops.embedding_fwd(ids, table[:, 1:9]),                       # rows off the 16-byte lines
                 lambda: ops.embedding_fwd(ids, table[:0]),                           # no rows
                 lambda: ops.embedding_bwd(dout, ids[:3], 10),
                 lambda: ops.embedding_bwd(dout, ids, 10, accumulate=True),
                 lambda: ops.embedding_bwd(dout, ids, 10, out=torch.empty(9, 16, device=device)),
                 lambda: ops.embedding_bwd(dout, ids, 10, out=torch.empty(10, 32, device=device)[:, :16]),    # a stride without accumulate
                 lambda: ops.embedding_bwd(dout, ids, 10, out=torch.empty(10, 16, device=device), out_dtype=bf16),
                 lambda: ops.embedding_bwd(dout, ids, 10, out_dtype=f16),
                 lambda: ops.embedding_bwd(dout[:, :12], ids, 10),
                 lambda: ops.embedding_bwd(dout.half(), ids, 10),
                 lambda: ops.embedding_bwd(dout, ids, 10, padding_idx=-1),
                 lambda: ops.embedding_bwd(dout, ids, 10, padding_idx=10),
                 lambda: ops.embedding_bwd(dout, ids, 0)):
        with pytest.raises(err):
            call()


# ------------------------------------------------------------------------------------ linear cross entropy
def plain_linear_xent(x, w, target, bias, smoothing, ignore, mean):
    """the operator in 64 bits, and how far bf16 / fp32 arithmetic may be off it: (loss, rows, dx, dw, db), (tolerances of the same)"""
    x, w = x.double(), w.double()
    V, D = w.shape
    b = torch.zeros(V, dtype=f64, device=w.device) if bias is None else bias.double()
    z = x @ w.t() + b
    counted = target != ignore
    bad = counted & ((target < 0) | (target >= V))
    t = torch.where(counted & ~bad, target, torch.zeros_like(target))
    q = torch.full_like(z, smoothing / V)
    q[torch.arange(len(t), device=t.device), t] += 1.0 - smoothing
    lse = torch.logsumexp(z, 1)
    smooth = smoothing * (lse - z.mean(1)) if smoothing > 0 else 0.0            # no 0 * inf where a class is masked out
    rows = (1.0 - smoothing) * (lse - z.gather(1, t[:, None])[:, 0]) + smooth
    rows[~counted] = 0.0
    rows[bad] = math.nan
    n = int(counted.sum())
    g = (1.0 / n if mean else 1.0) if n else 0.0
    loss = rows.sum() * g
    p = (z - lse[:, None]).exp()
    dz = p - q
    dz[~counted], p[~counted] = 0.0, 0.0
    # a logit is an fp32 sum of D products of bf16 factors, plus the bias
    zerr = ((D + 2) * U32 * (x.abs() @ w.abs().t() + torch.where(b.isinf(), torch.zeros_like(b), b.abs()))).max(1).values
    # its exponential: relative error of the argument's error and of the exponent's rounding; sums over at most V of them
    perr = 2 * zerr + (V / 64 + 200) * U32 * (1 + torch.where(lse.isfinite(), lse.abs(), torch.zeros_like(lse)))
    rtol = perr * (1 + smoothing)
    # the kept factor is fp16 relative to its piece's maximum, the gradient factor bf16
    E = p * (2.0 ** -11 + perr[:, None]) * 1.01 + 2.0 ** -24 + dz.abs() * 2.0 ** -8 * 1.01
    E[~counted] = 0.0
    dx, dw, db = g * (dz @ w), g * (dz.t() @ x), g * dz.sum(0)
    dxt = g * (E @ w.abs() + (V + 4) * U32 * (dz.abs() @ w.abs()))
    dwt = g * (E.t() @ x.abs() + (len(t) + 4) * U32 * (dz.abs().t() @ x.abs()))
    dbt = g * (E.sum(0) + (len(t) + 4) * U32 * dz.abs().sum(0))
    lt = rtol[counted].sum() * g + 4 * U32 * abs(loss)
    return (loss, rows, dx, dw, db), (lt, rtol, dxt, dwt, dbt)


def check_linear_xent(r, x, w, target, bias=None, smoothing=0.0, ignore=-100, mean=True, grad=True):
    want, tol = plain_linear_xent(x, w, target, bias, smoothing, ignore, mean)
    for name, got, v, t in zip(("loss", "rows", "dx", "dweight", "dbias"), r, want, tol):
        if not grad and name[0] == "d":
            assert got is None
            continue
        if name == "dbias" and bias is None:
            assert got is None
            continue
        got = got.to(v.device)
        extra = half_ulp(got.dtype) * 1.01 * (v.abs() + t) + (2.0 ** -133 if got.dtype == bf16 else 0.0)
        off = (got.double() - v).abs()
        bad = ~(off <= t + extra) & ~(got.double() == v)
        assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / (t + extra)).nan_to_num(9e9).max()):.3g} of its tolerance"


def xent_inputs(T, V, D, g, ignored=0.2, sharp=1.0):
    w = (torch.randn(V, D, generator=g) * (2.0 / math.sqrt(D))).to(bf16)
    target = torch.randint(0, V, (T,), generator=g)
    x = (torch.randn(T, D, generator=g) + sharp * w[target].float()).to(bf16)
    target[torch.rand(T, generator=g) < ignored] = -100
    return x, w, target


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,D", [(1, 1, 8), (1, 1000, 192), (3, 2, 16), (17, 63, 64), (64, 64, 72), (65, 257, 128), (255, 300, 136), (256, 256, 64), (257, 1023, 200),
                                   (300, 5000, 64), (700, 700, 384), (40, 33000, 64), (1500, 130, 1032)])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
@pytest.mark.parametrize("btype", [None, bf16, f32])
def test_linear_xent(device, T, V, D, smoothing, btype):
    ops = _ops()
    g = torch.Generator().manual_seed(T * 7 + V + D)
    x, w, target = xent_inputs(T, V, D, g)
    bias = None if btype is None else (torch.randn(V, generator=g) * 0.5).to(btype)
    args = (x.to(device), w.to(device), target.to(device), None if bias is None else bias.to(device))
    r = ops.linear_xent(*args, smoothing=smoothing)
    check_linear_xent(r, x, w, target, bias, smoothing)
    alone = ops.linear_xent(*args, smoothing=smoothing, want_grad=False)
    assert torch.equal(alone.loss, r.loss) and torch.equal(alone.rows, r.rows) and alone.dx is None
    again = ops.linear_xent(*args, smoothing=smoothing)
    assert all(a is None or torch.equal(a, b) for a, b in zip(again, r))
    s = ops.linear_xent(*args, smoothing=smoothing, reduction="sum", dweight_dtype=f32)
    assert s.dweight.dtype == f32
    check_linear_xent(s, x, w, target, bias, smoothing, mean=False)


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,D,block_bytes", [(1099, 24921, 424, 2 << 30), (8275, 8906, 392, 2 << 30), (8275, 8906, 392, 100 << 20), (16583, 8692, 168, 2 << 30),
                                               (1680, 21915, 720, 2 << 30), (6800, 6618, 2384, 2 << 30), (3615, 3627, 2240, 40 << 20), (8062, 7972, 2048, 2 << 30),
                                               (5225, 7940, 1896, 2 << 30)])
def test_linear_xent_large(device, T, V, D, block_bytes):
    """sizes that reach the large kernels: whole rounds of tiles, tiles cut into ranges of the contraction with and without whole rounds before
    them, tile columns in teams of 2 to 8, several blocks of rows; the plain form in 64 bits runs on the GPU"""
    ops = _ops()
    g = torch.Generator().manual_seed(T + V + D)
    x, w, target = (t.to(device) for t in xent_inputs(T, V, D, g))
    bias = (torch.randn(V, generator=g) * 0.5).to(device) if D % 16 else None
    smoothing = 0.1 if T % 2 else 0.0
    wtype = f32 if V % 2 else bf16
    r = ops.linear_xent(x, w, target, bias, smoothing=smoothing, dweight_dtype=wtype, block_bytes=block_bytes)
    check_linear_xent(r, x, w, target, bias, smoothing)
    again = ops.linear_xent(x, w, target, bias, smoothing=smoothing, dweight_dtype=wtype, block_bytes=block_bytes)
    assert all(a is None or torch.equal(a, b) for a, b in zip(again, r))
    alone = ops.linear_xent(x, w, target, bias, smoothing=smoothing, want_grad=False)
    assert torch.equal(alone.rows, r.rows)


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,D", [(3909, 8328, 432), (2534, 14114, 568), (6893, 5240, 600), (5541, 9060, 216)])      # logits by two kernels: split by classes, by rows
def test_linear_xent_logits_by_two_kernels(device, T, V, D):
    ops = _ops()
    g = torch.Generator().manual_seed(T + D)
    x, w, target = (t.to(device) for t in xent_inputs(T, V, D, g))
    check_linear_xent(ops.linear_xent(x, w, target), x, w, target)
    bias = (torch.randn(V, generator=g) * 0.5).to(bf16).to(device)
    r = ops.linear_xent(x, w, target, bias, smoothing=0.1)
    check_linear_xent(r, x, w, target, bias, 0.1)
    e = ops.linear_xent(x, w, target, bias, smoothing=0.1, want_grad=False)
    assert torch.equal(e.rows, r.rows) and torch.equal(e.loss, r.loss)
    few = ops.linear_xent(x[-100:], w, target[-100:], bias, smoothing=0.1, want_grad=False)       # the same rows by one kernel alone
    assert torch.equal(few.rows, r.rows[-100:])


@pytest.mark.gpu
@pytest.mark.parametrize("wtype", [bf16, f32])
def test_linear_xent_in_several_blocks_of_rows(device, wtype):
    ops = _ops()
    g = torch.Generator().manual_seed(5)
    x, w, target = xent_inputs(1300, 700, 72, g)
    bias = torch.randn(700, generator=g)
    args = (x.to(device), w.to(device), target.to(device), bias.to(device))
    whole = ops.linear_xent(*args, smoothing=0.1, dweight_dtype=wtype)
    for block_bytes in (1, 768 * 2 * 600):                  # 256 rows, 512 rows at a time
        r = ops.linear_xent(*args, smoothing=0.1, dweight_dtype=wtype, block_bytes=block_bytes)
        check_linear_xent(r, x, w, target, bias, 0.1)
        assert torch.equal(r.rows, whole.rows) and torch.equal(r.loss, whole.loss)
        e = ops.linear_xent(*args, smoothing=0.1, want_grad=False, block_bytes=block_bytes)
        assert torch.equal(e.rows, whole.rows) and torch.equal(e.loss, whole.loss)


@pytest.mark.gpu
def test_linear_xent_strides(device):
    ops = _ops()
    g = torch.Generator().manual_seed(6)
    x, w, target = xent_inputs(100, 300, 64, g)
    bx, bw = torch.full((100, 96), math.nan, dtype=bf16), torch.full((300, 80), math.nan, dtype=bf16)
    bx[:, 16:80], bw[:, 8:72] = x, w
    tg = torch.stack([target, target + 1], 1).to(device)[:, 0]
    r = ops.linear_xent(bx.to(device)[:, 16:80], bw.to(device)[:, 8:72], tg)
    check_linear_xent(r, x, w, target)
    assert all(torch.equal(a, b) for a, b in zip(r, ops.linear_xent(x.to(device), w.to(device), target.to(device))) if a is not None)


@pytest.mark.gpu
def test_linear_xent_rows_that_do_not_count_and_labels_that_are_none(device):
    ops = _ops()
    g = torch.Generator().manual_seed(7)
    x, w, target = xent_inputs(70, 500, 64, g)
    dev = lambda t: ops.linear_xent(x.to(device), w.to(device), t.to(device), ignore_index=3)          # noqa: E731
    target[target < 0] = 5
    target[10:40] = 3
    check_linear_xent(dev(target), x, w, target, ignore=3)
    nothing = dev(torch.full_like(target, 3))
    assert all(torch.all(t == 0) for t in (nothing.loss, nothing.rows, nothing.dx, nothing.dweight))
    bad = target.clone()
    bad[0], bad[1] = 500, -7
    r = dev(bad)
    ok = torch.ones(70, dtype=torch.bool)
    ok[:2] = False
    assert torch.isnan(r.loss) and torch.isnan(r.rows[:2]).all() and torch.isnan(r.dx[:2]).all() and torch.isnan(r.dweight).all()
    assert torch.equal(r.rows[2:], dev(target).rows[2:]) and torch.isfinite(r.dx[2:]).all() and torch.all(r.dx[10:40] == 0)
    one = ops.linear_xent(x[:0].to(device), w.to(device), target[:0].to(device))
    assert one.loss.item() == 0 and one.rows.shape == (0,) and one.dx.shape == (0, 64) and torch.all(one.dweight == 0)


@pytest.mark.gpu
def test_linear_xent_extreme_logits(device):
    ops = _ops()
    g = torch.Generator().manual_seed(8)
    x, w, target = xent_inputs(60, 400, 64, g, ignored=0.0)
    # classes that a bias masks out: with -inf, with the type's lowest value; whole pieces of 64 columns among them
    for low in (-math.inf, torch.finfo(f32).min):
        bias = torch.randn(400, generator=g)
        bias[64:200] = low
        t = target.clone()
        t[(t >= 64) & (t < 200)] = 1
        r = ops.linear_xent(x.to(device), w.to(device), t.to(device), bias.to(device))
        check_linear_xent(r, x, w, t, torch.where(bias < -1e30, torch.full_like(bias, -math.inf), bias))
        assert torch.all(r.dweight[64:200] == 0) and torch.all(r.dbias[64:200] == 0)
    # logits of thousands: one class has everything
    big = (x.float() * 40).to(bf16)
    r = ops.linear_xent(big.to(device), (w.float() * 40).to(bf16).to(device), target.to(device))
    check_linear_xent(r, big, (w.float() * 40).to(bf16), target)
    # equal logits everywhere
    zero = torch.zeros_like(x)
    r = ops.linear_xent(zero.to(device), w.to(device), target.to(device))
    check_linear_xent(r, zero, w, target)
    assert torch.all((r.rows - math.log(400)).abs() < 1e-5)
    # NaN and infinity in one row stay in that row (and in dweight)
    y = x.clone()
    y[3, 5] = math.nan
    y[4, 5] = math.inf
    r = ops.linear_xent(y.to(device), w.to(device), target.to(device))
    assert torch.isnan(r.rows[3:5]).all() and torch.isnan(r.loss) and torch.isnan(r.dx[3:5]).all()
    keep = [i for i in range(60) if i not in (3, 4)]
    clean = ops.linear_xent(x.to(device), w.to(device), target.to(device))
    assert torch.equal(r.rows[keep], clean.rows[keep]) and torch.equal(r.dx[keep], clean.dx[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,D", [(300, 200, 64), (1680, 21915, 72)])                   # logits by the small and by the large kernel
def test_linear_xent_gradient_of_classes_far_below_a_neighbour(device, T, V, D):
    """every class has a row of dweight and an entry of dbias of its own, in which no larger class stands beside it: a probability is held to so many
    bits of ITSELF, 40 powers of e below the largest of its neighbours too"""
    ops = _ops()
    g = torch.Generator().manual_seed(T)
    x, w = (torch.randn(T, D, generator=g) * 0.3).to(bf16).to(device), (torch.randn(V, D, generator=g) * 0.3).to(bf16).to(device)
    target = (torch.randint(64, V, (T,), generator=g)).to(device)                        # never one of the first 64 classes
    bias = torch.randn(V, generator=g)
    bias[0], bias[1:64] = 8.0, 8.0 - torch.linspace(2.0, 40.0, 63)
    bias = bias.to(device)
    r = ops.linear_xent(x, w, target, bias, reduction="sum", dweight_dtype=f32)
    z = x.double() @ w.double().t() + bias.double()
    lse = torch.logsumexp(z, 1)
    p = (z[:, :64] - lse[:, None]).exp()
    # as in plain_linear_xent, without anything that does not shrink with p
    zerr = ((D + 2) * U32 * (x.double().abs() @ w.double().abs().t() + bias.double().abs())).max()
    perr = 2 * zerr + (V / 64 + 200) * U32 * (1 + lse.abs().max())
    E = p * (2.0 ** -11 + 2.0 ** -8 + perr + (T + 4) * U32) * 1.01
    assert torch.all((r.dweight[:64].double() - p.t() @ x.double()).abs() <= E.t() @ x.double().abs())
    assert torch.all((r.dbias[:64].double() - p.sum(0)).abs() <= E.sum(0))
    assert float(p.sum(0)[63] / p.sum(0)[0]) < 1e-16 and torch.all(r.dbias[:64] > 0)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [2.0 ** 9, 2.0 ** 12, 2.0 ** 15])
def test_linear_xent_of_logits_of_millions(device, scale):
    """one class has everything, however large the logits: whole numbers here, so that fp32 holds them exactly"""
    ops = _ops()
    g = torch.Generator().manual_seed(3)
    x, w = torch.randint(-8, 9, (90, 64), generator=g).to(bf16), torch.randint(-8, 9, (300, 64), generator=g).to(bf16)
    x, w = (x * scale).to(device), (w * scale).to(device)                                # logits in units of scale^2 = 2^18 .. 2^30
    z = x.double() @ w.double().t()
    first, second = z.topk(2, 1).values.unbind(1)
    x, z = x[first > second], z[first > second]                                          # without ties
    assert len(x) > 60 and z.abs().max() < 2.0 ** 24 * scale ** 2
    target = z.argmax(1)
    target[::2] = 7
    r = ops.linear_xent(x, w, target, dweight_dtype=f32, reduction="sum")
    want = z.max(1).values - z.gather(1, target[:, None])[:, 0]
    assert torch.all((r.rows.double() - want).abs() <= 8 * U32 * z.abs().max())
    dz = torch.nn.functional.one_hot(z.argmax(1), 300).double() - torch.nn.functional.one_hot(target, 300).double()
    assert torch.equal(r.dweight.double(), dz.t() @ x.double())
    assert torch.equal(r.dx.double(), (dz @ w.double()).to(bf16).double())


@pytest.mark.gpu
@pytest.mark.parametrize("top", [65, 1000, 10000])
def test_linear_xent_loss_of_certain_rows(device, top):
    """the loss of a row does not know how large its logits are: log(1 + k e^-gap) to fp32's rounding of numbers near 1"""
    ops = _ops()
    V, D = 700, 64
    x, w = torch.zeros(40, D), torch.zeros(V, D)
    w[:, 0], w[:, 1] = 1.0, 0.0
    w[torch.arange(0, V, 5), 1] = 1.0                                                    # every fifth class is `gap` above the others
    gap = torch.arange(40) % 20
    x[:, 0], x[:, 1] = (top // 8) * 8 if top > 256 else top, gap
    w[333, 2], x[:, 2] = 1.0, 2.0 * gap                                                  # the target: as much again above those
    x, w = x.to(bf16).to(device), w.to(bf16).to(device)
    z = x.double() @ w.double().t()
    assert torch.equal(z, (x.float() @ w.float().t()).double())                          # whole numbers: nothing is rounded on the way
    target = torch.full((40,), 333, device=device)
    want = torch.log1p(((z - z[:, 333:334]).exp().sum(1) - 1.0))
    for smoothing in (0.0, 0.1):
        r = ops.linear_xent(x, w, target, smoothing=smoothing, want_grad=False)
        exact = (1 - smoothing) * want + smoothing * (want + z[:, 333] - z.mean(1))
        # the sum s: an exponential and its argument, V / 64 sums; its logarithm; with smoothing the mean, of the logits' size
        tol = (V / 64 + 16) * U32 * (1 + want) + smoothing * 16 * U32 * z.abs().max()
        assert torch.all((r.rows.double() - exact).abs() <= tol)
    # whatever the logits, no loss is negative
    g = torch.Generator().manual_seed(top)
    x, w = torch.randn(500, 64, generator=g).to(bf16).to(device), torch.randn(90, 64, generator=g).to(bf16).to(device)
    x = x * (top / 65.0)
    rows = ops.linear_xent(x, w, (x @ w.t()).argmax(1), want_grad=False).rows
    assert torch.all(rows >= 0) and (rows < 1e-3).any()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [2, 3, 6, 13])
@pytest.mark.parametrize("grad", [False, True])
def test_linear_xent_loss_of_few_classes(device, V, grad):
    """few terms to a sum: nothing averages a rounding out"""
    ops = _ops()
    g = torch.Generator().manual_seed(V)
    x, w = torch.zeros(400, 8), torch.zeros(V, 8)
    x[:, :3], w[:, :3] = torch.randint(-2, 3, (400, 3), generator=g).float(), torch.randint(-1, 2, (V, 3), generator=g).float()
    x, w = x.to(bf16).to(device), w.to(bf16).to(device)
    target = torch.randint(0, V, (400,), generator=g).to(device)
    r = ops.linear_xent(x, w, target, want_grad=grad)
    z = x.double() @ w.double().t()                                                      # whole numbers up to 6
    want = torch.logsumexp(z, 1) - z.gather(1, target[:, None])[:, 0]
    # exp(-d): the argument's rounding, d e^-d < 0.4, and the exponential's own ulp; the sum, its logarithm, ln 2, the result
    assert torch.all((r.rows.double() - want).abs() <= 8 * U32 * (1 + want))


@pytest.mark.gpu
def test_linear_xent_row_whose_mask_leaves_nothing(device):
    """every class masked out with the type's lowest value: equal logits, as a softmax has it; with -inf: NaN, as a softmax has it"""
    ops = _ops()
    g = torch.Generator().manual_seed(4)
    x, w, target = (t.to(device) for t in xent_inputs(50, 300, 64, g, ignored=0.0))
    r = ops.linear_xent(x, w, target, torch.full((300,), torch.finfo(f32).min, device=device))
    assert torch.all((r.rows - math.log(300)).abs() <= 8 * U32 * math.log(300))
    p = torch.full((50, 300), 1 / 300, dtype=f64, device=device) - torch.nn.functional.one_hot(target, 300).double()
    assert torch.all((r.dx.double() - p @ w.double() / 50).abs() <= (2.0 ** -11 + 2.0 ** -7) * 1.01 * (p.abs() @ w.double().abs() / 50))
    r = ops.linear_xent(x, w, target, torch.full((300,), -math.inf, device=device))
    assert torch.isnan(r.rows).all() and torch.isnan(r.dx).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,D,block_bytes", [(1, 1000, 192, 1 << 30), (70, 500, 64, 1 << 30), (700, 3000, 192, 1 << 30), (2050, 12001, 520, 1 << 30), (1500, 2000, 72, 1 << 20)])
def test_linear_xent_ignored_rows_may_hold_anything(device, T, V, D, block_bytes):
    ops = _ops()
    g = torch.Generator().manual_seed(T + V)
    x, w, target = (t.to(device) for t in xent_inputs(T, V, D, g, ignored=0.4))
    target[-1] = -100                                                                     # the last row of x too: short blocks repeat it
    bias = torch.randn(V, generator=g).to(device)
    dirty, clean = x.clone(), x.clone()
    ignored = target == -100
    dirty[ignored] = torch.tensor([math.nan, math.inf, -math.inf, 3e38], device=device).to(bf16).repeat(int(ignored.sum()), D // 4)
    clean[ignored] = 0.0
    for smoothing in (0.0, 0.1):
        got = ops.linear_xent(dirty, w, target, bias, smoothing=smoothing, dweight_dtype=f32, block_bytes=block_bytes)
        want = ops.linear_xent(clean, w, target, bias, smoothing=smoothing, dweight_dtype=f32, block_bytes=block_bytes)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.isfinite(t).all() for t in got) and torch.all(got.dx[ignored] == 0)
        check_linear_xent(want, clean, w, target, bias, smoothing)


@pytest.mark.gpu
def test_linear_xent_gradient_against_differences(device):
    ops = _ops()
    g = torch.Generator().manual_seed(9)
    x, w, target = xent_inputs(90, 310, 48, g)
    bias = torch.randn(310, generator=g)
    r = ops.linear_xent(x.to(device), w.to(device), target.to(device), bias.to(device), smoothing=0.1, dweight_dtype=f32)
    _, tol = plain_linear_xent(x, w, target, bias, 0.1, -100, True)
    loss = lambda a, b, c: plain_linear_xent(a, b, target, c, 0.1, -100, True)[0][0]            # noqa: E731
    h = 1e-5
    for k in range(3):
        args = [x.double(), w.double(), bias.double()]
        u = torch.randn(args[k].shape, generator=g, dtype=f64)
        up, down = list(args), list(args)
        up[k], down[k] = args[k] + h * u, args[k] - h * u
        slope = (loss(*up) - loss(*down)) / (2 * h)
        got = r[2 + k].cpu().double()
        # every element may be off by its own tolerance; the difference quotient of the 64-bit function by 1e-8
        allow = ((tol[2 + k] + half_ulp(r[2 + k].dtype) * (got.abs() + tol[2 + k])) * u.abs()).sum()
        assert abs((got * u).sum() - slope) <= allow + 1e-8
        assert allow < 0.2 * (got * u).abs().sum()                                             # the bound says something


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,D", [(3, 1 << 22, 8), (3000001, 2, 8), (1, 2, 2000), (4097, 1, 64)])
def test_linear_xent_longest_sides(device, T, V, D):
    ops = _ops()
    g = torch.Generator().manual_seed(T + V)
    x, w, target = (t.to(device) for t in xent_inputs(T, V, D, g))
    check_linear_xent(ops.linear_xent(x, w, target), x, w, target)


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,D", [(33000, 70001, 256), (600, 2200001, 1024)])           # probabilities, then weights and their gradient past 4 GiB
def test_linear_xent_offsets_past_32_bits(device, T, V, D):
    ops = _ops()
    x = torch.randn(T, D, device=device).to(bf16)
    w = (torch.randn(V, D, device=device) / math.sqrt(D)).to(bf16)
    target = torch.randint(0, V, (T,), device=device)
    r = ops.linear_xent(x, w, target, reduction="sum", block_bytes=8 << 30)
    k = 64
    rows = torch.cat([torch.arange(k), torch.arange(T - k, T)]).to(device)                # first and last rows of x, of the weight
    cols = torch.cat([torch.arange(k), torch.arange(V - k, V)]).to(device)
    lse = torch.full((T,), -math.inf, dtype=f64, device=device)
    dx = torch.zeros(2 * k, D, dtype=f64, device=device)
    step = max(1, (1 << 27) // T)
    for c in range(0, V, step):
        lse = torch.logaddexp(lse, torch.logsumexp(x.double() @ w[c:c + step].double().t(), 1))
    dxt = torch.zeros_like(dx)
    perr = 2 * (D + 2) * U32 * (x.abs().float().sum(1).max() * w.abs().max()).double() + (V / 64 + 200) * U32 * (1 + lse.abs().max())
    err = lambda p, dz: p * (2.0 ** -11 + perr) * 1.01 + 2.0 ** -24 + dz.abs() * 2.0 ** -8 * 1.01              # noqa: E731   (see plain_linear_xent)
    for c in range(0, V, 1 << 16):
        wd = w[c:c + (1 << 16)].double()
        p = (x[rows].double() @ wd.t() - lse[rows, None]).exp()
        dz = p - (target[rows, None] == torch.arange(c, c + len(wd), device=device)).double()
        dx += dz @ wd
        dxt += err(p, dz) @ wd.abs() + (V + 4) * U32 * (dz.abs() @ wd.abs())
    p = (x.double() @ w[cols].double().t() - lse[:, None]).exp()
    dz = p - (target[:, None] == cols).double()
    dw, dwt = dz.t() @ x.double(), err(p, dz).t() @ x.double().abs() + (T + 4) * U32 * (dz.abs().t() @ x.double().abs())
    nll = lse - (x.double() * w[target].double()).sum(1)
    assert torch.all((r.rows.double() - nll).abs() <= perr)
    for got, want, tol in ((r.dx[rows], dx, dxt), (r.dweight[cols], dw, dwt)):
        assert torch.all((got.double() - want).abs() <= tol + 2.0 ** -8 * 1.01 * (want.abs() + tol) + 2.0 ** -133)


@pytest.mark.gpu
def test_linear_xent_large_in_a_graph_and_on_two_streams_at_once(device):
    ops = _ops()
    g = torch.Generator().manual_seed(12)
    sets = [tuple(t.to(device) for t in xent_inputs(*shape, g)) for shape in ((2050, 12001, 520), (1100, 25000, 424))]
    eager = [ops.linear_xent(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    both = [[], []]
    for k in range(3):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                both[i].append(ops.linear_xent(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(u, v) for r in both[i] for u, v in zip(r, eager[i]) if u is not None)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    got = []
    for graph, s in zip(graphs, sets):
        with torch.cuda.graph(graph):
            got.append(ops.linear_xent(*s))
    for k in range(3):
        for s in sets:
            s[0].copy_(torch.randn(s[0].shape, generator=g))
        torch.cuda.synchronize()
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for r, s in zip(got, sets):
            assert all(torch.equal(u, v) for u, v in zip(r, ops.linear_xent(*s)) if u is not None)


@pytest.mark.gpu
def test_linear_xent_in_a_graph_on_another_stream(device):
    ops = _ops()
    g = torch.Generator().manual_seed(10)
    x, w, target = (t.to(device) for t in xent_inputs(600, 900, 64, g))
    ops.linear_xent(x, w, target)
    ops.linear_xent(x[:5], w, target[:5])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, few = ops.linear_xent(x, w, target), ops.linear_xent(x[:5], w, target[:5])
    side = torch.cuda.Stream()
    for k in range(3):
        a, _, c = xent_inputs(600, 900, 64, g)
        x.copy_(a), target.copy_(c)
        if k == 2:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
            torch.cuda.current_stream().wait_stream(side)
        else:
            graph.replay()
        want, want_few = ops.linear_xent(x, w, target), ops.linear_xent(x[:5], w, target[:5])
        torch.cuda.synchronize()
        assert all(u is None or torch.equal(u, v) for u, v in zip((*got, *few), (*want, *want_few)))


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,D,block_bytes", [(40, 500, 64, 1 << 30), (700, 3000, 192, 1 << 30), (2050, 12001, 520, 1 << 30), (1500, 2000, 72, 1 << 20)])
def test_linear_xent_some_of_the_gradients(device, T, V, D, block_bytes):
    ops = _ops()
    g = torch.Generator().manual_seed(T + V)
    x, w, target = (t.to(device) for t in xent_inputs(T, V, D, g))
    bias = torch.randn(V, generator=g).to(device)
    args = dict(smoothing=0.1, block_bytes=block_bytes)
    full = ops.linear_xent(x, w, target, bias, **args)
    check_linear_xent(full, x, w, target, bias, 0.1)
    for grads in ((), ("x",), ("weight",), ("bias",), ("x", "bias"), ("weight", "bias"), ["x", "weight"]):
        r = ops.linear_xent(x, w, target, bias, grads=grads, **args)
        assert torch.equal(r.loss, full.loss) and torch.equal(r.rows, full.rows)
        for name, got, want in (("x", r.dx, full.dx), ("weight", r.dweight, full.dweight), ("bias", r.dbias, full.dbias)):
            assert torch.equal(got, want) if name in grads else got is None
    head = w.float().requires_grad_(True)                               # frozen features, then a frozen head
    from vision_transformers_torch_xla_amd import losses
    losses.linear_cross_entropy(x, head, target, bias, smoothing=0.1).backward()
    assert close(head.grad, full.dweight.cpu(), 0.005)
    feats = x.clone().requires_grad_(True)
    losses.linear_cross_entropy(feats, w, target, bias, smoothing=0.1).backward()
    assert close(feats.grad, full.dx.cpu(), 0.005)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [300, 1024, 1025, 5000])
@pytest.mark.parametrize("V", [40, 1000, 3001])
def test_linear_xent_bias_gradient_keeps_the_hits(device, T, V):
    """1 - smoothing is no bf16 number: a hit must not be off by its rounding in the same direction every time"""
    ops = _ops()
    g = torch.Generator().manual_seed(T + V)
    x, w = (torch.randn(T, 64, generator=g) * 0.05).to(bf16), (torch.randn(V, 64, generator=g) * 0.05).to(bf16)
    target = torch.randint(0, 8, (T,), generator=g) * (V // 8)
    target[::7] = -100
    bias = torch.zeros(V)
    for reduction in ("sum", "mean"):
        r = ops.linear_xent(x.to(device), w.to(device), target.to(device), bias.to(device), smoothing=0.1, reduction=reduction, grads=("bias",))
        (_, _, _, _, db), _ = plain_linear_xent(x, w, target, bias, 0.1, -100, reduction == "mean")
        counted = target != -100
        p = torch.softmax(x[counted].double() @ w.double().t(), 1)
        n = int(counted.sum())
        # fp16 and bf16 roundings of what is not a hit, of the size of p; the sums
        tol = 1.01 * (2.0 ** -9 + 2.0 ** -8) * (p + 0.1 / V).sum(0) + n * 2.0 ** -24 + (n + 4) * U32 * (p.sum(0) + torch.bincount(target[counted], minlength=V))
        assert torch.all((r.dbias.cpu().double() - db).abs() <= tol * (1.0 / n if reduction == "mean" else 1.0))
        hit = db[target[counted][0]].abs()
        assert (tol * (1.0 / n if reduction == "mean" else 1.0)).min() < 0.0017 * hit or V == 40        # it would see 0.9 rounded to bf16


@pytest.mark.gpu
@pytest.mark.parametrize("T,V", [(2000, 3001), (900, 21843), (700, 100003)])
def test_linear_xent_smoothing_is_not_rounded_the_same_way_in_every_row(device, T, V):
    """1 - smoothing at the targets and smoothing / V at all other classes are no bf16 numbers (0.9 is off by 0.17 %, 0.1 / 21843 by 0.25 %): sums over many rows must
    not be off by the rounding of a constant"""
    ops = _ops()
    g = torch.Generator().manual_seed(V)
    D = 64
    x = (1.0 + 0.3 * torch.randn(T, D, generator=g)).to(bf16).to(device)                 # all of one sign: nothing averages out in dweight
    w = (torch.randn(V, D, generator=g) * 0.02).to(bf16).to(device)
    target = (torch.randint(0, 8, (T,), generator=g) * (V // 8)).to(device)
    bias = torch.zeros(V)
    never = torch.arange(1, V // 8)                                                      # classes of a probability of nothing: smoothing / V is all they get
    bias[never] = -60.0
    never, bias = never.to(device), bias.to(device)
    r = ops.linear_xent(x, w, target, bias, smoothing=0.1, reduction="sum", dweight_dtype=f32)
    X, W, u = x.double(), w.double(), 0.1 / V
    p = torch.softmax(X @ W.t() + bias.double(), 1)
    hits = torch.nn.functional.one_hot(target, V).double()
    dz = p - u - 0.9 * hits
    # as in plain_linear_xent, but at a target what is rounded is no constant: at most what stands there beside 0.9, p + u, is lost; and
    # what a class of no probability gets, u, is held to 2e-4 (of these three V: lx_factor, 8e-6, 1.1e-4 and 8e-7)
    E = (p * 2.0 ** -11 + (p - u).abs() * 2.0 ** -8) * 1.01 * (1 - hits) + (p + u) * hits + (T + 300) * U32 * dz.abs() + 2.0 ** -30 * p
    E[:, never] = 2e-4 * u
    for got, want, tol in ((r.dweight, dz.t() @ X, E.t() @ X.abs()), (r.dbias, dz.sum(0), E.sum(0))):
        assert torch.all((got.double() - want).abs() <= tol)
        hit = target.unique()
        assert (tol[hit] / want[hit].abs()).max() < 1.2e-3                               # it would see 0.9 rounded to bf16
    # dx: its own rounding to bf16 is as far and has either sign; over all T * D elements it leaves 2^-8 / sqrt(3 T D) < 1.1e-5 of their size (six times
    # that is allowed), a constant's rounding all of itself.  At the target p - u beside 0.9 is lost here too: of a want that is 0.9 of W's row, up to
    # the other classes' share, that is (p + u) / 0.9
    want = dz @ W
    lost = float((hits * (p + u)).sum(1).max()) / 0.9
    assert lost < 1.2e-3 and abs(float((r.dx.double() * want).sum() / (want * want).sum()) - 1) <= 6.6e-5 + 1.02 * lost


@pytest.mark.gpu
@pytest.mark.parametrize("smoothing", [1e-6, 0.5, 0.97, 1.0])
def test_linear_xent_any_smoothing(device, smoothing):
    ops = _ops()
    g = torch.Generator().manual_seed(2)
    x, w, target = xent_inputs(130, 333, 64, g)
    bias = torch.randn(333, generator=g)
    dev = [t.to(device) for t in (x, w, target, bias)]
    for reduction in ("mean", "sum"):
        r = ops.linear_xent(*dev, smoothing=smoothing, reduction=reduction, dweight_dtype=f32)
        check_linear_xent(r, x, w, target, bias, smoothing, mean=reduction == "mean")


@pytest.mark.gpu
def test_linear_xent_refuses(device):
    ops, err = _ops(), _error()
    x, w, t = torch.randn(6, 16, device=device).to(bf16), torch.randn(9, 16, device=device).to(bf16), torch.zeros(6, dtype=torch.int64, device=device)
    b = torch.zeros(9, device=device)
    for call in (lambda: ops.linear_xent(x.float(), w, t), lambda: ops.linear_xent(x, w.half(), t), lambda: ops.linear_xent(x, w, t.int()),
                 lambda: ops.linear_xent(x, w, t[:5]), lambda: ops.linear_xent(x, w[:, :8], t), lambda: ops.linear_xent(x[:, :12], w[:, :12], t),
                 lambda: ops.linear_xent(x, w, t, b[:8]), lambda: ops.linear_xent(x, w, t, b.half()), lambda: ops.linear_xent(x, w, t.cpu()),
                 lambda: ops.linear_xent(x, w, t, smoothing=1.5), lambda: ops.linear_xent(x, w, t, smoothing=math.nan),
                 lambda: ops.linear_xent(x, w, t, reduction="none"), lambda: ops.linear_xent(x, w, t, dweight_dtype=f16),
                 lambda: ops.linear_xent(x[:, ::2], w[:, ::2], t), lambda: ops.linear_xent(x[:, 1:9], w[:, 1:9], t), lambda: ops.linear_xent(x, w[:0], t),
                 lambda: ops.linear_xent(x, w, t, grads="x"), lambda: ops.linear_xent(x, w, t, grads=("x", "w")),
                 lambda: ops.linear_xent(x, w, t, block_bytes=0), lambda: ops.linear_xent(x[:1].expand(6, 16), w, t)):
        with pytest.raises(err):
            call()


@pytest.mark.gpu
def test_linear_xent_without_rows_checks_its_arguments(device):
    ops, err = _ops(), _error()
    x, w, t = torch.empty(0, 16, device=device, dtype=bf16), torch.zeros(9, 16, device=device, dtype=bf16), torch.empty(0, dtype=torch.int64, device=device)
    assert ops.linear_xent(x, w, t, smoothing=0.1).loss.item() == 0.0
    for kw in ({"smoothing": 1.5}, {"smoothing": math.nan}, {"smoothing": -0.1}, {"reduction": "none"}, {"block_bytes": 0}):
        with pytest.raises(err):
            ops.linear_xent(x, w, t, **kw)


# --------------------------------------------------------------------------------------- modules and the path
def close(got, want, rel):
    got, want = got.detach().double().cpu(), want.double()
    return float((got - want).norm() / want.norm()) <= rel


@pytest.mark.gpu
@pytest.mark.parametrize("wtype", [f32, bf16])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
def test_linear_cross_entropy_module(device, wtype, reduction):
    from vision_transformers_torch_xla_amd.losses import LinearCrossEntropy
    g = torch.Generator().manual_seed(3)
    torch.manual_seed(3)
    m = LinearCrossEntropy(64, 211, smoothing=0.1, ignore_index=-1, reduction=reduction).to(device)
    assert m.weight.dtype == f32 and m.weight.std() < 0.03 and torch.all(m.bias == 0)
    with torch.no_grad():
        m.weight.copy_(torch.randn(211, 64, generator=g) * 0.3)
        m.bias.copy_(torch.randn(211, generator=g))
    m = m.to(wtype)
    x = torch.randn(6, 20, 64, generator=g).to(device, bf16).requires_grad_(True)
    t = torch.randint(-1, 211, (6, 20), generator=g)
    loss = m(x, t.to(device))
    (3.0 * loss).backward()
    (want, _, dx, dw, db), (lt, _, dxt, dwt, dbt) = plain_linear_xent(x.detach().cpu().view(-1, 64), m.weight.detach().to(bf16).cpu(), t.view(-1),
                                                                     m.bias.detach().cpu(), 0.1, -1, reduction == "mean")
    assert abs(loss.item() - want) <= lt + U32 * abs(want)
    for got, v, tol in ((x.grad.view(-1, 64), dx, dxt), (m.weight.grad, dw, dwt), (m.bias.grad, db, dbt)):
        # the gradient and its product with the upstream 3 are rounded to the type
        assert torch.all((got.cpu().double() - 3 * v).abs() <= 3 * (tol + 2.02 * half_ulp(got.dtype) * (v.abs() + tol) + 1e-38))
        assert got.dtype == (bf16 if got.shape == x.grad.view(-1, 64).shape and got.data_ptr() == x.grad.data_ptr() else wtype)
    with torch.no_grad():
        assert torch.equal(m(x, t.to(device)), loss)
    again = m(x, t.to(device))
    again.backward(retain_graph=True)
    with pytest.raises(_error(), match="second time"):
        again.backward()


@pytest.mark.gpu
def test_upstream_scalar_is_not_rounded_to_the_gradients_type(device):
    from vision_transformers_torch_xla_amd import losses
    g = torch.Generator().manual_seed(13)
    x, w, t = (v.to(device) for v in xent_inputs(90, 50, 32, g))
    bias = torch.randn(50, generator=g).to(device, bf16)
    up = 1.0 + 2.0 ** -8 + 2.0 ** -9                                 # bf16 has 1 + 2^-7 for it
    want = _ops().linear_xent(x, w, t, bias)
    leaves = [v.clone().requires_grad_(True) for v in (x, w, bias)]
    (up * losses.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2])).backward()
    for leaf, v in zip(leaves, want[2:]):
        assert torch.equal(leaf.grad, (v.float() * up).to(bf16))


def test_upstream_scalar_is_multiplied_in_place():
    """a gradient of the weight's size is not held twice"""
    from vision_transformers_torch_xla_amd.losses import _times
    for g, go in ((torch.randn(8, 16), torch.tensor(0.7)), (torch.randn(40), torch.tensor(0.7, dtype=f64)), (torch.randn(40).to(bf16), torch.tensor(0.7))):
        want = (g.float() * go.float()).to(g.dtype)
        got = _times(g, go)
        assert got is g and torch.equal(g, want)
    assert _times(None, torch.tensor(2.0)) is None


@pytest.mark.gpu
def test_linear_cross_entropy_inputs_of_every_layout(device, monkeypatch):
    from vision_transformers_torch_xla_amd import losses
    g = torch.Generator().manual_seed(8)
    x, w, t = xent_inputs(24, 90, 32, g)
    dev = [v.to(device) for v in (x, w, t)]
    want = losses.linear_cross_entropy(*dev)
    # fp32 holders of the same values, rows with an odd stride, a start between 16-byte lines, columns first, one row for all
    odd = torch.zeros(24, 33, device=device, dtype=bf16)
    odd[:, 1:] = dev[0]
    line = torch.zeros(24 * 32 + 1, device=device)
    line[1:] = dev[0].float().reshape(-1)
    for v in (dev[0].float(), odd[:, 1:], line[1:].view(24, 32), dev[0].t().contiguous().t(), dev[0].view(4, 6, 32)):
        v.requires_grad_(True)
        got = losses.linear_cross_entropy(v, dev[1].float(), dev[2].view(v.shape[:-1]))
        assert torch.equal(got, want)
        got.backward()
        assert v.grad.shape == v.shape and v.grad.dtype == v.dtype
    row = dev[0][:1].detach().clone().requires_grad_(True)
    losses.linear_cross_entropy(row.expand(24, 32), dev[1], dev[2]).backward()
    (_, _, dx, _, _), (_, _, dxt, _, _) = plain_linear_xent(x[:1].expand(24, 32), w, t, None, 0.0, -100, True)
    # 24 gradients, each rounded to bf16, then torch's sum of them in bf16
    assert torch.all((row.grad.cpu().double() - dx.sum(0)).abs() <= dxt.sum(0) + 4 * 2.0 ** -8 * dx.abs().sum(0))
    empty = dev[0][:0].detach().requires_grad_(True)
    weight = dev[1].float().requires_grad_(True)
    losses.linear_cross_entropy(empty, weight, dev[2][:0]).backward()
    assert empty.grad.shape == (0, 32) and torch.all(weight.grad == 0)
    # the gradients are computed where somebody can ask for them, and only there
    asked = []
    real = losses.ops.linear_xent
    monkeypatch.setattr(losses.ops, "linear_xent", lambda *a, **k: (asked.append(k["want_grad"]), real(*a, **k))[1])
    losses.linear_cross_entropy(dev[0], dev[1], dev[2])
    losses.linear_cross_entropy(dev[0], weight, dev[2])
    with torch.no_grad():
        losses.linear_cross_entropy(dev[0], weight, dev[2])
    assert asked == [False, True, False]


@pytest.mark.gpu
def test_modules_in_a_graph(device):
    """forward and backward of lookup and loss captured and replayed; the eager graph of the same parameters is gone before the capture"""
    from vision_transformers_torch_xla_amd.embedding import TokenEmbedding
    from vision_transformers_torch_xla_amd.losses import LinearCrossEntropy
    torch.manual_seed(9)
    emb, head = TokenEmbedding(120, 32).to(device), LinearCrossEntropy(32, 120).to(device)
    with torch.no_grad():
        emb.weight.mul_(30), head.weight.mul_(30)
    params = [*emb.parameters(), *head.parameters()]
    ids, target = torch.randint(0, 120, (200,), device=device), torch.randint(0, 120, (200,), device=device)

    def step():
        for p in params:
            p.grad = None
        loss = head(emb(ids), target)
        loss.backward()
        return loss.detach()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(), step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    held = [p.grad for p in params]
    for k in range(3):
        ids.copy_(torch.randint(0, 120, (200,), device=device)), target.copy_(torch.randint(0, 120, (200,), device=device))
        graph.replay()
        got = [loss.clone(), *(h.clone() for h in held)]
        want = [step(), *(p.grad for p in params)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_token_embedding_module(device):
    from vision_transformers_torch_xla_amd.embedding import TokenEmbedding
    torch.manual_seed(4)
    m = TokenEmbedding(50, 16, scale=4.0, padding_idx=-1).to(device)
    assert torch.all(m.weight[49] == 0)
    with torch.no_grad():
        m.weight[49] = 1.0
    ids = torch.randint(0, 50, (7, 30), device=device)
    ids[0] = 49
    out = m(ids)
    assert out.dtype == bf16 and torch.equal(out, (m.weight.detach()[ids] * 4.0).to(bf16))
    up = torch.randn(7, 30, 16, device=device).to(bf16)
    out.backward(up)
    check_embedding_grad(m.weight.grad, up.cpu(), ids.cpu(), 50, 4.0, 49)
    assert torch.all(m.weight.grad[49] == 0)
    # a gradient that is one broadcast row
    m.weight.grad = None
    m(ids).sum().backward()
    check_embedding_grad(m.weight.grad, torch.ones(7, 30, 16), ids.cpu(), 50, 4.0, 49)


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [bf16, f32])
def test_token_embedding_backward_of_every_layout(device, out_dtype):
    """what autograd hands to the lookup's backward where the vectors are summed, averaged or joined with others"""
    from vision_transformers_torch_xla_amd.embedding import TokenEmbedding
    torch.manual_seed(7)
    m = TokenEmbedding(50, 16, scale=2.0, out_dtype=out_dtype).to(device)
    ids = torch.randint(0, 50, (30,), device=device)
    other = torch.ones(30, 3, device=device, dtype=out_dtype)
    up = torch.randn(30, 40, device=device).to(out_dtype)
    row = torch.randn(16, device=device).to(out_dtype)
    cases = {
        "summed over the tokens": (ids, lambda e: (e.sum(0), row), row.expand(30, 16)),
        "one sequence, summed": (ids[None], lambda e: (e.sum(1)[0], row), row.expand(30, 16)),
        "one sequence of several, summed": (ids.view(5, 6), lambda e: (e.sum(1), up[:5, :16]), up[:5, None, :16].expand(5, 6, 16)),
        "before others": (ids, lambda e: (torch.cat([e, other], 1), up[:, :19]), up[:, :16]),
        "behind others": (ids, lambda e: (torch.cat([other, e], 1), up[:, :19]), up[:, 3:19]),
        "one token, behind others": (ids[:1], lambda e: (torch.cat([other[:1], e], 1), up[:1, :19]), up[:1, 3:19]),
        "columns first": (ids, lambda e: (e.t(), up[:16, :30]), up[:16, :30].t()),
        "no token": (ids[:0], lambda e: (e.sum(0), row), row.expand(0, 16)),
    }
    for name, (i, use, dout) in cases.items():
        m.weight.grad = None
        out, v = use(m(i))
        out.backward(v)
        if i.numel() == 0:
            assert torch.all(m.weight.grad == 0)
        else:
            check_embedding_grad(m.weight.grad, dout.cpu(), i.cpu(), 50, 2.0, None)


def test_module_arguments_are_checked():
    from vision_transformers_torch_xla_amd.embedding import TokenEmbedding, embedding
    from vision_transformers_torch_xla_amd.losses import LinearCrossEntropy, linear_cross_entropy
    err = _error()
    w, i = torch.zeros(8, 16), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: TokenEmbedding(0, 16), lambda: TokenEmbedding(8, 12), lambda: TokenEmbedding(8, 16, padding_idx=8),
                 lambda: embedding(i, w, padding_idx=-9), lambda: embedding(i, w), lambda: LinearCrossEntropy(12, 8), lambda: LinearCrossEntropy(16, 0),
                 lambda: LinearCrossEntropy(16, 8, smoothing=2.0), lambda: LinearCrossEntropy(16, 8, reduction="none"),
                 lambda: linear_cross_entropy(torch.zeros(3, 16), w, i), lambda: linear_cross_entropy(torch.zeros(2, 16), w, i),
                 lambda: linear_cross_entropy(torch.zeros(3, 16, dtype=f64), w, i)):
        with pytest.raises(err):
            call()


@pytest.mark.gpu
def test_lookup_loss_clip_and_step_together(device):
    """one training step of the smallest model that has all of it: tokens -> table -> the same table as the head -> loss, the two gradients of
    the shared table, their common norm with a second parameter, the clipped step of the fused AdamW"""
    from vision_transformers_torch_xla_amd import engine, ops
    from vision_transformers_torch_xla_amd.embedding import embedding
    from vision_transformers_torch_xla_amd.losses import linear_cross_entropy
    g = torch.Generator().manual_seed(12)
    V, D, T = 300, 64, 500
    table = (torch.randn(V, D, generator=g) * 0.3).to(bf16).float()          # bf16 values, so that the plain form has the same products
    gain = torch.ones(D) * 1.5
    ids, target = torch.randint(0, V, (T,), generator=g), torch.randint(0, V, (T,), generator=g)
    target[::5] = -100

    p, q = torch.nn.Parameter(table.to(device)), torch.nn.Parameter(gain.to(device))
    x = embedding(ids.to(device), p, scale=2.0) * q                            # bf16 * fp32 -> fp32
    loss = linear_cross_entropy(x, p, target.to(device))
    loss.backward()
    norm = engine.clip_grad_norm_([p, [q], p], 0.05)                            # p is reached twice and counts once

    P, Q = table.double().requires_grad_(True), gain.double().requires_grad_(True)
    X = P[ids] * 2.0 * Q
    keep = target >= 0
    L = torch.nn.functional.cross_entropy(X[keep] @ P.t(), target[keep])
    L.backward()
    N = torch.sqrt(P.grad.pow(2).sum() + Q.grad.pow(2).sum())
    # x is rounded to bf16 before the products, its gradient and the loss factor too: three roundings of 2^-8 at most, incoherent
    tol = 3 * 2.0 ** -8
    assert abs(loss.item() - L.item()) <= 2 * 2.0 ** -8 * abs(L.item())
    assert abs(norm.item() / N.item() - 1) <= tol and N > 0.05
    coef = 0.05 / (N + 1e-6)
    assert close(p.grad, P.grad * coef, 2 * tol) and close(q.grad, Q.grad * coef, 2 * tol)
    clipped = math.sqrt(float(p.grad.double().pow(2).sum() + q.grad.double().pow(2).sum()))
    assert abs(clipped / 0.05 - 1) <= 1e-4
    m, v = torch.zeros_like(p.data), torch.zeros_like(p.data)
    before, grad = p.data.clone(), p.grad.clone()
    ops.adamw_step(p.data, grad, m, v, lr=0.1, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1)
    # the first step moves every weight with a gradient by lr against its sign
    big = grad.abs() > 1e-6
    assert torch.all((p.data - before)[big].sign() == -grad.sign()[big])


@pytest.mark.gpu
def test_clip_grad_norm_takes_modules_and_parameters(device):
    from vision_transformers_torch_xla_amd import engine
    from vision_transformers_torch_xla_amd.vit import create_model
    torch.manual_seed(5)
    lin = torch.nn.Linear(24, 40).to(device)
    other = torch.nn.Parameter(torch.zeros(33, device=device, dtype=bf16))
    unused = torch.nn.Parameter(torch.zeros(5, device=device))
    for t in (lin.weight, lin.bias, other):
        t.grad = torch.randn_like(t)
    want = [t.grad.double().cpu() for t in (lin.weight, lin.bias, other)]
    norm, clipped = plain_clip(want, 0.7)
    got = engine.clip_grad_norm_((lin, other, unused), 0.7)
    assert abs(got.item() - norm) <= 2 * U32 * norm
    check_clipped([lin.weight.grad, lin.bias.grad, other.grad], clipped)
    assert engine.clip_grad_norm_(unused, 1.0).item() == 0.0
    # a flat-buffer model beside a head with parameters of its own
    model = create_model("vit_tiny_patch16_224", num_classes=8, depth=1).to(device)
    flat = model._ensure_grad_buffer()
    flat.copy_(torch.randn(flat.shape, device=device))
    lin.weight.grad, lin.bias.grad = torch.randn_like(lin.weight), torch.randn_like(lin.bias)
    norm, clipped = plain_clip([flat.cpu(), lin.weight.grad.cpu(), lin.bias.grad.cpu()], 1.0)
    assert abs(engine.clip_grad_norm_([model, lin], 1.0).item() / norm - 1) <= 2 * U32
    check_clipped([flat, lin.weight.grad, lin.bias.grad], clipped)


@pytest.mark.gpu
def test_train_one_epoch_with_a_criterion_that_holds_the_head(device):
    from vision_transformers_torch_xla_amd import engine
    from vision_transformers_torch_xla_amd.embedding import TokenEmbedding
    from vision_transformers_torch_xla_amd.losses import LinearCrossEntropy
    torch.manual_seed(6)
    model, criterion = TokenEmbedding(100, 32).to(device), LinearCrossEntropy(32, 100).to(device)
    with torch.no_grad():
        model.weight.mul_(20)
        criterion.weight.mul_(20)
    opt = torch.optim.SGD([*model.parameters(), *criterion.parameters()], lr=0.5)
    data = [(torch.randint(0, 100, (64,)), torch.randint(0, 100, (64,))) for _ in range(3)]
    want_model, want_head = model.weight.detach().double().cpu(), criterion.weight.detach().double().cpu()
    bias = torch.zeros(100, dtype=f64)
    losses = []
    for ids, t in data:
        a, w, b = want_model.clone().requires_grad_(True), want_head.clone().requires_grad_(True), bias.clone().requires_grad_(True)
        loss = torch.nn.functional.cross_entropy(a[ids] @ w.t() + b, t)
        loss.backward()
        norm = math.sqrt(sum(float(v.grad.pow(2).sum()) for v in (a, w, b)))
        c = min(1.0, 0.1 / (norm + 1e-6))
        assert c < 1.0
        want_model, want_head, bias = (v.detach() - 0.5 * c * v.grad for v in (a, w, b))
        losses.append(loss.item())
    start = model.weight.detach().double().cpu()
    stats = engine.train_one_epoch(model, criterion, data, opt, device, 0, max_norm=0.1)
    assert "class_acc" not in stats and abs(stats["loss"] - sum(losses) / 3) <= 2 * 2.0 ** -8 * sum(losses) / 3
    # the weights have moved by three clipped steps of 0.05 in all; a step is off by a few roundings of 2^-8
    assert float((model.weight.detach().double().cpu() - want_model).norm()) <= 3 * 0.05 * 6 * 2.0 ** -8
    assert float((criterion.weight.detach().double().cpu() - want_head).norm()) <= 3 * 0.05 * 6 * 2.0 ** -8
    assert float((want_model - start).norm()) > 0.01


# --------------------------------------------------------------------------------------- checks without a GPU
def test_cpu_tensors_are_refused():
    ops, err = _ops(), _error()
    x = torch.zeros(4, 16)
    ids = torch.zeros(4, dtype=torch.int64)
    for call in (lambda: ops.clip_grads([x], 1.0), lambda: ops.embedding_fwd(ids, x), lambda: ops.embedding_bwd(x, ids, 4),
                 lambda: ops.linear_xent(x.to(bf16), x.to(bf16), ids)):
        with pytest.raises(err, match="GPU"):
            call()


def test_entry_points_check_before_they_launch():
    import ctypes as C
    from tests.test_abi_and_host import _lib
    lib = _lib().load()
    buf = C.create_string_buffer(65536)
    p = (C.cast(buf, C.c_void_p).value + 255) // 256 * 256
    one = lambda v, t: (t * 1)(v)          # noqa: E731
    src, n, ty = one(p, C.c_void_p), one(4, C.c_int64), one(0, C.c_int)
    need = lib.vitk_clip_grads_workspace(1)
    assert need > 0 and lib.vitk_clip_grads_workspace(300) > need and lib.vitk_clip_grads_workspace(-1) == 0
    assert lib.vitk_clip_grads(src, src, n, ty, 1, 1.0, p, p, 16, None) == -28
    assert lib.vitk_clip_grads(src, src, n, ty, 1, -1.0, p, p, need, None) == -22
    assert lib.vitk_clip_grads(src, src, n, one(3, C.c_int), 1, 1.0, p, p, need, None) == -22
    assert lib.vitk_clip_grads(one(p + 2, C.c_void_p), src, n, ty, 1, 1.0, p, p, need, None) == -22
    assert lib.vitk_clip_grads(src, src, one(-1, C.c_int64), ty, 1, 1.0, p, p, need, None) == -22
    assert lib.vitk_clip_grads(src, src, n, ty, 1, 1.0, None, p, need, None) == -22
    assert lib.vitk_embedding_fwd(p, 1, p, 0, 12, p, 0, 16, 4, 4, 12, 1.0, None) == -22 and b"multiples of 8" in lib.vitk_last_error()
    assert lib.vitk_embedding_fwd(p, 1, p, 2, 16, p, 0, 16, 4, 4, 16, 1.0, None) == -22
    assert lib.vitk_embedding_fwd(p, 1, p + 4, 0, 16, p, 0, 16, 4, 4, 16, 1.0, None) == -22
    assert lib.vitk_embedding_fwd(None, 1, None, 0, 16, None, 0, 16, 0, 4, 16, 1.0, None) == 0          # nothing to do
    need = lib.vitk_embedding_bwd_workspace(2000, 4, 16)
    assert need > 0 and lib.vitk_embedding_bwd(p, 0, 16, p, 1, p, 0, 16, 2000, 4, 16, 1.0, -1, 0, p, need - 1, None) == -28
    assert lib.vitk_embedding_bwd(p, 0, 16, p, 1, p, 0, 16, 2000, 4, 16, 1.0, -1, 0, None, need, None) == -22
    assert lib.vitk_embedding_bwd(p, 0, 16, p, 1, p, 0, 24, 4, 4, 16, 1.0, -1, 0, p, need, None) == -22
    assert lib.vitk_embedding_bwd(p, 0, 8, p, 1, p, 0, 16, 4, 4, 16, 1.0, -1, 0, p, need, None) == -22
    assert lib.vitk_embedding_bwd(None, 0, 16, p, 1, p, 0, 16, 4, 4, 16, 1.0, -1, 0, p, need, None) == -22
    need = lib.vitk_linear_xent_workspace(4, 4, 16, 1, 0, 0, 0, 1 << 20)

    def xent(x=p, ldx=16, w=p, V=4, D=16, eps=0.0, dx=p, dw=p, db=None, nbytes=need, T=4, ld=16):
        return lib.vitk_linear_xent(x, ldx, w, 16, None, 0, p, T, V, D, eps, -100, 1, p, p, dx, ld, dw, ld, 0, db, 0, p, nbytes, 1 << 20, None)
    assert need > 0 and lib.vitk_linear_xent_workspace(0, 4, 16, 1, 0, 0, 0, 1 << 20) == 0
    assert xent(nbytes=need - 1) == -28
    for kw in ({"x": None}, {"ldx": 12}, {"D": 12}, {"V": 0}, {"V": 1 << 23}, {"eps": -0.1}, {"eps": 1.1}, {"dx": None, "dw": None, "db": p}, {"db": p}, {"dx": p + 8}, {"dw": p + 8}, {"x": p + 8}, {"T": 0}, {"ld": 8}):
        assert xent(**kw) == -22, kw


def test_linear_xent_workspace_stays_within_its_blocks():
    from tests.test_abi_and_host import _lib
    size = _lib().load().vitk_linear_xent_workspace
    budget = 1 << 30
    for T, V, D in ((8192, 100003, 2048), (1 << 20, 100003, 64), (100352, 8192, 768), (1, 4000000, 8), (300, 1 << 22, 64)):
        n = size(T, V, D, 1, 1, 0, 0, budget)
        rows256 = 256 * ((V + 255) // 256 * 256) * 2.25
        other = 4 * V * D + 8 * 256 * 256 * max(1, D // 256) * 256                 # the fp32 sum of dw, the partial sums of dx
        assert n <= max(budget, rows256) + other + (1 << 20), (T, V, D, n)
