"""The linear head's cross entropy (nnh_linear_cross_entropy_*) on the GPU against the formula in 64 bits, within the bounds of
its roundings."""
import math

import pytest
import torch

from lm_reference import assert_within, linear_cross_entropy

pytestmark = pytest.mark.gpu
T = {"f32": torch.float32, "bf16": torch.bfloat16}


def inputs(dtype, rows, D, V, bias, seed=0, skip=0.2, wide=1.0):
    gen = torch.Generator().manual_seed(seed)
    t = T[dtype]
    x = torch.randn(rows, D, generator=gen).to(t)
    w = (torch.randn(V, D, generator=gen) * (wide / math.sqrt(D))).to(t)
    targets = torch.randint(0, V, (rows,), generator=gen).int()
    targets[torch.rand(rows, generator=gen) < skip] = -1
    b = (torch.randn(V, generator=gen) * 0.5).to(t) if bias else None
    return x, w, targets, b


def check(dtype, rows, D, V, bias=False, reduction="mean", g=None, **more):
    import nnh
    print(dtype, rows, D, V, bias, reduction, flush=True)
    x, w, targets, b = inputs(dtype, rows, D, V, bias, **more)
    dev = [None if y is None else y.cuda() for y in (x, w, targets, b)]
    gd = None if g is None else g.cuda()
    want = linear_cross_entropy(x, w, targets, b, reduction, g)
    loss, lse = nnh.linear_cross_entropy_forward(*dev, reduction=reduction)
    assert_within(loss, want["loss"], "loss")
    assert_within(lse, want["lse"], "lse")
    got = nnh.linear_cross_entropy_backward(gd, dev[0], dev[1], dev[2], lse, dev[3], reduction)
    for name, y in zip(("dx", "dw", "db"), got):
        if y is not None:
            assert_within(y, want[name], name)
    want = linear_cross_entropy(x, w, targets, b, reduction, g, kept=True)
    got = nnh.linear_cross_entropy_train(*dev, reduction=reduction, g=gd)
    for name, y in zip(("loss", "dx", "dw", "db"), got):
        if y is not None:
            assert_within(y, want[name], "train " + name)


SHAPES = [(1, 1, 1), (1, 8, 2), (3, 64, 65), (130, 72, 300), (257, 128, 129), (64, 13, 1000), (100, 200, 511), (1000, 64, 64), (5, 256, 5000),
          (300, 33, 2049)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("bias", [False, True])
def test_shapes(gpu, dtype, shape, bias):
    check(dtype, *shape, bias=bias, skip=0.0 if shape[0] == 1 else 0.2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("given", [False, True])
def test_reductions(gpu, dtype, reduction, given):
    g = None
    if given:
        g = torch.randn(90, generator=torch.Generator().manual_seed(4)) if reduction == "none" else torch.tensor(-0.37)
    check(dtype, 90, 64, 333, bias=True, reduction=reduction, g=g)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_large_tiles(gpu, dtype):
    """Enough 256 x 256 tiles that the scores and dw take them, sizes that they do not divide; peaked scores."""
    check(dtype, 1111, 96, 12001, bias=True, wide=3.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_without_targets(gpu, dtype):
    """None at all: the mean is NaN, the sum 0, the gradients 0. A target past the vocabulary: a NaN loss, no gradient."""
    import nnh
    x, w, targets, b = (y.cuda() for y in inputs(dtype, 40, 24, 50, True))
    none = torch.full_like(targets, -1)
    for red in ("mean", "sum", "none"):
        loss, dx, dw, db = nnh.linear_cross_entropy_train(x, w, none, b, reduction=red)
        assert bool(torch.isnan(loss).all()) if red == "mean" else bool((loss == 0).all())
        assert not any(bool(y.any()) for y in (dx, dw, db))
    check(dtype, 40, 24, 50, True, skip=1.1, reduction="sum")
    past = targets.clone()
    past[3] = 50
    loss, lse = nnh.linear_cross_entropy_forward(x, w, past, b, reduction="none")
    assert bool(torch.isnan(loss[3])) and int(torch.isnan(loss).sum()) == 1 and bool(torch.isfinite(lse).all())
    dx, dw, db = nnh.linear_cross_entropy_backward(None, x, w, past, lse, b, reduction="none")
    assert not bool(dx[3].any())
    without = targets.clone()
    without[3] = -1
    for y, z in zip((dx, dw, db), nnh.linear_cross_entropy_backward(None, x, w, without, lse, b, reduction="none")):
        assert torch.equal(y, z)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_no_rows(gpu, dtype):
    import nnh
    x, w, targets = torch.zeros(0, 16, dtype=T[dtype], device="cuda"), torch.ones(20, 16, dtype=T[dtype], device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    loss, lse = nnh.linear_cross_entropy_forward(x, w, targets, reduction="sum")
    assert float(loss) == 0.0 and lse.shape == (0,)
    dx, dw, db = nnh.linear_cross_entropy_backward(None, x, w, targets, lse, w[:, 0].contiguous(), reduction="mean")
    assert dx.shape == (0, 16) and not bool(dw.any()) and not bool(db.any())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_that_are_not_finite(gpu, dtype):
    """A row without a target may hold anything: the gradients of the others and of the weight stay as they are. An infinite
    or NaN score in a row that counts makes that row's loss NaN."""
    import nnh
    x, w, targets, _ = (None if y is None else y.cuda() for y in inputs(dtype, 70, 32, 100, False))
    targets[5], targets[6] = -1, 7
    x[5] = 0
    want = nnh.linear_cross_entropy_train(x, w, targets, reduction="sum")
    lse = nnh.linear_cross_entropy_forward(x, w, targets, reduction="sum")[1]
    second = nnh.linear_cross_entropy_backward(None, x, w, targets, lse, reduction="sum")
    x[5, 3] = math.nan
    got = nnh.linear_cross_entropy_train(x, w, targets, reduction="sum")
    assert torch.equal(got[0], want[0])
    again = nnh.linear_cross_entropy_backward(None, x, w, targets, lse, reduction="sum")
    for y, z in ((got, want[1:3]), (again, second[:2])):
        for a, b in zip(y[1:3] if y is got else y[:2], z):
            assert torch.equal(a, b)
    assert not bool(got[1][5].any())
    x[5, 3] = 0.0
    x[6, 3] = math.nan
    loss, _ = nnh.linear_cross_entropy_forward(x, w, targets, reduction="none")
    assert bool(torch.isnan(loss[6])) and int(torch.isnan(loss).sum()) == 1


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_accumulation_and_leading_axes(gpu, dtype):
    import nnh
    x, w, targets, b = (y.cuda() for y in inputs(dtype, 96, 40, 77, True))
    want = linear_cross_entropy(x, w, targets, b, "sum", kept=True)
    old = [torch.randn_like(y.float()).to(y.dtype) for y in (x, w, b)]
    total = [y.clone() for y in old]
    x3, t3 = x.view(4, 24, 40), targets.view(4, 24)
    out = nnh.linear_cross_entropy_train(x3, w, t3, b, reduction="sum", dx=total[0].view(4, 24, 40), dx_first=False, dw=total[1],
                                         dw_first=False, db=total[2], db_first=False)
    assert out[1].shape == x3.shape
    u = torch.finfo(T[dtype]).eps / 2
    for name, was, now in zip(("dx", "dw", "db"), old, total):
        value, bound = want[name]
        was = was.double().cpu()
        assert_within(now.view_as(was), (value + was, bound + 2 * u * (value + was).abs() + u * bound), name)
    loss, lse = nnh.linear_cross_entropy_forward(x3, w, t3, b, reduction="none")
    assert loss.shape == lse.shape == (4, 24)


def test_views_that_are_not_aligned(gpu):
    """bf16 rows at odd addresses are copied first."""
    import nnh
    x, w, targets, _ = inputs("bf16", 50, 64, 90, False)
    want = linear_cross_entropy(x, w, targets, kept=True)

    def moved(y):
        room = torch.zeros(y.numel() + 1, dtype=y.dtype, device="cuda")
        room[1:] = y.flatten()
        return room[1:].view(y.shape)

    for a, b in ((moved(x), w.cuda()), (x.cuda(), moved(w)), (moved(x), moved(w))):
        dw = moved(torch.zeros_like(w))
        got = nnh.linear_cross_entropy_train(a, b, targets.cuda(), dw=dw)
        for name, y in zip(("loss", "dx", "dw"), got):
            assert_within(y, want[name], name)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_pieces(gpu, dtype):
    """So many rows that the vocabulary is cut: the backward in pieces of at most 1 GiB, the one call in more than the 4 GiB
    that it keeps. Rows repeat a few, so that the 64-bit form stays small: dw and db are those of the few, times their
    number."""
    import nnh
    rows, D, V, few = (2 ** 20 + 64, 16, 2111, 64)
    x, w, targets, b = inputs(dtype, few, D, V, True, skip=0.1)
    many = rows // few
    g = torch.full((), 1.0)
    want = linear_cross_entropy(x, w, targets, b, "sum", g, kept=True)
    dev = [y.cuda() for y in (x, w, targets, b)]
    X, Y = dev[0].repeat(many, 1), dev[2].repeat(many)
    loss, lse = nnh.linear_cross_entropy_forward(X, dev[1], Y, dev[3], reduction="none")
    assert torch.equal(lse.view(many, few), lse[:few].expand(many, few)) and torch.equal(loss.view(many, few), loss[:few].expand(many, few))
    assert_within(lse[:few], want["lse"], "lse")
    second = nnh.linear_cross_entropy_backward(None, X, dev[1], Y, lse, dev[3], reduction="sum")
    one = nnh.linear_cross_entropy_train(X, dev[1], Y, dev[3], reduction="sum")[1:]
    for got in (second, one):
        assert torch.equal(got[0].view(many, few, D), got[0][:few].expand(many, few, D))
        assert_within(got[0][:few], want["dx"], "dx")
        for name, y in (("dw", got[1]), ("db", got[2])):
            value, bound = want[name]
            # sums over `rows` terms instead of `few`: rows u32 of the terms' sizes, at most 1 |x| each
            size = x.double().abs().amax() if name == "dw" else 1.0
            extra = (rows + 8) * 2.0 ** -24 * (value.abs() + bound + few * 2.0 ** -7 * size / few)
            assert_within(y.double() / many, (value, bound + extra), name)


def test_capture(gpu):
    """Captured once with a workspace of its own and replayed on new inputs, with eager calls between; refused without one."""
    import nnh
    x, w, targets, b = (y.cuda() for y in inputs("bf16", 300, 64, 1000, True))
    size = nnh.workspace_size("linear_cross_entropy", nnh.BF16, 300, 64, 1000, 2, 1)
    room = torch.empty(size, dtype=torch.uint8, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    nnh.set_workspace(room, side)
    try:
        with torch.cuda.graph(graph, stream=side):
            got = nnh.linear_cross_entropy_train(x, w, targets, b)
        for seed in range(3):
            new = [y.cuda() for y in inputs("bf16", 300, 64, 1000, True, seed=seed)]
            for y, z in zip((x, w, targets, b), new):
                y.copy_(z)
            want = nnh.linear_cross_entropy_train(x, w, targets, b)
            graph.replay()
            torch.cuda.synchronize()
            for y, z in zip(got, want):
                assert torch.equal(y, z)
    finally:
        nnh.set_workspace(None, side)
    other = torch.cuda.CUDAGraph()
    with pytest.raises(nnh.NnhError, match="registered workspace"):
        with torch.cuda.graph(other, stream=side):
            nnh.linear_cross_entropy_train(x, w, targets, b)
