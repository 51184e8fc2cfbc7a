"""The linear head's cross entropy on the GPU where its gradients' products take another path than at small sizes, against the formula in
64 bits: tiles of 256 x 256 (from 200 of them on, or in runs of the depth that make up for fewer), runs of 128 x 128 ones, rows that
are stored whole or not."""
import pytest
import torch

from lm_reference import assert_within, linear_cross_entropy
from test_linear_cross_entropy_gpu import T, check, inputs

pytestmark = pytest.mark.gpu


def tiles(inner, outer, side):
    return -(-inner // side) * -(-outer // side)


@pytest.mark.parametrize("D", [1032, 1030])
@pytest.mark.parametrize("bias", [False, True])
def test_large_gradient_tiles(gpu, D, bias):
    """dw takes 255 tiles of 256 x 256, stored in whole rows where they are multiples of 16 bytes; dx ten of them in 25 runs of the
    vocabulary. Peaked scores."""
    rows, V = 500, 12900
    assert tiles(D, V, 256) >= 200 and tiles(D, rows, 256) * min(-(-256 // tiles(D, rows, 256)), V // 512) >= 192
    check("bf16", rows, D, V, bias=bias, wide=2.0)


@pytest.mark.parametrize("D", [1032, 1030])
def test_large_gradient_tiles_added(gpu, D):
    import nnh
    rows, V = 500, 12900
    x, w, targets, b = (y.cuda() for y in inputs("bf16", rows, D, V, True))
    want = linear_cross_entropy(x, w, targets, b, "sum", kept=True)
    old = [torch.randn_like(y.float()).bfloat16() for y in (x, w, b)]
    total = [y.clone() for y in old]
    nnh.linear_cross_entropy_train(x, w, targets, b, reduction="sum", dx=total[0], dx_first=False, dw=total[1], dw_first=False, db=total[2],
                                   db_first=False)
    u = torch.finfo(torch.bfloat16).eps / 2
    for name, was, now in zip(("dx", "dw", "db"), old, total):
        value, bound = want[name]
        was = was.double().cpu()
        assert_within(now, (value + was, bound + 2 * u * (value + was).abs() + u * bound), name)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,D,V", [(5000, 64, 300), (5003, 40, 77), (70, 520, 9001)])
def test_gradients_in_runs(gpu, dtype, rows, D, V):
    """Few tiles over many rows (dw) or words (dx): the depth in runs, rows without a target among them."""
    check(dtype, rows, D, V, bias=True, reduction="sum")


@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_a_large_vocabulary_in_32_bits(gpu, reduction):
    check("f32", 90, 72, 50257, bias=True, reduction=reduction, wide=3.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_without_targets_in_runs(gpu, dtype):
    """Whole runs of rows without a target, whose values are not finite."""
    import nnh
    x, w, targets, _ = inputs(dtype, 5000, 64, 300, False)
    targets[600:2900] = -1
    want = linear_cross_entropy(x, w, targets, None, "sum", kept=True)
    x[600:2900] = float("nan")
    x, w, targets = x.cuda(), w.cuda(), targets.cuda()
    loss, dx, dw, _ = nnh.linear_cross_entropy_train(x, w, targets, reduction="sum")
    for name, y in (("loss", loss), ("dx", dx), ("dw", dw)):
        assert_within(y, want[name], name)
    lse = nnh.linear_cross_entropy_forward(x, w, targets, reduction="sum")[1]
    dx, dw, _ = nnh.linear_cross_entropy_backward(None, x, w, targets, lse, reduction="sum")
    for name, y in (("dx", dx), ("dw", dw)):
        assert_within(y, want[name], name)
    assert T[dtype] == dw.dtype
