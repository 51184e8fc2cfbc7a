"""Linears in 8-bit integers on the GPU: codes and scales exactly, products within the roundings of their scales."""
import math

import pytest
import torch

from lm_reference import assert_within
from serving_reference import T, codes_of, draw, linear_int8

pytestmark = pytest.mark.gpu


def weight(seed, V, D):
    """Codes at a pitch that is a multiple of 16, what is behind a row's codes not zero."""
    gen = torch.Generator().manual_seed(seed)
    w = torch.randint(-128, 128, (V, -(-D // 16) * 16), generator=gen, dtype=torch.int8)
    return w, torch.rand(V, generator=gen) / (64 * math.sqrt(max(1, D)))


def check(dtype, rows, D, V, bias=True, seed=0):
    import nnh
    print(dtype, rows, D, V, bias, flush=True)
    t = T[dtype]
    x = draw(seed, rows, D, dtype=t) * torch.exp(draw(seed + 1, rows, 1)).to(t)
    w, s = weight(seed + 2, V, D)
    b = draw(seed + 3, V, dtype=t) if bias else None
    y = nnh.linear_int8(x.cuda(), w.cuda()[:, :D], s.cuda(), None if b is None else b.cuda())
    assert_within(y, linear_int8(x, w[:, :D], s, b), "y")


SHAPES = [(1, 1, 1), (1, 16, 16), (1, 4096, 100), (3, 100, 33), (16, 64, 64), (17, 1000, 257), (32, 48, 130), (33, 65, 17), (64, 2047, 129), (65, 64, 64), (100, 1000, 257),
          (130, 33, 130), (257, 129, 300), (65, 5000, 64), (300, 4096, 520), (2, 8192, 8200), (20, 300, 16400), (70, 131, 1), (2, 4000, 300), (4, 4080, 33), (4, 4081, 33), (16, 960, 16384), (5, 1000, 8200), (1, 16300, 20), (3, 5, 16385),
          (24, 130, 5000), (40, 200, 5000), (50, 130, 9000), (64, 65, 16384), (64, 65, 16385), (32, 40, 40000)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("bias", [True, False])
def test_shapes(gpu, dtype, shape, bias):
    check(dtype, *shape, bias=bias)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,V", [(1000, 300), (200, 9000), (130, 17000)])
def test_rows_by_themselves(gpu, dtype, D, V):
    """A row's result does not depend on what it is computed with: whole, few rows' and tiles' forms give the same bits."""
    import nnh
    x = (draw(1, 200, D, dtype=T[dtype]) * torch.exp(draw(2, 200, 1)).to(T[dtype])).cuda()
    w, s = weight(3, V, D)
    w, s, b = w.cuda()[:, :D], s.cuda(), draw(4, V, dtype=T[dtype]).cuda()
    all_rows = nnh.linear_int8(x, w, s, b)
    for rows in (1, 7, 16, 17, 32, 40, 64, 65):
        assert torch.equal(nnh.linear_int8(x[100:100 + rows], w, s, b), all_rows[100:100 + rows]), rows


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [16384, 16383])
def test_large_tiles(gpu, dtype, V):
    """256 x 256 tiles, with a last one seen in part, and several stages of depth."""
    check(dtype, 850, 1100, V)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [1, 7, 8, 16, 100, 1000, 1024, 1032, 1030, 5000])
@pytest.mark.parametrize("rows", [1, 5, 300])
def test_codes(gpu, dtype, D, rows):
    import nnh
    x = draw(D, rows, D, dtype=T[dtype])
    for pitch in (D, -(-D // 16) * 16, D + 29):
        codes = torch.full((rows, pitch), 77, dtype=torch.int8, device="cuda")
        nnh.quantize_rows(x.cuda(), codes=codes[:, :D])
        want, scale = codes_of(x)
        got, s = nnh.quantize_rows(x.cuda())
        assert torch.equal(s.cpu(), scale)
        assert torch.equal(got.cpu().double(), want) and torch.equal(codes[:, :D].cpu().double(), want)
        assert bool((codes[:, D:] == 77).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_borders_between_codes(gpu, dtype):
    """Values half way between two codes go to the even one, values next to that to their own side; codes stay within 127."""
    import nnh
    t = T[dtype]
    scales = [1.0, 0.0078125, 3.0, 1 / 3, 2.0 ** -120, 2.0 ** -126, 2.0 ** -140, 1.7e38 / 127, 0.1]
    rows = []
    for s in scales:
        top = torch.tensor(127.0 * s).to(t)
        unit = (top.float() / 127).double()
        half = ((torch.arange(-127, 127) + 0.5).double() * unit).to(t)
        near = [half, torch.nextafter(half, torch.full_like(half, math.inf)), torch.nextafter(half, torch.full_like(half, -math.inf))]
        rows.append(torch.cat([top.reshape(1), -top.reshape(1)] + [x[x.abs() <= top] for x in near]))
    n = min(r.numel() for r in rows)
    x = torch.stack([r[:n] for r in rows])
    got, s = nnh.quantize_rows(x.cuda())
    want, scale = codes_of(x)
    assert torch.equal(s.cpu(), scale) and torch.equal(got.cpu().double(), want)
    tiny = torch.full((3, 20), 0.0).float()
    tiny[0, 3], tiny[1, 4], tiny[1, 5], tiny[2, 0] = 2.0 ** -149, 190 * 2.0 ** -149, -64 * 2.0 ** -149, 2.0 ** -126
    got, s = nnh.quantize_rows(tiny.cuda())
    want, scale = codes_of(tiny)
    assert torch.equal(s.cpu(), scale) and torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [3, 70])
def test_not_finite(gpu, dtype, rows):
    """A row with an infinity or NaN gives NaN, a row of zeros the bias; the others are not touched."""
    import nnh
    t = T[dtype]
    x = draw(0, rows, 100, dtype=t)
    x[0, 99], x[1] = math.inf, 0
    x[2, 3] = math.nan
    w, s = weight(1, 40, 100)
    b = draw(2, 40, dtype=t)
    y = nnh.linear_int8(x.cuda(), w.cuda()[:, :100], s.cuda(), b.cuda()).cpu()
    assert y[0].isnan().all() and y[2].isnan().all() and torch.equal(y[1], b)
    value, bound = linear_int8(x, w[:, :100], s, b)
    assert_within(y[3:], (value[3:], bound[3:]), "y")
    codes, scale = nnh.quantize_rows(x.cuda())
    assert scale[:3].isnan().tolist() == [True, False, True] and bool((codes[:3] == 0).all())


def test_full_range(gpu):
    """The largest sums that 32 bits hold: 131071 products of -128 and 127."""
    import nnh
    D = 131071
    for rows in (1, 65):
        x = torch.full((rows, D), -127.0)
        x[:, ::2] = 127.0
        w = torch.full((3, D + 1), -128, dtype=torch.int8)
        w[1, ::2] = 127
        w[2] = 127
        y = nnh.linear_int8(x.cuda(), w.cuda()[:, :D], torch.ones(3).cuda())
        assert_within(y, linear_int8(x, w[:, :D], torch.ones(3)), "y")
        x[:] = 127.0
        y = nnh.linear_int8(x.cuda(), w.cuda()[:, :D], torch.ones(3).cuda())
        assert y[0, 0].item() == float(torch.tensor(-127.0 * 128 * D).float())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 20, 100, 900])
def test_pitches_and_depth_zero(gpu, dtype, rows):
    import nnh
    t = T[dtype]
    x = draw(0, rows, 3, 104, dtype=t)
    xd = torch.empty(rows, 3, 104, dtype=t, device="cuda").copy_(x)[:, 1, 1:98]
    w, s = weight(1, 133, 97)
    out = torch.full((rows, 2, 150), 7.0, dtype=t, device="cuda")
    nnh.linear_int8(xd, w.cuda()[:, :97], s.cuda(), out=out[:, 1, 3:136])
    assert_within(out[:, 1, 3:136], linear_int8(x[:, 1, 1:98], w[:, :97], s), "y")
    out[:, 1, 3:136] = 7
    assert bool((out == 7).all())
    b = draw(2, 133, dtype=t).cuda()
    empty = torch.empty(133, 0, dtype=torch.int8, device="cuda")
    y = nnh.linear_int8(torch.empty(rows, 0, dtype=t, device="cuda"), empty, s.cuda(), b)
    assert torch.equal(y, b.expand(rows, -1))
    assert nnh.linear_int8(torch.empty(0, 97, dtype=t, device="cuda"), w.cuda()[:, :97], s.cuda()).shape == (0, 133)
    y3 = nnh.linear_int8(x.cuda().view(rows, 3, 104)[:, :, :96].contiguous(), w.cuda()[:, :96], s.cuda())
    assert y3.shape == (rows, 3, 133)


def test_quantised_weight(gpu):
    """A weight quantised by the same call: as near to the product in 32 bits as the two quantisations' steps allow."""
    import nnh
    x, w = draw(0, 90, 500), draw(1, 70, 500)
    codes, scale = nnh.quantize_rows(w.cuda())
    y = nnh.linear_int8(x.cuda(), codes, scale).cpu().double()
    xc, xs = codes_of(x)
    wc, ws = codes_of(w)
    xs, ws = xs.double()[:, None], ws.double()[:, None]
    # |x w - x' w'| <= |x| |w - w'| + |w'| |x - x'|, a code being off by at most half a scale
    bound = x.double().abs() @ (ws.expand(-1, 500) / 2).t() + (xs.expand(-1, 500) / 2) @ (wc * ws).abs().t()
    want = x.double() @ w.double().t()
    assert bool(((y - want).abs() <= bound * (1 + 1e-5)).all())


@pytest.mark.parametrize("rows,D,V", [(4, 300, 200), (20, 300, 200), (100, 4096, 300)])
def test_captured_and_on_two_streams(gpu, rows, D, V):
    """Where the rows' codes need scratch: captured with exactly the size asked for, refused without."""
    import nnh
    w, s = weight(1, V, D)
    w, s = w.cuda()[:, :D], s.cuda()
    x = [draw(i, rows, D, dtype=torch.bfloat16).cuda() for i in range(2)]
    size = nnh.workspace_size("linear_int8", rows, D, V)
    assert (size > 0) == (rows > 4)
    room = torch.full((size + 4096,), 7, dtype=torch.uint8, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    if size:
        with pytest.raises(nnh.NnhError, match="workspace"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                nnh.linear_int8(x[0], w, s)
    if size:
        nnh.set_workspace(room[:size], side)
    try:
        with torch.cuda.graph(graph, stream=side):
            y = nnh.linear_int8(x[0], w, s)
        for seed in range(3):
            x[0].copy_(draw(10 + seed, rows, D, dtype=torch.bfloat16))
            want = nnh.linear_int8(x[0], w, s)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)
        assert bool((room[size:] == 7).all())
    finally:
        nnh.set_workspace(None, side)
    want = [nnh.linear_int8(t, w, s) for t in x]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [nnh.linear_int8(t, w, s, stream=st) for t, st in zip(x, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
