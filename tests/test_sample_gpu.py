"""The choice of tokens on the GPU against a plain form in 64 bits. The kernel's weights are rounded to 2^-bits of the largest, so where
a sum of weights is that near to its border (u's or top_p's) the next token is right too; elsewhere, and where the weights are exact,
it has to be the same."""
import math

import pytest
import torch

from serving_reference import T, draw, ints, sample_row

pytestmark = pytest.mark.gpu


def run(logits, u, **o):
    import nnh
    dev = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in o.items()}
    return nnh.sample(logits if logits.is_cuda else logits.cuda(), u.cuda(), **dev)


def check(logits, u, exact=False, got=None, **o):
    tokens, logprob = got or run(logits, u, **o)
    tokens, logprob = tokens.cpu(), logprob.cpu()
    V = logits.shape[1]
    bits = min(51, 62 - max(0, (V - 1).bit_length()))
    for r in range(logits.shape[0]):
        one = {n: x[r].item() for n, x in o.items() if x is not None}
        ways = [sample_row(logits[r].cpu(), u[r].item(), **one)]
        if not exact:  # half of 2^-bits for each of the weights, beside a sum of 1 at least
            e = V * 2.0 ** -bits
            for du in (-e, e):
                for dp in (-e, 0.0, e) if "top_p" in one else (0.0,):
                    moved = dict(one, top_p=one["top_p"] + dp) if "top_p" in one else one
                    ways.append(sample_row(logits[r].cpu(), max(0.0, u[r].item() + du), **moved))
        hit = [w for w in ways if w[0] == int(tokens[r])]
        assert hit, (r, int(tokens[r]), ways, one, u[r].item())
        want = hit[0][1]
        # the result is rounded to 32 bits; the sums' own error, relative to 1 at least, is V 2^-bits at most
        assert abs(float(logprob[r]) - want) <= 2.0 ** -24 * abs(want) + V * 2.0 ** -bits + 1e-12 or float(logprob[r]) == want, (r, float(logprob[r]), want)
    return tokens


def uniform(seed, rows, lo=0.0, hi=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (lo + (hi - lo) * torch.rand(rows, generator=gen)).clamp(max=1 - 2.0 ** -24)


FILTERS = {"none": {}, "k": {"k": 40}, "p": {"p": 0.9}, "m": {"m": 0.02}, "kp": {"k": 300, "p": 0.8}, "km": {"k": 20, "m": 0.01}, "all": {"k": 500, "p": 0.95, "m": 0.001},
           "one": {"k": 1}, "p0": {"p": 0.0}, "wide": {"k": 3000, "p": 0.999}}


def options(name, rows, seed=5):
    f, o = FILTERS[name], {}
    if "k" in f:
        o["top_k"] = torch.randint(1, f["k"] + 1, (rows,), generator=torch.Generator().manual_seed(seed)).int()
        o["top_k"][0] = f["k"]
    if "p" in f:
        o["top_p"] = f["p"] * uniform(seed + 1, rows, 0.8, 1.0)
    if "m" in f:
        o["min_p"] = f["m"] * uniform(seed + 2, rows, 0.5, 1.0)
    return o


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 63, 64, 1000, 8192, 8193, 50257])
@pytest.mark.parametrize("name", sorted(FILTERS))
def test_filters(gpu, dtype, V, name):
    rows = 5
    z = draw(V, rows, V, dtype=T[dtype], scale=2.5)
    check(z, uniform(V + 1, rows), temperature=uniform(V + 2, rows, 0.3, 1.5), **options(name, rows))
    check(z, uniform(V + 3, rows), **options(name, rows, 9))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("wide", [0.0, 1e-6, 0.01, 20.0, 1e4])
@pytest.mark.parametrize("name", ["none", "kp", "p", "wide"])
def test_other_distributions(gpu, dtype, wide, name):
    """All logits alike or nearly (bins with more elements than the list), a few tokens with all of the weight."""
    z = draw(3, 4, 20000, dtype=T[dtype], scale=wide)
    check(z, uniform(1, 4), **options(name, 4))
    check(z + 5, uniform(2, 4), temperature=torch.tensor([1e-3, 1.0, 50.0, 1e30]), **options(name, 4))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [7, 3000, 40000])
def test_equal_logits(gpu, dtype, V):
    """Equal logits are taken in the order of their index; weights are exact, so are the borders: u and top_p at whole shares and next
    to them."""
    n = V // 2
    z = torch.zeros(9, V, dtype=T[dtype])
    u = torch.tensor([0.0, 0.5, 0.25, 1 / 3, 1 - 2.0 ** -24, 2.0 ** -24, 2.0 ** -130, 0.75, 0.5 - 2.0 ** -25])
    tokens = check(z, u, exact=True)
    assert tokens[0] == 0 and tokens[1] == -(-V // 2) - (V % 2) and tokens[4] == V - 1
    check(z, u, exact=True, top_p=torch.full((9,), 0.5))
    check(z, u, exact=True, top_k=torch.full((9,), n + 1, dtype=torch.int32), top_p=torch.tensor([0.1, 0.5, 1.0, 2.0, -1.0, 0.25, 2.0 ** -24, 0.9, math.nan]).nan_to_num(1.0))
    z[:, n:] = 1
    check(z, u, exact=False, top_k=torch.full((9,), n + 3, dtype=torch.int32))
    z[:, :] = -math.inf
    z[:, 1::2] = -0.0
    z[:, 3::4] = 0.0
    check(z, u, exact=True, top_k=torch.full((9,), max(1, n // 2), dtype=torch.int32))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [5, 9000])
def test_values_that_are_not_finite(gpu, dtype, V):
    z = draw(1, 8, V, dtype=T[dtype])
    z[0] = -math.inf
    z[1] = math.nan
    z[2, :-1] = math.nan
    z[3, 1], z[3, 4] = math.inf, math.inf
    z[4, 2] = math.nan
    z[5, 3] = -math.inf
    z[6, :4] = torch.tensor([-math.inf, math.nan, math.inf, math.inf])
    u = uniform(3, 8)
    tokens = check(z, u)
    assert tokens[:3].tolist() == [-1, -1, V - 1] and int(tokens[3]) in (1, 4) and int(tokens[6]) in (2, 3)
    check(z, u, temperature=torch.zeros(8))
    check(z, u, temperature=torch.tensor([-1.0, 0.0, 0.0, 0.0, 0.0, -math.inf, 0.0, 0.5]))
    check(z, u, top_k=torch.tensor([3, 3, 3, 1, 2, 0, -5, 2 ** 31 - 1], dtype=torch.int32), min_p=torch.tensor([0.1, 0.1, 0.1, 0.1, 2.0, 1.0, -1.0, 0.0]))
    # NaN is off; NaN as temperature takes the largest
    import nnh
    nan = torch.full((8,), math.nan).cuda()
    a = nnh.sample(z.cuda(), u.cuda(), top_p=nan, min_p=nan)
    b = nnh.sample(z.cuda(), u.cuda())
    assert torch.equal(a[0], b[0])
    c, d = nnh.sample(z.cuda(), u.cuda(), temperature=nan), nnh.sample(z.cuda(), u.cuda(), temperature=torch.zeros(8).cuda())
    assert torch.equal(c[0], d[0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [100, 30001])
def test_pitch_and_alignment(gpu, dtype, V):
    t = T[dtype]
    z = draw(1, 6, V, dtype=t, scale=2.0)
    for pitch, shift in ((V, 0), (V + 3, 0), (-(-V // 8) * 8 + 8, 0), (-(-V // 8) * 8 + 8, 1)):
        room = torch.full((6 * pitch + 16,), 100.0, dtype=t, device="cuda")[shift:shift + 6 * pitch].view(6, pitch)
        room[:, :V] = z.cuda()
        o = options("kp", 6)
        check(z, uniform(2, 6), got=run(room[:, :V], uniform(2, 6), **o), **o)


@pytest.mark.parametrize("wide", [3.0, 0.05, 1e-3, 300.0])
@pytest.mark.parametrize("name", ["none", "kp", "all"])
def test_values_that_are_counted(gpu, wide, name):
    """16-bit logits of few values and of magnitudes below 2^-8 and above 2^8, whose weights are found in another way."""
    z = draw(8, 6, 30000, dtype=torch.bfloat16, scale=wide)
    z[1] = z[1].round()
    z[2, ::3] = -z[2, ::3].abs()
    z[3, 5::7] = 0.0
    z[4, ::2] = -math.inf
    t = torch.tensor([1.0, 0.5, 1.0, wide, 1.0, 100.0]) * max(1.0, wide / 3)
    check(z, uniform(9, 6), temperature=t, **options(name, 6))


def test_frequencies(gpu):
    """Every token comes up for the share of u that is its own."""
    V, n = 6, 1 << 12
    z = torch.tensor([0.1, 2.0, -1.0, 2.0, 0.0, -3.0])
    u = (torch.arange(n).float() + 0.5) / n
    tokens, logprob = run(z.repeat(n, 1), u)
    p = torch.softmax(z.double(), 0)
    for i in range(V):
        assert abs(int((tokens == i).sum()) - float(p[i]) * n) <= 1
    assert (logprob.cpu().double() - torch.log(p)[tokens.cpu().long()]).abs().max() < 1e-6


@pytest.mark.parametrize("rows,V", [(20, 40000), (3, 500), (300, 9000)])
def test_captured_and_on_two_streams(gpu, rows, V):
    """Large vocabularies need scratch: captured with exactly the size asked for, refused without."""
    import nnh
    z = [draw(i, rows, V, dtype=torch.bfloat16).cuda() for i in range(2)]
    u, k = uniform(1, rows).cuda(), torch.full((rows,), min(V, 2000), dtype=torch.int32, device="cuda")
    size = nnh.workspace_size("sample", nnh.BF16, rows, V)
    assert (size > 0) == (V > 8192)
    room = torch.full((size + 4096,), 7, dtype=torch.uint8, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    if size:
        with pytest.raises(nnh.NnhError, match="workspace"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                nnh.sample(z[0], u, top_k=k)
        nnh.set_workspace(room[:size], side)
    try:
        with torch.cuda.graph(graph, stream=side):
            got = nnh.sample(z[0], u, top_k=k)
        for seed in range(3):
            z[0].copy_(draw(10 + seed, rows, V, dtype=torch.bfloat16))
            want = nnh.sample(z[0], u, top_k=k)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert bool((room[size:] == 7).all())
    finally:
        nnh.set_workspace(None, side)
    want = [nnh.sample(x, u, top_k=k) for x in z]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        outs = [nnh.sample(x, u, top_k=k, stream=s) for x, s in zip(z, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) for a, b in zip(outs, want))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,V", [(130, 20001), (300, 20001), (1100, 8200)])
def test_more_rows(gpu, dtype, rows, V):
    """Rows that share the GPU in slices, two to a row, rows of one workgroup each, more of them than are done at a time."""
    z = draw(4, rows, V, dtype=T[dtype], scale=3.0)
    t = uniform(5, rows, 0.2, 1.2)
    t[3] = 0
    z[5] = -math.inf
    check(z, uniform(6, rows), temperature=t)
    check(z, uniform(7, rows), temperature=t, **options("all", rows))


def test_rows_past_32_bits(gpu):
    """Rows that begin past 2^31 and 2^32 elements."""
    import nnh
    V, rows = 131072, (1 << 32) // 131072 + 2
    z = torch.zeros(rows, V, dtype=torch.bfloat16, device="cuda")
    at = [0, rows // 2 + 1, rows - 1]
    for i, r in enumerate(at):
        z[r, 77 + i] = 60
    tokens, _ = nnh.sample(z[rows - 3:], torch.full((3,), 0.5, device="cuda"))
    assert int(tokens[2]) == 79
    tokens, _ = nnh.sample(z, torch.full((rows,), 0.5, device="cuda"), top_k=torch.full((rows,), 1, dtype=torch.int32, device="cuda"))
    assert [int(tokens[r]) for r in at] == [77, 78, 79] and int(tokens[1]) == 0
