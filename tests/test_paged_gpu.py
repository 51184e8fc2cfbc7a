"""The paged cache on the GPU: new tokens into their pages, and attention over them against the formula in 64 bits, within the bounds
of its roundings."""
import math

import pytest
import torch

from lm_reference import assert_within
from serving_reference import T, Batch, draw, ints

pytestmark = pytest.mark.gpu


def attend(b, most=None, out=None, lse=None, cache=None, **rule):
    import nnh
    dev = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in rule.items()}
    r = nnh.AttentionRule(k_lens=b.lens.cuda(), **dev)
    return nnh.paged_attention(b.q.cuda(), cache or b.cache(nnh), b.starts.cuda(), max(b.new) if most is None else most, r, out=out, lse=lse)


def check(b, absent=None, most=None, cache=None, **rule):
    print(b.t, b.new, b.held, b.page, b.H, b.Hkv, b.D, b.layout, sorted(rule), flush=True)
    out = torch.full((b.rows, b.H, b.D), 7.0, dtype=b.t, device="cuda")
    lse = torch.full((b.rows, b.H), 7.0, device="cuda")
    attend(b, most, out, lse, cache, **rule)
    torch.cuda.synchronize()
    (o, eo), (l, el) = b.want(absent, **rule)
    live = int(b.starts[-1])
    assert_within(lse[:live], (l[:live], el[:live]), "lse")
    assert_within(out[:live], (o[:live], eo[:live]), "out")
    assert bool((out[live:] == 7).all()) and bool((lse[live:] == 7).all())
    return out, lse


SHAPES = [([1], [1], 16, 1, 1, 64), ([1, 1, 1], [1, 33, 500], 16, 8, 2, 128), ([3, 1], [3, 90], 8, 4, 4, 32), ([70], [70], 16, 4, 1, 64),
          ([129, 1, 40], [300, 77, 40], 24, 4, 2, 80), ([200, 0, 5], [200, 10, 5], 100, 6, 2, 96), ([33], [1000], 1, 4, 1, 64),
          ([2, 300], [700, 300], 7, 3, 3, 40), ([64, 65], [64, 65], 64, 2, 2, 13), ([1, 1], [2000, 65], 33, 12, 1, 1), ([17], [50], 256, 8, 2, 30)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
def test_shapes(gpu, dtype, shape, causal):
    check(Batch(dtype, *shape), causal=causal)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["cap", "slopes", "window", "window_only", "prefix", "scale", "all"])
@pytest.mark.parametrize("D", [64, 96, 128, 20])
def test_rules(gpu, dtype, kind, D):
    """One batch of single tokens, short chunks and long ones under each rule."""
    H, Hkv, every = 4, 2, kind == "all"
    o = {"causal": kind != "window_only"}
    if kind == "cap" or every:
        o["cap"] = 5.0
    if kind == "slopes" or every:
        o["slopes"] = torch.exp2(-torch.arange(1.0, H + 1))
    if kind in ("window", "window_only") or every:
        o["window"] = 37
    if kind == "prefix" or every:
        o["prefix"] = ints(0, 70, 5000, 3)
    if kind == "scale":
        o["scale"] = 0.37
    check(Batch(dtype, [1, 20, 150, 1], [400, 90, 290, 1], 24, H, Hkv, D, scale_q=2.0), **o)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["heads", "pair"])
@pytest.mark.parametrize("D", [64, 20])
def test_layouts(gpu, dtype, layout, D):
    import nnh
    b = Batch(dtype, [1, 100], [333, 140], 16, 4, 2, D, layout=layout)
    check(b, causal=True)
    # the new tokens taken out and stored again
    full = b.cache(nnh)
    for x in (b.k, b.v):
        x.fill_(math.nan)
    b.store(1)
    cache = b.cache(nnh)
    k, v = (torch.cat([b.tokens[n][i][b.held[n] - b.new[n]:] for n in range(2)] + [draw(5, 2, 2, D, dtype=b.t)]).cuda() for i in (0, 1))
    nnh.paged_append(cache, k, v, b.starts.cuda(), b.lens.cuda())
    assert torch.equal(cache.k.nan_to_num(9.0), full.k.nan_to_num(9.0)) and torch.equal(cache.v.nan_to_num(9.0), full.v.nan_to_num(9.0))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [128, 13])
@pytest.mark.parametrize("page", [1, 16, 24])
def test_append(gpu, dtype, D, page):
    """Rows of strides of their own; rows of no sequence, tokens behind the table and pages that are none are stored nowhere."""
    import nnh
    t = T[dtype]
    starts, lens = ints(1, 4, 4, 30, 31), ints(3, 50, 40, 3 * page + 1)  # row 0 belongs to no sequence; the last token has no place
    table = torch.arange(4 * 3 * 60 // page).int()[:4 * -(-60 // page)].view(4, -1)[:, :max(3, -(-60 // page))].contiguous()
    if page == 16:
        table[2, 1] = -1
        table[2, 2] = 10 ** 6
    if table.shape[1] * page >= 3 * page + 1:
        table = table[:, :3].contiguous() if page > 1 else table
    pages = 200
    k, v = (draw(s, 40, 3, 2, 2 * D, dtype=t)[:, 1, :, :D] for s in (1, 2))
    pool = [torch.full((pages, page, 2, D), 5.0, dtype=t) for _ in range(2)]
    cache = nnh.PagedCache(pool[0].cuda(), pool[1].cuda(), table.cuda())
    kd, vd = (torch.empty(40, 3, 2, 2 * D, dtype=t, device="cuda")[:, 1, :, :D].copy_(x) for x in (k, v))
    nnh.paged_append(cache, kd, vd, starts.cuda(), lens.cuda())
    for n in range(4):
        for row in range(int(starts[n]), int(starts[n + 1])):
            pos = int(lens[n]) - int(starts[n + 1]) + row
            if pos < 0 or pos >= table.shape[1] * page:
                continue
            p = int(table[n, pos // page])
            if 0 <= p < pages:
                pool[0][p, pos % page], pool[1][p, pos % page] = k[row], v[row]
    assert torch.equal(cache.k.cpu(), pool[0]) and torch.equal(cache.v.cpu(), pool[1])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [128, 64, 30])
@pytest.mark.parametrize("new", [1, 120])
def test_pages_that_are_none(gpu, dtype, D, new):
    """Tokens whose page is gone are not seen, whatever else lies there; a sequence without any."""
    b = Batch(dtype, [new, new, 1], [300, 200, 40], 16, 4, 2, D)
    gone = {(0, 0), (0, 7), (0, 8), (1, 3)} | {(2, i) for i in range(3)}
    for n, i in gone:
        b.table[n, i] = (-1, 10 ** 7, -2 ** 31)[i % 3]
    check(b, absent=gone, causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("new", [1, 90])
def test_not_finite_in_masked_places(gpu, dtype, bad, new):
    """Keys and values that a row does not see are not finite; a value that some rows see and others do not."""
    import nnh
    b = Batch(dtype, [new, 2], [190, 80], 24, 4, 2, 64)
    (o, eo), (l, el) = b.want(causal=True, window=100)
    for n in range(2):
        page, slot = b.places(n)
        dead = torch.arange(b.held[n]) < b.held[n] - b.new[n] - 99  # before every row's window
        b.k[page[dead], slot[dead]] = bad
        b.v[page[dead], slot[dead]] = bad
    out, lse = attend(b, causal=True, window=100)
    live = int(b.starts[-1])
    assert_within(lse[:live], (l[:live], el[:live]), "lse")
    assert_within(out[:live], (o[:live], eo[:live]), "out")
    if new > 1:  # the last token's value: only the last row sees it
        page, slot = b.places(0)
        cache = b.cache(nnh)
        cache.v[int(page[-1]), int(slot[-1]), 1, 3] = bad
        out, _ = attend(b, cache=cache, causal=True, window=100)
        assert_within(out[:new - 1], (o[:new - 1], eo[:new - 1]), "rows before")
        assert not torch.isfinite(out[new - 1, 2:, 3]).any() and torch.isfinite(out[new - 1, :2]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_without_keys(gpu, dtype):
    """More rows than tokens (the first ones are before position 0), sequences of no tokens, of no rows, no pages at all, most below a
    sequence's rows."""
    import nnh
    b = Batch(dtype, [5, 0, 100, 3], [2, 0, 50, 0], 16, 4, 2, 64)
    out, lse = attend(b, causal=True)
    (o, eo), (l, el) = b.want(causal=True)
    assert_within(out[:108], (o[:108], eo[:108]), "out")
    assert_within(lse[:108], (l[:108], el[:108]), "lse")
    assert bool((out[:3] == 0).all()) and bool((lse[:3] == -math.inf).all()) and bool((out[105:108] == 0).all())
    empty = nnh.PagedCache(torch.empty(0, 16, 2, 64, dtype=b.t, device="cuda"), torch.empty(0, 16, 2, 64, dtype=b.t, device="cuda"), b.table.cuda())
    out, lse = attend(b, cache=empty, causal=True)
    assert bool((out[:108] == 0).all()) and bool((lse[:108] == -math.inf).all())
    out = torch.full((b.rows, 4, 64), 7.0, dtype=b.t, device="cuda")
    attend(b, most=4, out=out, causal=True)
    done = [0, 1, 2, 3, *range(5, 9), 105, 106, 107]
    assert_within(out[done], (o[done], eo[done]), "most")
    assert bool((out[4] == 7).all()) and bool((out[9:105] == 7).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new,held", [(1, 5000), (16, 5000), (40, 5000), (200, 6000)])
def test_keys_divided(gpu, dtype, new, held):
    """Few rows over long caches, whose keys are divided over the GPU, in either form; beside a sequence whose keys are few."""
    check(Batch(dtype, [new, 1], [held, 3], 16, 4, 1, 64), causal=True, cap=9.0)
    check(Batch(dtype, [new], [held], 24, 8, 8, 128, pad=0), causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides(gpu, dtype):
    """q and out as parts of wider rows, a cache of a wider pool's heads; two tokens off alignment."""
    import nnh
    t = T[dtype]
    b = Batch(dtype, [1, 100], [200, 130], 16, 4, 2, 64)
    (o, eo), _ = b.want(causal=True)
    for shift in (0, 1):
        q = torch.zeros(b.rows, 3, 4, 72, dtype=t, device="cuda")[:, 1, :, shift:64 + shift].copy_(b.q)
        out = torch.full((b.rows, 3, 4, 72), 7.0, dtype=t, device="cuda")
        k, v = (torch.zeros(x.shape[0], 16, 5, 72, dtype=t, device="cuda")[:, :, 1:3, shift:64 + shift].copy_(x) for x in (b.k, b.v))
        r = nnh.AttentionRule(causal=True, k_lens=b.lens.cuda())
        nnh.paged_attention(q, nnh.PagedCache(k, v, b.table.cuda()), b.starts.cuda(), 100, r, out=out[:, 1, :, shift:64 + shift])
        assert_within(out[:101, 1, :, shift:64 + shift], (o[:101], eo[:101]), "out")
        out[:, 1, :, shift:64 + shift] = 7
        assert bool((out == 7).all())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_captured(gpu, dtype):
    """A step (append, then attention) captured with a workspace of exactly the size asked for, replayed as sequences grow; refused
    without one."""
    import nnh
    N, page, H, Hkv, D, width, t = 3, 16, 4, 2, 64, 60, T[dtype]
    pool = [torch.zeros(N * width, page, Hkv, D, dtype=t, device="cuda") for _ in range(4)]
    table = torch.randperm(N * width).int().view(N, width).cuda()
    one, two = nnh.PagedCache(pool[0], pool[1], table), nnh.PagedCache(pool[2], pool[3], table)
    k, v, q = (torch.zeros(70, h, D, dtype=t, device="cuda") for h in (Hkv, Hkv, H))
    starts, lens = ints(0, 0, 0, 0).cuda(), ints(0, 0, 0).cuda()
    rule = nnh.AttentionRule(causal=True, k_lens=lens)
    size = nnh.workspace_size("paged_attention", N, 70, 64, width * page, H, Hkv, D)
    assert size > 0
    room = torch.full((size + 4096,), 7, dtype=torch.uint8, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()

    def step(cache, out, lse):
        nnh.paged_append(cache, k, v, starts, lens)
        return nnh.paged_attention(q, cache, starts, 64, rule, out=out, lse=lse)

    outs = [(torch.zeros(70, H, D, dtype=t, device="cuda"), torch.zeros(70, H, device="cuda")) for _ in range(2)]
    with pytest.raises(nnh.NnhError, match="workspace"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            step(one, *outs[0])
    nnh.set_workspace(room[:size], side)
    try:
        with torch.cuda.graph(graph, stream=side):
            step(one, *outs[0])
        for seed, new, held in [(1, [64, 3, 0], [64, 3, 0]), (2, [1, 60, 1], [65, 63, 1]), (3, [1, 1, 1], [66, 64, 2]), (4, [5, 5, 5], [900, 800, 7])]:
            for i, x in enumerate((k, v, q)):
                x.copy_(draw(10 * seed + i, *x.shape, dtype=t))
            starts.copy_(ints(0, new[0], new[0] + new[1], sum(new)))
            lens.copy_(ints(*held))
            step(two, *outs[1])
            graph.replay()
            torch.cuda.synchronize()
            for x, y in zip(outs[0] + (one.k, one.v), outs[1] + (two.k, two.v)):
                assert torch.equal(x, y)
        assert bool((room[size:] == 7).all())
    finally:
        nnh.set_workspace(None, side)


@pytest.mark.parametrize("new", [1, 100])
def test_two_streams(gpu, new):
    """Calls on two streams at once, each with scratch of its own, repeat bit for bit."""
    import nnh
    b = [Batch("bf16", [new, 1], [3000, 500], 16, 4, 2, 128, seed=s) for s in (0, 50)]
    caches, q, starts, lens = [x.cache(nnh) for x in b], [x.q.cuda() for x in b], [x.starts.cuda() for x in b], [x.lens.cuda() for x in b]

    def call(i, stream=None):
        return nnh.paged_attention(q[i], caches[i], starts[i], new, nnh.AttentionRule(causal=True, k_lens=lens[i]), stream=stream)

    want = [call(i) for i in (0, 1)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = [call(i, streams[i]) for i in (0, 1)]
        torch.cuda.synchronize()
        for x, y, z in zip(want, got, b):
            live = int(z.starts[-1])
            assert torch.equal(x[0][:live], y[0][:live]) and torch.equal(x[1][:live], y[1][:live])


def test_places_past_32_bits(gpu):
    """Pages whose elements lie past 2^31 and 2^32 of the pool's start."""
    import nnh
    D, Hkv, page = 128, 8, 256
    pages = (1 << 32) // (D * Hkv * page) + 40
    pool = [torch.zeros(pages, page, Hkv, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    b = Batch("bf16", [1, 40], [1000, 300], page, 8, 8, D, extra=0)
    far = torch.tensor([pages - 1 - i if i % 2 else pages // 2 + i for i in range(b.k.shape[0])])
    pool[0][far.cuda()], pool[1][far.cuda()] = b.k.cuda(), b.v.cuda()
    table = torch.where(b.table >= 0, far.int()[b.table.clamp(min=0).long()], -1)
    (o, eo), _ = b.want(causal=True)
    cache = nnh.PagedCache(pool[0], pool[1], table.cuda())
    out, _ = attend(b, cache=cache, causal=True)
    assert_within(out[:41], (o[:41], eo[:41]), "out")
    k, v = (torch.cat([b.tokens[n][i][b.held[n] - b.new[n]:] for n in range(2)]).cuda() for i in (0, 1))
    for x in pool:
        x.zero_()
    nnh.paged_append(cache, k, v, b.starts[:3].cuda(), b.lens.cuda())
    for n in range(2):
        p, s = b.places(n)
        new = slice(b.held[n] - b.new[n], None)
        assert torch.equal(pool[0][far[p[new]].cuda(), s[new].cuda()].cpu(), b.tokens[n][0][new])
        assert torch.equal(pool[1][far[p[new]].cuda(), s[new].cuda()].cpu(), b.tokens[n][1][new])
