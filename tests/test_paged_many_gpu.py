"""The paged cache on the GPU with many sequences and long caches: sequences past the 64 that a wave looks at in one go, each form of few
columns (by the number of workgroups, keys divided or not), keys in more than 64 parts and in several rounds, joins of several heads to a
wave. Against the formula in 64 bits, within the bounds of its roundings."""
import math
import random

import pytest
import torch

from lm_reference import assert_within, masked_attention
from serving_reference import Batch, draw, ints
from test_paged_gpu import attend, check

pytestmark = pytest.mark.gpu


def divided(b, most=None):
    import nnh
    return nnh.workspace_size("paged_attention", b.N, b.rows, most or max(b.new), b.table.shape[1] * b.page, b.H, b.Hkv, b.D) > 0


def lengths(N, longest, seed, chunks=(), long=()):
    """New and held tokens of N sequences: mostly one new token, some of none about the 64th and at the end; chunks: sequences of 80 new
    ones, long: sequences that hold 600 to 1000."""
    rng = random.Random(seed)
    new = [rng.choice([0, 1, 1, 1, 1, 1, 2, 5]) for _ in range(N)]
    for n in (62, 63, N - 2):
        new[n] = 0
    new[64] = new[N - 1] = 3
    for n in chunks:
        new[n] = 80
    held = [max(x, rng.randint(1, longest)) for x in new]
    for n in long:
        held[n] = rng.randint(600, 1000)
    return new, held


# 65 sequences of two key heads are fewer than 256 workgroups, 130 fewer than 1024, 130 of eight key heads more
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 20])
@pytest.mark.parametrize("N,H,Hkv", [(65, 4, 2), (130, 4, 2), (130, 8, 8)])
def test_keys_not_divided(gpu, dtype, D, N, H, Hkv):
    b = Batch(dtype, *lengths(N, 150, N), 16, H, Hkv, D)
    assert not divided(b)
    check(b, causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 128, 20])
@pytest.mark.parametrize("N", [65, 130, 200])
def test_keys_divided_over_sequences(gpu, dtype, D, N):
    """Long sequences before and behind the 64th, of single tokens and of chunks: both forms have parts on either side."""
    new, held = lengths(N, 150, N + 1, chunks=(5, 64, N - 1), long=(0, 5, 40, 64, N - 4, N - 1))
    b = Batch(dtype, new, held, 16, 4, 2, D, width=64)
    assert divided(b)
    check(b, causal=True)
    check(b, causal=True, window=300, prefix=torch.randint(0, 200, (N,), generator=torch.Generator().manual_seed(N)).int())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N", [65, 130])
def test_append(gpu, dtype, N):
    """New tokens of sequences on either side of the 64th, taken out and stored again."""
    import nnh
    b = Batch(dtype, *lengths(N, 60, N + 2, chunks=(3, 66) if N > 66 else (3,)), 24, 4, 2, 24)
    full = b.cache(nnh)
    for x in (b.k, b.v):
        x.fill_(math.nan)
    b.store(1)
    cache = b.cache(nnh)
    k, v = (torch.cat([b.tokens[n][i][b.held[n] - b.new[n]:] for n in range(N)] + [draw(5, 2, 2, 24, dtype=b.t)]).cuda() for i in (0, 1))
    nnh.paged_append(cache, k, v, b.starts.cuda(), b.lens.cuda())
    assert torch.equal(cache.k.nan_to_num(9.0), full.k.nan_to_num(9.0)) and torch.equal(cache.v.nan_to_num(9.0), full.v.nan_to_num(9.0))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_sequences_under_a_wide_table(gpu, dtype):
    """So many that their keys are not divided, whatever the table has room for."""
    b = Batch(dtype, *lengths(770, 40, 3), 16, 8, 8, 8, width=64)
    assert not divided(b)
    check(b, causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("H,Hkv", [(15, 3), (16, 16)])
def test_several_heads_to_a_wave_of_the_join(gpu, dtype, H, Hkv):
    """rows H of more than 8192 (two heads to a wave: one is left over of 15) with keys in parts, in both forms."""
    rng = random.Random(H)
    new, held = [500] + [1] * 60, [1500] + [rng.randint(1, 1400) for _ in range(60)]
    b = Batch(dtype, new, held, 24, H, Hkv, 16)
    assert divided(b) and 8192 <= b.rows * H < 12288
    check(b, causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("new", [1, 40])
def test_more_parts_than_lanes(gpu, dtype, new):
    """36000 keys of one key head: parts of 256 keys, 140 of them."""
    b = Batch(dtype, [new, 2], [36000, 40], 64, 4, 1, 16)
    assert divided(b)
    check(b, causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rounds_of_few_columns(gpu, dtype):
    """Three rounds of workgroups: 70 sequences of 3500 keys on 16 key heads, 7700 tiles for the 48 workgroups a key head that make one."""
    rng = random.Random(9)
    b = Batch(dtype, [1] * 69 + [3], [rng.randint(2000, 5000) for _ in range(70)], 16, 16, 16, 8)
    assert divided(b) and sum(-(-h // 32) for h in b.held) > 3 * 48 * 48
    check(b, causal=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rounds_of_a_chunk(gpu, dtype):
    """Two rounds: 1000 tokens over 26000 keys on 16 key heads, 8 groups of 407 tiles for 32 workgroups a key head; some of its rows."""
    b = Batch(dtype, [1000], [26000], 64, 16, 16, 8)
    assert divided(b) and 8 * (26000 // 64) > 2 * 32 * 48
    out, lse = attend(b, causal=True)
    k, v = b.tokens[0]
    for first, last in ((0, 3), (126, 130), (511, 514), (895, 898), (997, 1000)):
        want = masked_attention(b.q[None, first:last], k[None], v[None], q_start=ints(25000 + first), causal=True)
        assert_within(out[first:last], [x[0] for x in want["out"]], "out")
        assert_within(lse[first:last], [x[0].t() for x in want["lse"]], "lse")
