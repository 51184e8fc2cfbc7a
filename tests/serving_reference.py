"""Plain forms of the serving operators (a paged cache, attention over it, linears in 8-bit integers, sampling), in 64 bits and on the
CPU, and random batches to run them on."""
import math

import numpy as np
import torch

from lm_reference import U32, masked_attention, unit

T = {"f32": torch.float32, "bf16": torch.bfloat16}


def draw(seed, *shape, dtype=torch.float32, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * scale).to(dtype)


def ints(*values):
    return torch.tensor(values, dtype=torch.int32)


class Batch:
    """Sequences of `new` rows each that hold `held` tokens with them, in pages dealt out in a random order; slots that no sequence has
    hold NaN. pad: rows behind the last sequence; extra: pages that nobody has; layout: "plain", "heads" ({pages, Hkv, page, D}
    in memory) or "pair" (keys and values of a page side by side)."""

    def __init__(self, dtype, new, held, page, H, Hkv, D, pad=2, extra=2, seed=0, layout="plain", width=0, scale_q=1.0):
        t = T[dtype]
        self.t, self.new, self.held, self.page = t, list(new), list(held), page
        self.H, self.Hkv, self.D, self.N = H, Hkv, D, len(new)
        used = [-(-h // page) for h in held]
        pages = sum(used) + extra
        gen = torch.Generator().manual_seed(seed + 77)
        order = torch.randperm(max(1, pages), generator=gen).int()
        self.table = torch.full((self.N, max([width, 1] + used)), -7, dtype=torch.int32)
        at = 0
        for n, count in enumerate(used):
            self.table[n, :count] = order[at:at + count]
            at += count
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.rows = starts[-1] + pad
        self.starts, self.lens = ints(*starts), ints(*held)
        self.tokens = [[draw(seed + 3 * n + i, held[n], Hkv, D, dtype=t) for i in (1, 2)] for n in range(self.N)]
        shape = (max(1, pages), page, Hkv, D)
        if layout == "plain":
            self.k, self.v = torch.full(shape, math.nan, dtype=t), torch.full(shape, math.nan, dtype=t)
        elif layout == "heads":
            self.k, self.v = (torch.full((shape[0], Hkv, page, D), math.nan, dtype=t).transpose(1, 2) for _ in range(2))
        else:
            both = torch.full((shape[0], 2, page, Hkv, D), math.nan, dtype=t)
            self.k, self.v = both[:, 0], both[:, 1]
        self.layout = layout
        self.store(0)
        self.q = draw(seed + 1000, self.rows, H, D, dtype=t, scale=scale_q)

    def places(self, n):
        j = torch.arange(self.held[n])
        return self.table[n].long()[j // self.page], j % self.page

    def store(self, skip):
        """The sequences' tokens into their pages, all but the last skip * new."""
        for n in range(self.N):
            page, slot = self.places(n)
            live = self.held[n] - skip * self.new[n]
            ok = (page >= 0) & (page < self.k.shape[0]) & (torch.arange(self.held[n]) < live)
            self.k[page[ok], slot[ok]] = self.tokens[n][0][ok]
            self.v[page[ok], slot[ok]] = self.tokens[n][1][ok]

    def cache(self, nnh):
        """On the device, in the same memory layout."""
        if self.layout == "plain":
            k, v = self.k.cuda(), self.v.cuda()
        elif self.layout == "heads":
            k, v = (x.transpose(1, 2).contiguous().cuda().transpose(1, 2) for x in (self.k, self.v))
        else:
            both = torch.stack([self.k, self.v], 1).cuda()
            k, v = both[:, 0], both[:, 1]
        return nnh.PagedCache(k, v, self.table.cuda())

    def want(self, absent=None, **rule):
        """out {rows, H, D} and lse {rows, H} with their bounds, NaN behind the last sequence. absent: {(sequence, page index)} without a
        page."""
        out = torch.full((2, self.rows, self.H, self.D), math.nan, dtype=torch.float64)
        lse = torch.full((2, self.rows, self.H), math.nan, dtype=torch.float64)
        for n in range(self.N):
            a, b = int(self.starts[n]), int(self.starts[n + 1])
            if a == b:
                continue
            o = dict(rule)
            if "prefix" in o:
                o["prefix"] = o["prefix"][n:n + 1]
            if absent:
                docs = torch.zeros(1, self.held[n], dtype=torch.int32)
                for m, i in absent:
                    if m == n:
                        docs[:, i * self.page:(i + 1) * self.page] = -1
                o["k_docs"], o["q_docs"] = docs, torch.zeros(1, b - a, dtype=torch.int32)
            k, v = self.tokens[n]
            w = masked_attention(self.q[None, a:b], k[None], v[None], q_start=ints(self.held[n] - (b - a)), **o)
            for i in range(2):
                out[i, a:b] = w["out"][i][0]
                lse[i, a:b] = w["lse"][i][0].t()
        return out, lse


def codes_of(x):
    """Rows as 8-bit codes with a scale each: scale = max |x| / 127 in 32 bits, codes the nearest to x / scale, ties to even. A row with a
    value that is not finite has codes of 0 and a scale of NaN."""
    x = x.double()
    fine = torch.isfinite(x).all(1)
    top = torch.where(fine[:, None], x.abs(), 0.0).amax(1) if x.shape[1] else x.sum(1)
    scale = (top.float() / 127).float()
    s = scale.double()[:, None]
    codes = torch.where(fine[:, None] & (s > 0), x / torch.where(s > 0, s, 1.0), 0.0).round().clamp(-127, 127)
    return codes, torch.where(fine, scale, math.nan)


def linear_int8(x, w, w_scale, bias=None):
    """(value, bound): the sums are whole numbers; what rounds is their way to 32 bits, the two scales, the bias and the result."""
    codes, scale = codes_of(x)
    prod = (codes @ w.double().t()) * scale.double()[:, None] * w_scale.double()[None, :]
    y = prod + (bias.double()[None, :] if bias is not None else 0.0)
    bound = 4 * U32 * prod.abs() + 2 * U32 * y.abs()
    return y, bound + (unit(x.dtype) if x.dtype != torch.float32 else 0.0) * (y.abs() + bound)


def sample_row(z, u, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """(token, log-probability) of one row of logits; ties in the order of the index."""
    z = z.double().numpy()
    z = np.where(np.isnan(z), -math.inf, z)
    top = z.max()
    if top == -math.inf:
        return -1, -math.inf
    order = np.argsort(-z, kind="stable")
    if not temperature > 0:
        return int(order[0]), 0.0
    z = z[order]
    if top == math.inf:
        far = np.where(z == top, 0.0, math.inf)
    else:
        far = (top - z) / temperature
    w = np.exp(-far)
    keep = len(w)
    if min_p is not None and min_p > 0:
        keep = max(1, int((w >= min_p).sum()))
    if top_k is not None and top_k > 0:
        keep = min(keep, top_k)
    total = w[:keep].cumsum()
    if top_p is not None and top_p < 1:
        keep = max(1, int((total - w[:keep] < top_p * total[-1]).sum()))
    total = total[:keep]
    n = min(int((total <= u * total[-1]).sum()), keep - 1)
    while w[n] == 0.0:
        n -= 1
    return int(order[n]), float(-far[n] - math.log(total[-1]))
