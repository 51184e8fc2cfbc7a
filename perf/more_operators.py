"""Operators that serve a language model as cases that can be timed and checked: what a step of many sequences over a paged
cache does, from the linears in 8-bit integers to the choice of the next tokens.

A case is a dict of plain values; "op" says which operator it runs.

  append   new keys and values of many sequences (rows packed one sequence after another) into the pages of a cache
  paged    attention of the new tokens of many sequences, one or a chunk of them each, over the pages that hold their keys
  int8     a linear layer with weights in 8-bit integers, a scale for each output, and activations quantised row by row
  sample   the next token of each row of logits: temperature, min-p, top-k and top-p, from a given random number

With `own` false, `run` computes them from elementary torch operations in 32 bits (codes and the choice of a token in 64, so that
values next to a border fall on their own side); with `own` true, by the framework's calls.
"""
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def _append(name, dtype, seqs, new, held, page, kv_heads, dh):
    c = {"op": "append", "dtype": dtype, "seqs": seqs, "new": new, "held": held, "page": page, "kv_heads": kv_heads, "dh": dh}
    return dict(c, name=name) if name else c


def _paged(name, dtype, seqs, new, riders, held, page, heads, kv_heads, dh, cap=0.0, window=0, slopes=False):
    c = {"op": "paged", "dtype": dtype, "seqs": seqs, "new": new, "riders": riders, "held": held, "page": page, "heads": heads,
         "kv_heads": kv_heads, "dh": dh, "cap": cap, "window": window, "slopes": slopes}
    return dict(c, name=name) if name else c


def _int8(name, dtype, rows, d, outs, bias=False):
    c = {"op": "int8", "dtype": dtype, "rows": rows, "d": d, "outs": outs, "bias": bias}
    return dict(c, name=name) if name else c


def _sample(name, dtype, rows, vocab, wide, k=0, p=1.0, min_p=0.0):
    c = {"op": "sample", "dtype": dtype, "rows": rows, "vocab": vocab, "wide": wide, "k": k, "p": p, "min_p": min_p}
    return dict(c, name=name) if name else c


def listed():
    return [
        # Prompts being read: chunks of eight sequences go into the pool in one call.
        _append("append_chunks", "bf16", 8, 2048, 4096, 16, 8, 128),
        # The benchmark's attention heads, one token of each of four sequences: latency.
        _append("append_one_f32", "f32", 4, 1, 300, 32, 8, 64),
        # Serving: one token of each of 64 sequences of unlike length.
        _paged("paged_decode_64", "bf16", 64, 1, 0, 8192, 16, 32, 8, 128),
        # A chunk of one prompt beside the single tokens of 31 other sequences; heads and pages that no tile divides.
        _paged("paged_mixed_80", "bf16", 32, 1021, 31, 4096, 24, 12, 4, 80, cap=50.0),
        # A long prompt read in chunks: 4096 tokens over the 16384 that the cache then holds, bound by its products.
        _paged("paged_chunk_16384", "bf16", 1, 4096, 0, 16384, 128, 32, 8, 128),
        # One user's next token against a short cache, in 32 bits: latency.
        _paged("paged_one_f32", "f32", 1, 1, 0, 300, 16, 8, 8, 64, slopes=True),
        # One token through a square projection: the weights' bytes and latency.
        _int8("int8_1x4096", "bf16", 1, 4096, 4096),
        # A batch of 32 tokens through an MLP's first layer.
        _int8("int8_32x16384", "bf16", 32, 4096, 16384, bias=True),
        # A prompt's tokens through the same layer: the largest product.
        _int8("int8_8192x16384", "bf16", 8192, 4096, 16384),
        # One user's next token from a vocabulary that no tile divides.
        _sample("sample_1x50257", "f32", 1, 50257, 2.5, k=50, p=0.9),
        # A full batch over a large vocabulary, the kept set found by its probability alone.
        _sample("sample_256x128000", "bf16", 256, 128000, 3.0, p=0.95, min_p=0.001),
        # A batch that draws from the whole distribution.
        _sample("sample_64x32000", "f32", 64, 32000, 2.0),
    ]


def _log(rng, lo, hi):
    """A size between lo and hi over the logarithm: half of them as they come, half multiples of 16."""
    v = max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))
    return v if rng.random() < 0.5 or v < 32 else v // 16 * 16


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "chunk", "chunk", "int8", "int8", "int8", "sample", "sample", "sample"])
    dtype = rng.choice(["f32", "bf16", "bf16"])
    kv, group = rng.choice([(1, 8), (2, 4), (4, 3), (8, 1), (8, 4), (12, 1)])
    dh, page = rng.choice([32, 64, 80, 96, 128, 128]), rng.choice([8, 16, 16, 24, 32, 64, 100, 128, 256])
    if op == "append":
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, 16384 // seqs))
        return _append(None, dtype, seqs, new, new + _log(rng, 1, 4096), page, kv, dh)
    if op == "decode":
        held = _log(rng, 16, 32768)
        seqs = _log(rng, 1, max(1, min(128, 524288 // held)))
        return _paged(None, dtype, seqs, rng.choice([1, 1, 1, 2, 4]), 0, held, page, kv * group, kv, dh, cap=rng.choice([0.0, 0.0, 30.0]),
                      window=_log(rng, 8, held) if rng.random() < 0.2 else 0, slopes=rng.random() < 0.3)
    if op == "chunk":
        new = _log(rng, 8, 2048)
        held = new + _log(rng, 1, 8192)
        seqs = _log(rng, 1, max(1, min(64, int((4e7 if dtype == "bf16" else 5e6) * 32 / (kv * group) / (new * held)), 262144 // held)))
        return _paged(None, dtype, seqs, new, rng.choice([0, 0, seqs // 2, seqs - 1]), held, page, kv * group, kv, dh,
                      cap=rng.choice([0.0, 0.0, 50.0]), window=_log(rng, 8, held) if rng.random() < 0.2 else 0, slopes=rng.random() < 0.3)
    if op == "int8":
        rows, d = _log(rng, 1, 4096), _log(rng, 64, 8192)
        outs = _log(rng, 64, max(64, min(50257, int(2e11 / (rows * d)))))
        return _int8(None, dtype, rows, d, outs, rng.random() < 0.4)
    vocab = _log(rng, 64, 131072)
    rows = _log(rng, 1, max(1, min(512, 16_000_000 // vocab)))
    return _sample(None, dtype, rows, vocab, rng.choice([0.5, 1.5, 2.5, 4.0]), k=rng.choice([0, 0, _log(rng, 1, 1000)]),
                   p=rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]), min_p=rng.choice([0.0, 0.0, 0.001, 0.05]))


# ---- inputs ----

def _generator(seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def _lens(c, seed):
    """Each sequence's new tokens and the keys it holds with them: lengths that differ by up to four times, in an order of the
    seed's. Riders bring one token."""
    rng = random.Random(7919 * c["seqs"] + c["held"])
    new, held = [], []
    for b in range(c["seqs"]):
        ridden = b < c.get("riders", 0)
        n = 1 if ridden else c["new"] if c["seqs"] == 1 or c["new"] <= 4 else rng.randint(max(1, c["new"] // 2), c["new"])
        new.append(n)
        held.append(c["held"] if c["seqs"] == 1 else rng.randint(max(n, c["held"] // 4), c["held"]))
    order = list(range(c["seqs"]))
    random.Random(seed).shuffle(order)
    return [new[b] for b in order], [held[b] for b in order]


def _prepare_cache(c, seed):
    gen, t = _generator(seed), _TYPES[c["dtype"]]
    new, held = _lens(c, seed)
    width = -(-max(held) // c["page"])
    used = [-(-h // c["page"]) for h in held]
    pages = sum(used) + 3  # a few that no sequence has
    where = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)  # pages are handed out in any order
    table, at = torch.zeros((c["seqs"], width), dtype=torch.int32, device="cuda"), 0
    for b, n in enumerate(used):
        table[b, :n] = where[at:at + n]
        at += n

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(t)

    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s = {"k": normal(pages, c["page"], c["kv_heads"], c["dh"]), "v": normal(pages, c["page"], c["kv_heads"], c["dh"]), "table": table,
         "new": new, "held": held, "most": max(new),
         "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"), "lens": torch.tensor(held, dtype=torch.int32, device="cuda")}
    rows = starts[-1] + (0 if c["seqs"] == 1 else 3)  # a batch's rows are padded: what is behind the last sequence is left alone
    return s, rows, normal


def _prepare_append(c, seed):
    s, rows, normal = _prepare_cache(c, seed)
    s["new_k"], s["new_v"] = normal(rows, c["kv_heads"], c["dh"]), normal(rows, c["kv_heads"], c["dh"])
    return s


def _prepare_paged(c, seed):
    s, rows, normal = _prepare_cache(c, seed)
    s["q"] = normal(rows, c["heads"], c["dh"])
    if c["cap"]:  # wide scores, as a model with capped ones has them
        s["q"] *= 3
    s["out"] = torch.zeros_like(s["q"])
    s["lse"] = torch.zeros((rows, c["heads"]), dtype=torch.float32, device="cuda")
    s["slopes"] = torch.exp2(-8.0 * torch.arange(1, c["heads"] + 1, device="cuda") / c["heads"]) if c["slopes"] else None
    return s


def _prepare_int8(c, seed):
    gen, t = _generator(seed), _TYPES[c["dtype"]]
    x = torch.randn((c["rows"], c["d"]), generator=gen, device="cuda")
    x *= torch.exp(torch.randn((c["rows"], 1), generator=gen, device="cuda"))  # tokens differ in size
    pitch = -(-c["d"] // 16) * 16
    w = torch.zeros((c["outs"], pitch), dtype=torch.int8, device="cuda")  # rows begin at multiples of 16 bytes
    w[:, :c["d"]] = (torch.randn((c["outs"], c["d"]), generator=gen, device="cuda") * 40).round_().clamp_(-127, 127).to(torch.int8)
    scale = (0.5 + torch.rand(c["outs"], generator=gen, device="cuda")) / (40 * math.sqrt(c["d"]))
    bias = (0.3 * torch.randn(c["outs"], generator=gen, device="cuda")).to(t) if c["bias"] else None
    return {"x": x.to(t), "w": w[:, :c["d"]], "scale": scale, "b": bias}


def _prepare_sample(c, seed):
    gen, t = _generator(seed), _TYPES[c["dtype"]]
    rows = c["rows"]

    def uniform(lo, hi):
        return lo + (hi - lo) * torch.rand(rows, generator=gen, device="cuda")

    s = {"logits": (torch.randn((rows, c["vocab"]), generator=gen, device="cuda") * c["wide"]).to(t), "u": uniform(0.0, 1.0).clamp_(max=1 - 2.0 ** -24),
         "temperature": uniform(0.5, 1.3), "k": None, "p": None, "min_p": None}
    s["logits"][:, 1::97] = -math.inf  # tokens that a grammar rules out
    if rows > 3:
        s["temperature"][rows // 2] = 0.0  # some users want the most likely token
    if c["k"]:
        s["k"] = torch.randint(1, c["k"] + 1, (rows,), generator=gen, device="cuda", dtype=torch.int32)
        s["k"][0] = c["k"]
    if c["p"] < 1:
        s["p"] = c["p"] * uniform(0.9, 1.0)
    if c["min_p"]:
        s["min_p"] = c["min_p"] * uniform(0.5, 1.0)
    return s


def prepare(case, seed):
    s = {"append": _prepare_append, "paged": _prepare_paged, "int8": _prepare_int8, "sample": _prepare_sample}[case["op"]](case, seed)
    s["case"] = case
    return s


# ---- one pass, plain ----

def _plain_append(s):
    c = s["case"]
    starts, lens, table = s["starts"].long(), s["lens"].long(), s["table"].long()
    row = torch.arange(s["new_k"].shape[0], device=table.device)
    seq = torch.searchsorted(starts[1:], row, right=True)
    live = seq < c["seqs"]
    row, seq = row[live], seq[live]
    pos = lens[seq] - starts[seq + 1] + row
    page, slot = table[seq, pos // c["page"]], pos % c["page"]
    s["k"][page, slot] = s["new_k"][row]
    s["v"][page, slot] = s["new_v"][row]
    return {"k": s["k"], "v": s["v"]}


def _plain_paged(s):
    c = s["case"]
    group, at = c["heads"] // c["kv_heads"], 0
    for b, (n, held) in enumerate(zip(s["new"], s["held"])):
        pages = s["table"][b, :-(-held // c["page"])].long()
        k = s["k"][pages].flatten(0, 1)[:held].float().transpose(0, 1).contiguous()  # {kv, held, dh}
        v = s["v"][pages].flatten(0, 1)[:held].float().transpose(0, 1).contiguous()
        pos = held - n + torch.arange(n, device=k.device)
        far = pos[:, None] - torch.arange(held, device=k.device)[None, :]
        seen = far >= 0
        if c["window"]:
            seen &= far < c["window"]
        heads = 1 if n * held > 1 << 24 else c["kv_heads"]  # as many key heads at once as leave the scores a reasonable size
        for h in range(0, c["kv_heads"], heads):
            q = s["q"][at:at + n, h * group:(h + heads) * group].float().view(n, heads, group, c["dh"]).permute(1, 2, 0, 3).reshape(heads, group * n, c["dh"])
            z = torch.matmul(q, k[h:h + heads].transpose(1, 2).contiguous()).view(heads, group, n, held).mul_(1.0 / math.sqrt(c["dh"]))
            if c["cap"]:
                z = torch.tanh(z / c["cap"]) * c["cap"]
            if s["slopes"] is not None:
                z = z - s["slopes"][h * group:(h + heads) * group].view(heads, group, 1, 1) * far
            z = z.masked_fill_(~seen, -math.inf)
            top = z.amax(-1, keepdim=True)
            z = torch.exp(z.sub_(top))
            total = z.sum(-1, keepdim=True)
            o = torch.matmul(z.view(heads, group * n, held), v[h:h + heads]).view(heads, group, n, c["dh"]) / total
            s["out"][at:at + n, h * group:(h + heads) * group] = o.permute(2, 0, 1, 3).reshape(n, heads * group, c["dh"]).to(s["out"].dtype)
            s["lse"][at:at + n, h * group:(h + heads) * group] = (top + torch.log(total)).view(heads * group, n).t()
        at += n
    return {"out": s["out"], "lse": s["lse"]}


def _plain_int8(s):
    x = s["x"].float()
    scale = x.abs().amax(1) / 127
    codes = torch.where(scale[:, None] > 0, x.double() / scale.double()[:, None], 0.0).round().float()
    y = torch.matmul(codes, s["w"].float().t()) * scale[:, None] * s["scale"][None, :]
    if s["b"] is not None:
        y += s["b"].float()
    return {"y": y.to(s["x"].dtype)}


def _plain_sample(s):
    z = s["logits"].double()
    rows, vocab = z.shape
    greedy = s["temperature"] <= 0
    t = torch.where(greedy, 1.0, s["temperature"].double())
    z, order = z.sort(dim=1, descending=True, stable=True)
    w = torch.exp((z - z[:, :1]) / t[:, None])
    if s["min_p"] is not None:
        w = torch.where(w >= s["min_p"].double()[:, None], w, 0.0)
    if s["k"] is not None:
        w = torch.where(torch.arange(vocab, device=z.device)[None, :] < s["k"][:, None], w, 0.0)
    total = w.cumsum(1)
    if s["p"] is not None:
        w = torch.where(total - w < s["p"].double()[:, None] * total[:, -1:], w, 0.0)
        total = w.cumsum(1)
    at = (total <= s["u"].double()[:, None] * total[:, -1:]).sum(1).clamp(max=vocab - 1)
    at = torch.where(greedy, 0, at)[:, None]
    logprob = torch.where(greedy, 0.0, torch.log(w.gather(1, at) / total[:, -1:]).squeeze(1))
    return {"tokens": order.gather(1, at).squeeze(1).to(torch.int32), "logprob": logprob.float()}


# ---- one pass, the framework's calls ----

def _nnh():
    path = os.path.join(_ROOT, "nn-cpp_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import nnh
    return nnh


def _own_cache(s):
    if "cache" not in s:  # as a program keeps one
        s["cache"] = _nnh().PagedCache(s["k"], s["v"], s["table"])
    return s["cache"]


def _own_append(s):
    _nnh().paged_append(_own_cache(s), s["new_k"], s["new_v"], s["starts"], s["lens"])
    return {"k": s["k"], "v": s["v"]}


def _own_paged(s):
    nnh, c = _nnh(), s["case"]
    rule = nnh.AttentionRule(causal=True, window=c["window"], cap=c["cap"], slopes=s["slopes"], k_lens=s["lens"])
    out, lse = nnh.paged_attention(s["q"], _own_cache(s), s["starts"], s["most"], rule, out=s["out"], lse=s["lse"])
    return {"out": out, "lse": lse}


def _own_int8(s):
    return {"y": _nnh().linear_int8(s["x"], s["w"], s["scale"], s["b"])}


def _own_sample(s):
    tokens, logprob = _nnh().sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["k"], top_p=s["p"], min_p=s["min_p"])
    return {"tokens": tokens, "logprob": logprob}


def run(state):
    if own:
        return {"append": _own_append, "paged": _own_paged, "int8": _own_int8, "sample": _own_sample}[state["case"]["op"]](state)
    return {"append": _plain_append, "paged": _plain_paged, "int8": _plain_int8, "sample": _plain_sample}[state["case"]["op"]](state)


# ---- what a pass cannot do without ----

def work(case):
    c = case
    size = 2 if c["dtype"] == "bf16" else 4
    if c["op"] == "append":
        new, _ = _lens(c, 0)
        return {"bytes": sum(new) * c["kv_heads"] * c["dh"] * size * 4, "flops": 0}
    if c["op"] == "paged":
        new, held = _lens(c, 0)
        pairs = keys = 0
        for n, h in zip(new, held):
            most = min(h, c["window"]) if c["window"] else h  # what the last of its rows sees; the first sees n - 1 positions less far
            keys += min(h, most + n - 1)
            pairs += sum(min(most, h - n + 1 + i) for i in range(n))
        return {"bytes": size * c["dh"] * (2 * keys * c["kv_heads"] + 2 * sum(new) * c["heads"]) + 4 * sum(new) * c["heads"],
                "flops": 4 * pairs * c["heads"] * c["dh"]}
    if c["op"] == "int8":
        return {"bytes": c["rows"] * c["d"] * size + c["outs"] * (c["d"] + 4) + c["rows"] * c["outs"] * size,
                "flops": 2 * c["rows"] * c["d"] * c["outs"]}
    return {"bytes": c["rows"] * (c["vocab"] * size + 16), "flops": 0}


# ---- the same from the definitions, in 64 bits ----

def _exact_append(c, seed):
    s = _prepare_append(c, seed)
    at = 0
    k, v, table = s["k"].double(), s["v"].double(), s["table"].tolist()
    for b, (n, held) in enumerate(zip(s["new"], s["held"])):
        pos = held - n
        while pos < held:  # a page at a time
            slot = pos % c["page"]
            m = min(c["page"] - slot, held - pos)
            k[table[b][pos // c["page"]], slot:slot + m] = s["new_k"][at:at + m].double()
            v[table[b][pos // c["page"]], slot:slot + m] = s["new_v"][at:at + m].double()
            at, pos = at + m, pos + m
    return {"k": k, "v": v}


def _exact_paged(c, seed):
    s = _prepare_paged(c, seed)
    out, lse = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda"), torch.zeros(s["lse"].shape, dtype=torch.float64, device="cuda")
    group, first = c["heads"] // c["kv_heads"], 0
    for b, (n, held) in enumerate(zip(s["new"], s["held"])):
        j = torch.arange(held, device="cuda")
        page, slot = s["table"][b].long()[j // c["page"]], j % c["page"]
        for h in range(c["heads"]):
            k, v = s["k"][page, slot, h // group].double(), s["v"][page, slot, h // group].double()
            for a in range(0, n, 1024):
                m = min(1024, n - a)
                gap = (held - n + a + torch.arange(m, device="cuda"))[:, None] - j[None, :]
                z = s["q"][first + a:first + a + m, h].double() @ k.t() / math.sqrt(c["dh"])
                z = c["cap"] * torch.tanh(z / c["cap"]) if c["cap"] else z
                z = z - float(s["slopes"][h]) * gap if c["slopes"] else z
                z = torch.where((gap >= 0) & ((gap < c["window"]) if c["window"] else True), z, -math.inf)
                norm = torch.logsumexp(z, 1)
                out[first + a:first + a + m, h] = torch.exp(z - norm[:, None]) @ v
                lse[first + a:first + a + m, h] = norm
        first += n
    return {"out": out, "lse": lse}


def _exact_int8(c, seed):
    s = _prepare_int8(c, seed)
    y = torch.empty((c["rows"], c["outs"]), dtype=torch.float64, device="cuda")
    w = s["w"].double().t().contiguous()
    for a in range(0, c["rows"], 1024):
        x = s["x"][a:a + 1024].double()
        unit = (x.abs().amax(1, keepdim=True).float() / 127).double()  # a scale is a number in 32 bits
        low = torch.floor(x / unit)
        rest = x / unit - low
        codes = low + ((rest > 0.5) | ((rest == 0.5) & (low % 2 != 0))).double()
        y[a:a + 1024] = (codes @ w) * unit * s["scale"].double()[None, :] + (s["b"].double()[None, :] if c["bias"] else 0.0)
    return {"y": y}


def _exact_sample(c, seed):
    s = _prepare_sample(c, seed)
    tokens, logprob = [], []
    for r in range(c["rows"]):
        z, t = s["logits"][r].double(), float(s["temperature"][r])
        best = float(z.max())
        if t <= 0:
            tokens.append(int((z == best).nonzero()[0]))
            logprob.append(0.0)
            continue
        p = torch.softmax(z / t, 0)
        keep = torch.ones(c["vocab"], dtype=torch.bool, device="cuda")
        if s["min_p"] is not None:
            keep &= p / p.max() >= float(s["min_p"][r])
        # by descending logits; among equal ones the lowest index comes first
        rank = torch.argsort(z, descending=True, stable=True)
        rank = rank[keep[rank]]
        if s["k"] is not None:
            rank = rank[:int(s["k"][r])]
        q = p[rank] / p[rank].sum()
        if s["p"] is not None:
            before = torch.cat([q.new_zeros(1), q.cumsum(0)[:-1]])
            rank = rank[before < float(s["p"][r])]
            q = p[rank] / p[rank].sum()
        i = min(int((q.cumsum(0) <= float(s["u"][r])).sum()), len(rank) - 1)
        tokens.append(int(rank[i]))
        logprob.append(math.log(float(q[i])))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "logprob": torch.tensor(logprob, dtype=torch.float64)}


def exact(case, seed):
    return {"append": _exact_append, "paged": _exact_paged, "int8": _exact_int8, "sample": _exact_sample}[case["op"]](case, seed)
