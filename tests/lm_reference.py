"""Plain 64-bit forms of the operators of language models, with a bound on what rounding may do to each output.

A rounding to a type t is off by at most u(t) = finfo(t).eps / 2 of the value. The bounds below add up, to first order, what
the formulas' roundings can do: products accumulated in fp32 over K terms (K u32 of the sum of absolute values), the
exponential and the capped score's tanh (a few u32), and, for bf16 operands, the roundings that the kernels document: the
probabilities and score gradients as operands of a product, and the stored results."""
import math

import torch

U32 = torch.finfo(torch.float32).eps / 2


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def visible(N, Tq, Tk, causal=False, window=0, q_start=None, k_lens=None, prefix=None, q_docs=None, k_docs=None):
    i = torch.arange(Tq)[None, :, None] + (torch.zeros(N, dtype=torch.long) if q_start is None else q_start.long().cpu())[:, None, None]
    j = torch.arange(Tk)[None, None, :]
    see = torch.ones(N, Tq, Tk, dtype=torch.bool)
    if causal:
        see &= j <= i
    if window:
        see &= (i - j).abs() < window
    if prefix is not None:
        see |= j < prefix.long().cpu()[:, None, None]
    if k_lens is not None:
        see &= j < k_lens.long().cpu()[:, None, None]
    if q_docs is not None:
        qd, kd = q_docs.cpu()[:, :, None], k_docs.cpu()[:, None, :]
        see &= (qd == kd) & (kd >= 0)
    return see, (i - j).abs().double()


def masked_attention(q, k, v, g=None, scale=0.0, cap=0.0, slopes=None, **mask):
    """{name: (value, bound)} of out, lse and, with g, dq, dk, dv; q {N, Tq, H, D}, k and v {N, Tk, Hkv, D}. Values of keys
    and queries that no pair uses do not matter, finite or not."""
    t = q.dtype
    u = unit(t) if t != torch.float32 else 0.0
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    N, Tq, H, D = q.shape
    Tk, grp = k.shape[1], H // k.shape[2]
    scale = scale or 1.0 / math.sqrt(D)
    see, far = visible(N, Tq, Tk, **mask)
    kq = see.any(2)  # queries and keys that are in use
    kk = see.any(1)
    q = torch.where(kq[:, :, None, None], q, 0.0)
    k, v = (torch.where(kk[:, :, None, None], x, 0.0) for x in (k, v))
    Q, K, V = q.transpose(1, 2), k.transpose(1, 2).repeat_interleave(grp, 1), v.transpose(1, 2).repeat_interleave(grp, 1)
    see, far = see[:, None], far[:, None]
    s = scale * Q @ K.transpose(2, 3)
    es = (D + 2) * U32 * scale * (Q.abs() @ K.abs().transpose(2, 3))
    th = torch.tanh(s / cap) if cap else None
    z = cap * th if cap else s
    # the 16-bit kernels' tanh is off by up to 4 u32 of 1 (its reciprocal and exponential), the 32-bit ones' by as much of it
    ez = es + (4 * U32 * (cap if t != torch.float32 else (cap * th).abs()) + 4 * U32 * z.abs() if cap else 2 * U32 * z.abs())
    if slopes is not None:
        b = slopes.double().cpu()[None, :, None, None] * far
        z = z - b
        ez = ez + 4 * U32 * (b + z.abs())
    z = torch.where(see, z, -math.inf)
    lse = torch.logsumexp(z, 3)
    p = torch.where(see, torch.exp(z - torch.where(lse == -math.inf, 0.0, lse)[..., None]), 0.0)
    ez = torch.where(see, ez + 4 * U32 * (1 + z.abs().nan_to_num(posinf=0.0)), 0.0)
    worst = ez.amax(3, keepdim=True) if Tk else ez.sum(3, keepdim=True)  # of a row's scores: what its maximum and sum can be off by
    ep = p * (ez + worst + (Tk + 8) * U32)
    o = p @ V
    eo = (ep + p * (u + Tk * U32)) @ V.abs()
    back = lambda x: x.transpose(1, 2)  # noqa: E731
    stored = lambda x, e: (back(x), back(e + (u + 2 * U32) * (x.abs() + e)))  # noqa: E731
    res = {"out": stored(o, eo), "lse": (lse, worst[..., 0] + (Tk + 4) * U32 + 4 * U32 * lse.abs().nan_to_num(posinf=0.0))}
    if g is None:
        return res
    G = torch.where(kq[:, :, None, None], g.detach().cpu().double(), 0.0).transpose(1, 2)
    dp = G @ V.transpose(2, 3)
    delta = (G * o).sum(3, keepdim=True)
    # delta is taken from the stored out
    ed = (G.abs() * (eo + (u + 2 * U32) * (o.abs() + eo))).sum(3, keepdim=True) + D * U32 * (G.abs() * o.abs()).sum(3, keepdim=True)
    edp = (D + 2) * U32 * (G.abs() @ V.abs().transpose(2, 3))
    ep = ep + 4 * U32 * p * (1 + lse.abs().nan_to_num(posinf=0.0))[..., None]
    bend = 1.0 - th * th if cap else torch.ones_like(s)
    ds = p * (dp - delta) * bend
    eds = ep * (dp - delta).abs() * bend + p * (edp + ed) * bend + (u + 6 * U32) * ds.abs()
    if cap:
        eds = eds + p * (dp - delta).abs() * 12 * U32 + p * (dp - delta).abs() * 2 * th.abs() * es / cap
    fold = lambda x: x.view(N, H // grp, grp, Tk, D).sum(2)  # noqa: E731
    res["dq"] = stored(scale * ds @ K, scale * (eds + Tk * U32 * ds.abs()) @ K.abs())
    st, est = ds.transpose(2, 3), (eds + Tq * grp * U32 * ds.abs()).transpose(2, 3)
    res["dk"] = stored(fold(scale * st @ Q), fold(scale * est @ Q.abs()))
    pt, ept = p.transpose(2, 3), (ep + p * (u + Tq * grp * U32)).transpose(2, 3)
    res["dv"] = stored(fold(pt @ G), fold(ept @ G.abs()))
    return res


def assert_within(got, want, what=""):
    """got (a tensor) against (value, bound), not finite values included."""
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    fine = torch.isfinite(value)
    assert torch.equal(torch.isnan(got), torch.isnan(value)), f"{what}: NaN in other places"
    assert torch.equal(got[~fine].nan_to_num(nan=0.0), value[~fine].nan_to_num(nan=0.0)), f"{what}: infinities differ"
    over = (got - value).abs()[fine] - bound[fine]
    if over.numel() and over.max() > 0:
        at = int(over.argmax())
        raise AssertionError(f"{what}: {int((over > 0).sum())} of {over.numel()} out of bounds; worst: got "
                             f"{got[fine][at].item()}, want {value[fine][at].item()} within {bound[fine][at].item()}")


# ---- AdamW ----

E4M3 = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()  # 0 .. 448


def nearest_e4m3(x):
    """The nearest e4m3 values of |x| <= 448, ties to the even code."""
    border, a = (E4M3[1:] + E4M3[:-1]) / 2, x.abs()
    low, high = torch.searchsorted(border, a), torch.searchsorted(border, a, right=True)
    return torch.copysign(E4M3[torch.where(low % 2 == 0, low, high)], x)


def block_codes(x, root):
    """Moments as 8-bit codes and scale bytes (root: x is v, kept as its square root), and the values they stand for."""
    n = x.numel()
    y = torch.nn.functional.pad(x.sqrt() if root else x, (0, -n % 64)).view(-1, 64)
    fine = torch.where(torch.isfinite(y), y, 0.0)
    top = fine.abs().amax(1, keepdim=True)
    e = torch.where(top > 0, (torch.frexp(top).exponent - 8 + 127).clamp(0, 254), 0)
    unit = torch.tensor([math.ldexp(1.0, k - 127) for k in range(255)], dtype=torch.float64)[e.long()]
    q = nearest_e4m3(fine / unit)
    if root:
        q = torch.where((fine > 0) & (q == 0), 2.0 ** -9, q)
    q = torch.where(torch.isfinite(y), q, math.nan)
    return q.view(-1)[:n], e.view(-1).to(torch.uint8), (q * unit).view(-1)[:n]


def adamw(p, g, m, v, step, lr, beta1, beta2, eps, weight_decay, scale=1.0):
    """One step in 64 bits: new p, m and v."""
    p, g, m, v = p.double(), g.double() * scale, m.double(), v.double()
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    new = p - lr * weight_decay * p - lr * (m / (1 - beta1 ** step)) / ((v / (1 - beta2 ** step)).sqrt() + eps)
    return new, m, v


# ---- linear cross entropy ----

def linear_cross_entropy(x, w, targets, bias=None, reduction="mean", g=None, kept=False):
    """{name: (value, bound)} of loss, lse, dx, dw and, with a bias, db. kept: the call that rounds exp(z) to bf16 before dz."""
    t = x.dtype
    u = unit(t) if t != torch.float32 else 0.0
    x, w, targets = x.detach().cpu().double(), w.detach().cpu().double(), targets.cpu().long()
    b = torch.zeros(w.shape[0], dtype=torch.float64) if bias is None else bias.detach().cpu().double()
    D, V, rows = x.shape[1], w.shape[0], x.shape[0]
    z = x @ w.t() + b
    ez = (D + 2) * U32 * (x.abs() @ w.abs().t() + b.abs()) + 4 * U32 * (1 + z.abs())
    worst = ez.amax(1, keepdim=True)
    lse = torch.logsumexp(z, 1)
    el = worst[:, 0] + (V + 8) * U32 + 4 * U32 * lse.abs()
    live = (targets >= 0) & (targets < V)
    count = int((targets >= 0).sum())
    at = targets.clamp(0, V - 1)[:, None]
    each = torch.where(live, lse - z.gather(1, at)[:, 0], torch.where(targets < 0, 0.0, math.nan))
    ee = (el + ez.gather(1, at)[:, 0] + 2 * U32 * (lse.abs() + each.abs().nan_to_num())) * live
    up = torch.ones(rows if reduction == "none" else (), dtype=torch.float64) if g is None else g.detach().cpu().double()
    # the 32-bit calls' last sums are in 64 bits
    if reduction == "none":
        loss, eloss, f = each, ee, up[:, None]
    elif reduction == "sum":
        loss, eloss, f = each.sum(), ee.sum() + 2 * U32 * each.sum().abs(), up
    else:
        loss = each.sum() / count if count else torch.tensor(math.nan, dtype=torch.float64)
        eloss, f = ee.sum() / max(1, count) + 2 * U32 * loss.abs(), up / max(1, count)
    p = torch.exp(z - lse[:, None])
    ep = p * (ez + el[:, None] + 4 * U32 * (1 + z.abs() + lse.abs()[:, None]))
    hot = torch.zeros_like(p)
    hot[live, targets[live]] = 1.0
    dz, edz = (p - hot) * live[:, None], (ep + 2 * U32 * (p + hot)) * live[:, None]
    edz = edz + (u * p if kept else 0.0) + u * (dz.abs() + edz)
    if reduction == "none":  # a factor for each row is part of dz
        dz, edz, f = dz * f, (edz + 2 * U32 * dz.abs()) * f.abs(), 1.0
    f = torch.as_tensor(f, dtype=torch.float64)

    def stored(v, e):
        v, e = f * v, f.abs() * e
        return v, e + (u + 6 * U32) * (v.abs() + e) + 1e-45

    res = {"loss": (loss, eloss), "lse": (lse, el)}
    res["dx"] = stored(dz @ w, (edz + V * U32 * dz.abs()) @ w.abs())
    res["dw"] = stored(dz.t() @ x, (edz + rows * U32 * dz.abs()).t() @ x.abs())
    if bias is not None:
        res["db"] = stored(dz.sum(0), (edz + rows * U32 * dz.abs()).sum(0))
    return res
