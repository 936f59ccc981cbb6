"""Definitions in 64 bits (CPU) of the operators for adapting a matcher, and how far a computation may be from them.

Bounds.  u = finfo(type).eps / 2 is the relative error of one rounding (at least half of the smallest subnormal, `tiny`, in
absolute terms).  fp32 arithmetic over n terms whose exponents' arguments reach x is given e = 2^-24 (n + 64 + 16 x): n for the
sums, 16 x for arguments of exp2 (each of a handful of roundings of a number of size x log2(e) moves the result by its own size), 64
for everything that happens a fixed number of times."""
import math

import torch

INF = math.inf


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def attention(q, k, v, causal=False, scale=None, q_lens=None, k_lens=None, do=None):
    """o, lse (and dq, dk, dv) with the bounds of each: dict name -> (value, bound).  Inputs: CPU tensors of the tested type."""
    dt = q.dtype
    u, t = unit(dt), tiny(dt)
    B, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G = Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    out = {n: (torch.zeros(s, dtype=torch.float64), torch.zeros(s, dtype=torch.float64))
           for n, s in (("o", q.shape), ("dq", q.shape), ("dk", k.shape), ("dv", v.shape))}
    out["lse"] = (torch.full((B, Hq, Lq), -INF, dtype=torch.float64), torch.zeros((B, Hq, Lq), dtype=torch.float64))
    round_p = 0.0 if dt == torch.float32 else u            # the probabilities and ds are rounded for the second product
    # exp2 gives 0 where its result is below fp32's smallest normal 2^-126, and so does a conversion to bf16 of such a number: an error
    # of up to 2^-126 in a probability, and with it of 2^-126 (|dp| + |delta|) in ds
    tiny_p = max(t, 2.0 ** -126)
    for b in range(B):
        nq = Lq if q_lens is None else min(max(int(q_lens[b]), 0), Lq)
        nk = Lk if k_lens is None else min(max(int(k_lens[b]), 0), Lk)
        if nq == 0 or nk == 0:
            continue
        see = torch.ones(nq, nk, dtype=torch.bool)
        if causal:
            see = torch.arange(nk)[None, :] <= torch.arange(nq)[:, None] + (nk - nq)
        some = see.any(1, keepdim=True)
        for h in range(Hq):
            Q, K, V = (x.double() for x in (q[b, :nq, h], k[b, :nk, h // G], v[b, :nk, h // G]))
            x = scale * (Q @ K.T)
            size = float((scale * (Q.abs() @ K.abs().T)).max())
            x = x.masked_fill(~see, -INF)
            top = x.amax(1, keepdim=True).masked_fill(~some, 0.0)
            p = torch.exp(x - top)
            total = p.sum(1, keepdim=True)
            p = p / total.masked_fill(~some, 1.0)
            lse = (top + total.log()).squeeze(1)
            biggest = max(size, float(lse[some[:, 0]].abs().max()) if some.any() else 0.0)
            e = 2.0 ** -24 * (nk + nq * G + 2 * D + 64 + 16 * biggest)
            mass = p @ V.abs()
            out["o"][0][b, :nq, h] = p @ V
            out["o"][1][b, :nq, h] = (round_p + e) * mass + tiny_p * (see.double() @ V.abs()) + u * (p @ V).abs() + t
            out["lse"][0][b, h, :nq] = lse
            out["lse"][1][b, h, :nq] = e * (1 + lse.abs().nan_to_num(0, 0, 0))
            if do is None:
                continue
            g = do[b, :nq, h].double()
            dp, delta = g @ V.T, (g * (p @ V)).sum(1, keepdim=True)
            ds = p * (dp - delta)
            # delta is taken from the rounded o; dp and delta are sums of D terms
            o_err = out["o"][1][b, :nq, h]
            ds_err = p * ((g.abs() * o_err).sum(1, keepdim=True) + e * (g.abs() @ V.abs().T + (g.abs() * mass).sum(1, keepdim=True))) \
                + (round_p + e) * ds.abs() + tiny_p * see * (1 + dp.abs() + delta.abs())
            out["dq"][0][b, :nq, h] = scale * (ds @ K)
            out["dq"][1][b, :nq, h] = scale * ((ds_err + e * ds.abs()) @ K.abs())
            out["dk"][0][b, :nk, h // G] += scale * (ds.T @ Q)
            out["dk"][1][b, :nk, h // G] += scale * ((ds_err + e * ds.abs()).T @ Q.abs())
            out["dv"][0][b, :nk, h // G] += p.T @ g
            out["dv"][1][b, :nk, h // G] += ((round_p + 2 * e) * p + tiny_p * see).T @ g.abs()
    for n in ("dq", "dk", "dv"):
        out[n] = (out[n][0], out[n][1] + u * out[n][0].abs() + t)
    return out if do is not None else {n: out[n] for n in ("o", "lse")}


def _row_error(z, classes):
    finite = z[torch.isfinite(z)]
    return 2.0 ** -24 * (classes / 64 + 64 + 16 * (float(finite.abs().max()) if finite.numel() else 0.0))


def log_probs(logits, targets=None, top=0, scale=1.0, d_log_prob=None, d_entropy=None):
    """dict name -> (value, bound); top_index has no bound.  targets [R, n]."""
    u, t = unit(logits.dtype), tiny(logits.dtype)
    scale = float(torch.tensor(scale, dtype=torch.float32))
    z = scale * logits.double()
    R, V = z.shape
    e = _row_error(z, V)
    broken = (torch.isnan(z) | (z == INF)).any(1)
    empty = (z < -2.0 ** 100).all(1)                       # allows nothing
    lse = torch.where(empty, -INF, torch.logsumexp(z, 1))
    lp = torch.where(empty[:, None], torch.full_like(z, -INF), z - lse[:, None])
    p = torch.where(lp == -INF, torch.zeros_like(lp), lp.exp())
    plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
    H = -plp.sum(1)
    lse, H = torch.where(broken, torch.nan, lse), torch.where(broken, torch.nan, H)
    lp = torch.where(broken[:, None], torch.nan, lp)

    def around(x):
        return e * (1 + x.abs().nan_to_num(0, 0, 0))

    out = {"lse": (lse, around(lse)), "entropy": (H, 4 * e * (1 + H.nan_to_num(0) + (p * lp.nan_to_num(0, 0, 0) ** 2).nan_to_num(0).sum(1)))}
    if targets is not None:
        at = targets.long()
        inside = (at >= 0) & (at < V)
        w = torch.where(inside, lp.gather(1, at.clamp(0, V - 1)), 0.0)
        out["log_prob"] = (w, around(w))
    if top:
        order = torch.sort(logits.double() + 0.0, dim=1, descending=True, stable=True)[1][:, :top]
        w = lp.gather(1, order)
        out["top_index"] = (torch.where(broken[:, None], -1, order), None)
        out["top_log_prob"] = (w, around(w))
    if d_log_prob is not None or d_entropy is not None:
        d, size = torch.zeros_like(z), torch.zeros_like(z)
        live = (~empty)[:, None]
        if d_log_prob is not None:
            at = targets.long()
            g = torch.where((at >= 0) & (at < V) & live, d_log_prob.double(), 0.0)
            d = d - p * g.sum(1, keepdim=True)
            size = size + p * g.abs().sum(1, keepdim=True)
            d.scatter_add_(1, at.clamp(0, V - 1), g)
            size.scatter_add_(1, at.clamp(0, V - 1), g.abs())
        if d_entropy is not None:
            h = torch.where(live[:, 0], d_entropy.double(), 0.0)[:, None]
            d = d - h * (plp + p * H[:, None])
            size = size + h.abs() * (p * (1 + H.abs()[:, None]) + plp.abs())
        d = torch.where(broken[:, None], torch.nan, d * scale)
        out["d_logits"] = (d, (u * d.abs() + 4 * e * scale * size).nan_to_num(0) + t)
    return out


def distill(logits, index, value, temperature=1.0, tail=False, d_loss=None):
    u, t = unit(logits.dtype), tiny(logits.dtype)
    scale = float(torch.tensor(1.0 / temperature, dtype=torch.float32))
    z = scale * logits.double()
    R, V = z.shape
    e = _row_error(z, V) + _row_error(torch.where((index >= 0) & (index < V), value, 0.0).double(), 1)
    used = (index >= 0) & (index < V)
    at = index.long().clamp(0, V - 1)
    lse = torch.logsumexp(z, 1)
    lq = (z - lse[:, None]).gather(1, at)
    a = torch.where(used, value.double(), -INF)
    if tail:
        lp, p = a, a.exp()
    else:
        a = a * scale
        none = ~used.any(1, keepdim=True)
        lp = a - torch.logsumexp(a.masked_fill(none, 0.0), 1, keepdim=True)
        p = torch.where(used & ~none, lp.exp(), 0.0)
    terms = torch.where(p > 0, p * (lp - lq), 0.0)
    size = torch.where(p > 0, p * (1 + lp.abs() + lq.abs()), 0.0).sum(1)
    loss, mass = terms.sum(1), p.sum(1)
    share = torch.zeros_like(z).scatter_add_(1, at, p)
    q = (z - lse[:, None]).exp()
    spread = q * mass[:, None] + share
    if tail:
        rest = (1 - mass).clamp(min=0)
        rest = torch.where(rest < 2.0 ** -20, 0.0, rest)
        named = torch.zeros_like(z).scatter_add_(1, at, used.double()) > 0
        log_tail = torch.logsumexp(z.masked_fill(named, -INF), 1) - lse
        loss = loss + torch.where(rest > 0, rest * (rest.clamp(min=1e-300).log() - log_tail), 0.0)
        size = size + torch.where(rest > 0, rest * (1 + log_tail.abs().nan_to_num(0, 0, 0) + rest.clamp(min=1e-300).log().abs()), 0.0)
        mass = mass + rest
        w = torch.where(named, 0.0, (z - lse[:, None] - log_tail.nan_to_num(0, 0, 0)[:, None]).exp())
        share = share + rest[:, None] * w
        spread = q * mass[:, None] + share
    out = {"loss": (loss, 4 * e * (1 + size)), "lse": (lse, e * (1 + lse.abs()))}
    if tail:
        out["log_tail"] = (log_tail, 2 * e * (1 + log_tail.abs().nan_to_num(0, 0, 0)))
    if d_loss is not None:
        g = d_loss.double()[:, None] * scale
        d = g * (q * mass[:, None] - share)
        out["d_logits"] = (d, u * d.abs() + 4 * e * g.abs() * spread + t)
    return out


def check(got, want, what=""):
    """every name of `want` within its bound of the GPU's (or any) tensor in `got`"""
    for name, (value, bound) in want.items():
        x = got[name].detach().cpu()
        assert x.shape == value.shape, (what, name, x.shape, value.shape)
        if bound is None:
            assert torch.equal(x.long(), value.long()), (what, name, (x.long() != value.long()).nonzero()[:4])
            continue
        x = x.double()
        same = torch.isnan(value) & torch.isnan(x) | (value == x)
        off = torch.where(same, torch.zeros_like(x), (x - value).abs())
        bad = ~(off <= bound) & ~same
        assert not bad.any(), (what, name, int(bad.sum()), "of", x.numel(), "first", bad.nonzero()[0].tolist(),
                               float(x[tuple(bad.nonzero()[0])]), float(value[tuple(bad.nonzero()[0])]), float(bound[tuple(bad.nonzero()[0])]))
