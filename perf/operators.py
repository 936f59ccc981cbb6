"""Cases of the matcher-training operators: attention with its backward pass, log probabilities of given candidates, and
distillation from a teacher's top alternatives.

`run` computes a case in plain torch (32 bits, rounded once at the end) while `own` is false, and through the package's entry
points when it is true.  `exact` is the definition of the same outputs in 64 bits; its gradients come from autograd.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------ cases
def _attn(name, op, dtype, batch, q_heads, kv_heads, q_len, k_len, head_dim, causal=False, ragged=0.0):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "q_len": q_len,
            "k_len": k_len, "head_dim": head_dim, "causal": causal, "ragged": ragged}


def _rows(name, op, dtype, rows, classes, stride=0, top=0, scale=1.0, masked=0.0):
    return {"name": name, "op": op, "dtype": dtype, "rows": rows, "classes": classes, "stride": stride or classes, "top": top,
            "scale": scale, "masked": masked}


def _distill(name, dtype, rows, classes, stride=0, listed_per_row=8, temperature=1.0, tail=False, unused=0.0):
    return {"name": name, "op": "distill", "dtype": dtype, "rows": rows, "classes": classes, "stride": stride or classes,
            "top": listed_per_row, "temperature": temperature, "tail": tail, "unused": unused}


def listed():
    return [
        # a fine-tuning step of one matcher layer: the images of eight pairs, four heads of 64, up to 1024 keypoints each
        _attn("attn-train-matcher", "attn_train", "bf16", 16, 4, 4, 1024, 1024, 64, ragged=0.25),
        # the same arithmetic over a long token sequence, causal, key heads shared by four query heads
        _attn("attn-train-causal-shared", "attn_train", "bf16", 2, 16, 4, 4096, 4096, 128, causal=True),
        # cross attention of ragged batches, odd lengths and a head size between the usual ones
        _attn("attn-train-odd", "attn_train", "f16", 3, 6, 2, 517, 1333, 80, ragged=0.6),
        # training in the matcher's own 32 bits, 1000 keypoints (the default of the detector)
        _attn("attn-train-f32", "attn_train", "f32", 4, 4, 4, 1000, 1000, 64),
        # one pair of frames through one layer: where latency counts
        _attn("attn-one-pair", "attn", "f16", 2, 4, 4, 512, 512, 64, ragged=0.3),
        # one new token per sequence against a long ragged cache
        _attn("attn-single-token", "attn", "bf16", 32, 32, 8, 1, 16384, 128, causal=True, ragged=0.5),
        # the next token of one sequence, with the alternatives a user is shown
        _rows("logp-one-token", "logp", "bf16", 1, 131072, top=20),
        # scoring a batch of given sequences; rows of an odd length, so most start off a 16-byte boundary
        _rows("logp-prompt", "logp", "bf16", 2048, 100003, top=5, scale=1 / 0.7),
        # the log-assignments of eight pairs: 1024 keypoints and the dustbin, the matcher's padded rows
        _rows("logp-assignment", "logp", "f32", 8 * 1025, 1025, stride=1028, top=4),
        # a policy step: log probability and entropy with their gradients, an eighth of the vocabulary masked out
        _rows("logp-train-masked", "logp_train", "f16", 1024, 50257, masked=0.125),
        # a student of the matcher: the teacher's eight best candidates of each keypoint and one bucket for the rest
        _distill("distill-assignment", "f32", 8 * 1025, 1025, stride=1028, tail=True, unused=0.2),
        # a student over a large vocabulary, 64 of the teacher's logits kept
        _distill("distill-vocabulary", "bf16", 2048, 131072, listed_per_row=64, temperature=2.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn_train", "attn_train", "attn", "attn", "logp", "logp", "logp_train", "distill", "distill"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op in ("attn_train", "attn"):
        kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 1, 2, 4, 8])
        head_dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
        causal, ragged = rng.random() < 0.5, rng.choice([0.0, 0.0, 0.3, 0.9])
        k_len = _log(rng, 1, 8192 if op == "attn_train" else 32768)
        q_len = 1 if op == "attn" and rng.random() < 0.4 else min(_log(rng, 1, 8192), k_len) if causal else _log(rng, 1, 8192)
        # at most half of the largest listed case's scores, and tensors of at most 2^27 elements
        most = (1 << 28) if dtype != "f32" else (1 << 26)
        while q_len * k_len * kv_heads * group > most:
            q_len, k_len = max(1, q_len * 2 // 3), max(1, k_len * 2 // 3)
        batch = max(1, min(_log(rng, 1, 48), most // (q_len * k_len * kv_heads * group), (1 << 27) // (k_len * kv_heads * head_dim),
                           (1 << 27) // (q_len * kv_heads * group * head_dim)))
        c = _attn("", op, dtype, batch, kv_heads * group, kv_heads, q_len, k_len, head_dim, causal, ragged)
    else:
        classes = _log(rng, 2, 200000)
        rows = max(1, min(_log(rng, 1, 16384), (1 << 26) // classes))
        stride = classes + rng.choice([0, 0, 0, 3, 16])
        top = min(classes, rng.choice([1, 4, 8, 20, 32, 64]))
        if op == "distill":
            c = _distill("", dtype, rows, classes, stride, top, rng.choice([1.0, 1.0, 2.0]), top < classes // 2 and rng.random() < 0.5,
                         rng.choice([0.0, 0.3]))
        else:
            c = _rows("", op, dtype, rows, classes, stride, rng.choice([0, top]) if op == "logp" else 0, rng.choice([1.0, 1 / 0.7]),
                      rng.choice([0.0, 0.0, 0.3]))
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def _lengths(c, length, step):
    """Rows in use of each sequence: between (1 - ragged) and all of `length`, the same for every seed."""
    if not c["ragged"]:
        return None
    return [max(1, length - int(c["ragged"] * length * ((b * step) % 1.0))) for b in range(c["batch"])]


def _as_tensor(lengths):
    return None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dt)

    s = {"case": dict(case)}
    if case["op"] in ("attn", "attn_train"):
        B, D = case["batch"], case["head_dim"]
        s["q"] = normal(B, case["q_len"], case["q_heads"], D)
        s["k"] = normal(B, case["k_len"], case["kv_heads"], D)
        s["v"] = normal(B, case["k_len"], case["kv_heads"], D)
        s["q_lens"] = _as_tensor(None if case["q_len"] == 1 else _lengths(case, case["q_len"], 0.381966))
        s["k_lens"] = _as_tensor(_lengths(case, case["k_len"], 0.618034))
        if case["op"] == "attn_train":
            s["do"] = normal(B, case["q_len"], case["q_heads"], D)
        return s
    R, V = case["rows"], case["classes"]
    # a few candidates stand out of each row, as a trained model's do
    z = torch.randn((R, case["stride"]), generator=g, device="cuda").mul_(2.0)
    peaks = torch.randint(0, V, (R, 4), generator=g, device="cuda")
    z.scatter_add_(1, peaks, torch.rand((R, 4), generator=g, device="cuda") * 12)
    if case["op"] == "distill":
        K = case["top"]
        teacher = z[:, :V] + torch.randn((R, V), generator=g, device="cuda")
        s["teacher_value"], index = torch.topk(teacher, K, dim=1)
        if case["tail"]:
            s["teacher_value"] = s["teacher_value"] / case["temperature"] - torch.logsumexp(teacher / case["temperature"], 1, keepdim=True)
        if case["unused"]:
            drop = torch.rand((R, K), generator=g, device="cuda") < case["unused"]
            index = torch.where(drop, torch.full_like(index, -1), index)
        s["teacher_index"] = index.to(torch.int32)
        s["d_loss"] = torch.rand(R, generator=g, device="cuda")      # of a scaled sum
        s["logits"] = z.to(dt)[:, :V]
        return s
    s["targets"] = torch.where(torch.rand(R, generator=g, device="cuda") < 0.5, peaks[:, 0],
                               torch.randint(0, V, (R,), generator=g, device="cuda")).to(torch.int32)
    if case["masked"]:
        kept = z.gather(1, peaks[:, :1])          # a grammar leaves a token to choose
        z.masked_fill_(torch.rand(z.shape, generator=g, device="cuda") < case["masked"], -math.inf)
        z.scatter_(1, peaks[:, :1], kept)
    s["logits"] = z.to(dt)[:, :V]
    if case["op"] == "logp_train":
        s["d_log_prob"] = torch.randn(R, generator=g, device="cuda")
        s["d_entropy"] = torch.randn(R, generator=g, device="cuda")
    return s


# ------------------------------------------------------------------ plain forms
def _visible(c, q_lens, k_lens, device):
    """[B or 1, 1, q_len, k_len]: query row i of a sequence sees key j"""
    i = torch.arange(c["q_len"], device=device).view(1, -1, 1)
    j = torch.arange(c["k_len"], device=device).view(1, 1, -1)
    nq = c["q_len"] if q_lens is None else q_lens.view(-1, 1, 1)
    nk = c["k_len"] if k_lens is None else k_lens.view(-1, 1, 1)
    see = (i < nq) & (j < nk)
    if c["causal"]:
        see = see & (j <= i + (nk - nq))
    return see.unsqueeze(1)


def _plain_attention(s):
    c = s["case"]
    B, Hq, Hk, Lq, Lk, D = c["batch"], c["q_heads"], c["kv_heads"], c["q_len"], c["k_len"], c["head_dim"]
    G, scale = Hq // Hk, 1 / math.sqrt(D)

    def heads(x):      # [B, L, Hk * G, D] -> [B, Hk, G * L, D]
        return x.float().view(B, x.shape[1], Hk, -1, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)

    def back(x, L):    # [B, Hk, G * L, D] -> [B, L, Hk * G, D] in the inputs' type
        return x.view(B, Hk, -1, L, D).permute(0, 3, 1, 2, 4).reshape(B, L, -1, D).to(s["q"].dtype)

    q, k, v = heads(s["q"]), heads(s["k"]), heads(s["v"])
    see = _visible(c, s["q_lens"], s["k_lens"], q.device).unsqueeze(1)
    x = torch.matmul(q, k.transpose(2, 3)).mul_(scale).view(B, Hk, G, Lq, Lk)
    x = torch.where(see, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    lse = torch.log(total) + top
    p = (p / torch.where(total == 0, 1.0, total)).view(B, Hk, G * Lq, Lk)
    o = torch.matmul(p, v)
    out = {"o": back(o, Lq), "lse": lse.view(B, Hq, Lq)}
    if c["op"] == "attn_train":
        do = heads(s["do"])
        dp = torch.matmul(do, v.transpose(2, 3))
        ds = p * (dp - (do * o).sum(-1, keepdim=True)) * scale
        # rows behind the sequences' ends have no probabilities: they add nothing
        out["dq"] = back(torch.matmul(ds, k), Lq)
        out["dk"] = back(torch.matmul(ds.transpose(2, 3), q), Lk)
        out["dv"] = back(torch.matmul(p.transpose(2, 3), do), Lk)
    return out


def _plain_log_probs(s):
    c = s["case"]
    z = s["logits"].float() * c["scale"]
    top = z.amax(1, keepdim=True)
    x = z - top
    e = torch.exp(x)
    total = e.sum(1, keepdim=True)
    lp = x - torch.log(total)
    p = e / total
    plp = torch.where(p > 0, p * lp, 0.0)
    entropy = -plp.sum(1)
    at = s["targets"].long().view(-1, 1)
    out = {"log_prob": lp.gather(1, at).view(-1), "entropy": entropy, "lse": (torch.log(total) + top).view(-1)}
    if c["top"]:
        # the order of the logits themselves, equal ones by index
        index = torch.sort(s["logits"].float(), dim=1, descending=True, stable=True)[1][:, :c["top"]]
        out["top_index"], out["top_log_prob"] = index.to(torch.int32), lp.gather(1, index)
    if c["op"] == "logp_train":
        g, h = s["d_log_prob"].view(-1, 1), s["d_entropy"].view(-1, 1)
        d = -g * p - h * (plp + p * entropy.view(-1, 1))
        d.scatter_add_(1, at, g)
        out["d_logits"] = (d * c["scale"]).to(s["logits"].dtype)
    return out


def _plain_distill(s):
    c = s["case"]
    T = c["temperature"]
    z = s["logits"].float() / T
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    q = e / total
    used = s["teacher_index"] >= 0
    at = torch.where(used, s["teacher_index"], 0).long()
    lq = (z - top).gather(1, at) - torch.log(total)
    a = s["teacher_value"].float()
    if c["tail"]:
        p = torch.where(used, torch.exp(a), 0.0)
        lp = a
    else:
        a = torch.where(used, a / T, -math.inf)
        most = a.amax(1, keepdim=True)
        ea = torch.where(used, torch.exp(a - most), 0.0)
        sum_a = ea.sum(1, keepdim=True)
        p = ea / torch.where(sum_a == 0, 1.0, sum_a)
        lp = a - most - torch.log(sum_a)
    loss = torch.where(p > 0, p * (lp - lq), 0.0).sum(1, keepdim=True)
    mass = p.sum(1, keepdim=True)
    spare = torch.zeros_like(q)
    spare.scatter_add_(1, at, p)                 # unused entries add zero
    if c["tail"]:
        rest = (1 - p.double().sum(1, keepdim=True)).clamp(min=0).float()
        rest = torch.where(rest < 2.0 ** -20, 0.0, rest)
        named = torch.zeros_like(q)
        named.scatter_add_(1, at, used.float())
        rest_e = torch.where(named > 0, 0.0, e)
        rest_total = rest_e.sum(1, keepdim=True)
        log_tail = torch.log(rest_total) - torch.log(total)
        loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - log_tail), 0.0)
        mass = mass + rest
        spare = spare + rest * rest_e / torch.where(rest_total > 0, rest_total, 1.0)
    d = (q * mass - spare) * (s["d_loss"].view(-1, 1) / T)
    return {"loss": loss.view(-1), "lse": (torch.log(total) + top).view(-1), "d_logits": d.to(s["logits"].dtype)}


# ------------------------------------------------------------------ the package's operators
def _operators():
    import __graft_entry__
    return __graft_entry__.load_pkg().operators


def _own_attention(s):
    O, c = _operators(), s["case"]
    o, lse = O.attention(s["q"], s["k"], s["v"], causal=c["causal"], q_lens=s["q_lens"], k_lens=s["k_lens"])
    out = {"o": o, "lse": lse}
    if c["op"] == "attn_train":
        out["dq"], out["dk"], out["dv"] = O.attention_backward(s["do"], s["q"], s["k"], s["v"], o, lse, causal=c["causal"],
                                                               q_lens=s["q_lens"], k_lens=s["k_lens"])
    return out


def _own_log_probs(s):
    O, c = _operators(), s["case"]
    r = O.log_probs(s["logits"], s["targets"], top=c["top"], scale=c["scale"])
    out = {"log_prob": r.log_prob, "entropy": r.entropy, "lse": r.lse}
    if c["top"]:
        out["top_index"], out["top_log_prob"] = r.top_index, r.top_log_prob
    if c["op"] == "logp_train":
        out["d_logits"] = O.log_probs_backward(s["logits"], s["targets"], r.lse, r.entropy, d_log_prob=s["d_log_prob"],
                                               d_entropy=s["d_entropy"], scale=c["scale"])
    return out


def _own_distill(s):
    O, c = _operators(), s["case"]
    r = O.distill(s["logits"], s["teacher_index"], s["teacher_value"], temperature=c["temperature"], tail=c["tail"])
    d = O.distill_backward(s["d_loss"], s["logits"], s["teacher_index"], s["teacher_value"], r.lse, r.log_tail,
                           temperature=c["temperature"], tail=c["tail"])
    return {"loss": r.loss, "lse": r.lse, "d_logits": d}


def run(state):
    op = state["case"]["op"]
    if op in ("attn", "attn_train"):
        return _own_attention(state) if own else _plain_attention(state)
    if op in ("logp", "logp_train"):
        return _own_log_probs(state) if own else _plain_log_probs(state)
    return _own_distill(state) if own else _plain_distill(state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] in ("attn", "attn_train"):
        B, Hq, Hk, D = case["batch"], case["q_heads"], case["kv_heads"], case["head_dim"]
        nq = (None if case["q_len"] == 1 else _lengths(case, case["q_len"], 0.381966)) or [case["q_len"]] * B
        nk = _lengths(case, case["k_len"], 0.618034) or [case["k_len"]] * B
        pairs = 0
        for a, b in zip(nq, nk):
            if case["causal"]:
                seen = np.clip(np.arange(a) + 1 + b - a, 0, b)
                pairs += int(seen.sum())
            else:
                pairs += a * b
        q, kv = sum(nq) * Hq * D, sum(nk) * Hk * D
        out_q, out_kv = B * case["q_len"] * Hq * D, B * case["k_len"] * Hk * D
        if case["op"] == "attn":
            return {"bytes": e * (q + 2 * kv + out_q) + 4 * B * Hq * case["q_len"], "flops": 4 * D * Hq * pairs}
        return {"bytes": e * (2 * q + 2 * kv + 2 * out_q + 2 * out_kv) + 4 * B * Hq * case["q_len"], "flops": 14 * D * Hq * pairs}
    R, V, K = case["rows"], case["classes"], case["top"]
    if case["op"] == "logp":
        return {"bytes": R * (V * e + 16 + 8 * K), "flops": 6 * R * V}
    if case["op"] == "logp_train":
        return {"bytes": R * (2 * V * e + 24), "flops": 12 * R * V}
    return {"bytes": R * (2 * V * e + 8 * K + 12), "flops": 10 * R * V}


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_attention(s):
    c = s["case"]
    train = c["op"] == "attn_train"
    if c["batch"] * c["q_heads"] * c["q_len"] * c["k_len"] > 1 << 30:
        return None
    Hq, G, scale = c["q_heads"], c["q_heads"] // c["kv_heads"], c["head_dim"] ** -0.5
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    o, lse = torch.zeros_like(q), torch.full((c["batch"], Hq, c["q_len"]), -math.inf, dtype=torch.float64, device=q.device)
    dq, dk, dv = (torch.zeros_like(x) for x in (q, k, v))
    for b in range(c["batch"]):
        nq = c["q_len"] if s["q_lens"] is None else int(s["q_lens"][b])
        nk = c["k_len"] if s["k_lens"] is None else int(s["k_lens"][b])
        first = max(0, nq - nk) if c["causal"] else 0      # the rows before it see no key
        if first >= nq:
            continue
        hidden = torch.ones(nq - first, nk, dtype=torch.bool, device=q.device).triu(nk - nq + first + 1) if c["causal"] else None
        for h in range(Hq):
            x, y, w = (t.detach().clone().requires_grad_(train) for t in (q[b, first:nq, h], k[b, :nk, h // G], v[b, :nk, h // G]))
            a = (x @ y.t()) * scale
            if hidden is not None:
                a = a.masked_fill(hidden, -math.inf)
            r = torch.softmax(a, 1) @ w
            o[b, first:nq, h], lse[b, h, first:nq] = r.detach(), torch.logsumexp(a, 1).detach()
            if train:
                r.backward(s["do"][b, first:nq, h].double())
                dq[b, first:nq, h] = x.grad
                dk[b, :nk, h // G] += y.grad
                dv[b, :nk, h // G] += w.grad
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv} if train else {"o": o, "lse": lse}


def _in_chunks(s, names, one):
    """one(rows of the named tensors, in 64 bits) over chunks of rows, joined"""
    parts, step = [], max(1, (1 << 25) // s["case"]["classes"])
    for r in range(0, s["case"]["rows"], step):
        parts.append(one(*(s[n][r:r + step].double() if s[n].is_floating_point() else s[n][r:r + step].long() for n in names)))
    return {n: torch.cat([p[n] for p in parts]) for n in parts[0]}


def _exact_log_probs(s):
    c = s["case"]
    train = c["op"] == "logp_train"

    def one(z, at, *grads):
        z = z.detach().requires_grad_(train)
        lse = torch.logsumexp(z * c["scale"], 1, keepdim=True)
        d = z * c["scale"] - lse
        hidden = torch.isinf(d)
        shown = torch.where(hidden, 0.0, d)
        entropy = -torch.where(hidden, 0.0, shown.exp() * shown).sum(1)
        lp = d.gather(1, at.view(-1, 1)).view(-1)
        out = {"log_prob": lp, "entropy": entropy, "lse": lse.view(-1)}
        if train:
            torch.autograd.backward([lp, entropy], list(grads))
            out["d_logits"] = z.grad
        return {n: t.detach() for n, t in out.items()}

    out = _in_chunks(s, ["logits", "targets"] + (["d_log_prob", "d_entropy"] if train else []), one)
    if c["top"]:
        value, index = torch.sort(s["logits"], dim=1, descending=True, stable=True)
        out["top_index"] = index[:, :c["top"]].to(torch.int32)
        out["top_log_prob"] = value[:, :c["top"]].double() * c["scale"] - out["lse"].view(-1, 1)
    return out


def _exact_distill(s):
    c = s["case"]

    def one(z, at, a, g):
        z = z.detach().requires_grad_(True)
        lse = torch.logsumexp(z / c["temperature"], 1, keepdim=True)
        used = at >= 0
        at = at.clamp(min=0)
        lq = (z / c["temperature"]).gather(1, at) - lse
        if c["tail"]:
            lp = a
        else:
            lp = torch.log_softmax((a / c["temperature"]).masked_fill(~used, -1e300), 1)
        p = lp.exp() * used
        loss = (p * (lp - lq)).masked_fill(~used, 0.0).sum(1)
        if c["tail"]:
            named = torch.zeros_like(z, dtype=torch.long).scatter_add_(1, at, used.long()) > 0
            tail = torch.logsumexp((z / c["temperature"]).masked_fill(named, -math.inf), 1) - lse.view(-1)
            rest = (1 - p.sum(1)).clamp(min=0.0)
            loss = loss + torch.where(rest >= 2.0 ** -20, rest * (rest.clamp(min=1e-300).log() - tail), torch.zeros_like(rest))
        loss.backward(g)
        return {"loss": loss.detach(), "lse": lse.detach().view(-1), "d_logits": z.grad}

    return _in_chunks(s, ["logits", "teacher_index", "teacher_value", "d_loss"], one)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("attn", "attn_train"):
        return _exact_attention(s)
    return _exact_log_probs(s) if case["op"] in ("logp", "logp_train") else _exact_distill(s)
