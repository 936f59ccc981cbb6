"""The operators for adapting a matcher on the GPU (-m gpu) against their definitions in 64 bits (operators_reference.py: elementwise
bounds from the arithmetic): lengths from nothing to several ranges, head layouts, strides, masks that leave rows empty, what may lie
behind a sequence's end, ties, adversarial orders, other streams, graphs, and a run of all of them together."""
import math

import numpy as np
import pytest
import torch

import operators_reference as R

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
INF = math.inf


@pytest.fixture(scope="module")
def O(U):
    assert U._lib.lib().urf_device_count() >= 1, "GPU tests need an MI355X"
    return U.operators


def cuda(t):
    return None if t is None else t.cuda()


def normal(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def lens(values):
    return None if values is None else torch.tensor(values, dtype=torch.int32)


def run_attention(O, q, k, v, do, causal=False, scale=None, q_lens=None, k_lens=None):
    o, lse = O.attention(q, k, v, causal=causal, scale=scale, q_lens=q_lens, k_lens=k_lens)
    dq, dk, dv = O.attention_backward(do, q, k, v, o, lse, causal=causal, scale=scale, q_lens=q_lens, k_lens=k_lens)
    return {"o": o, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


# batch, rows, keys, query heads, key heads, head size, causal, rows in use, keys in use
SHAPES = [
    (1, 1, 1, 1, 1, 8, False, None, None),
    (2, 1, 77, 4, 2, 64, True, None, [77, 5]),
    (1, 33, 130, 3, 1, 40, False, None, None),
    (2, 129, 257, 4, 4, 64, True, None, None),
    (1, 200, 64, 2, 1, 128, True, None, None),            # the first 136 rows see nothing
    (3, 17, 300, 6, 2, 80, False, [17, 0, 9], [300, 12, 0]),
    (1, 5, 0, 2, 2, 64, False, None, None),               # no key at all
    (2, 70, 65, 8, 8, 96, True, [70, 31], [3, 65]),
    (1, 300, 520, 2, 2, 32, False, None, None),
    (1, 1500, 1300, 1, 1, 64, False, None, None),         # few workgroups: ranges of rows and keys
    (1, 700, 700, 5, 1, 128, True, None, None),
    (40, 3, 40, 2, 2, 24, True, None, None),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:6])) + ("c" if s[6] else ""))
def test_attention_and_gradients(O, shape, dtype):
    B, Lq, Lk, Hq, Hk, D, causal, nq, nk = shape
    q, do = normal((B, Lq, Hq, D), dtype, 1), normal((B, Lq, Hq, D), dtype, 2)
    k, v = normal((B, Lk, Hk, D), dtype, 3), normal((B, Lk, Hk, D), dtype, 4)
    got = run_attention(O, cuda(q), cuda(k), cuda(v), cuda(do), causal, None, cuda(lens(nq)), cuda(lens(nk)))
    R.check(got, R.attention(q, k, v, causal, None, nq, nk, do), shape)
    again = run_attention(O, cuda(q), cuda(k), cuda(v), cuda(do), causal, None, cuda(lens(nq)), cuda(lens(nk)))
    assert all(torch.equal(got[n], again[n]) for n in got), "two runs differ"


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_single_row_over_a_long_cache_is_split(O, dtype):
    q, k, v = normal((2, 1, 8, 128), dtype, 1), normal((2, 9001, 2, 128), dtype, 2), normal((2, 9001, 2, 128), dtype, 3)
    n = [9001, 4100]
    o, lse = O.attention(cuda(q), cuda(k), cuda(v), causal=True, k_lens=cuda(lens(n)))
    R.check({"o": o, "lse": lse}, R.attention(q, k, v, True, None, None, n))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_strides_and_what_lies_behind_the_ends(O, dtype):
    """head-major and packed layouts, a batch that is broadcast, NaN behind every sequence's end and in the tensors' gaps"""
    B, Lq, Lk, H, D = 3, 40, 52, 4, 72
    nq, nk = [40, 11, 0], [9, 52, 30]
    big = torch.full((B, H, Lq + 3, D + 8), torch.nan, dtype=dtype)
    big[:, :, :Lq, :D] = normal((B, H, Lq, D), dtype, 1)
    q = cuda(big)[:, :, :Lq, :D].permute(0, 2, 1, 3)
    packed = torch.full((1, Lk, 2, H, D), torch.nan, dtype=dtype)
    packed[:] = normal(packed.shape, dtype, 2)
    kv = cuda(packed)
    k, v = kv[:, :, 0].expand(B, -1, -1, -1), kv[:, :, 1].expand(B, -1, -1, -1)
    do = cuda(normal((B, Lq, H, D), dtype, 3))
    want = R.attention(q.cpu(), k.cpu(), v.cpu(), False, 0.2, nq, nk, do.cpu())
    R.check(run_attention(O, q, k, v, do, False, 0.2, cuda(lens(nq)), cuda(lens(nk))), want)
    # now with the unused rows poisoned, every tensor of its own
    k, v, q, do = (t.clone() for t in (k, v, q, do))
    for b in range(B):
        q[b, nq[b]:], do[b, nq[b]:] = torch.nan, INF
        k[b, nk[b]:], v[b, nk[b]:] = INF, torch.nan
    got = run_attention(O, q, k, v, do, False, 0.2, cuda(lens(nq)), cuda(lens(nk)))
    R.check(got, want)
    assert all(bool((got["o"][b, nq[b]:] == 0).all()) and bool((got["dq"][b, nq[b]:] == 0).all()) for b in range(B))
    assert all(bool((got["dk"][b, nk[b]:] == 0).all()) and bool((got["dv"][b, nk[b]:] == 0).all()) for b in range(B))


def test_attention_lengths_beyond_the_tensors_are_clamped(O):
    q, k, v, do = (normal((3, 20, 2, 64), torch.bfloat16, s) for s in range(4))
    over, under = cuda(lens([99, 20, -7])), cuda(lens([20, 1 << 30, -1]))
    R.check(run_attention(O, cuda(q), cuda(k), cuda(v), cuda(do), False, None, over, under),
            R.attention(q, k, v, False, None, [20, 20, 0], [20, 20, 0], do))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("group", [1, 3])
def test_attention_rows_that_see_nothing_may_hold_anything(O, dtype, group):
    """causal with more rows than keys: the first rows' q and do are not used, in their own gradient or in the keys'"""
    nq, nk = [150, 90, 41], [60, 0, 70]
    q, do = (normal((3, 150, 2 * group, 64), dtype, s) for s in (1, 2))
    k, v = (normal((3, 70, 2, 64), dtype, s) for s in (3, 4))
    want = R.attention(q, k, v, True, None, nq, nk, do)
    for b in range(3):
        blind = max(0, nq[b] - nk[b])
        q[b, :blind], do[b, :blind] = torch.nan, INF
    R.check(run_attention(O, cuda(q), cuda(k), cuda(v), cuda(do), True, None, cuda(lens(nq)), cuda(lens(nk))), want)


def test_attention_offsets_beyond_32_bits(O):
    """rows 2^26 elements apart: the last ones lie 5 GB behind the first"""
    L, D, step = 40, 64, 1 << 26
    store = torch.empty(step * (L - 1) + D, dtype=torch.bfloat16, device="cuda")
    k = store.as_strided((1, L, 1, D), (0, step, 0, 1))
    k.copy_(cuda(normal((1, L, 1, D), torch.bfloat16, 1)))
    q, v, do = (normal((1, L, 1, D), torch.bfloat16, s) for s in (2, 3, 4))
    R.check(run_attention(O, cuda(q), k, cuda(v), cuda(do), True), R.attention(q, k.cpu(), v, True, None, None, None, do))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_large_and_small_scores(O, dtype):
    """scores of some hundreds either way: the running maximum has to move, and rows far below zero keep their probabilities"""
    q, k, v, do = (normal((2, 90, 2, 64), dtype, s) for s in range(4))
    q = q * 12
    k = k * 4
    k[:, 40:] *= 3
    q[1] = -q[1].abs()
    k[1] = k[1].abs()
    R.check(run_attention(O, cuda(q), cuda(k), cuda(v), cuda(do), True), R.attention(q, k, v, True, None, None, None, do))


def test_attention_gradients_against_differences(O):
    """fp32: the change of sum(o * do) along a direction is what the gradients say"""
    B, Lq, Lk, H, D = 1, 37, 45, 2, 16
    x = [normal(s, torch.float32, i) for i, s in enumerate([(B, Lq, H, D), (B, Lk, H, D), (B, Lk, H, D)])]
    way = [normal(t.shape, torch.float32, 7 + i) for i, t in enumerate(x)]
    do = normal((B, Lq, H, D), torch.float32, 11)
    got = run_attention(O, *map(cuda, x), cuda(do), True)
    slope = sum(float((got[n].cpu().double() * w.double()).sum()) for n, w in zip(("dq", "dk", "dv"), way))
    want = R.attention(*x, True, None, None, None, do)
    grad_err = sum(float((want[n][1] * w.double().abs()).sum()) for n, w in zip(("dq", "dk", "dv"), way))
    h = 2.0 ** -7
    value, exact, err = [], [], 0.0
    for s in (h, -h):
        y = [(t + s * w) for t, w in zip(x, way)]
        o = O.attention(*map(cuda, y), causal=True)[0]
        value.append(float((o.cpu().double() * do.double()).sum()))
        ref = R.attention(*y, True)["o"]
        exact.append(float((ref[0] * do.double()).sum()))
        err += float((ref[1] * do.double().abs()).sum())
    # the truncation of the difference is known from the definition; the rest is the rounding of both evaluations
    truth = sum(float((want[n][0] * w.double()).sum()) for n, w in zip(("dq", "dk", "dv"), way))
    truncation = abs((exact[0] - exact[1]) / (2 * h) - truth)
    assert abs((value[0] - value[1]) / (2 * h) - slope) <= truncation + err / (2 * h) + grad_err


# ------------------------------------------------------------------ rows of scores
ROWS = [(1, 1, 0), (3, 2, 0), (5, 7, 3), (4, 64, 0), (9, 1025, 3), (3, 2049, 0), (2, 9001, 0), (1, 70001, 0), (530, 2501, 5), (7, 513, 0), (4100, 300, 3), (2051, 2047, 0),
        (3, 40001, 3), (128, 32771, 1), (2, 300007, 0)]


def rows_of(R_, V, pad, dtype, seed, masked=0.0):
    """scores of rows V + pad elements apart, the first one (pad + 1) / 2 elements behind a boundary"""
    z = normal((R_, V + pad), torch.float32, seed) * 3
    at = (pad + 1) // 2
    if masked:
        z[torch.rand(z.shape, generator=torch.Generator().manual_seed(seed + 1)) < masked] = -INF
        z[:, at] = 0.25
    return z.to(dtype)[:, at:at + V], cuda(z.to(dtype))[:, at:at + V]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,classes,pad", ROWS)
@pytest.mark.parametrize("masked", [0.0, 0.4])
def test_log_probs_and_gradients(O, rows, classes, pad, dtype, masked):
    z, zc = rows_of(rows, classes, pad, dtype, 5, masked)
    g = torch.Generator().manual_seed(3)
    targets = torch.randint(-1, classes + 1, (rows, 3), generator=g, dtype=torch.int32)       # none, and one beyond the classes
    targets[:, 2] = targets[:, 0]                                                             # the same one twice
    top, scale = min(64, classes, 1 + classes // 3), 0.7
    r = O.log_probs(zc, cuda(targets), top=top, scale=scale)
    d_lp, d_h = normal((rows, 3), torch.float32, 6), normal((rows,), torch.float32, 7)
    d = O.log_probs_backward(zc, cuda(targets), r.lse, r.entropy, d_log_prob=cuda(d_lp), d_entropy=cuda(d_h), scale=scale)
    R.check({**r._asdict(), "d_logits": d}, R.log_probs(z, targets, top, scale, d_lp, d_h), (rows, classes))
    only = O.log_probs_backward(zc, None, r.lse, r.entropy, d_entropy=cuda(d_h), scale=scale)
    R.check({"d_logits": only}, {"d_logits": R.log_probs(z, None, 0, scale, None, d_h)["d_logits"]})
    other = O.log_probs_backward(zc, cuda(targets), r.lse, r.entropy, d_log_prob=cuda(d_lp), scale=scale)
    R.check({"d_logits": other}, {"d_logits": R.log_probs(z, targets, 0, scale, d_lp, None)["d_logits"]})


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("classes,copies", [(100, 1), (1500, 1), (5000, 1), (20000, 1), (50000, 1), (100, 200), (1500, 180)])
def test_log_probs_alternatives_of_awkward_rows(O, dtype, classes, copies):
    """ties, -0 and +0, ascending and descending rows, one value everywhere, few scores that are not masked, all that is large in one
    lane's reach, NaN, +inf, nothing at all; copies: enough rows for two a wave, different kinds side by side"""
    i = torch.arange(classes, dtype=torch.float32)
    few = torch.full((classes,), -INF)
    few[[3, classes // 2, classes - 1]] = torch.tensor([1.0, 1.0, 2.0])
    near = torch.zeros(classes)
    near[:8] = 5 + torch.arange(8.0)
    near[512:520] = 5.0
    z = torch.stack([i / classes, -i / classes, torch.zeros(classes), torch.where(i % 2 == 0, -0.0, 0.0), i % 3, few, near,
                     torch.full((classes,), -INF), torch.where(i == 7, torch.nan, i % 5), torch.where(i == classes - 1, INF, i % 5),
                     torch.full((classes,), torch.finfo(dtype).min), torch.full((classes,), INF)]).to(dtype).repeat(copies, 1)
    targets = torch.full((len(z), 1), 7, dtype=torch.int32)
    for top in (1, 20, 32, 64):
        got = O.log_probs(cuda(z), cuda(targets), top=top)
        R.check(got._asdict(), R.log_probs(z, targets, top), top)
    one = torch.ones(len(z), 1)
    d = O.log_probs_backward(cuda(z), cuda(targets), got.lse, got.entropy, d_log_prob=cuda(one), d_entropy=cuda(one[:, 0].contiguous()))
    R.check({"d_logits": d}, {"d_logits": R.log_probs(z, targets, 0, 1.0, one, one[:, 0])["d_logits"]})


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,classes,pad", [r for r in ROWS if r[1] > 1])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_and_gradients(O, rows, classes, pad, dtype, tail):
    z, zc = rows_of(rows, classes, pad, dtype, 8)
    K, T = min(64, max(1, classes // 2)), 1.5
    teacher = z.float() + normal(z.shape, torch.float32, 9)
    t = O.log_probs(cuda(teacher), top=K, scale=1 / T)
    index, value = t.top_index.cpu(), t.top_log_prob.cpu()
    if not tail:
        value = teacher.gather(1, index.long())
    drop = torch.rand(index.shape, generator=torch.Generator().manual_seed(4)) < 0.2
    index[drop], value[drop] = -1, torch.nan                    # unused: the value is not looked at
    if rows > 1:
        index[-1] = -1                                          # nothing is listed
        index[0, 0] = classes                                   # beyond the classes: unused too
    g = normal((rows,), torch.float32, 10)
    r = O.distill(zc, cuda(index), cuda(value), temperature=T, tail=tail)
    d = O.distill_backward(cuda(g), zc, cuda(index), cuda(value), r.lse, r.log_tail, temperature=T, tail=tail)
    R.check({"loss": r.loss, "lse": r.lse, "log_tail": r.log_tail, "d_logits": d}, R.distill(z, index, value, T, tail, g), (rows, classes))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("tail", [False, True])
def test_distill_edges(O, dtype, tail):
    """an alternative listed twice, every class listed, a student far from (and in agreement with) its teacher, masked scores"""
    V, K = 40, 40
    z = normal((5, V), torch.float32, 1).to(dtype)
    z[1, :] = -60.0
    z[1, 5] = 60.0                                              # the unlisted rest is 2^-170 of the student's probability
    z[2, 7:20] = -INF
    index = torch.arange(K, dtype=torch.int32).repeat(5, 1)
    value = torch.log_softmax(normal((5, K), torch.float32, 2), 1)
    index[1, 1:], value[1, 0] = -1, math.log(0.5)
    index[1, 0] = 5
    index[2, 1:], value[2, 0] = -1, math.log(0.9)
    index[3, :] = -1
    index[3, :3], value[3, :3] = torch.tensor([4, 4, 9], dtype=torch.int32), torch.tensor([0.2, 0.3, 0.4]).log()
    index[4, 1:], value[4, 0] = -1, 0.0                         # the teacher is certain: no rest
    g = torch.tensor([1.0, -2.0, 0.5, 1.0, 3.0])
    r = O.distill(cuda(z), cuda(index), cuda(value), tail=tail)
    d = O.distill_backward(cuda(g), cuda(z), cuda(index), cuda(value), r.lse, r.log_tail, tail=tail)
    R.check({"loss": r.loss, "lse": r.lse, "log_tail": r.log_tail, "d_logits": d}, R.distill(z, index, value, 1.0, tail, g))


def test_rows_gradients_against_differences(O):
    rows, V, K = 6, 300, 5
    z, way = normal((rows, V), torch.float32, 1) * 2, normal((rows, V), torch.float32, 2)
    t = O.log_probs(cuda(z + normal((rows, V), torch.float32, 3)), top=K)
    index, value, targets = t.top_index, t.top_log_prob, cuda(torch.randint(0, V, (rows,), dtype=torch.int32))
    g, h = normal((rows,), torch.float32, 4), normal((rows,), torch.float32, 5)

    def plain(x):       # the three scalars in 64 bits on the CPU
        a = R.log_probs(x, targets.cpu()[:, None])
        b = R.distill(x, index.cpu(), value.cpu(), 1.0, True)
        return float((a["log_prob"][0][:, 0] * g).sum() + (a["entropy"][0] * h).sum() + (b["loss"][0] * g).sum()), \
            float((a["log_prob"][1][:, 0] * g.abs()).sum() + (a["entropy"][1] * h.abs()).sum() + (b["loss"][1] * g.abs()).sum())

    def ours(x):
        a, b = O.log_probs(cuda(x), targets), O.distill(cuda(x), index, value, tail=True)
        return float((a.log_prob.cpu().double() * g).sum() + (a.entropy.cpu().double() * h).sum() + (b.loss.cpu().double() * g).sum())

    a, b = O.log_probs(cuda(z), targets), O.distill(cuda(z), index, value, tail=True)
    d = O.log_probs_backward(cuda(z), targets, a.lse, a.entropy, d_log_prob=cuda(g), d_entropy=cuda(h)).cpu().double() \
        + O.distill_backward(cuda(g), cuda(z), index, value, b.lse, b.log_tail, tail=True).cpu().double()
    wa = R.log_probs(z, targets.cpu()[:, None], 0, 1.0, g[:, None], h)["d_logits"]
    wb = R.distill(z, index.cpu(), value.cpu(), 1.0, True, g)["d_logits"]
    step = 2.0 ** -7
    (p0, e0), (p1, e1) = plain(z + step * way), plain(z - step * way)
    truncation = abs((p0 - p1) / (2 * step) - float(((wa[0] + wb[0]) * way).sum()))
    got = (ours(z + step * way) - ours(z - step * way)) / (2 * step)
    assert abs(got - float((d * way).sum())) <= truncation + (e0 + e1) / (2 * step) + float(((wa[1] + wb[1]) * way.abs()).sum())


# ------------------------------------------------------------------ callers
def _all_operators(O, s):
    a = run_attention(O, s["q"], s["k"], s["v"], s["do"], True, None, s["nq"], s["nk"])
    logits = a["o"].float().reshape(s["q"].shape[0] * s["q"].shape[1], -1)
    r = O.log_probs(logits, s["targets"], top=9)
    t = O.distill(logits, s["index"], s["value"], tail=True)
    d = O.log_probs_backward(logits, s["targets"], r.lse, r.entropy, d_log_prob=s["g"], d_entropy=s["g"])
    e = O.distill_backward(s["g"], logits, s["index"], s["value"], t.lse, t.log_tail, tail=True)
    return {**a, "lp": r.log_prob, "h": r.entropy, "ti": r.top_index, "tp": r.top_log_prob, "loss": t.loss, "tail": t.log_tail, "d": d, "e": e}


def _inputs(seed, long=False):
    B, L, Lk = (1, 700, 700) if long else (2, 60, 90)
    s = {n: cuda(normal((B, L if n in ("q", "do") else Lk, 4 if n in ("q", "do") else 2, 64), torch.bfloat16, seed + i))
         for i, n in enumerate(("q", "k", "v", "do"))}
    rows = B * L
    s["nq"], s["nk"] = cuda(lens([L, L // 2][:B])), cuda(lens([Lk - 3, Lk][:B]))
    s["targets"] = cuda(torch.randint(0, 256, (rows,), generator=torch.Generator().manual_seed(seed), dtype=torch.int32))
    s["g"] = cuda(normal((rows,), torch.float32, seed + 9))
    s["index"] = cuda(torch.stack([torch.randperm(256, generator=torch.Generator().manual_seed(seed + r))[:6] for r in range(rows)]).to(torch.int32))
    s["value"] = cuda(torch.log_softmax(normal((rows, 7), torch.float32, seed + 8), 1)[:, :6].contiguous())
    return s


@pytest.mark.parametrize("long", [False, True])
def test_captured_and_replayed(O, long):
    """one graph of all calls, workspaces included, replayed on other inputs with eager work between the replays"""
    s = _inputs(1, long)
    for _ in range(2):
        _all_operators(O, s)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        _all_operators(O, s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _all_operators(O, s)
    for seed in (21, 31, 41, 1):
        other = _inputs(seed, long)
        for n in s:
            s[n].copy_(other[n])
        want = _all_operators(O, other)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out[n].nan_to_num(7.0), want[n].nan_to_num(7.0)) for n in want), seed


def test_two_streams_at_once(O):
    inputs = [_inputs(1, True), _inputs(51, True)]
    want = [_all_operators(O, s) for s in inputs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(_all_operators(O, inputs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(g[n], want[i][n]) for n in g), i


def test_few_rows_in_parts_captured_and_on_two_streams(O):
    """single tokens over long keys and a few long rows of scores: two graphs, each with the workspaces of its own capture, replayed at
    the same time, and the same calls eagerly on two streams"""
    def inputs(seed):
        return {"q": cuda(normal((2, 1, 8, 64), torch.bfloat16, seed)), "k": cuda(normal((2, 5000, 2, 64), torch.bfloat16, seed + 1)),
                "v": cuda(normal((2, 5000, 2, 64), torch.bfloat16, seed + 2)), "z": cuda(normal((3, 60001), torch.bfloat16, seed + 3))}

    def calls(s):
        o, lse = O.attention(s["q"], s["k"], s["v"], causal=True)
        return {"o": o, "lse": lse, **{n: t for n, t in O.log_probs(s["z"], top=9)._asdict().items() if t is not None and n != "lse"}}

    sets = [inputs(1), inputs(50)]
    for s in sets:
        calls(s)
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(calls(s))
    for seed in (7, 90, 1):
        for i, s in enumerate(sets):
            for n, t in inputs(seed + 400 * i).items():
                s[n].copy_(t)
        want = [calls(s) for s in sets]
        torch.cuda.synchronize()
        eager = [None, None]
        for _ in range(4):
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    graphs[i].replay()
                    eager[i] = calls(sets[i])
        torch.cuda.synchronize()
        for i in range(2):
            for n in want[i]:
                assert torch.equal(outs[i][n], want[i][n]) and torch.equal(eager[i][n], want[i][n]), (seed, i, n)


def test_refusals(O):
    q = torch.zeros((1, 4, 2, 64), dtype=torch.bfloat16, device="cuda")
    z, t, f = torch.zeros((2, 50), device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros(2, device="cuda")
    ix, val = torch.zeros((2, 3), dtype=torch.int32, device="cuda"), torch.zeros((2, 3), device="cuda")
    o, lse = O.attention(q, q, q)
    bad = [lambda: O.attention(q.cpu(), q, q), lambda: O.attention(q, q.float(), q), lambda: O.attention(q[0], q, q),
           lambda: O.attention(q, q[:, :, :1], q), lambda: O.attention(q.double(), q.double(), q.double()),
           lambda: O.attention(q[:, :, :, 4:], q[:, :, :, 4:], q[:, :, :, 4:]), lambda: O.attention(q, q, q, scale=-1.0),
           lambda: O.attention(q, q, q, k_lens=torch.zeros(2, dtype=torch.int32, device="cuda")),
           lambda: O.attention(q, q, q, k_lens=torch.zeros(1, dtype=torch.int64, device="cuda")),
           lambda: O.attention(q, q, q, q_lens=torch.zeros(1, dtype=torch.int32)),
           lambda: O.attention(q.transpose(1, 3), q.transpose(1, 3), q.transpose(1, 3)),
           lambda: O.attention(q.clone().requires_grad_(), q, q),
           lambda: O.attention_backward(q[:, :2], q, q, q, o, lse), lambda: O.attention_backward(q, q, q, q, o, lse[:, :1]),
           lambda: O.log_probs(z[0]), lambda: O.log_probs(z.T), lambda: O.log_probs(z, t.long()), lambda: O.log_probs(z, t[:1]),
           lambda: O.log_probs(z, top=51), lambda: O.log_probs(z, top=-1), lambda: O.log_probs(z, scale=0.0), lambda: O.log_probs(z.cpu()),
           lambda: O.log_probs(z, torch.zeros((2, 65), dtype=torch.int32, device="cuda")),
           lambda: O.log_probs_backward(z, None, f, f, d_log_prob=f), lambda: O.log_probs_backward(z, t, f[:1], f, d_log_prob=f),
           lambda: O.distill(z, ix, val[:, :2]), lambda: O.distill(z, ix.long(), val), lambda: O.distill(z, ix, val, temperature=0.0),
           lambda: O.distill(z, torch.zeros((2, 65), dtype=torch.int32, device="cuda"), torch.zeros((2, 65), device="cuda")),
           lambda: O.distill_backward(f, z, ix, val, f, None, tail=True)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was accepted")
    for head_dim in (4, 62, 136):                          # past the wrapper's own checks: the C ABI's
        w = torch.zeros((1, 4, 2, head_dim + head_dim % 4), dtype=torch.float32, device="cuda")[..., :head_dim]
        with pytest.raises(RuntimeError):
            O.attention(w, w, w)
    three = torch.zeros((1, 4, 3, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError):
        O.attention(three, q, q)
    with pytest.raises(RuntimeError):
        O.attention(q[..., :0], q[..., :0], q[..., :0])
    none = O.log_probs(z[:0], t[:0], top=3)
    assert none.lse.shape == (0,) and none.top_index.shape == (0, 3)
    assert O.attention(q[:, :0], q, q)[0].shape == (1, 0, 2, 64)
    assert bool((O.attention_backward(q[:, :0], q[:, :0], q, q, q[:, :0], lse[:, :, :0])[1] == 0).all())


# ------------------------------------------------------------------ the matcher's own path, and a step of a student
def test_matcher_log_probs_of_the_last_pair(U, O, sg_blob):
    from conftest import make_features
    F = U.frontend
    rng = np.random.default_rng(3)
    f0 = make_features(rng, 90)
    f1 = make_features(rng, 70, f0, 40)
    sg = F.SuperGlue(F.SuperGlueConfig())
    assert sg.build(sg_blob)
    pm = F.PointMatching(F.SuperGlueConfig())
    a, b = pm.NormalizeKeypoints(f0, 640, 512), pm.NormalizeKeypoints(f1, 640, 512)
    with pytest.raises(RuntimeError):
        sg.match_log_probs()
    i0, i1, m0, m1, Z = sg.infer(a, b, want_scores=True)
    targets = np.where(i0 >= 0, i0, 70).astype(np.int32)
    targets[5] = -1
    lp, entropy, index, value = sg.match_log_probs(targets, top=3)
    want = R.log_probs(torch.from_numpy(Z[:90]), torch.from_numpy(targets)[:, None], 3)
    R.check({"log_prob": torch.from_numpy(lp)[:, None], "entropy": torch.from_numpy(entropy), "top_index": torch.from_numpy(index),
             "top_log_prob": torch.from_numpy(value)}, {n: want[n] for n in ("log_prob", "entropy", "top_index", "top_log_prob")})
    matched = (i0 >= 0) & (targets >= 0)
    assert matched.sum() >= 10 and np.array_equal(index[matched, 0], i0[matched])     # a match is its keypoint's best candidate
    assert sg.match_log_probs()[1].shape == (90,)
    with pytest.raises(ValueError):
        sg.match_log_probs(targets[:3])
    with pytest.raises(RuntimeError):
        sg.match_log_probs(top=65)
    sg.infer(a, b)                                                                    # no log-assignment kept
    with pytest.raises(RuntimeError):
        sg.match_log_probs()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_a_students_step_together(U, O, sg_blob, dtype):
    """The teacher is the matcher: its best candidates of each keypoint.  The student is one attention layer between the two images'
    descriptors and a product of its outputs: its loss's gradient with respect to the layer's inputs goes through the distillation, a
    plain product and the attention, and equals autograd's in 64 bits up to the roundings of the stages."""
    from conftest import make_features
    F = U.frontend
    rng = np.random.default_rng(5)
    n0, n1, K = 90, 70, 6
    f0 = make_features(rng, n0)
    f1 = make_features(rng, n1, f0, 40)
    sg = F.SuperGlue(F.SuperGlueConfig())
    assert sg.build(sg_blob)
    pm = F.PointMatching(F.SuperGlueConfig())
    assert sg.infer(pm.NormalizeKeypoints(f0, 640, 512), pm.NormalizeKeypoints(f1, 640, 512), want_scores=True) is not None
    _, _, index, value = sg.match_log_probs(top=K)
    index, value = torch.from_numpy(index), torch.from_numpy(value)
    H, D = 4, 64
    q = torch.from_numpy(f0[:, 3:]).float().mul(8).to(dtype).view(1, n0, H, D)
    kv = torch.from_numpy(f1[:, 3:]).float().mul(8).to(dtype).view(1, n1, H, D)
    W = normal((H * D, n1 + 1), torch.float32, 1) / 16
    o, lse = O.attention(cuda(q), cuda(kv), cuda(kv))
    logits = o.view(n0, H * D).float() @ cuda(W)
    r = O.distill(logits, cuda(index), cuda(value), tail=True)
    d_logits = O.distill_backward(torch.full((n0,), 1.0 / n0, device="cuda"), logits, cuda(index), cuda(value), r.lse, r.log_tail, tail=True)
    do = (d_logits @ cuda(W).T.contiguous()).to(dtype).view(1, n0, H, D)
    dq, dk, dv = O.attention_backward(do, cuda(q), cuda(kv), cuda(kv), o, lse)
    # 64 bits, from the same inputs
    x, y = q.double().requires_grad_(), kv.double().requires_grad_()
    a = torch.softmax(torch.einsum("bihd,bjhd->bhij", x, y) * D ** -0.5, -1)
    z = torch.einsum("bhij,bjhd->bihd", a, y).reshape(n0, H * D) @ W.double()
    lp = torch.log_softmax(z, 1)
    p = value.double().exp()
    rest = (1 - p.sum(1)).clamp(min=0)
    named = torch.zeros_like(lp).scatter_(1, index.long(), 1.0) > 0
    tail = torch.logsumexp(lp.masked_fill(named, -INF), 1)
    loss = (p * (value.double() - lp.gather(1, index.long()))).sum(1) + torch.where(rest >= 2.0 ** -20, rest * (rest.clamp(min=1e-300).log() - tail), 0.0)
    loss.mean().backward()
    # four roundings of 16-bit types lie on the way (the probabilities, o, do, and the gradient's own), each relative to terms whose
    # sizes add up to at most a few times the result's: the 2-norm of the difference is taken against 8 of them, fp32 against 2^-24 times
    # the number of terms of the longest sums
    tol = 8 * R.unit(dtype) if dtype != torch.float32 else 2.0 ** -24 * (n0 + n1 + H * D + 64)
    for got, want in ((dq, x.grad), (dk + dv, y.grad)):
        assert float((got.cpu().double() - want).norm() / want.norm()) <= tol
    assert float((r.loss.cpu().double() - loss.detach()).abs().max()) <= tol * (1 + float(loss.detach().abs().max()))
