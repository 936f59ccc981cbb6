"""Values at the edges of the operators' ranges on the GPU (-m gpu): NaN, infinities and scores that overflow among the rows and keys
in use, small and large gradients in f16, scales outside of 32 bits, what torch records that these calls do not."""
import math

import pytest
import torch

import operators_reference as R
from test_gpu_operators import DTYPES, INF, cuda, lens, normal, run_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def O(U):
    assert U._lib.lib().urf_device_count() >= 1, "GPU tests need an MI355X"
    return U.operators


# batch, rows, keys, query heads, key heads, head size: the forward kernel's three forms (128 rows a workgroup, 32, ranges of keys)
FORMS = {"wide": (33, 1000, 70, 8, 8, 64), "narrow": (2, 150, 200, 4, 2, 64), "ranges": (2, 1, 3000, 4, 2, 128), "ranges of rows": (1, 300, 2500, 2, 1, 72)}


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("what", ["nan query", "nan key", "infinite score"])
def test_attention_of_values_that_are_not_finite(O, dtype, form, what):
    """A row in use with a NaN or a score of +infinity has no distribution: o, lse and dq are NaN there, and so are dk and dv of the
    keys that it sees.  Other heads and sequences are what they are without it, and so are the head's other rows where a query is bad."""
    B, Lq, Lk, Hq, Hk, D = FORMS[form]
    G, h, row, key = Hq // Hk, 1, Lq - 1, Lk // 2 + 1
    hk = h // G
    q, do = normal((B, Lq, Hq, D), dtype, 1), normal((B, Lq, Hq, D), dtype, 2)
    k, v = normal((B, Lk, Hk, D), dtype, 3), normal((B, Lk, Hk, D), dtype, 4)
    clean = {n: t.cpu() for n, t in run_attention(O, cuda(q), cuda(k), cuda(v), cuda(do)).items()}
    bound = {n: w[1] for n, w in R.attention(q[:1], k[:1], v[:1], False, None, None, None, do[:1]).items()}
    head = torch.zeros((B, Lq, Hq), dtype=torch.bool)          # rows that share keys with the bad one
    head[0, :, hk * G:hk * G + G] = True
    bad = torch.zeros_like(head)
    bad[0, row, h] = True
    if what == "nan query":
        q[0, row, h, D - 3] = torch.nan
    elif what == "nan key":
        k[0, key, hk, 5] = torch.nan
        bad = head
    elif dtype == torch.float16:             # products of f16 values stay below fp32's largest: an infinity among the inputs
        q[0, row, h, 0] = INF
        k[0, :, hk, 0] = 0.5 + k[0, :, hk, 0].abs()
    else:                                    # finite inputs whose product overflows, for one key alone
        q[0, row, h], k[0, key, hk] = 2.0 ** 66, 2.0 ** 66
    got = {n: t.cpu() for n, t in run_attention(O, cuda(q), cuda(k), cuda(v), cuda(do)).items()}
    for t in (got, clean):
        t["lse"] = t["lse"].transpose(1, 2)
    bound["lse"] = bound["lse"].transpose(1, 2)
    for n in ("o", "lse", "dq"):
        assert bool(got[n][bad].isnan().all()), n
        assert torch.equal(got[n][~head], clean[n][~head]), n
        if what == "nan query":              # (the running maximum moves for a wave's rows together: not the same bits)
            rest = (head & ~bad)[0]
            assert bool(((got[n][0][rest].double() - clean[n][0][rest].double()).abs() <= 2 * bound[n][0][rest]).all()), n
    keys = torch.zeros((B, Lk, Hk), dtype=torch.bool)
    keys[0, :, hk] = True
    for n in ("dk", "dv"):
        assert bool(got[n][keys].isnan().all()) and torch.equal(got[n][~keys], clean[n][~keys]), n


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_rows_that_see_nothing_beside_keys_that_are_not_finite(O, dtype, form, causal):
    """o and dq of rows behind the end, and of causal rows before the first key, are 0 and lse is -infinity whatever the keys in use hold"""
    B, Lq, Lk, Hq, Hk, D = FORMS[form]
    nq = [Lq // 2 if b % 2 else max(1, Lq - 3) for b in range(B)]
    nk = [min(Lk, max(1, nq[b] - 1 - b % 3)) if causal else Lk for b in range(B)]
    q, do = normal((B, Lq, Hq, D), dtype, 1), normal((B, Lq, Hq, D), dtype, 2)
    k, v = normal((B, Lk, Hk, D), dtype, 3), normal((B, Lk, Hk, D), dtype, 4)
    k[:, :, :, 3], v[:, 0], v[:, 1:] = torch.nan, torch.nan, INF
    got = run_attention(O, cuda(q), cuda(k), cuda(v), cuda(do), causal, None, cuda(lens(nq)), cuda(lens(nk)))
    blind = torch.stack([(torch.arange(Lq) >= nq[b]) | ((torch.arange(Lq) < nq[b] - nk[b]) if causal else False) for b in range(B)])
    assert bool(blind.any())
    blind = blind.cuda()
    assert bool((got["o"][blind] == 0).all()) and bool((got["dq"][blind] == 0).all())
    assert bool((got["lse"].transpose(1, 2)[blind] == -INF).all())
    assert bool(got["lse"].transpose(1, 2)[~blind].isnan().all()) and bool(got["o"][~blind].isnan().all())


# The probabilities (for dv) and the gradients of the scores (for dq and dk) are rounded to f16 once before the sum, and the sum once
# more.  Terms and result are numbers of f16's full precision if the kernel keeps them in range, so that both roundings have the same
# distribution relative to what they round; the terms' errors are independent and add up in squares: to at most the error of one
# rounding of the result where the terms do not cancel (the keys and queries are random: |sum|^2 is sum |term|^2 on average).  Together
# sqrt(2) times the error of one rounding at the end; delta's error (from the rounded o, whose entries are sqrt(e / keys) of v's) is
# scale = 1 / sqrt(head size) of one rounding in dq, less in dk, and fp32's is far below.  2 leaves room for the draw.  (Rounded without their range in mind the terms are subnormal: 3 to 11 times.)
SMALL = [(1, 1024, 8192, 1, 1, 64, False), (1, 256, 8192, 2, 1, 128, True), (16, 512, 4096, 8, 4, 64, False), (2, 1000, 1300, 2, 2, 40, True)]


@pytest.mark.parametrize("shape", SMALL, ids=lambda s: "x".join(map(str, s[:6])) + ("c" if s[6] else ""))
@pytest.mark.parametrize("size", [1e-4, 1e-3, 1e-2, 1.0, 30.0])
def test_attention_f16_gradients_of_any_size(O, shape, size):
    B, Lq, Lk, Hq, Hk, D, causal = shape
    q, do = normal((B, Lq, Hq, D), torch.float16, 1), (normal((B, Lq, Hq, D), torch.float32, 2) * size).to(torch.float16)
    k, v = normal((B, Lk, Hk, D), torch.float16, 3), normal((B, Lk, Hk, D), torch.float16, 4)
    got = run_attention(O, cuda(q), cuda(k), cuda(v), cuda(do), causal)
    b = B - 1                                # the definition of one sequence: 64 bits on the CPU
    want = R.attention(*(t[b:b + 1] for t in (q, k, v)), causal, None, None, None, do[b:b + 1])
    for n in ("dq", "dk", "dv"):
        x = want[n][0]
        once = float((x.to(torch.float16).double() - x).norm())
        off = float((got[n][b:b + 1].cpu().double() - x).norm())
        assert off <= 2 * once, (n, off / float(x.norm()), once / float(x.norm()))


@pytest.mark.parametrize("shape", SMALL[:1] + SMALL[2:], ids=lambda s: "x".join(map(str, s[:6])) + ("c" if s[6] else ""))
def test_attention_f16_products_beyond_its_largest_number(O, shape):
    """do . v reaches some 10^6: the products before the sum need not fit f16, the gradients do.  Rows of very different sizes side by side."""
    B, Lq, Lk, Hq, Hk, D, causal = shape
    B = min(B, 2)
    q, do = normal((B, Lq, Hq, D), torch.float16, 1) / 8, normal((B, Lq, Hq, D), torch.float32, 2)
    k, v = normal((B, Lk, Hk, D), torch.float16, 3) / 8, normal((B, Lk, Hk, D), torch.float16, 4) * 64
    do[:, ::2] *= 1e-3
    do[:, 1::2] *= 2000
    do = do.to(torch.float16)
    got = run_attention(O, cuda(q), cuda(k), cuda(v), cuda(do), causal)
    b = B - 1
    want = R.attention(*(t[b:b + 1] for t in (q, k, v)), causal, None, None, None, do[b:b + 1])
    assert float((do[b, :, 0].double() @ v[b, :, 0].double().T).abs().max()) > 2 * 65504
    for n in ("dq", "dk", "dv"):
        x = want[n][0]
        assert float(x.abs().max()) < 65504
        for part in ((x[:, ::2], got[n][b:b + 1, ::2]), (x[:, 1::2], got[n][b:b + 1, 1::2])) if n == "dq" else ((x, got[n][b:b + 1]),):
            once = float((part[0].to(torch.float16).double() - part[0]).norm())
            assert float((part[1].cpu().double() - part[0]).norm()) <= 2 * once, n


@pytest.mark.parametrize("form", ["wide", "ranges"])
def test_attention_f16_small_probabilities_add_up(O, form):
    """One key takes 0.99 of a row, 300000 others 2^-25 of its probability each: together 0.009, whose values are 1 where the first one's is
    0.  In f16's numbers next to 1 those that come behind it round to nothing.  Here they are taken times 2^9, 251 steps of f16's smallest: half a step is
    0.002 of each, fp32's sums of n / 16 equal steps for o and the row's sum are off by 2^-24 per step at most, o is rounded once."""
    n = 300000
    B, Lq = (256, 64) if form == "wide" else (1, 8)
    q = torch.zeros((B, Lq, 1, 64), dtype=torch.float16)
    q[..., 0] = 8.0
    k = torch.zeros((1, n, 1, 64), dtype=torch.float16)
    k[0, n // 2, 0, 0] = 17.375                                 # score: 17.375, exp(-17.375) = 0.478 of 2^-24
    v = torch.ones((1, n, 1, 64), dtype=torch.float16)
    v[0, n // 2] = 0.0
    share = math.exp(-17.375)
    want = (n - 1) * share / (1 + (n - 1) * share)
    o, lse = O.attention(cuda(q), cuda(k).expand(B, -1, -1, -1), cuda(v).expand(B, -1, -1, -1))
    off = float((o.double() / want - 1).abs().max())
    tol = 0.5 * 2.0 ** -24 / (share * 2.0 ** 9) + 2 * n / 16 * 2.0 ** -24 + R.unit(torch.float16)
    assert off <= tol
    # the row's sum takes in n / 64 tiles one after the other, each addition rounded by at most 2^-24 of the whole sum, which is 1 with the
    # large key in it (not of the small keys' share): d(lse) = d(sum) / sum
    assert float((lse.double() - (17.375 + math.log1p((n - 1) * share))).abs().max()) <= 2.0 ** -24 * (64 + 16 * 20 + n / 64)


@pytest.mark.parametrize("form", [*FORMS.values(), (40, 100, 4, 4, 2, 64)], ids=[*FORMS, "few keys"])
def test_attention_lse_of_16_bit_inputs_has_32(O, form):
    """The same numbers as f16, bf16 and fp32 give the same scores and sums, all in 32 bits: one lse is as good as the other.  (Products of
    16-bit numbers are exact, the order of sums differs: twice the fp32 call's error and a rounding of lse.)"""
    B, Lq, Lk, Hq, Hk, D = form
    q, k, v = (normal(s, torch.bfloat16, i).float().to(torch.float16) for i, s in enumerate([(B, Lq, Hq, D), (B, Lk, Hk, D), (B, Lk, Hk, D)]))
    want = R.attention(q[-1:].float(), k[-1:].float(), v[-1:].float())["lse"][0]
    off = {t: float((O.attention(cuda(q.to(t)), cuda(k.to(t)), cuda(v.to(t)))[1][-1:].cpu().double() - want).norm() / want.norm()) for t in DTYPES}
    assert off[torch.float32] < 1e-6
    for t in (torch.float16, torch.bfloat16):
        assert off[t] <= 2 * off[torch.float32] + 2.0 ** -24, off


# Two roundings, of the terms (as above) and of the result, are sqrt(2) of one.  delta has to add little to that: from the rounded o it is off
# by u |o|, which with n keys is sqrt(e / n) of what it is subtracted from, so that rows of 65 keys and more stay below sqrt(2 + 0.06), and
# rows of fewer need a better one.  The terms' share is a sum of squares over few terms where there are few rows and keys: an error e is
# uniform, e^2 has 0.8 of its mean squared as variance (second moment 1.8), and the terms' own sizes, products of a normal number and a
# softmax weight, have a fourth moment of about 8 times the squared second: a relative standard deviation of sqrt(1.8 * 8 / terms), of
# which three are allowed (16 for 14.4).  In dq the terms cancel a little: the keys a row prefers lie towards q, by 2 scale q among the terms
# (weighted by p^2) and by scale q around their mean, so that sum |term|^2 is (1 + 4 / D) / (1 + 1 / D) = 1.05 of |sum|^2 for queries of
# unit entries and 1.2 for those twice as long, which weigh more.  0.06 and, between the two, 0.14 make 2.2.
@pytest.mark.parametrize("dtype", DTYPES[1:], ids=str)
@pytest.mark.parametrize("keys", [2, 3, 15, 30, 64, 65, 90, 300])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("ragged", [False, True])
def test_attention_gradients_of_rows_with_few_keys(O, dtype, keys, causal, ragged):
    """16-bit dq and dk are no worse where rows see a handful of keys; rows of the first tile, of later ones, of shared heads"""
    B, Lq, Hq, Hk, D = 16, min(keys, 150) if causal else 150, 8, 4, 64
    nk = [max(2, keys - b % 4 * keys // 5) for b in range(B)] if ragged else None
    nq = [Lq - b % 3 for b in range(B)] if ragged and Lq > 3 else None
    q, do = normal((B, Lq, Hq, D), dtype, 1), normal((B, Lq, Hq, D), dtype, 2)
    k, v = normal((B, keys, Hk, D), dtype, 3), normal((B, keys, Hk, D), dtype, 4)
    got = run_attention(O, cuda(q), cuda(k), cuda(v), cuda(do), causal, None, cuda(lens(nq)), cuda(lens(nk)))
    want = R.attention(q, k, v, causal, None, nq, nk, do)
    terms = sum(Hq * (min(max(0, i + 1 + c - a), c) if causal else c) for a, c in zip(nq or [Lq] * B, nk or [keys] * B) for i in range(a))
    for n in ("dq", "dk", "dv"):
        x = want[n][0]
        once = float((x.to(dtype).double() - x).norm())
        off = float((got[n].cpu().double() - x).norm())
        assert off <= math.sqrt(2.2 + 3 * math.sqrt(16 / terms)) * once, (n, off / once)
    R.check(got, want)


@pytest.mark.parametrize("rows,classes,pad", [(9000, 1025, 3), (5000, 2048, 0), (6, 1500, 1), (300, 777, 0), (5000, 300, 0), (4100, 1025, 0)])
@pytest.mark.parametrize("tail", [None, False, True], ids=["log_probs", "distill", "distill with the rest"])
def test_fp32_gradients_are_not_off_by_the_rounding_of_lse(O, rows, classes, pad, tail):
    """lse is about 20: rounded to 32 bits it is off by up to 16 times 2^-24, and a probability by as much of itself.  What the kernels may
    lose, per probability p = exp(x), in units of 2^-24: two roundings of x (|x| each), one of the exponential (2), the sum's (5 after
    some 26 additions of random errors) and the products' (2), each 0.58 of that in the mean: at most 2 + |x|; of what is listed,
    one.  Student and teacher nearly agree."""
    g = torch.Generator().manual_seed(rows)
    teacher = torch.randn((rows, classes + pad), generator=g)[:, :classes] * 2 + 10
    z = (teacher + 0.2 * torch.randn((rows, classes), generator=g)).contiguous()
    zc = torch.zeros((rows, classes + pad), device="cuda")[:, :classes].copy_(cuda(z))
    x = z.double() - torch.logsumexp(z.double(), 1, keepdim=True)
    p = x.exp()
    if tail is None:
        w, at = torch.rand(rows, generator=g), torch.randint(0, classes, (rows, 1), generator=g, dtype=torch.int32)
        r = O.log_probs(zc, cuda(at))
        got = O.log_probs_backward(zc, cuda(at), r.lse, r.entropy, d_log_prob=cuda(w[:, None].contiguous()))
        want = torch.zeros_like(p).scatter_add_(1, at.long(), torch.ones((rows, 1), dtype=torch.float64)) - p
        # what is subtracted is 1: the gradient of the target itself is 1 - p, rounded
        room = (2 + x.abs()) * p + want.abs()
        want, room = want * w[:, None].double(), room * w[:, None].double()
    else:
        t = O.log_probs(cuda(teacher.contiguous()), top=20)
        index, value = t.top_index, t.top_log_prob
        if not tail:
            value = cuda(teacher).gather(1, index.long())
        w = torch.rand(rows, generator=g)
        r = O.distill(zc, index, value, tail=tail)
        got = O.distill_backward(cuda(w), zc, index, value, r.lse, r.log_tail, tail=tail)
        want = R.distill(z, index.cpu(), value.cpu(), 1.0, tail, w)["d_logits"][0]
        share = torch.zeros_like(p).scatter_add_(1, index.cpu().long(), torch.softmax(value.double().cpu(), 1))
        room = ((2 + x.abs()) * p + 2 * share) * w[:, None].double()
    off = float((got.cpu().double() - want).norm())
    assert off <= 2.0 ** -24 * float(room.norm()), off / (2.0 ** -24 * float(room.norm()))


@pytest.mark.parametrize("dtype", DTYPES[1:], ids=str)
def test_attention_rows_of_one_key_have_no_gradient(O, dtype):
    """p = 1 whatever the score: dq and dk are 0, and not what rounding leaves of do . v - delta"""
    for B, Lq, Lk, Hq, Hk, D, causal, nk in ((5, 200, 1, 4, 2, 64, False, None), (3, 30, 9, 4, 1, 96, False, [1, 9, 1]), (2, 700, 700, 2, 2, 128, True, None)):
        q, do = normal((B, Lq, Hq, D), dtype, 1), normal((B, Lq, Hq, D), dtype, 2)
        k, v = normal((B, Lk, Hk, D), dtype, 3), normal((B, Lk, Hk, D), dtype, 4)
        got = run_attention(O, cuda(q), cuda(k), cuda(v), cuda(do), causal, None, None, cuda(lens(nk)))
        R.check(got, R.attention(q, k, v, causal, None, None, nk, do))
        for b in range(B):
            if causal:
                assert bool((got["dq"][b, 0] == 0).all())
            elif nk is None or nk[b] == 1:
                assert bool((got["dq"][b] == 0).all()) and bool((got["dk"][b] == 0).all())


def test_scales_outside_of_32_bits_are_refused(O):
    """a scale that 32 bits hold as 0 would be read as the default; one that they hold as infinity (or whose product with log2(e) they do) has no exponentials"""
    q, z = torch.zeros((1, 4, 2, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros((2, 50), device="cuda")
    ix, val, f = torch.zeros((2, 3), dtype=torch.int32, device="cuda"), torch.zeros((2, 3), device="cuda"), torch.zeros(2, device="cuda")
    o, lse = O.attention(q, q, q)
    for s in (1e-46, 2.0 ** -150, 1e39, 3.3e38, 1e400, -1e-46, 0.0):
        for call in (lambda: O.attention(q, q, q, scale=s), lambda: O.attention_backward(q, q, q, q, o, lse, scale=s), lambda: O.log_probs(z, scale=s),
                     lambda: O.log_probs_backward(z, None, f, f, d_entropy=f, scale=s)):
            with pytest.raises(ValueError):
                call()
    for t in (1e46, 1e-39, 0.0, -1.0, 5e-324, math.nan):
        for call in (lambda: O.distill(z, ix, val, temperature=t), lambda: O.distill_backward(f, z, ix, val, f, temperature=t)):
            with pytest.raises(ValueError):
                call()


def test_a_tiny_scale_is_not_the_default(O):
    q, k, v = (normal((1, 40, 2, 64), torch.float32, s) for s in (1, 2, 3))
    o, lse = O.attention(cuda(q), cuda(k), cuda(v), scale=1e-44)
    R.check({"o": o, "lse": lse}, R.attention(q, k, v, False, 1e-44))


def test_what_torch_would_record_is_refused(O):
    """tangents of forward mode and traces would be cut silently"""
    from torch.autograd import forward_ad
    q = torch.zeros((1, 4, 2, 64), device="cuda")
    z, f, t = torch.zeros((2, 50), device="cuda"), torch.zeros(2, device="cuda"), torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    with forward_ad.dual_level():
        d, e, g = (forward_ad.make_dual(x, torch.ones_like(x)) for x in (q, z, f))
        for call in (lambda: O.attention(d, q, q), lambda: O.attention(q, q, d), lambda: O.log_probs(e), lambda: O.distill(e, t, f[:, None]),
                     lambda: O.distill(z, t, g[:, None]), lambda: O.distill_backward(g, z, t, f[:, None], f)):
            with pytest.raises(ValueError):
                call()
        O.log_probs(z)                       # no tangent: as ever
    for call in (lambda x: O.attention(x, x, x)[0], lambda x: O.log_probs(x[0, 0]).lse):
        with pytest.raises(ValueError):
            torch.jit.trace(call, q)
    for call in (lambda: torch.func.jvp(lambda x: O.log_probs(x).lse, (z,), (z,)), lambda: torch.func.vmap(lambda x: O.log_probs(x).lse)(z[None]),
                 lambda: torch.func.grad(lambda x: O.log_probs(x).lse.sum())(z)):
        with pytest.raises((ValueError, RuntimeError)):
            call()


def test_tensors_whose_memory_is_not_their_values_are_refused(O):
    """torch puts a negation off (the memory holds the opposite), and a tensor of zeros may have no memory at all"""
    q, z, f = (normal(s, torch.float32, 1).cuda() for s in ((1, 4, 2, 64), (2, 50), (2,)))
    t, ix = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    o, lse = O.attention(q, q, q)
    none = torch._efficientzerotensor
    for call in (lambda: O.attention(torch._neg_view(q), q, q), lambda: O.attention_backward(torch._neg_view(q), q, q, q, o, lse),
                 lambda: O.attention_backward(q, q, q, q, o, torch._neg_view(lse)), lambda: O.log_probs(torch._neg_view(z)),
                 lambda: O.distill_backward(torch._neg_view(f), z, ix, torch.zeros((2, 3), device="cuda"), f),
                 lambda: O.attention(q, q, q, k_lens=none((1,), dtype=torch.int32, device="cuda")),
                 lambda: O.log_probs(z, none((2,), dtype=torch.int32, device="cuda")), lambda: O.log_probs(none((2, 50), device="cuda"))):
        with pytest.raises((ValueError, RuntimeError)):      # (the second: where the C ABI finds the null pointer)
            call()


def test_sizes_beyond_32_bits_are_refused(O):
    """broadcast views reach them without the memory"""
    q, k, z = torch.zeros((1, 4, 2, 64), device="cuda"), torch.zeros((1, 1, 2, 64), device="cuda"), torch.zeros((1, 5), device="cuda")
    f, ix = torch.zeros(1, device="cuda").expand(1 << 31), torch.zeros((1, 1), dtype=torch.int32, device="cuda").expand(1 << 31, 1)
    long, many = k.expand(1, 1 << 31, 2, 64), z.expand(1 << 31, 5)
    for call in (lambda: O.attention(q, long, long), lambda: O.attention(q[:, :1].expand(1 << 32, 1, 2, 64), k.expand(1 << 32, 1, 2, 64), k.expand(1 << 32, 1, 2, 64)),
                 lambda: O.log_probs(many), lambda: O.log_probs(z[:, :1].expand(1, 1 << 31)), lambda: O.distill(many, ix, f[:, None]),
                 lambda: O.log_probs_backward(many, None, f, f, d_entropy=f)):
        with pytest.raises(ValueError):
            call()
