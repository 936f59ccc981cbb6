"""Refusals of the operators for adapting a matcher at the C ABI and in operators.py (no GPU: every check comes before the device is
touched), and the 64-bit definitions the GPU tests compare with against autograd."""
import ctypes as C
import math

import pytest
import torch

import operators_reference as R


class Attn:
    """a valid forward / backward call on addresses that are never followed"""

    def __init__(self, U, **change):
        self.L, self.O = U._lib.lib(), U.operators
        c = dict(dtype=2, batch=2, q_heads=4, kv_heads=2, head_dim=64, q_len=10, k_len=20, causal=0, scale=0.0, device=0)
        c.update({k: v for k, v in change.items() if k in c})
        self.cfg = self.O._ATTN_CONFIG.pack(*c.values())
        self.c, self.change = c, change

    def view(self, name, rows, heads):
        base = {"q": 1 << 20, "k": 2 << 20, "v": 3 << 20, "o": 4 << 20, "do": 5 << 20, "dq": 6 << 20, "dk": 7 << 20, "dv": 8 << 20}[name]
        v = [base, rows * heads * 64, heads * 64, 64]
        for i, key in enumerate(("p", "sb", "sr", "sh")):
            v[i] = self.change.get(f"{name}_{key}", v[i])
        return None if v[0] is None else self.O._ATTN_TENSOR.pack(*v)

    def views(self, names):
        return [self.view(n, self.c["q_len"] if n in ("q", "o", "do", "dq") else self.c["k_len"],
                          self.c["q_heads"] if n in ("q", "o", "do", "dq") else self.c["kv_heads"]) for n in names]

    def forward(self):
        return self.L.urf_attn_forward(self.cfg, *self.views("qkv"), None, None, *self.views(["o"]), self.change.get("lse", 1 << 24),
                                       self.change.get("work", 1 << 25), self.change.get("bytes", 1 << 30), None)

    def backward(self):
        return self.L.urf_attn_backward(self.cfg, *self.views("qkvo"), self.change.get("lse", 1 << 24), *self.views(["do"]), None, None,
                                        *self.views(["dq", "dk", "dv"]), self.change.get("work", 1 << 25),
                                        self.change.get("bytes", 1 << 30), None)


BOTH = [dict(dtype=3), dict(dtype=-1), dict(batch=0), dict(q_len=0), dict(k_len=-1), dict(kv_heads=0), dict(kv_heads=3), dict(q_heads=0),
        dict(head_dim=0), dict(head_dim=12), dict(head_dim=136), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
        dict(q_p=None), dict(v_p=0), dict(q_p=(1 << 20) + 8), dict(k_sr=130), dict(v_sh=4), dict(q_sb=1), dict(lse=None),
        dict(q_len=1 << 30, q_heads=8, kv_heads=1), dict(batch=1 << 30), dict(batch=1 << 22, kv_heads=4), dict(q_len=1 << 27), dict(k_len=1 << 28),
        dict(batch=1 << 15, q_len=1 << 10), dict(batch=1 << 30, q_heads=1 << 30, kv_heads=1 << 30), dict(k_len=(1 << 31) - 1)]
FORWARD = [dict(o_p=None), dict(o_p=1 << 20), dict(o_sr=0), dict(o_sh=32), dict(o_sb=0), dict(o_sr=64), dict(o_sb=64 * 4 * 9), dict(o_sr=128, o_sh=64), dict(o_sr=64, o_sh=64 * 9),
           dict(o_sb=-64), dict(o_sb=1 << 61), dict(work=None, q_len=1, k_len=5000),
           dict(bytes=16, q_len=1, k_len=5000), dict(work=(1 << 25) + 4, q_len=1, k_len=5000)]
BACKWARD = [dict(do_p=None), dict(o_p=None), dict(dq_p=None), dict(dk_p=2 << 20), dict(dq_p=5 << 20), dict(dv_p=7 << 20), dict(dk_sr=0),
            dict(dv_sb=0), dict(dk_sr=64), dict(dq_sb=64 * 39), dict(work=None), dict(bytes=0), dict(work=(1 << 25) + 8)]


@pytest.mark.parametrize("change", BOTH, ids=str)
def test_attention_refuses(U, change):
    a = Attn(U, **change)
    assert a.forward() == -2 and a.backward() == -2
    assert U._lib.lib().urf_last_error()


@pytest.mark.parametrize("change", FORWARD, ids=str)
def test_attention_forward_refuses(U, change):
    assert Attn(U, **change).forward() == -2


@pytest.mark.parametrize("change", BACKWARD, ids=str)
def test_attention_backward_refuses(U, change):
    assert Attn(U, **change).backward() == -2


def test_attention_workspace(U):
    L, O, n = U._lib.lib(), U.operators, C.c_size_t(7)

    def size(backward, **c):
        a = Attn(U, **c)
        assert L.urf_attn_workspace(a.cfg, backward, C.byref(n)) == 0
        return n.value

    assert L.urf_attn_workspace(None, 0, C.byref(n)) == -2 and L.urf_attn_workspace(Attn(U).cfg, 0, None) == -2
    assert L.urf_attn_workspace(Attn(U, dtype=9).cfg, 0, C.byref(n)) == -2
    assert size(0, batch=64, q_len=1024, k_len=1024) == 0                            # enough workgroups: nothing to join
    assert size(0, batch=1, q_len=1, k_len=8192) >= 2 * 4 * (64 + 2) * 4             # two ranges at least
    assert size(1) >= 2 * 4 * 10 * 4                                                 # delta
    assert size(1, k_len=0) >= 2 * 4 * 10 * 4


class Rows:
    def __init__(self, U, **change):
        self.L = U._lib.lib()
        c = dict(dtype=0, rows=4, classes=50, row_stride=50, scale=1.0, device=0)
        c.update({k: v for k, v in change.items() if k in c})
        self.cfg, self.x = U.operators._ROWS_CONFIG.pack(*c.values()), change

    def a(self, name, default):
        return self.x.get(name, default)

    def log_probs(self):
        return self.L.urf_log_probs(self.a("cfg", self.cfg), self.a("z", 4096), self.a("t", 1 << 16), self.a("n", 1), self.a("top", 3),
                                    self.a("lp", 1 << 17), self.a("h", 1 << 18), self.a("lse", 1 << 19), self.a("ti", 1 << 20), self.a("tp", 1 << 21),
                                    self.a("work", 1 << 25), self.a("bytes", 1 << 30), None)

    def log_probs_backward(self):
        return self.L.urf_log_probs_backward(self.a("cfg", self.cfg), self.a("z", 4096), self.a("t", 1 << 16), self.a("n", 1), self.a("lse", 1 << 19),
                                             self.a("h", 1 << 18), self.a("g", 1 << 22), self.a("gh", 1 << 23), self.a("d", 1 << 24), self.a("ds", 50), None)

    def distill(self):
        return self.L.urf_distill(self.a("cfg", self.cfg), self.a("z", 4096), self.a("ix", 1 << 16), self.a("v", 1 << 17), self.a("k", 5), self.a("tail", 1),
                                  self.a("loss", 1 << 18), self.a("lse", 1 << 19), self.a("lt", 1 << 20), None)

    def distill_backward(self):
        return self.L.urf_distill_backward(self.a("cfg", self.cfg), self.a("z", 4096), self.a("ix", 1 << 16), self.a("v", 1 << 17), self.a("k", 5),
                                           self.a("tail", 1), self.a("lse", 1 << 19), self.a("lt", 1 << 20), self.a("g", 1 << 22), self.a("d", 1 << 24),
                                           self.a("ds", 50), None)


ALL = ["log_probs", "log_probs_backward", "distill", "distill_backward"]
GRAD = ["log_probs_backward", "distill_backward"]


@pytest.mark.parametrize("calls,change", [
    (ALL, dict(cfg=None)), (ALL, dict(dtype=7)), (ALL, dict(rows=-1)), (ALL, dict(classes=0)), (ALL, dict(classes=(1 << 31) - 1)), (ALL, dict(scale=0.0)), (ALL, dict(rows=1 << 24, row_stride=0)),
    (ALL, dict(scale=-2.0)), (ALL, dict(scale=math.nan)), (ALL, dict(z=None)), (ALL, dict(z=4098)), (ALL, dict(lse=None)),
    (["log_probs", "log_probs_backward"], dict(n=65)), (["log_probs", "log_probs_backward"], dict(n=-1)), (["log_probs", "log_probs_backward"], dict(t=None)),
    (["log_probs"], dict(top=65)), (["log_probs"], dict(top=-1)), (["log_probs"], dict(top=51)), (["log_probs"], dict(lp=None)),
    (["log_probs"], dict(h=None)), (["log_probs"], dict(ti=None)), (["log_probs"], dict(classes=100000, row_stride=0, work=None)),
    (["log_probs"], dict(classes=100000, row_stride=0, bytes=1000)), (["log_probs"], dict(classes=100000, row_stride=0, work=(1 << 25) + 8)), (["log_probs"], dict(tp=None)),
    (["log_probs_backward"], dict(h=None)), (["log_probs_backward"], dict(g=None)),
    (["distill", "distill_backward"], dict(k=0)), (["distill", "distill_backward"], dict(k=65)), (["distill", "distill_backward"], dict(ix=None)),
    (["distill", "distill_backward"], dict(v=None)), (["distill", "distill_backward"], dict(lt=None)), (["distill"], dict(loss=None)),
    (["distill_backward"], dict(g=None)), (GRAD, dict(d=None)), (GRAD, dict(d=(1 << 24) + 2)), (GRAD, dict(ds=49)), (GRAD, dict(d=4096)),
    (GRAD, dict(d=4096 + 4 * 150)), (GRAD, dict(d=4096 - 4 * 10)),
], ids=str)
def test_rows_refuse(U, calls, change):
    for call in calls:
        assert getattr(Rows(U, **change), call)() == -2, call


def test_log_probs_workspace(U):
    L, n = U._lib.lib(), C.c_size_t()

    def size(top, **c):
        assert L.urf_log_probs_workspace(Rows(U, **c).cfg, top, C.byref(n)) == 0
        return n.value

    assert size(3) == 0 and size(3, rows=5000, classes=100000) == 0 and size(0, rows=0, classes=100000) == 0
    assert size(5, rows=1, classes=100000) >= 2 * (5 * 8 + 12)                       # two parts at least
    for c, top in ((dict(dtype=9), 0), (dict(), 51), (dict(), -1), (dict(), 65)):
        assert L.urf_log_probs_workspace(Rows(U, **c).cfg, top, C.byref(n)) == -2
    assert L.urf_log_probs_workspace(None, 0, C.byref(n)) == -2 and L.urf_log_probs_workspace(Rows(U).cfg, 0, None) == -2


def test_rows_of_no_rows_are_nothing_to_do(U):
    for call in ALL:
        assert getattr(Rows(U, rows=0, z=None, d=None, t=None, ix=None, v=None), call)() == 0, call


def test_match_log_probs_refuses(U):
    assert U._lib.lib().urf_sg_match_log_probs(None, None, 0, None, None, None, None) == -2


def test_python_refuses_what_is_not_on_the_gpu(U):
    O = U.operators
    q, z = torch.zeros((1, 2, 1, 64)), torch.zeros((2, 5))
    t = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: O.attention(q, q, q), lambda: O.attention_backward(q, q, q, q, q, q), lambda: O.log_probs(z, t), lambda: O.attention(1, q, q),
                 lambda: O.log_probs_backward(z, t, z[:, 0], z[:, 0], d_log_prob=z[:, 0]), lambda: O.distill(z, t[:, None], z[:, :1]),
                 lambda: O.distill_backward(z[:, 0], z, t[:, None], z[:, :1], z[:, 0]), lambda: O.log_probs(None)):
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------ the definitions themselves
def test_reference_attention_is_autograds():
    g = torch.Generator().manual_seed(0)
    q, k, v, do = (torch.randn(s, generator=g, dtype=torch.float32) for s in ((2, 9, 4, 8), (2, 13, 2, 8), (2, 13, 2, 8), (2, 9, 4, 8)))
    for causal, nq, nk in ((False, None, None), (True, None, None), (True, [9, 4], [5, 13])):
        want = R.attention(q, k, v, causal, 0.3, nq, nk, do)
        x, y, w = (t.double().requires_grad_() for t in (q, k, v))
        total = 0
        for b in range(2):
            a, c = (9, 13) if nq is None else (nq[b], nk[b])
            for h in range(4):
                s = 0.3 * x[b, :a, h] @ y[b, :c, h // 2].T
                if causal:
                    s = s.masked_fill(torch.arange(c)[None] > torch.arange(a)[:, None] + (c - a), -math.inf)
                rows = torch.isfinite(s).any(1)
                o = torch.softmax(s[rows], 1) @ w[b, :c, h // 2]
                assert torch.allclose(o, want["o"][0][b, :a, h][rows], atol=1e-12)
                assert bool((want["o"][0][b, :a, h][~rows] == 0).all())
                total = total + (o * do[b, :a, h][rows].double()).sum()
        total.backward()
        for t, n in ((x, "dq"), (y, "dk"), (w, "dv")):
            assert torch.allclose(t.grad, want[n][0], atol=1e-12)


def test_reference_rows_are_autograds():
    g = torch.Generator().manual_seed(0)
    z = (torch.randn((4, 30), generator=g) * 2)
    z[1, 3:9] = -math.inf
    targets = torch.tensor([[1, 1], [4, -1], [29, 30], [0, 7]])
    gl, gh = torch.randn((4, 2), generator=g), torch.randn(4, generator=g)
    x = z.double().requires_grad_()
    lp = torch.log_softmax(0.5 * x, 1)
    p = lp.exp()
    H = -(p * lp.masked_fill(p == 0, 0.0)).sum(1)
    ok = (targets >= 0) & (targets < 30)
    picked = lp.gather(1, targets.clamp(0, 29))
    picked = torch.where(ok & torch.isfinite(picked), picked, 0.0)
    assert torch.isfinite(picked).all()
    gl = torch.where(torch.isfinite(lp.gather(1, targets.clamp(0, 29))), gl, 0.0)
    ((picked * gl).sum() + (H * gh).sum()).backward()
    assert torch.allclose(R.log_probs(z, targets, 0, 0.5, gl, gh)["d_logits"][0], x.grad, atol=1e-12)
    index = torch.tensor([[3, 3, -1], [20, 12, 11], [-1, -1, -1], [5, 29, 0]], dtype=torch.int32)
    value = torch.log(torch.tensor([[0.2, 0.3, 0.1], [0.5, 0.1, 0.1], [0.3, 0.3, 0.3], [0.4, 0.4, 0.2]]))
    for tail in (False, True):
        x = z.double().requires_grad_()
        want = R.distill(z, index, value, 2.0, tail, gh)
        lq = torch.log_softmax(x / 2, 1)
        total = 0
        for r in range(4):
            use = [(int(i), float(a)) for i, a in zip(index[r], value[r].double()) if i >= 0]
            w = [math.exp(a) for _, a in use] if tail else torch.softmax(torch.tensor([a / 2 for _, a in use], dtype=torch.float64), 0).tolist() if use else []
            loss = sum(b * (math.log(b) - lq[r, i]) for b, (i, _) in zip(w, use))
            rest = 1 - sum(w)
            if tail and rest >= 2.0 ** -20:
                others = [i for i in range(30) if i not in {j for j, _ in use}]
                loss = loss + rest * (math.log(rest) - torch.logsumexp(lq[r, others], 0))
            assert abs(float(torch.as_tensor(loss).detach()) - float(want["loss"][0][r])) < 1e-9
            total = total + loss * float(gh[r])
        total.backward()
        assert torch.allclose(x.grad, want["d_logits"][0], atol=1e-9)
