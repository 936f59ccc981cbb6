"""The operators for adapting a matcher (include/urf.h: urf_attn_*, urf_log_probs*, urf_distill*) on torch tensors.

Every function enqueues its kernels on the current stream of its tensors' device and returns tensors allocated there, workspaces
included, from torch's allocator: calls on several streams share nothing, and a call may be captured into a graph.  Forward and
backward are separate calls, as in the C ABI; nothing here records for autograd (inputs that require a gradient are refused while
it is enabled, rather than silently cut from the graph).
"""
import collections
import ctypes as C
import math

import torch

from . import _lib
from ._lib import AttnConfig, AttnTensor, RowsConfig, check

TOP_MAX = 64                                                          # URF_TOP_MAX
LogProbs = collections.namedtuple("LogProbs", "log_prob entropy lse top_index top_log_prob")
Distill = collections.namedtuple("Distill", "loss lse log_tail")
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}      # URF_F32, URF_F16, URF_BF16


def _require(cond, text):
    if not cond:
        raise ValueError(text)


def _floats(who, **tensors):
    """the tensors' common device, after the checks every operator makes"""
    first = None
    for name, t in tensors.items():
        _require(isinstance(t, torch.Tensor) and t.is_cuda, f"{who}: {name} has to be a tensor on the GPU")
        _require(t.dtype in DTYPES, f"{who}: {name} is {t.dtype} (float32, float16 or bfloat16)")
        _require(not (torch.is_grad_enabled() and t.requires_grad),
                 f"{who}: {name} requires a gradient, which this call would not record: call it under torch.no_grad() with "
                 "detached tensors, and the backward call for the gradients")
        first = first if first is not None else t
        _require(t.device == first.device, f"{who}: {name} is on {t.device}, not on {first.device}")
    return first.device


def _ints(who, name, t, shape, device):
    if t is None:
        return None
    _require(isinstance(t, torch.Tensor) and t.dtype == torch.int32 and t.device == device and tuple(t.shape) == tuple(shape)
             and t.is_contiguous(), f"{who}: {name} has to be a contiguous int32 tensor {tuple(shape)} on {device}")
    return t


def _p(t):
    return None if t is None else C.c_void_p(t.data_ptr())


def _stream(device):
    return C.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _view(t):
    return AttnTensor(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def _heads(who, name, t, dtype):
    _require(t.dim() == 4, f"{who}: {name} has to be [batch, rows, heads, head size]")
    _require(t.dtype == dtype, f"{who}: {name} is {t.dtype}, not {dtype}")
    _require(t.stride(3) == 1 or t.shape[3] == 1, f"{who}: the last dimension of {name} has to be contiguous")
    per = 16 // t.element_size()
    _require(t.data_ptr() % 16 == 0 and all(t.stride(d) % per == 0 for d in range(3) if t.shape[d] > 1),
             f"{who}: base and strides of {name} have to be multiples of 16 bytes (make it contiguous)")
    return t


def _attn_config(who, q, k, v, causal, scale, q_lens, k_lens):
    for name, t in (("q", q), ("k", k), ("v", v)):
        _heads(who, name, t, q.dtype)
    _require(k.shape == v.shape and k.shape[0] == q.shape[0] and k.shape[3] == q.shape[3], f"{who}: shapes of q, k and v do not fit")
    _require(scale is None or (math.isfinite(scale) and scale > 0), f"{who}: scale {scale}")
    _ints(who, "q_lens", q_lens, q.shape[:1], q.device)
    _ints(who, "k_lens", k_lens, q.shape[:1], q.device)
    return AttnConfig(DTYPES[q.dtype], q.shape[0], q.shape[2], k.shape[2], q.shape[3], q.shape[1], k.shape[1], int(bool(causal)),
                      scale or 0.0, q.device.index)


def _workspace(cfg, backward, device):
    n = C.c_size_t()
    check(_lib.lib().urf_attn_workspace(C.byref(cfg), backward, C.byref(n)), "urf_attn_workspace")
    return torch.empty(n.value, dtype=torch.uint8, device=device) if n.value else None, n


def attention(q, k, v, *, causal=False, scale=None, q_lens=None, k_lens=None):
    """o, lse = softmax(scale q k^T) v over [batch, rows, heads, head size] tensors (any strides of the first three dimensions
    that are multiples of 16 bytes); lse is [batch, heads, rows], float32.  k and v may have fewer heads (shared by consecutive
    query heads) and another length.  q_lens / k_lens: int32 [batch] on the GPU, rows / keys in use; scale defaults to
    1 / sqrt(head size); causal aligns the last row in use with the last key in use.  Rows without a visible key: o = 0,
    lse = -inf."""
    who = "attention"
    device = _floats(who, q=q, k=k, v=v)
    cfg = _attn_config(who, q, k, v, causal, scale, q_lens, k_lens)
    o = torch.empty(q.shape, dtype=q.dtype, device=device)
    lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=device)
    if not q.numel():
        return o, lse
    work, n = _workspace(cfg, 0, device)
    check(_lib.lib().urf_attn_forward(C.byref(cfg), C.byref(_view(q)), C.byref(_view(k)), C.byref(_view(v)), _p(q_lens), _p(k_lens),
                                      C.byref(_view(o)), _p(lse), _p(work), n, _stream(device)), "urf_attn_forward")
    return o, lse


def attention_backward(do, q, k, v, o, lse, *, causal=False, scale=None, q_lens=None, k_lens=None):
    """dq, dk, dv for the gradient `do` of attention()'s o; o, lse and the other arguments are that call's."""
    who = "attention_backward"
    device = _floats(who, q=q, do=do, k=k, v=v, o=o, lse=lse)
    cfg = _attn_config(who, q, k, v, causal, scale, q_lens, k_lens)
    for name, t in (("do", do), ("o", o)):
        _require(_heads(who, name, t, q.dtype).shape == q.shape, f"{who}: {name} has to be of q's shape")
    _require(lse.dtype == torch.float32 and lse.is_contiguous() and tuple(lse.shape) == (q.shape[0], q.shape[2], q.shape[1]),
             f"{who}: lse has to be attention()'s")
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=device) for t in (q, k, v))
    if not q.numel():
        return dq, dk.zero_(), dv.zero_()
    work, n = _workspace(cfg, 1, device)
    check(_lib.lib().urf_attn_backward(C.byref(cfg), C.byref(_view(q)), C.byref(_view(k)), C.byref(_view(v)), C.byref(_view(o)),
                                       _p(lse), C.byref(_view(do)), _p(q_lens), _p(k_lens), C.byref(_view(dq)), C.byref(_view(dk)),
                                       C.byref(_view(dv)), _p(work), n, _stream(device)), "urf_attn_backward")
    return dq, dk, dv


def _rows_config(who, logits, scale):
    _require(logits.dim() == 2, f"{who}: logits has to be [rows, classes]")
    _require(logits.shape[1] >= 1 and (logits.stride(1) == 1 or logits.shape[1] == 1), f"{who}: the rows of logits have to be contiguous")
    _require(math.isfinite(scale) and scale > 0, f"{who}: scale {scale} (positive)")
    return RowsConfig(DTYPES[logits.dtype], logits.shape[0], logits.shape[1], logits.stride(0), scale, logits.device.index)


def _targets(who, targets, logits):
    if targets is None:
        return 0
    _require(isinstance(targets, torch.Tensor) and targets.dim() in (1, 2), f"{who}: targets has to be [rows] or [rows, n]")
    _ints(who, "targets", targets, (logits.shape[0],) + tuple(targets.shape[1:]), logits.device)
    n = targets.shape[1] if targets.dim() == 2 else 1
    _require(n <= TOP_MAX, f"{who}: {n} targets per row (at most {TOP_MAX})")
    return n


def _f32(who, name, t, shape, device):
    _require(isinstance(t, torch.Tensor) and t.dtype == torch.float32 and t.device == device and tuple(t.shape) == tuple(shape)
             and t.is_contiguous(), f"{who}: {name} has to be a contiguous float32 tensor {tuple(shape)} on {device}")
    return t


def log_probs(logits, targets=None, *, top=0, scale=1.0):
    """LogProbs(log_prob, entropy, lse, top_index, top_log_prob) of softmax(scale * logits) per row of [rows, classes].  targets: int32
    [rows] or [rows, n] (n <= 64; -1 = none, log probability 0); `top` <= 64 alternatives, descending, equal scores by index.  What was
    not asked for is None."""
    who = "log_probs"
    device = _floats(who, logits=logits)
    cfg = _rows_config(who, logits, scale)
    n = _targets(who, targets, logits)
    _require(0 <= top <= min(TOP_MAX, cfg.classes), f"{who}: top {top} (0 .. {TOP_MAX}, at most {cfg.classes} classes)")
    entropy, lse = (torch.empty(cfg.rows, dtype=torch.float32, device=device) for _ in range(2))
    log_prob = None if targets is None else torch.empty(targets.shape, dtype=torch.float32, device=device)
    top_index = torch.empty((cfg.rows, top), dtype=torch.int32, device=device) if top else None
    top_log_prob = torch.empty((cfg.rows, top), dtype=torch.float32, device=device) if top else None
    check(_lib.lib().urf_log_probs(C.byref(cfg), _p(logits), _p(targets), n, top, _p(log_prob), _p(entropy), _p(lse), _p(top_index),
                                   _p(top_log_prob), _stream(device)), "urf_log_probs")
    return LogProbs(log_prob, entropy, lse, top_index, top_log_prob)


def log_probs_backward(logits, targets, lse, entropy, *, d_log_prob=None, d_entropy=None, scale=1.0):
    """The gradient of sum(log_prob * d_log_prob) + sum(entropy * d_entropy) with respect to logits; lse and entropy are
    log_probs()'s for the same logits, targets and scale."""
    who = "log_probs_backward"
    device = _floats(who, logits=logits)
    cfg = _rows_config(who, logits, scale)
    if d_log_prob is None:
        targets = None
    n = _targets(who, targets, logits)
    _require((targets is None) == (d_log_prob is None), f"{who}: d_log_prob without targets")
    if targets is not None:
        _f32(who, "d_log_prob", d_log_prob, targets.shape, device)
    _f32(who, "lse", lse, (cfg.rows,), device)
    _f32(who, "entropy", entropy, (cfg.rows,), device)
    if d_entropy is not None:
        _f32(who, "d_entropy", d_entropy, (cfg.rows,), device)
    d = torch.empty(logits.shape, dtype=logits.dtype, device=device)
    check(_lib.lib().urf_log_probs_backward(C.byref(cfg), _p(logits), _p(targets), n, _p(lse), _p(entropy), _p(d_log_prob), _p(d_entropy),
                                            _p(d), C.c_longlong(cfg.classes), _stream(device)), "urf_log_probs_backward")
    return d


def _teacher(who, logits, index, value):
    _require(isinstance(index, torch.Tensor) and index.dim() == 2 and 1 <= index.shape[1] <= TOP_MAX,
             f"{who}: the teacher's indices have to be [rows, 1 .. {TOP_MAX}]")
    _ints(who, "teacher_index", index, (logits.shape[0], index.shape[1]), logits.device)
    _f32(who, "teacher_value", value, index.shape, logits.device)
    return index.shape[1]


def distill(logits, teacher_index, teacher_value, *, temperature=1.0, tail=False):
    """Distill(loss, lse, log_tail) per row: the divergence of softmax(logits / temperature) from a teacher known by its top
    alternatives (int32 indices, -1 = unused, and float32 values, both [rows, listed]).  tail=False: the values are logits, the listed
    alternatives are all there is.  tail=True: the values are log probabilities at this temperature (log_probs(teacher, top=...,
    scale=1 / temperature)), and what they leave is one more outcome.  log_tail is None without tail."""
    who = "distill"
    device = _floats(who, logits=logits)
    _require(math.isfinite(temperature) and temperature > 0, f"{who}: temperature {temperature}")
    cfg = _rows_config(who, logits, 1.0 / temperature)
    listed = _teacher(who, logits, teacher_index, teacher_value)
    loss, lse = (torch.empty(cfg.rows, dtype=torch.float32, device=device) for _ in range(2))
    log_tail = torch.empty(cfg.rows, dtype=torch.float32, device=device) if tail else None
    check(_lib.lib().urf_distill(C.byref(cfg), _p(logits), _p(teacher_index), _p(teacher_value), listed, int(bool(tail)), _p(loss), _p(lse),
                                 _p(log_tail), _stream(device)), "urf_distill")
    return Distill(loss, lse, log_tail)


def distill_backward(d_loss, logits, teacher_index, teacher_value, lse, log_tail=None, *, temperature=1.0, tail=False):
    """The gradient of sum(loss * d_loss) with respect to logits; lse, log_tail and the other arguments are distill()'s."""
    who = "distill_backward"
    device = _floats(who, logits=logits)
    _require(math.isfinite(temperature) and temperature > 0, f"{who}: temperature {temperature}")
    cfg = _rows_config(who, logits, 1.0 / temperature)
    listed = _teacher(who, logits, teacher_index, teacher_value)
    _f32(who, "d_loss", d_loss, (cfg.rows,), device)
    _f32(who, "lse", lse, (cfg.rows,), device)
    if tail:
        _f32(who, "log_tail", log_tail, (cfg.rows,), device)
    d = torch.empty(logits.shape, dtype=logits.dtype, device=device)
    check(_lib.lib().urf_distill_backward(C.byref(cfg), _p(logits), _p(teacher_index), _p(teacher_value), listed, int(bool(tail)), _p(lse),
                                          _p(log_tail if tail else None), _p(d_loss), _p(d), C.c_longlong(cfg.classes), _stream(device)),
          "urf_distill_backward")
    return d
