"""The operators for adapting a matcher (include/urf.h: urf_attn_*, urf_log_probs*, urf_distill*) on torch tensors.

Every function enqueues its kernels on the current stream of its tensors' device and returns tensors allocated there, workspaces
included, from torch's allocator: calls on several streams share nothing, and a call may be captured into a graph.  Forward and
backward are separate calls, as in the C ABI; nothing here records for autograd: inputs that require a gradient while it is enabled,
inputs with a tangent of forward mode, and calls under torch.jit.trace are refused, rather than silently cut from what is recorded.
"""
import collections
import functools
import math
import struct

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import check

TOP_MAX = 64                                                          # URF_TOP_MAX
DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}      # URF_F32, URF_F16, URF_BF16
LogProbs = collections.namedtuple("LogProbs", "log_prob entropy lse top_index top_log_prob")
Distill = collections.namedtuple("Distill", "loss lse log_tail")

# the C ABI's structs as bytes (a call takes microseconds on the GPU: ctypes objects would cost more than the kernels)
_ATTN_CONFIG = struct.Struct("=8ifi")        # urf_attn_config
_ATTN_TENSOR = struct.Struct("=Q3q")         # urf_attn_tensor
_ROWS_CONFIG = struct.Struct("@3i4xqfi")     # urf_rows_config


def _refuse(who, text):
    raise ValueError(f"{who}: {text}")


def _scale(who, name, x):
    """x, a factor that 32 bits hold neither as 0 (which the C ABI reads as a default) nor, times log2(e), as infinity"""
    if not 2.0 ** -150 < x < 2.0 ** 127:
        _refuse(who, f"{name} {x} (positive, in the range of 32 bits)")
    return x


def _config(who, layout, *values):
    try:
        return layout.pack(*values)
    except struct.error:
        _refuse(who, f"sizes beyond 32 bits: {values}")


def _untraced(who):
    if torch._C._get_tracing_state() is not None:
        _refuse(who, "a trace would not record this call")


def _given(who, name, t):
    """what the kernels would not see of a tensor"""
    if t.requires_grad and torch.is_grad_enabled():
        _refuse(who, f"{name} requires a gradient, which this call would not record: call it under torch.no_grad() or with detached "
                     "tensors, and the backward call for the gradients")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        _refuse(who, f"{name} has a tangent, which this call would not carry on")
    if t.is_neg():
        _refuse(who, f"{name} is a negation that was put off: materialise it first (clone())")


def _scores(who, name, t, device):
    """what every floating input has to be"""
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        _refuse(who, f"{name} has to be a tensor on the GPU")
    if t.dtype not in DTYPES:
        _refuse(who, f"{name} is {t.dtype} (float32, float16 or bfloat16)")
    if t.requires_grad or t.is_neg() or forward_ad._current_level >= 0:
        _given(who, name, t)
    if device is not None and t.device != device:
        _refuse(who, f"{name} is on {t.device}, not on {device}")
    return t.device


def _plain(who, name, t, dtype, shape, device):
    """a contiguous tensor of the given type and shape; its address"""
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.device == device and t.shape == shape and t.is_contiguous()):
        _refuse(who, f"{name} has to be a contiguous {dtype} tensor {tuple(shape)} on {device}")
    if t.requires_grad or t.is_neg() or forward_ad._current_level >= 0:
        _given(who, name, t)
    p = t.data_ptr()
    if not p and t.numel():
        _refuse(who, f"{name} has no memory")
    return p


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


# ------------------------------------------------------------------ attention
def _head_view(who, name, t, dtype, device):
    _scores(who, name, t, device)
    if t.dim() != 4:
        _refuse(who, f"{name} has to be [batch, rows, heads, head size]")
    if t.dtype is not dtype:
        _refuse(who, f"{name} is {t.dtype}, not {dtype}")
    (B, L, H, D), (sb, sr, sh, sd), p = t.shape, t.stride(), t.data_ptr()
    per = 4 if dtype is torch.float32 else 8
    if sd != 1 and D != 1:
        _refuse(who, f"the last dimension of {name} has to be contiguous")
    # the stride of a dimension of one says nothing
    sb, sr, sh = sb if B > 1 else 0, sr if L > 1 else 0, sh if H > 1 else 0
    if p % 16 or sb % per or sr % per or sh % per:
        _refuse(who, f"base and strides of {name} have to be multiples of 16 bytes (make it contiguous)")
    return _ATTN_TENSOR.pack(p, sb, sr, sh)


def _attn_config(who, q, k, v, causal, scale, q_lens, k_lens):
    """device, configuration, the views of q, k and v, the addresses of the lengths"""
    _untraced(who)
    device = _scores(who, "q", q, None)
    views = [_head_view(who, name, t, q.dtype, device) for name, t in (("q", q), ("k", k), ("v", v))]
    (B, Lq, Hq, D), (Bk, Lk, Hk, Dk) = q.shape, k.shape
    if k.shape != v.shape or Bk != B or Dk != D:
        _refuse(who, f"shapes {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)} of q, k and v do not fit")
    if scale is not None:
        _scale(who, "scale", scale)
    lens = [None if t is None else _plain(who, name, t, torch.int32, (B,), device) for name, t in (("q_lens", q_lens), ("k_lens", k_lens))]
    cfg = _config(who, _ATTN_CONFIG, DTYPES[q.dtype], B, Hq, Hk, D, Lq, Lk, 1 if causal else 0, scale or 0.0, device.index)
    return device, cfg, views, lens


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(cfg, backward):
    n = _lib.C.c_size_t()
    check(_lib.lib().urf_attn_workspace(cfg, backward, _lib.C.byref(n)), "urf_attn_workspace")
    return n.value


def _head_output(like, device):
    """a contiguous tensor of the shape and type of `like`, and its view"""
    B, L, H, D = like.shape
    sr = H * D
    sb = max(L, 1) * sr
    t = torch.empty_strided((B, L, H, D), (sb, sr, D, 1), dtype=like.dtype, device=device)
    return t, _ATTN_TENSOR.pack(t.data_ptr(), sb, sr, D)


def _floats(n, device):
    return torch.empty_strided((n,), (1,), dtype=torch.float32, device=device)


def attention(q, k, v, *, causal=False, scale=None, q_lens=None, k_lens=None):
    """o, lse = softmax(scale q k^T) v over [batch, rows, heads, head size] tensors (any strides of the first three dimensions
    that are multiples of 16 bytes); lse is [batch, heads, rows], float32.  k and v may have fewer heads (shared by consecutive
    query heads) and another length.  q_lens / k_lens: int32 [batch] on the GPU, rows / keys in use; scale defaults to
    1 / sqrt(head size); causal aligns the last row in use with the last key in use.  Rows without a visible key: o = 0,
    lse = -inf."""
    who = "attention"
    device, cfg, views, lens = _attn_config(who, q, k, v, causal, scale, q_lens, k_lens)
    B, Lq, Hq, _ = q.shape
    o, o_view = _head_output(q, device)
    lse = torch.empty_strided((B, Hq, Lq), (Hq * Lq, Lq, 1), dtype=torch.float32, device=device)
    if not B * Lq * Hq:
        return o, lse
    n = _workspace_bytes(cfg, 0)
    work = torch.empty(n, dtype=torch.uint8, device=device) if n else None
    check(_lib.lib().urf_attn_forward(cfg, *views, *lens, o_view, lse.data_ptr(), work.data_ptr() if n else None, n,
                                      _stream(device)), "urf_attn_forward")
    return o, lse


def attention_backward(do, q, k, v, o, lse, *, causal=False, scale=None, q_lens=None, k_lens=None):
    """dq, dk, dv for the gradient `do` of attention()'s o; o, lse and the other arguments are that call's."""
    who = "attention_backward"
    device, cfg, views, lens = _attn_config(who, q, k, v, causal, scale, q_lens, k_lens)
    B, Lq, Hq, _ = q.shape
    if not isinstance(do, torch.Tensor) or not isinstance(o, torch.Tensor) or do.shape != q.shape or o.shape != q.shape:
        _refuse(who, "do and o have to be of q's shape")
    o_view, do_view = _head_view(who, "o", o, q.dtype, device), _head_view(who, "do", do, q.dtype, device)
    lse = _plain(who, "lse", lse, torch.float32, (B, Hq, Lq), device)
    (dq, dq_view), (dk, dk_view), (dv, dv_view) = (_head_output(t, device) for t in (q, k, v))
    if not B * Lq * Hq:
        return dq, dk.zero_(), dv.zero_()
    n = _workspace_bytes(cfg, 1)
    work = torch.empty(n, dtype=torch.uint8, device=device)
    check(_lib.lib().urf_attn_backward(cfg, *views, o_view, lse, do_view, *lens, dq_view, dk_view, dv_view,
                                       work.data_ptr(), n, _stream(device)), "urf_attn_backward")
    return dq, dk, dv


# ------------------------------------------------------------------ rows of scores
def _rows_config(who, logits, scale):
    """device, rows, classes, configuration"""
    _untraced(who)
    device = _scores(who, "logits", logits, None)
    if logits.dim() != 2:
        _refuse(who, "logits has to be [rows, classes]")
    (R, V), (sr, sv) = logits.shape, logits.stride()
    if V < 1 or (sv != 1 and V > 1):
        _refuse(who, "the rows of logits have to be contiguous and not empty")
    _scale(who, "scale", scale)
    return device, R, V, _config(who, _ROWS_CONFIG, DTYPES[logits.dtype], R, V, sr, scale, device.index)


@functools.lru_cache(maxsize=1024)
def _log_probs_workspace(cfg, top):
    n = _lib.C.c_size_t()
    check(_lib.lib().urf_log_probs_workspace(cfg, top, _lib.C.byref(n)), "urf_log_probs_workspace")
    return n.value


def _targets(who, targets, R, device):
    """how many per row, and their address"""
    if targets is None:
        return 0, None
    if not (isinstance(targets, torch.Tensor) and targets.dim() in (1, 2)):
        _refuse(who, "targets has to be [rows] or [rows, n]")
    n = targets.shape[1] if targets.dim() == 2 else 1
    if n > TOP_MAX:
        _refuse(who, f"{n} targets per row (at most {TOP_MAX})")
    return n, _plain(who, "targets", targets, torch.int32, (R, *targets.shape[1:]), device)


def log_probs(logits, targets=None, *, top=0, scale=1.0):
    """LogProbs(log_prob, entropy, lse, top_index, top_log_prob) of softmax(scale * logits) per row of [rows, classes].  targets: int32
    [rows] or [rows, n] (n <= 64; -1 = none, log probability 0); `top` <= 64 alternatives, descending, equal scores by index.  What was
    not asked for is None."""
    who = "log_probs"
    device, R, V, cfg = _rows_config(who, logits, scale)
    n, at = _targets(who, targets, R, device)
    if not 0 <= top <= min(TOP_MAX, V):
        _refuse(who, f"top {top} (0 .. {TOP_MAX}, at most the {V} classes)")
    entropy, lse = _floats(R, device), _floats(R, device)
    log_prob = None if targets is None else torch.empty(targets.shape, dtype=torch.float32, device=device)
    top_index = torch.empty_strided((R, top), (top, 1), dtype=torch.int32, device=device) if top else None
    top_log_prob = torch.empty_strided((R, top), (top, 1), dtype=torch.float32, device=device) if top else None
    size = _log_probs_workspace(cfg, top)
    work = torch.empty(size, dtype=torch.uint8, device=device) if size else None
    check(_lib.lib().urf_log_probs(cfg, logits.data_ptr(), at, n, top, log_prob.data_ptr() if n else None, entropy.data_ptr(),
                                   lse.data_ptr(), top_index.data_ptr() if top else None, top_log_prob.data_ptr() if top else None,
                                   work.data_ptr() if size else None, size, _stream(device)), "urf_log_probs")
    return LogProbs(log_prob, entropy, lse, top_index, top_log_prob)


def log_probs_backward(logits, targets, lse, entropy, *, d_log_prob=None, d_entropy=None, scale=1.0):
    """The gradient of sum(log_prob * d_log_prob) + sum(entropy * d_entropy) with respect to logits; lse and entropy are
    log_probs()'s for the same logits, targets and scale."""
    who = "log_probs_backward"
    device, R, V, cfg = _rows_config(who, logits, scale)
    if d_log_prob is None:
        targets = None
    elif targets is None:
        _refuse(who, "d_log_prob without targets")
    n, at = _targets(who, targets, R, device)
    g = None if targets is None else _plain(who, "d_log_prob", d_log_prob, torch.float32, targets.shape, device)
    h = None if d_entropy is None else _plain(who, "d_entropy", d_entropy, torch.float32, (R,), device)
    lse, entropy = _plain(who, "lse", lse, torch.float32, (R,), device), _plain(who, "entropy", entropy, torch.float32, (R,), device)
    d = torch.empty((R, V), dtype=logits.dtype, device=device)
    check(_lib.lib().urf_log_probs_backward(cfg, logits.data_ptr(), at, n, lse, entropy, g, h, d.data_ptr(), V, _stream(device)),
          "urf_log_probs_backward")
    return d


def _teacher(who, index, value, R, device):
    """how many listed per row, the addresses of indices and values"""
    if not (isinstance(index, torch.Tensor) and index.dim() == 2 and 1 <= index.shape[1] <= TOP_MAX):
        _refuse(who, f"the teacher's indices have to be [rows, 1 .. {TOP_MAX}]")
    K = index.shape[1]
    return K, _plain(who, "teacher_index", index, torch.int32, (R, K), device), _plain(who, "teacher_value", value, torch.float32, (R, K), device)


def _inverse(who, temperature):
    if not 0 < temperature < math.inf:
        _refuse(who, f"temperature {temperature}")
    return _scale(who, "1 / temperature", 1.0 / temperature)


def distill(logits, teacher_index, teacher_value, *, temperature=1.0, tail=False):
    """Distill(loss, lse, log_tail) per row: the divergence of softmax(logits / temperature) from a teacher known by its top
    alternatives (int32 indices, -1 = unused, and float32 values, both [rows, listed]).  tail=False: the values are logits, the listed
    alternatives are all there is.  tail=True: the values are log probabilities at this temperature (log_probs(teacher, top=...,
    scale=1 / temperature)), and what they leave is one more outcome.  log_tail is None without tail."""
    who = "distill"
    device, R, V, cfg = _rows_config(who, logits, _inverse(who, temperature))
    K, index, value = _teacher(who, teacher_index, teacher_value, R, device)
    loss, lse = _floats(R, device), _floats(R, device)
    log_tail = _floats(R, device) if tail else None
    check(_lib.lib().urf_distill(cfg, logits.data_ptr(), index, value, K, 1 if tail else 0, loss.data_ptr(), lse.data_ptr(),
                                 log_tail.data_ptr() if tail else None, _stream(device)), "urf_distill")
    return Distill(loss, lse, log_tail)


def distill_backward(d_loss, logits, teacher_index, teacher_value, lse, log_tail=None, *, temperature=1.0, tail=False):
    """The gradient of sum(loss * d_loss) with respect to logits; lse, log_tail and the other arguments are distill()'s."""
    who = "distill_backward"
    device, R, V, cfg = _rows_config(who, logits, _inverse(who, temperature))
    K, index, value = _teacher(who, teacher_index, teacher_value, R, device)
    g, lse = _plain(who, "d_loss", d_loss, torch.float32, (R,), device), _plain(who, "lse", lse, torch.float32, (R,), device)
    log_tail = _plain(who, "log_tail", log_tail, torch.float32, (R,), device) if tail else None
    d = torch.empty((R, V), dtype=logits.dtype, device=device)
    check(_lib.lib().urf_distill_backward(cfg, logits.data_ptr(), index, value, K, 1 if tail else 0, lse, log_tail, g, d.data_ptr(), V,
                                          _stream(device)), "urf_distill_backward")
    return d
