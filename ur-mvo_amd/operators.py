"""The operators for adapting a matcher (include/urf.h: urf_attn_*, urf_log_probs*, urf_distill*) on torch tensors.

Every function enqueues its kernels on the current stream of its tensors' device and returns tensors allocated there, workspaces
included, from torch's allocator: calls on several streams share nothing, and a call may be captured into a graph.  Forward and
backward are separate calls, as in the C ABI; nothing here records for autograd (inputs that require a gradient are refused while
it is enabled, rather than silently cut from the graph).
"""
import ctypes as C
import math

import torch

from . import _lib
from ._lib import AttnConfig, AttnTensor, check

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
