"""8-bit integer linear layer (a 1x1 conv over NHWC pixels) with a scale for each token and each output
channel: HIP kernel + torch oracle.

``int8_linear(x, x_scale, w, w_scale, bias=None, out_dtype=torch.bfloat16)``:
    out[..., n] = x_scale[...] * w_scale[n] * sum_k x[..., k] * w[n, k]  (+ bias[n])
x (..., K) int8 and x_scale (...) fp32 come from ``rms_norm_int8`` (ops/rms_norm.py); w (N, K) int8 and
w_scale (N,) fp32 from ``quantize_weight`` once; bias (N,) fp32.  The sum is exact (int32; K up to
131071), scaled in fp32 and rounded once to ``out_dtype`` (bf16, fp16 or fp32).  For inference: no
gradient.  Operands whose rows start on 16 bytes (K a multiple of 16) take the fastest loads.
"""
import torch

from . import _ext

MAX_K = 131071
_CODES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def quantize_weight(weight):
    """(N, K) floating weight -> (int8 (N, K), fp32 scale (N,)), contiguous, symmetric per output channel; once, not
    per call.  A row with an infinity or NaN has a scale of infinity or NaN, and its 8 bits say nothing."""
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError('weight must be a floating (N, K) tensor, got %s %s' % (weight.dtype, tuple(weight.shape)))
    w = weight.detach().float()
    top = w.abs().amax(1, keepdim=True) if w.shape[1] else w.new_zeros(w.shape[0], 1)
    # (127 / top passes fp32's range for rows under 2^-121: they are raised by 2^64 first, exactly)
    up = torch.where(top < 2. ** -100, 2. ** 64, 1.).to(top.dtype)
    q = torch.round(w * up * torch.where(top == 0, torch.zeros_like(top), 127 / (top * up))).clamp_(-127, 127)
    # (rows of k one after the other, also for a transposed weight: int8_linear would copy it every call)
    return q.to(torch.int8).contiguous(), (top / 127).reshape(-1)


def torch_int8_linear(x, x_scale, w, w_scale, bias=None, out_dtype=torch.bfloat16):
    """Plain implementation (also the CPU path); 64-bit sums are exact like the kernel's."""
    y = (torch.matmul(x.double(), w.double().t()).float() * x_scale[..., None]) * w_scale
    return (y if bias is None else y + bias).to(out_dtype)


def int8_linear(x, x_scale, w, w_scale, bias=None, out_dtype=torch.bfloat16, impl='auto'):
    if impl != 'torch' and _ext.device_ok(x) and _ext.gpu_path_enabled(required=(impl == 'hip')):
        # (the checks are the operator's own: csrc/bindings_tokens.cpp)
        if out_dtype not in _CODES:
            raise TypeError('out_dtype must be bfloat16, float16 or float32, got %s' % out_dtype)
        return _ext.ops().int8_linear(x, x_scale, w, w_scale, bias, _CODES[out_dtype])
    if x.dtype != torch.int8 or w.dtype != torch.int8:
        raise TypeError('x and w must be int8, got %s and %s' % (x.dtype, w.dtype))
    if out_dtype not in _CODES:
        raise TypeError('out_dtype must be bfloat16, float16 or float32, got %s' % out_dtype)
    if x.dim() < 1 or w.dim() != 2 or x.shape[-1] != w.shape[1]:
        raise ValueError('x must be (..., K), w (N, K); got %s, %s' % (tuple(x.shape), tuple(w.shape)))
    n, k = w.shape
    if k > MAX_K:
        raise ValueError('K = %d could overflow the 32-bit sums (at most %d)' % (k, MAX_K))
    for name, t, shape in (('x_scale', x_scale, x.shape[:-1]), ('w_scale', w_scale, (n,)), ('bias', bias, (n,))):
        if t is None and name == 'bias':
            continue
        if t.dtype != torch.float32 or t.shape != tuple(shape):
            raise ValueError('%s must be float32 of shape %s, got %s %s' % (name, tuple(shape), t.dtype, tuple(t.shape)))
        if torch.is_grad_enabled() and t.requires_grad:
            raise RuntimeError('int8_linear has no gradient (%s requires one): call it under torch.no_grad()' % name)
    for name, t in (('x_scale', x_scale), ('w', w), ('w_scale', w_scale), ('bias', bias)):
        if t is not None and t.device != x.device:
            raise ValueError('%s is on %s, x on %s' % (name, t.device, x.device))
    if _ext.has_tangent(x_scale, w_scale, bias):
        raise RuntimeError('int8_linear has no forward-mode derivative')
    return torch_int8_linear(x, x_scale, w, w_scale, bias, out_dtype)
