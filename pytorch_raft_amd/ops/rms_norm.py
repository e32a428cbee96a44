"""Root-mean-square norm over the channels, with the residual's addition: HIP kernels + torch oracle.

``rms_norm(x, weight)`` -> y = x / sqrt(mean x^2 + eps) * weight.
``rms_norm(x, weight, residual=r)`` -> (y, h): h = x + r, rounded to the type of x (it is the stream
that the next residual adds to), and y is the norm of h as rounded.  Differentiable in x, residual and
weight by the backward pass, once on the GPU: second and forward-mode derivatives raise there (the
encoders' fused norms, ops/encoder.py, are the per-image and per-batch counterparts).

``rms_norm_int8(x, weight, residual=None)`` -> (q, scale, h): the same norm with an 8-bit output for
``int8_linear`` (ops/int8.py): q = rint(y * 127 / max|y|) int8 with one fp32 scale = max|y| / 127 per
row (both from the unrounded fp32 y; an all-zero row has scale 0; a row with an infinity or NaN has a scale
of infinity or NaN, and its 8 bits say nothing).
h is None without a residual.  For inference: it has no gradient.

x (..., C) bf16, fp16 or fp32, C up to 16384; weight (C,) fp32 or the type of x; statistics in fp32.
"""
import torch

from . import _ext

MAX_CHANNELS = 16384


def _torch_norm(x, weight, residual, eps):
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    h = x if residual is None else (x.to(wide) + residual.to(wide)).to(x.dtype)
    f = h.to(wide)
    return f * torch.rsqrt(f.square().mean(-1, keepdim=True) + eps) * weight.to(wide), h


def torch_rms_norm(x, weight, residual=None, eps=1e-6):
    """Plain implementation (also the CPU path)."""
    y, h = _torch_norm(x, weight, residual, eps)
    y = y.to(x.dtype)
    return y if residual is None else (y, h)


def torch_rms_norm_int8(x, weight, residual=None, eps=1e-6):
    y, h = _torch_norm(x, weight, residual, eps)
    top = y.abs().amax(-1, keepdim=True)
    # (127 / top passes fp32's range for rows under 2^-121)
    up = torch.where(top < 2. ** -100, 2. ** 64, 1.).to(top.dtype)
    q = torch.round(y * up * torch.where(top == 0, torch.zeros_like(top), 127 / (top * up))).clamp(-127, 127)
    return q.nan_to_num(0.).to(torch.int8), (top / 127).squeeze(-1), None if residual is None else h


def _check(x, weight, residual, eps):
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_CHANNELS:
        raise ValueError('x must be (..., C) with 1 .. %d channels, got %s' % (MAX_CHANNELS, tuple(x.shape)))
    if weight.shape != x.shape[-1:]:
        raise ValueError('weight %s does not match the channels of x %s' % (tuple(weight.shape), tuple(x.shape)))
    if weight.dtype not in (torch.float32, x.dtype):
        raise TypeError('weight must be float32 or %s, got %s' % (x.dtype, weight.dtype))
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError('residual %s %s does not match x %s %s'
                         % (residual.dtype, tuple(residual.shape), x.dtype, tuple(x.shape)))
    if not 0 <= eps < float('inf'):
        raise ValueError('eps must be finite and not negative, got %r' % eps)
    for name, t in (('weight', weight), ('residual', residual)):
        if t is not None and t.device != x.device:
            raise ValueError('%s is on %s, x on %s' % (name, t.device, x.device))


def _on_gpu(x, impl):
    return impl != 'torch' and _ext.device_ok(x) and _ext.gpu_path_enabled(required=(impl == 'hip'))


def rms_norm(x, weight, residual=None, eps=1e-6, impl='auto'):
    if _on_gpu(x, impl):
        # (checks and the autograd node are the operator's own: csrc/bindings_tokens.cpp)
        if residual is None:
            return _ext.ops().rms_norm(x, weight, eps)
        return _ext.ops().rms_norm_residual(x, weight, residual, eps)
    _check(x, weight, residual, eps)
    return torch_rms_norm(x, weight, residual, eps)


def rms_norm_int8(x, weight, residual=None, eps=1e-6, impl='auto'):
    if _on_gpu(x, impl):
        out = _ext.ops().rms_norm_int8(x, weight, residual, eps)
        return tuple(out) if residual is not None else (*out, None)
    _check(x, weight, residual, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError('rms_norm_int8 has no gradient: call it under torch.no_grad()')
    if _ext.has_tangent(x, weight, residual):
        raise RuntimeError('rms_norm_int8 has no forward-mode derivative')
    return torch_rms_norm_int8(x, weight, residual, eps)
