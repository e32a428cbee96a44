"""Softmax attention over tokens (flattened feature maps, or any sequence): HIP kernels + torch oracle.

``attention(q, k, v)``: q (B, Lq, H, D), k and v (B, Lk, Hkv, D) -> (B, Lq, H, D), where query head h
reads key head ``h // (H // Hkv)``.  A channels_last feature map (B, C, h, w) is such a tensor without
a copy: ``x.permute(0, 2, 3, 1).reshape(B, h * w, heads, C // heads)``; so are the parts of one q|k|v
projection.

* ``scale``: of the scores, default ``D ** -0.5``; positive, within fp32's range (2^-150 .. 2^127).
* ``lengths`` (B,) int32: item b holds keys 0 .. lengths[b] - 1; what lies behind is not read.
* ``causal``: query i of item b stands at key position ``q_offset[b] + i`` and sees the keys up to it;
  ``q_offset`` (B,) int32 defaults to ``Lk - Lq`` (the last query sees the last key).  A step over
  caches filled to ``lengths`` passes ``q_offset = lengths - Lq``.  Without ``causal`` it changes nothing.
* ``mask``: bool, broadcastable to (B, H, Lq, Lk), True where a query sees a key.  Keys hidden by a mask
  that has one row for all queries and heads (a padding mask (B, 1, 1, Lk), or that expanded: sizes and
  strides tell, not the values) may hold anything; under a mask with a row for each query or head, and under
  ``causal``, keys and values must be finite also where they are hidden.

A query that sees no key gets zeros, and zero gradients, and adds nothing to those of keys and values: it
and its output's gradient may hold anything.  Where a query sees a key, an infinity or NaN in it, in what
it sees or in its output's gradient may reach all gradients of its head.  bf16, fp16 and fp32; sums, maxima and
accumulators are fp32, the probabilities are rounded to the inputs' type for their product with v.
Differentiable in q, k and v by the backward pass, once on the GPU: second and forward-mode derivatives
raise there (the backward recomputes the probabilities from a saved log-sum-exp; the same inputs give the
same bits).  Head sizes up to 128 (others than multiples of 8 are padded by a copy); less than 2^22 pairs
of item and key head and less than 2^26 rows (B * H * Lq) a call.  Calls with at most 32 rows
(H / Hkv * Lq), e.g. single tokens over a cache, run a kernel that splits the keys.

The all-pairs correlation (ops/corr.py) is the same product of two feature maps without the softmax.
"""
import torch

from . import _ext

MAX_HEAD = 128
LOG2_E = 1.4426950408889634


def torch_attention(q, k, v, scale=None, causal=False, mask=None, lengths=None, q_offset=None):
    """Plain implementation in the inputs' precision (also the CPU path)."""
    b, lq, h, d = q.shape
    lk, hkv = k.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    dev = q.device
    j = torch.arange(lk, device=dev)
    see = torch.ones(b, 1, lq, lk, dtype=torch.bool, device=dev)
    if lengths is not None:
        see = see & (j < lengths[:, None])[:, None, None]
    if causal:
        first = q_offset if q_offset is not None else torch.full((b,), lk - lq, device=dev)
        pos = first[:, None] + torch.arange(lq, device=dev)
        see = see & (j <= pos[..., None])[:, None]
    if mask is not None:
        see = see & mask
    # keys that nobody sees may hold anything
    used = see.any(1).any(1)[:, :, None, None]
    k = torch.where(used, k, torch.zeros_like(k)).repeat_interleave(h // hkv, 2)
    v = torch.where(used, v, torch.zeros_like(v)).repeat_interleave(h // hkv, 2)
    # and so may queries that see no key, and their gradients
    none = ~see.any(-1, keepdim=True)
    q = q.masked_fill(none.transpose(1, 2), 0.)
    s = torch.matmul(q.transpose(1, 2).contiguous(), k.permute(0, 2, 3, 1).contiguous()) * scale
    p = torch.softmax(s.masked_fill(~see, float('-inf')).masked_fill(none, 0.), -1) if lk else s
    return torch.matmul(p, v.transpose(1, 2).contiguous()).transpose(1, 2).masked_fill(none.transpose(1, 2), 0.)


def _check(q, k, v, scale, mask, lengths, q_offset):
    """The operator's own checks (csrc/bindings_tokens.cpp) for the plain form; -> the scale."""
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise ValueError('q must be (B, Lq, H, D), k and v (B, Lk, Hkv, D); got %s, %s, %s'
                         % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    b, lq, h, d = q.shape
    if k.shape[0] != b or k.shape[3] != d:
        raise ValueError('q %s and k %s disagree on batch or head size' % (tuple(q.shape), tuple(k.shape)))
    if not k.shape[2] or not h or h % k.shape[2]:
        raise ValueError('the %d query heads must be a multiple of the %d key heads' % (h, k.shape[2]))
    if not 1 <= d <= MAX_HEAD:
        raise ValueError('head size must be 1 .. %d, got %d' % (MAX_HEAD, d))
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError('q, k and v must have one dtype, got %s, %s, %s' % (q.dtype, k.dtype, v.dtype))
    scale = d ** -0.5 if scale is None else float(scale)
    # (scores are formed in fp32, in units of log 2)
    if not 2. ** -150 < scale * LOG2_E <= torch.finfo(torch.float32).max:
        raise ValueError('scale must be positive and finite in fp32 (2^-150 .. 2^127), got %r' % scale)
    if mask is not None:
        if mask.dtype != torch.bool:
            raise TypeError('mask must be bool (True = seen), got %s' % mask.dtype)
        if mask.dim() > 4 or any(m not in (1, n) for m, n in zip(mask.shape[::-1], (k.shape[1], lq, h, b))):
            raise ValueError('mask %s does not broadcast to %s' % (tuple(mask.shape), (b, h, lq, k.shape[1])))
    for name, t in (('lengths', lengths), ('q_offset', q_offset)):
        if t is not None and (t.dtype != torch.int32 or t.shape != (b,)):
            raise ValueError('%s must be int32 of shape (%d,), got %s %s' % (name, b, t.dtype, tuple(t.shape)))
    for name, t in (('k', k), ('v', v), ('mask', mask), ('lengths', lengths), ('q_offset', q_offset)):
        if t is not None and t.device != q.device:
            raise ValueError('%s is on %s, q on %s' % (name, t.device, q.device))
    return scale


def attention(q, k, v, scale=None, causal=False, mask=None, lengths=None, q_offset=None, impl='auto'):
    if impl != 'torch' and _ext.device_ok(q) and _ext.gpu_path_enabled(required=(impl == 'hip')):
        # (checks, padding and the autograd node are the operator's own: csrc/bindings_tokens.cpp)
        return _ext.ops().attention(q, k, v, scale, causal, mask, lengths, q_offset)
    scale = _check(q, k, v, scale, mask, lengths, q_offset)
    return torch_attention(q, k, v, scale, causal, mask, lengths, q_offset)
