"""The token operators together: what a block's stages get from each other, each stage against an
independent result for the very inputs that it got, for a prompt and for single tokens over its cache; and
the same refusals from both paths of each operator.

Bounds for each stage are those of its own tests (test_rms_norm.py, test_int8.py, test_attention.py).
"""
import pytest
import torch

from pytorch_raft_amd.ops.attention import attention
from pytorch_raft_amd.ops.int8 import int8_linear, quantize_weight
from pytorch_raft_amd.ops.rms_norm import rms_norm, rms_norm_int8
from test_attention import close, formula

DEV = 'cuda'
W = 2.0 ** -24


def norm_stage(x, weight, r, got):
    """q within half a step of the exact quotient, scale and h within their roundings."""
    q, scale, h = (t.cpu().double() for t in got)
    c = x.shape[-1]
    e = W * (c / 2 + 6)
    exact = x.cpu().double() + r.cpu().double()
    assert ((h - exact).abs() <= 2.0 ** -8 * exact.abs()).all()
    y = h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * weight.cpu().double()
    top = y.abs().amax(-1)
    assert ((scale - top / 127).abs() <= (e + 2 * W) * top / 127).all()
    assert ((q - y * 127 / top[..., None]).abs() <= 0.5 + 127 * (2 * e + 4 * W)).all()


def product_stage(q, scale, weight, got):
    w, ws = (t.cpu().double() for t in weight)
    ref = q.cpu().double() @ w.t() * scale.cpu().double()[..., None] * ws
    assert ((got.cpu().double() - ref).abs() <= 1.01 * (2.0 ** -8 + 3 * W) * ref.abs() + 1e-37).all()


@pytest.mark.gpu
@pytest.mark.parametrize('heads,kv,d,l', [(4, 2, 64, 150), (3, 1, 40, 33), (2, 2, 128, 257)])
def test_stages_of_a_block(ext_ops, heads, kv, d, l):
    g = torch.Generator().manual_seed(11)
    mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    b, c, room = 2, heads * d, l + 9
    w1, w2 = (1 + 0.1 * mk(c)).to(DEV), (1 + 0.1 * mk(c)).to(DEV)
    # (weights as a layer keeps them, input channels first, turned for the product)
    qkv = [t.to(DEV) for t in quantize_weight((mk(c, (heads + 2 * kv) * d) / c ** 0.5).t())]
    up = [t.to(DEV) for t in quantize_weight((mk(c, 2 * c) / c ** 0.5).t())]
    assert qkv[0].is_contiguous()
    cache = [torch.full((b, room, kv, d), float('nan'), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    held = torch.tensor([l, l - 5], dtype=torch.int32, device=DEV)    # the second item's prompt is shorter

    def block(x, r, lengths, first):
        n, s, h = rms_norm_int8(x, w1, residual=r)
        norm_stage(x, w1, r, (n, s, h))
        p = int8_linear(n, s, *qkv)
        product_stage(n, s, qkv, p)
        q, k, v = p.view(*x.shape[:2], -1, d).split([heads, kv, kv], 2)
        for i in range(b):                                            # behind an item's end nothing is written
            m = min(x.shape[1], int(lengths[i]) - int(first[i]))
            for to, new in zip(cache, (k, v)):
                to[i, first[i]:first[i] + m] = new[i, :m]
        kw = dict(causal=True, lengths=lengths, q_offset=first)
        o = attention(q, *cache, **kw)
        close(o, formula(q, *cache, **kw), 'out')
        n, s, h2 = rms_norm_int8(o.reshape(x.shape), w2, residual=h)
        norm_stage(o.reshape(x.shape), w2, h, (n, s, h2))
        z = int8_linear(n, s, *up)
        product_stage(n, s, up, z)
        return h2

    with torch.no_grad():
        block(mk(b, l, c).to(torch.bfloat16).to(DEV), mk(b, l, c).to(torch.bfloat16).to(DEV), held,
              torch.zeros(b, dtype=torch.int32, device=DEV))
        for _ in range(3):                                            # single tokens
            first, held = held, held + 1
            block(mk(b, 1, c).to(torch.bfloat16).to(DEV), mk(b, 1, c).to(torch.bfloat16).to(DEV), held, first)
        assert all(torch.isnan(t[i, held[i]:]).all() for t in cache for i in range(b))


def refusals(dev):
    g = torch.Generator().manual_seed(0)
    mk = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    i8 = lambda *s: torch.randint(-9, 9, s, generator=g).to(torch.int8).to(dev)  # noqa: E731
    q, k, v = mk(2, 3, 4, 8), mk(2, 6, 2, 8), mk(2, 6, 2, 8)
    ints = torch.ones(2, dtype=torch.int32, device=dev)
    bools = lambda *s: torch.ones(*s, dtype=torch.bool, device=dev)  # noqa: E731
    f, value, kind = attention, ValueError, TypeError
    yield from ((f, a, kw, value) for a, kw in [
        ((q[0], k, v), {}), ((q, k[0], v[0]), {}), ((q, k[:1], v[:1]), {}), ((q, k, v[:, :5]), {}), ((q[:, :, :3], k, v), {}),
        ((q[:, :, :0], k, v), {}), ((q, k[:, :, :0], v[:, :, :0]), {}), ((q, k[..., :4], v[..., :4]), {}),
        ((q[..., :0], k[..., :0], v[..., :0]), {}), ((mk(1, 2, 1, 136),) * 3, {}),
        ((q, k, v), {'scale': 0.}), ((q, k, v), {'scale': -1.}), ((q, k, v), {'scale': float('inf')}),
        ((q, k, v), {'scale': float('nan')}), ((q, k, v), {'lengths': ints.long()}), ((q, k, v), {'lengths': ints[:1]}),
        ((q, k, v), {'lengths': ints[:, None]}), ((q, k, v), {'q_offset': ints.float()}), ((q, k, v), {'q_offset': ints[:0]}),
        ((q, k, v), {'mask': bools(3, 6, 3)}), ((q, k, v), {'mask': bools(1, 2, 4, 3, 6)}), ((q, k, v), {'mask': bools(3, 1, 1, 6)}),
        ((q, k, v), {'mask': bools(0)})])
    yield from ((f, a, kw, kind) for a, kw in [
        ((q, k.half(), v.half()), {}), ((q, k, v.half()), {}), ((q, k, v), {'mask': mk(3, 6)}), ((q, k, v), {'mask': ints[:1]})])
    x, r, w = mk(4, 16), mk(4, 16), mk(16)
    for f in (rms_norm, rms_norm_int8):
        yield from ((f, a, kw, value) for a, kw in [
            ((x, w[:8]), {}), ((x, w[None]), {}), ((x[0, 0], w), {}), ((x, w), {'residual': r[:3]}), ((x, w), {'residual': r[:1]}),
            ((x, w), {'residual': r.half()}), ((x, w), {'eps': -1.}), ((x, w), {'eps': float('nan')}),
            ((x, w), {'eps': float('inf')}), ((x[:, :0], w[:0]), {}), ((mk(1, 16385), mk(16385)), {})])
        yield f, (x, w.half()), {}, kind
        yield f, (x.half(), w.bfloat16()), {}, kind
    f, grad = int8_linear, RuntimeError
    x, xs, w, ws, bias = i8(5, 33), mk(5), i8(7, 33), mk(7), mk(7)
    yield from ((f, a, kw, value) for a, kw in [
        ((x[:, :32], xs, w, ws), {}), ((x, xs[:4], w, ws), {}), ((x, xs[:, None], w, ws), {}), ((x, xs, w[0], ws), {}),
        ((x, xs, w, ws[:4]), {}), ((x, xs, w, ws), {'bias': bias[:4]}), ((x, xs, w, ws), {'bias': bias.half()}),
        ((x, xs.double(), w, ws), {}), ((i8(1, 131072), xs[:1], i8(1, 131072), ws[:1]), {})])
    yield from ((f, a, kw, kind) for a, kw in [
        ((x.float(), xs, w, ws), {}), ((x, xs, w.float(), ws), {}), ((x, xs, w, ws), {'out_dtype': torch.int8})])
    yield f, (x, xs, w, ws.clone().requires_grad_(True)), {}, grad
    yield rms_norm_int8, (mk(4, 16).requires_grad_(True), mk(16)), {}, grad


def check_refusals(dev):
    for f, args, kw, error in refusals(dev):
        with pytest.raises(error):
            f(*args, **kw)


def test_refusals_of_the_plain_forms():
    check_refusals('cpu')


@pytest.mark.gpu
def test_refusals_of_the_kernels(ext_ops):
    check_refusals(DEV)
