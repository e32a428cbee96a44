"""8-bit integer linear layer (ops/int8.py): plain form, refusals, and the HIP kernel against the exact
integer sum in 64 bits.

The sum is an integer of at most 31 bits: its conversion to fp32 rounds once (w = 2^-24), the two scales
and the bias once each, the result once more to its type (u = eps / 2):
  |out - exact| <= (u + 3 w) |out| + 3 w |sum xs ws| + w |bias|  (+ 2^-25 under fp16's normal range)
"""
import pytest
import torch

from pytorch_raft_amd.ops.attention import attention
from pytorch_raft_amd.ops.int8 import int8_linear, quantize_weight
from pytorch_raft_amd.ops.rms_norm import rms_norm, rms_norm_int8

DEV = 'cuda'
DTS = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def inputs(m, n, k, dev=DEV, seed=0, top=False):
    g = torch.Generator().manual_seed(seed)
    x, w = (torch.randint(-128, 128, s, generator=g).to(torch.int8) for s in ((m, k), (n, k)))
    if top:
        x[:], w[:] = -128, -128
    return [t.to(dev) for t in (x, torch.rand(m, generator=g) * 0.01, w, torch.rand(n, generator=g) * 0.01, torch.randn(n, generator=g))]


def check(x, xs, w, ws, bias, dt):
    out = int8_linear(x, xs, w, ws, bias=bias, out_dtype=dt, impl='hip')
    assert out.dtype == dt and out.shape == (*x.shape[:-1], w.shape[0])
    xc, xsc, wc, wsc = (t.cpu().double() for t in (x, xs, w, ws))
    part = xc @ wc.t() * xsc[..., None] * wsc
    ref = part if bias is None else part + bias.cpu().double()
    f = 2.0 ** -24
    tol = (torch.finfo(dt).eps / 2 + 3 * f) * ref.abs() + 3 * f * part.abs() + (f * bias.cpu().double().abs() if bias is not None else 0)
    d = (out.cpu().double() - ref).abs()
    assert (d <= 1.01 * tol + (2.0 ** -25 if dt == torch.float16 else 1e-37)).all(), d.max()
    return out


def test_plain_form():
    x, xs, w, ws, b = inputs(5, 7, 33, dev='cpu')
    ref = (x.long() @ w.long().t()).double() * xs[:, None].double() * ws.double() + b.double()
    assert torch.allclose(int8_linear(x, xs, w, ws, bias=b, out_dtype=torch.float32).double(), ref, rtol=1e-6, atol=1e-6)


def test_quantize_weight():
    w = torch.randn(9, 50, generator=torch.Generator().manual_seed(0))
    w[4] = 0
    q, s = quantize_weight(w)
    assert q.dtype == torch.int8 and s[4] == 0 and (q[4] == 0).all()
    assert ((q.float() * s[:, None] - w).abs() <= 0.5001 * s[:, None]).all()
    with pytest.raises(ValueError):
        quantize_weight(w[0])


def test_refusals():
    x, xs, w, ws, b = inputs(5, 7, 33, dev='cpu')
    for args, kw in (((x[:, :32], xs, w, ws), {}), ((x, xs[:4], w, ws), {}), ((x, xs, w, ws[:4]), {}),
                     ((x, xs, w, ws), {'bias': b[:4]}), ((x, xs.double(), w, ws), {}),
                     ((torch.zeros(1, 131072, dtype=torch.int8), xs[:1], torch.zeros(1, 131072, dtype=torch.int8), ws[:1]), {})):
        with pytest.raises(ValueError):
            int8_linear(*args, **kw)
    for args, kw in (((x.float(), xs, w, ws), {}), ((x, xs, w.float(), ws), {}), ((x, xs, w, ws), {'out_dtype': torch.int8})):
        with pytest.raises(TypeError):
            int8_linear(*args, **kw)
    with pytest.raises(RuntimeError):
        int8_linear(x, xs, w, ws.requires_grad_(True))


@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
@pytest.mark.parametrize('m', [1, 5, 16, 17, 32, 33, 64, 65, 130, 333])
@pytest.mark.parametrize('n,k', [(1, 1), (16, 64), (17, 33), (100, 128), (130, 257), (259, 1040), (64, 2500)])
def test_sizes(ext_ops, dt, m, n, k):
    x, xs, w, ws, b = inputs(m, n, k)
    check(x, xs, w, ws, b, DTS[dt])
    check(x, xs, w, ws, None, DTS[dt])


@pytest.mark.gpu
@pytest.mark.parametrize('m,n,k', [(2100, 2050, 64), (4100, 4200, 160), (4097, 4099, 77), (2049, 2200, 130), (8200, 16400, 32), (8193, 16387, 15)])
def test_large_tiles(ext_ops, m, n, k):
    """Sizes that fill the GPU with 128 x 128 and 256 x 256 tiles, whole and ragged."""
    x, xs, w, ws, b = inputs(m, n, k)
    out = int8_linear(x, xs, w, ws, bias=b, out_dtype=torch.float32)
    ref = torch.matmul(x.float(), w.float().t())     # exact: |sum| < 2^24
    ref = ref * xs[:, None] * ws
    tol = 2.0 ** -24 * 5 * (ref.abs() + b.abs())
    assert ((out - (ref + b)).abs() <= tol + 1e-30).all()


@pytest.mark.gpu
@pytest.mark.parametrize('m', [3, 100])
def test_largest_sums(ext_ops, m):
    x, xs, w, ws, b = inputs(m, 20, 131071, top=True)
    check(x, xs, w, ws, b, torch.float32)
    w.fill_(127)
    check(x, xs, w, ws, None, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize('m', [4, 200])
def test_layouts(ext_ops, m):
    x, xs, w, ws, b = inputs(m, 96, 64)
    ref = check(x, xs, w, ws, b, torch.bfloat16)
    assert torch.equal(ref, check(x.t().contiguous().t(), xs, w.t().contiguous().t(), ws, b, torch.bfloat16))
    flat = torch.zeros(w.numel() + 1, dtype=torch.int8, device=DEV)
    flat[1:] = w.flatten()
    assert torch.equal(ref, check(x, xs, flat[1:].view(w.shape), ws, b, torch.bfloat16))
    out = int8_linear(x.view(2, m // 2, 64), xs.view(2, m // 2), w, ws, bias=b)
    assert torch.equal(out.view(m, 96), ref)
    assert int8_linear(x[:0], xs[:0], w, ws).shape == (0, 96)
    assert (int8_linear(x[:, :0], xs, w[:, :0], ws) == 0).all()


@pytest.mark.gpu
def test_block_of_the_operators(ext_ops):
    """norm -> 8-bit projection -> attention -> norm with the residual -> 8-bit projection, as a token
    block serves: a prompt, then a single token over the cache that the prompt left.  The single
    token's output is the prompt form's for the same token: the two kernels differ in the order of
    their sums (attention's output by 2 u relative of sum P|v|), which can move an 8-bit value by a
    step, 1 / 127 of a row's largest: 4 % of the output's rms over 256 channels bounds it."""
    g = torch.Generator().manual_seed(7)
    mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    b, l, heads, kv, d = 2, 150, 4, 2, 64
    c = heads * d
    w1, w2 = (1 + 0.1 * mk(c)).to(DEV), (1 + 0.1 * mk(c)).to(DEV)
    qkv = [t.to(DEV) for t in quantize_weight(mk((heads + 2 * kv) * d, c) / c ** 0.5)]
    up = [t.to(DEV) for t in quantize_weight(mk(2 * c, c) / c ** 0.5)]
    x = mk(b, l, c).to(torch.bfloat16).to(DEV)

    def block(x, cache=None, lengths=None):
        n, s, _ = rms_norm_int8(x, w1)
        q, k, v = int8_linear(n, s, *qkv).view(*x.shape[:2], -1, d).split([heads, kv, kv], 2)
        if cache is not None:
            at = (lengths - 1).long()
            rows = torch.arange(b, device=DEV)
            cache[0][rows, at], cache[1][rows, at] = k[:, 0], v[:, 0]
            o = attention(q, *cache, lengths=lengths)
        else:
            o = attention(q, k, v, causal=True)
        n, s, h = rms_norm_int8(o.reshape(x.shape), w2, residual=x)
        return int8_linear(n, s, *up), h, k, v

    with torch.no_grad():
        full, hfull, k, v = block(x)
        cache = [torch.full((b, 200, kv, d), float('nan'), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        cache[0][:, :l - 1], cache[1][:, :l - 1] = k[:, :-1], v[:, :-1]
        one, hone, _, _ = block(x[:, -1:], cache, torch.full((b,), l, dtype=torch.int32, device=DEV))
        wide = rms_norm(x.double().cpu(), w1.double().cpu(), impl='torch')
    assert torch.isfinite(one).all() and torch.isfinite(wide).all()
    assert (hone - hfull[:, -1:]).abs().max() <= 2.0 ** -7 * hfull.abs().max()
    assert (one - full[:, -1:]).abs().max() <= 0.04 * 4 * full.float().square().mean().sqrt()
