"""Token attention (ops/attention.py): the plain form on the CPU, refusals, and the HIP kernels against
the formula in 64 bits.

Tolerances are elementwise bounds, computed in 64 bits from the inputs: with u = eps / 2 of the type
(one rounding to nearest) and w = 2^-24 (one fp32 rounding),
  scores     e_s = w (D + 8) scale sum_d |q_d k_d| (fp32 accumulation of D products, scaling, exponent)
  out        (u + e) sum_j P|v| + u |out|,  e = 2 max_j e_s + w (Lk + 16): P rounded once, sums in fp32
  delta      sum_d |dout| tol_out + w (D + 1) sum_d |dout out|   (it is formed from the rounded out)
  dS         u |dS| + P (2 e (|dP| + |delta|) + w (D + 8) sum_d |dout v| + tol_delta)
  dv, dk, dq  sums of the above against |dout|, scale |q|, scale |k|, plus u of the result
fp16 adds its absolute steps: probabilities below 2^-14 of a row's reference are off by 2^-25 in the
forward; in the backward both operands are scaled to 2^14, so 2^-39 of their bounds.  A result under
fp16's least normal value 2^-14 is rounded to a multiple of 2^-24, off by up to 2^-25 whatever its size
(for bf16 and fp32 the same step is 2^-133 and 2^-149: nothing here comes near them).
"""
import math

import pytest
import torch

from pytorch_raft_amd.ops.attention import attention, torch_attention

DEV = 'cuda'
DTS = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}


def formula(q, k, v, do=None, scale=None, causal=False, mask=None, lengths=None, q_offset=None):
    """64-bit out, gradients and elementwise tolerances; loops over batch and heads, on the CPU."""
    u = torch.finfo(q.dtype).eps / 2
    w = 2.0 ** -24
    tiny = q.dtype == torch.float16
    b, lq, h, d = q.shape
    lk, hkv = k.shape[1:3]
    scale = d ** -0.5 if scale is None else scale
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    do = None if do is None else do.detach().cpu().double()
    res = {n: torch.zeros(b, lq, h, d, dtype=torch.float64) for n in ('out', 'dq', 't_out', 't_dq')}
    res.update({n: torch.zeros(b, lk, hkv, d, dtype=torch.float64) for n in ('dk', 'dv', 't_dk', 't_dv')})
    for i in range(b):
        n = lk if lengths is None else int(lengths[i])
        see = (torch.arange(lk) < n).expand(lq, lk).clone()
        if causal:
            first = lk - lq if q_offset is None else int(q_offset[i])
            see &= torch.arange(lk) <= (first + torch.arange(lq))[:, None]
        for j in range(h):
            m = see if mask is None else see & mask.cpu().expand(b, h, lq, lk)[i, j]
            used = m.any(0)
            kk, vv = (torch.where(used[:, None], t[i, :, j // (h // hkv)], torch.zeros(())) for t in (k, v))
            qq = q[i, :, j]
            s = torch.where(m, scale * qq @ kk.t(), torch.tensor(-math.inf, dtype=torch.float64))
            some = m.any(-1, keepdim=True)
            p = torch.softmax(torch.where(some, s, torch.zeros(())), -1) * m
            o = p @ vv
            es = w * (d + 8) * scale * (qq.abs() @ kk.abs().t()) * m
            e = 2 * (es.max(-1, keepdim=True).values if lk else 0) + w * (lk + 16)
            to = (u + e) * (p @ vv.abs()) + u * o.abs() + (2.0 ** -25 * (m.double() @ vv.abs()) if tiny else 0)
            res['out'][i, :, j], res['t_out'][i, :, j] = o, to
            if do is None:
                continue
            dd = do[i, :, j]
            delta = (dd * o).sum(-1, keepdim=True)
            tdelta = (dd.abs() * to).sum(-1, keepdim=True) + w * (d + 1) * (dd * o).abs().sum(-1, keepdim=True)
            dp = dd @ vv.t()
            ds = p * (dp - delta)
            tds = u * ds.abs() + p * (2 * e * (dp.abs() + delta.abs()) + w * (d + 8) * (dd.abs() @ vv.abs().t()) + tdelta)
            tp = (u + 2 * e) * p
            if tiny:
                tds = tds + 2.0 ** -38 * 2 * dd.norm(dim=-1).max() * vv.norm(dim=-1).max() * m
                tp = tp + 2.0 ** -38 * m
            g = j // (h // hkv)
            res['dv'][i, :, g] += p.t() @ dd
            res['t_dv'][i, :, g] += tp.t() @ dd.abs() + w * (lq * (h // hkv)) * (p.t() @ dd.abs())
            res['dk'][i, :, g] += scale * ds.t() @ qq
            res['t_dk'][i, :, g] += scale * (tds.t() @ qq.abs() + w * (lq * (h // hkv)) * (ds.abs().t() @ qq.abs()))
            res['dq'][i, :, j] = scale * ds @ kk
            res['t_dq'][i, :, j] = scale * (tds @ kk.abs() + w * lk * (ds.abs() @ kk.abs()))
    for n in ('dq', 'dk', 'dv'):
        res['t_' + n] += u * res[n].abs()
    if tiny:
        for n in ('out', 'dq', 'dk', 'dv'):
            res['t_' + n] += 2.0 ** -25
    return res


def close(got, res, name):
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), name
    over = (got - res[name]).abs() - 1.01 * res['t_' + name] - 1e-30
    assert (over <= 0).all(), '%s: off by %.3g where %.3g is allowed' % (
        name, (got - res[name]).abs().flatten()[over.argmax()], res['t_' + name].flatten()[over.argmax()])


def inputs(b, lq, lk, hkv, g, d, dt, seed=0, dev=DEV):
    gen = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=gen).to(dt).to(dev)  # noqa: E731
    return mk(b, lq, hkv * g, d), mk(b, lk, hkv, d), mk(b, lk, hkv, d), mk(b, lq, hkv * g, d)


def check(q, k, v, do=None, **kw):
    if do is not None:
        q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = attention(q, k, v, impl='hip', **kw)
    res = formula(q, k, v, do, **kw)
    close(out, res, 'out')
    if do is not None:
        for n, t in zip(('dq', 'dk', 'dv'), torch.autograd.grad(out, (q, k, v), do)):
            assert t.dtype == q.dtype
            close(t, res, n)
    return out


# ------------------------------------------------------------------------------------------- CPU
@pytest.mark.parametrize('kw', [{}, {'causal': True}, {'scale': 0.3}])
def test_plain_form_against_formula(kw):
    q, k, v, _ = inputs(2, 5, 9, 2, 2, 8, torch.float32, dev='cpu')
    lengths = torch.tensor([9, 4], dtype=torch.int32)
    mask = torch.rand(2, 4, 5, 9, generator=torch.Generator().manual_seed(1)) < 0.7
    mask[0, 1, 3] = False
    for more in ({}, {'lengths': lengths}, {'mask': mask}, {'mask': mask[:, :1, :1], 'lengths': lengths}):
        close(attention(q, k, v, **kw, **more), formula(q, k, v, **kw, **more), 'out')


def test_plain_form_hidden_keys_may_hold_anything():
    q, k, v, _ = inputs(2, 3, 6, 1, 2, 8, torch.float32, dev='cpu')
    k[0, 4:], v[0, 4:] = float('nan'), float('inf')
    lengths = torch.tensor([4, 6], dtype=torch.int32)
    close(attention(q, k, v, lengths=lengths), formula(q, k, v, lengths=lengths), 'out')


def test_plain_form_gradients_against_differences():
    q, k, v, do = (t.double().requires_grad_(True) for t in inputs(1, 3, 4, 1, 2, 8, torch.float32, dev='cpu'))
    mask = torch.tensor([[1, 0, 1, 1], [0, 0, 0, 0], [1, 1, 0, 1]]).bool()
    assert torch.autograd.gradcheck(lambda *t: torch_attention(*t, mask=mask), (q, k, v))


def test_refusals():
    q, k, v, _ = inputs(2, 3, 6, 2, 2, 8, torch.float32, dev='cpu')
    ints = torch.ones(2, dtype=torch.int32)
    bad = [((q[0], k, v), {}), ((q, k[:1], v[:1]), {}), ((q, k, v[:, :5]), {}), ((q[:, :, :3], k, v), {}),
           ((q, k[..., :4], v[..., :4]), {}), ((q, k, v), {'scale': 0.}), ((q, k, v), {'scale': -1.}),
           ((q, k, v), {'scale': float('inf')}), ((q, k, v), {'scale': float('nan')}),
           ((q, k, v), {'lengths': ints.long()}), ((q, k, v), {'lengths': ints[:1]}),
           ((q, k, v), {'q_offset': ints.float()}), ((q, k, v), {'mask': torch.ones(3, 6, 3).bool()}),
           ((q, k, v), {'mask': torch.ones(1, 2, 4, 3, 6).bool()}),
           ((torch.zeros(1, 2, 1, 136),) * 3, {})]
    for args, kw in bad:
        with pytest.raises(ValueError):
            attention(*args, **kw)
    with pytest.raises(TypeError):
        attention(q, k.half(), v.half())
    with pytest.raises(TypeError):
        attention(q, k, v, mask=torch.zeros(3, 6))


# ------------------------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
@pytest.mark.parametrize('d', [8, 32, 40, 64, 80, 96, 128])
def test_head_sizes(ext_ops, dt, d):
    check(*inputs(2, 70, 133, 2, 1, d, DTS[dt]))


@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
@pytest.mark.parametrize('lq,lk', [(1, 1), (1, 31), (1, 600), (2, 32), (31, 33), (32, 64), (33, 65), (64, 128),
                                   (127, 129), (128, 1), (129, 700), (300, 257)])
def test_lengths(ext_ops, dt, lq, lk):
    check(*inputs(1, lq, lk, 2, 1, 64, DTS[dt]))


@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
@pytest.mark.parametrize('hkv,g', [(1, 1), (1, 3), (3, 2), (2, 8)])
@pytest.mark.parametrize('lq,lk', [(1, 300), (4, 300), (77, 77), (150, 150)])
def test_shared_heads_causal(ext_ops, dt, hkv, g, lq, lk):
    check(*inputs(2, lq, lk, hkv, g, 32, DTS[dt]), causal=True)


@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
@pytest.mark.parametrize('lq', [1, 9, 140])
@pytest.mark.parametrize('causal', [False, True])
def test_ragged(ext_ops, dt, lq, causal):
    """Items of 0, 1, odd and all keys; NaN and infinities behind them; queries before the first key."""
    q, k, v, do = inputs(5, lq, 200, 2, 2, 64, DTS[dt])
    lengths = torch.tensor([0, 1, 67, 128, 200], dtype=torch.int32, device=DEV)
    behind = torch.arange(200, device=DEV) >= lengths[:, None]
    k[behind], v[behind] = float('nan'), float('inf')
    for q_offset in (None, lengths - lq) if causal else (None,):
        out = check(q, k, v, do, lengths=lengths, causal=causal, q_offset=q_offset)
        assert (out[0] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
@pytest.mark.parametrize('lq', [1, 20, 100])
def test_masks(ext_ops, dt, lq):
    b, lk, hkv, g = 2, 165, 2, 2
    q, k, v, do = inputs(b, lq, lk, hkv, g, 40, DTS[dt])
    gen = torch.Generator().manual_seed(5)
    full = (torch.rand(b, hkv * g, lq, lk, generator=gen) < 0.5).to(DEV)
    full[0, 1, lq // 2] = False                   # a row with nothing
    full[1, :, :, 64:128] = False                 # a whole tile
    shared = full[:, :1]                          # one mask for all heads
    single = full[0, 0]                           # for all items
    turned = full.transpose(2, 3).contiguous().transpose(2, 3)   # keys are not the fastest dimension
    for m in (full, shared, single, turned):
        check(q, k, v, do, mask=m)
        check(q, k, v, do, mask=m, causal=True, lengths=torch.tensor([165, 101], dtype=torch.int32, device=DEV))
    keys = full[:, :1, :1].clone()
    keys[1] = False                               # an item with nothing
    hidden = ~keys[:, 0, 0]
    k, v = k.clone(), v.clone()
    k[hidden], v[hidden] = float('inf'), float('nan')
    out = check(q, k, v, do, mask=keys)
    assert (out[1] == 0).all()
    check(q, k, v, do, mask=keys, causal=True, lengths=torch.tensor([165, 101], dtype=torch.int32, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
@pytest.mark.parametrize('lq', [3, 50])
def test_layouts(ext_ops, dt, lq):
    """Parts of one projection, heads before tokens, odd offsets, expanded heads, head sizes off 8."""
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(2, lq, 6, 48, generator=gen).to(DTS[dt]).to(DEV)
    q, k, v = x.split([2, 2, 2], 2)
    do = torch.randn(2, lq, 2, 48, generator=gen).to(DTS[dt]).to(DEV)
    ref = check(q.contiguous(), k.contiguous(), v.contiguous(), do)
    assert torch.equal(ref, check(q, k, v, do.transpose(1, 2).contiguous().transpose(1, 2)))
    assert torch.equal(ref, check(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)), do))
    assert torch.equal(ref, check(*(t.permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0) for t in (q, k, v)), do))
    flat = torch.zeros(q.numel() + 1, dtype=q.dtype, device=DEV)
    flat[1:] = q.reshape(-1)
    assert torch.equal(ref, check(flat[1:].view(q.shape), k, v, do))
    check(q, k[:, :, :1].expand_as(k), v[:, :1].expand_as(v), do.expand_as(do))
    check(*(t[..., :13] for t in (q, k, v, do)))
    out = attention(q.detach().requires_grad_(True), k, v)
    out.sum().backward()                          # an expanded gradient


@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
def test_magnitudes(ext_ops, dt):
    """Scores far apart (one key takes all), and gradients far under fp16's range before scaling."""
    q, k, v, do = inputs(1, 90, 140, 1, 2, 64, DTS[dt])
    check(q * 6, k, v, do)
    check(q, k, v, do * 2.0 ** -12)
    check(q, k, v, do * 2.0 ** 6)
    check(q, k, v, torch.zeros_like(do))


@pytest.mark.gpu
def test_nan_stays_in_its_rows(ext_ops):
    q, k, v, _ = inputs(2, 40, 50, 2, 1, 32, torch.bfloat16)
    ref = attention(q, k, v)
    q[0, 7, 1] = float('nan')
    out = attention(q, k, v)
    assert torch.isnan(out[0, 7, 1]).all()
    out[0, 7, 1] = ref[0, 7, 1]
    assert torch.equal(out, ref)


@pytest.mark.gpu
def test_empty(ext_ops):
    for b, lq, lk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q, k, v, do = inputs(b, lq, lk, 2, 1, 32, torch.bfloat16)
        q, k, v = (t.requires_grad_(True) for t in (q, k, v))
        out = attention(q, k, v)
        assert out.shape == q.shape and (out == 0).all()
        grads = torch.autograd.grad(out, (q, k, v), do)
        assert all((g == 0).all() and g.shape == t.shape for g, t in zip(grads, (q, k, v)))


@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
def test_split_keys(ext_ops, dt):
    """Few row tiles over many keys: the key ranges are split and joined."""
    check(*inputs(1, 1, 5000, 1, 4, 128, DTS[dt])[:3])
    q, k, v, do = inputs(1, 40, 4001, 1, 1, 64, DTS[dt])
    check(q, k, v, do)
    check(q, k, v, do, lengths=torch.tensor([300], dtype=torch.int32, device=DEV), causal=True,
          q_offset=torch.tensor([270], dtype=torch.int32, device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
@pytest.mark.parametrize('lq,lk,g', [(3, 1500, 2), (40, 1500, 1), (1500, 40, 2), (900, 130, 3), (1300, 1, 1)])
def test_split_walks_under_masks(ext_ops, dt, lq, lk, g):
    """One side long, the other short: forward and backward split the long walk; masks and lengths on top."""
    q, k, v, do = inputs(2, lq, lk, 1, g, 64, DTS[dt])
    gen = torch.Generator().manual_seed(6)
    full = (torch.rand(2, g, lq, lk, generator=gen) < 0.6).to(DEV)
    lengths = torch.tensor([lk, (lk + 1) // 2], dtype=torch.int32, device=DEV)
    check(q, k, v, do)
    check(q, k, v, do, mask=full)
    check(q, k, v, do, mask=full, lengths=lengths, causal=True, q_offset=lengths - lq)
    check(q, k, v, do, mask=full[:, :1, :1], lengths=lengths)


@pytest.mark.gpu
def test_same_bits_again_and_other_stream(ext_ops):
    q, k, v, do = inputs(2, 333, 333, 2, 2, 64, torch.float16)
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))

    def once():
        out = attention(q, k, v, causal=True)
        return (out, *torch.autograd.grad(out, (q, k, v), do))
    ref = once()
    assert all(torch.equal(a, b) for a, b in zip(ref, once()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = once()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))


@pytest.mark.gpu
@pytest.mark.parametrize('lq', [1, 200])
def test_graph_replays(ext_ops, lq):
    q, k, v, do = inputs(2, lq, 700, 2, 2, 64, torch.float16)
    lengths = torch.tensor([700, 333], dtype=torch.int32, device=DEV)
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))

    def once():
        out = attention(q, k, v, lengths=lengths)
        return (out, *torch.autograd.grad(out, (q, k, v), do))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = once()
    for step in range(4):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(step)).to(q))
            lengths.copy_(torch.tensor([700 - 100 * step, 1 + 50 * step], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        ref = once()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ref, static)), step


@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
def test_gradients_against_differences(ext_ops, dt):
    """Directional differences of the 64-bit forward: with a step of 2^-16 the central difference is
    off by its square (2^-32 relative) and by 2^-53 / 2^-16 of the sum, far under the gradients' own
    tolerance, which is summed against the direction."""
    q, k, v, do = inputs(1, 37, 45, 1, 2, 32, DTS[dt])
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(attention(*leaves, causal=True), leaves, do)
    res = formula(q, k, v, do, causal=True)
    gen = torch.Generator().manual_seed(3)
    wide = [t.detach().cpu().double() for t in (q, k, v)]
    h = 2.0 ** -16
    for n, (g, name) in enumerate(zip(grads, ('dq', 'dk', 'dv'))):
        way = torch.randn(g.shape, generator=gen, dtype=torch.float64)
        f = [(torch_attention(*(t + sign * h * way if i == n else t for i, t in enumerate(wide)), causal=True)
              * do.cpu().double()).sum() for sign in (1, -1)]
        diff = (f[0] - f[1]) / (2 * h)
        assert abs(diff - (g.cpu().double() * way).sum()) <= 1.01 * (res['t_' + name] * way.abs()).sum() + 1e-6


@pytest.mark.gpu
def test_offsets_past_32_bits(ext_ops):
    """One token over a cache of more than 2^31 values (4 GiB in bf16): keys and values in its last rows
    and its first ones decide the output."""
    heads, d = 8, 128
    lk = (1 << 31) // (heads * d) + 777
    cache = torch.zeros(1, lk, heads, d, dtype=torch.bfloat16, device=DEV)
    gen = torch.Generator().manual_seed(4)
    rows = torch.tensor([0, 5, lk - 300, lk - 2, lk - 1])
    vals = torch.randn(len(rows), heads, d, generator=gen).to(torch.bfloat16)
    cache[0, rows.to(DEV)] = vals.to(DEV)
    q = (vals[-1:].float() * 3).to(torch.bfloat16).view(1, 1, heads, d).to(DEV)
    out = attention(q, cache, cache, scale=0.1)
    # the other lk - 5 keys have score 0 and value 0
    s = 0.1 * torch.einsum('hd,jhd->hj', q[0, 0].cpu().double(), vals.double())
    top = s.amax(1, keepdim=True).clamp(min=0)
    p = (s - top).exp()
    total = p.sum(1, keepdim=True) + (lk - len(rows)) * (-top).exp()
    ref = torch.einsum('hj,jhd->hd', p / total, vals.double())
    # P and the output rounded once each, 2^-8 relative; 1e-6 for the fp32 sum of lk terms
    tol = 2.0 ** -7 * torch.einsum('hj,jhd->hd', p / total, vals.double().abs()) + 1e-6
    assert ((out[0, 0].cpu().double() - ref).abs() <= tol).all()
    last = attention(q, cache, cache, scale=0.1, lengths=torch.tensor([lk - 1], dtype=torch.int32, device=DEV))
    assert (last.float().norm() < out.float().norm())


@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('first,last', [(0, 130), (70, 290), (64, 256), (250, 400), (0, 400)])
def test_padding_masks_of_whole_tiles(ext_ops, dt, causal, first, last):
    """Keys first .. last - 1 of the first item hidden (the second item sees all), whatever they hold."""
    q, k, v, do = inputs(2, 150, 400, 2, 1, 64, DTS[dt])
    mask = torch.ones(2, 1, 1, 400, dtype=torch.bool, device=DEV)
    mask[0, ..., first:last] = False
    k[0, first:last], v[0, first:last] = float('nan'), float('inf')
    check(q, k, v, do, mask=mask, causal=causal, lengths=torch.tensor([400, 390], dtype=torch.int32, device=DEV))


@pytest.mark.gpu
def test_query_heads_far_apart(ext_ops):
    """160 heads of one group, 14 MB from each other: the last lies past 2^31 bytes of the first."""
    q, k, v, do = inputs(1, 5, 65, 1, 160, 8, torch.bfloat16)
    far = torch.zeros(160, 7_000_000, dtype=q.dtype, device=DEV)
    far[:, :40] = q[0].transpose(0, 1).reshape(160, 40)
    check(far[:, :40].unflatten(1, (5, 8)).transpose(0, 1)[None], k, v, do)


@pytest.mark.gpu
@pytest.mark.parametrize('lq', [1, 40])
def test_long_head_major_cache_is_not_copied(ext_ops, lq):
    n = 1 << 18
    cache = torch.randn(1, 20, n, 128, device=DEV, dtype=torch.bfloat16).transpose(1, 2)  # 1.3 GB
    q = torch.randn(1, lq, 20, 128, device=DEV, dtype=torch.bfloat16)
    lengths = torch.tensor([n - 3], dtype=torch.int32, device=DEV)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = attention(q, cache, cache, lengths=lengths, impl='hip')
    assert torch.cuda.max_memory_allocated() - before < 1 << 29
    # the same values in the other order of memory give the same bits
    assert torch.equal(out, attention(q, cache.contiguous(), cache.contiguous(), lengths=lengths, impl='hip'))


@pytest.mark.gpu
def test_one_derivative_only(ext_ops):
    q, k, v, do = inputs(1, 40, 40, 1, 1, 32, torch.float32)
    q.requires_grad_(True)
    out = attention(q, k, v)
    with pytest.raises(RuntimeError, match='second derivative'):
        torch.autograd.grad(out, q, do, create_graph=True)


@pytest.mark.gpu
def test_two_streams_at_once(ext_ops):
    """Calls on two streams share nothing: each gives what it gives alone."""
    sets = [inputs(2, n, 900, 2, 2, 64, torch.bfloat16, seed=n) for n in (1, 130)]

    def once(q, k, v, do):
        q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
        out = attention(q, k, v)
        return (out, *torch.autograd.grad(out, (q, k, v), do))
    alone = [once(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(5):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(once(*s))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, alone[i % 2]))


@pytest.mark.gpu
def test_gpu_refusals(ext_ops):
    q, k, v, _ = inputs(1, 3, 6, 1, 1, 8, torch.float32)
    with pytest.raises(TypeError):
        attention(q.double(), k.double(), v.double())
    with pytest.raises(ValueError):
        attention(q, k.cpu(), v.cpu())
    with pytest.raises(ValueError):
        attention(q, k, v, lengths=torch.ones(1, dtype=torch.int32))
    with pytest.raises(RuntimeError):
        ext_ops.attn_fwd(q, k, v[:, :5], 1.0, False, None, None, None, False)
    with pytest.raises(RuntimeError):
        ext_ops.attn_fwd(q, k, v, -1.0, False, None, None, None, False)


@pytest.mark.gpu
def test_most_heads_of_a_call(ext_ops):
    many = torch.zeros(1 << 22, 1, 1, 8, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError):
        attention(many, many, many)
    many[-1] = 2
    q = many[1:].requires_grad_(True)
    out = attention(q, q, q)
    assert out[:-1].count_nonzero() == 0 and (out[-1] == 2).all()
    out.backward(torch.ones_like(out))
    assert (q.grad == 1).all()  # one key: dv = dout, no gradient through the scores
