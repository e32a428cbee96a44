"""Token attention (ops/attention.py) at the edges of what its documentation allows: queries that see no
key and hold anything, single keys, scales at the ends of fp32's range, forward-mode derivatives, and
the accuracy that the backward's row sums owe to the unrounded output.
"""
import pytest
import torch

from pytorch_raft_amd.ops.attention import attention
from test_attention import DEV, DTS, close, formula, inputs


def unseen_cases(dev):
    """(mask, lengths, causal, q_offset, which queries (B, H, Lq) see a key) over 2 items, 2 x 2 heads,
    150 queries and 170 keys: rows hidden by a mask for each row, causal rows before the first key (with
    and without lengths), and causal rows whose keys up to their own position are all padding."""
    b, h, lq, lk = 2, 4, 150, 170
    gen = torch.Generator().manual_seed(8)
    full = torch.rand(b, h, lq, lk, generator=gen) < 0.6
    full[0, :, 17] = False
    full[1, 2, 64:131] = False          # more than a whole tile of rows, one head
    full[1, :, 149] = False
    pos = torch.arange(lq)
    before = torch.tensor([-70, -1], dtype=torch.int32)
    lengths = torch.tensor([170, 3], dtype=torch.int32)
    left = torch.ones(b, 1, 1, lk, dtype=torch.bool)
    left[0, ..., :75] = False
    left[1, ..., :1] = False
    at = torch.tensor([0, 0], dtype=torch.int32)
    all_heads = lambda t: t[:, None].expand(b, h, lq)  # noqa: E731
    return [
        (full.to(dev), None, False, None, full.any(-1)),
        (None, None, True, before.to(dev), all_heads(pos + before[:, None] >= 0)),
        (None, lengths.to(dev), True, before.to(dev), all_heads(pos + before[:, None] >= 0)),
        (left.to(dev), None, True, at.to(dev), all_heads(pos >= torch.tensor([75, 1])[:, None])),
        (full.to(dev), lengths.to(dev), True, at.to(dev),
         (full & (torch.arange(lk) <= pos[:, None]) & (torch.arange(lk) < lengths[:, None, None, None])).any(-1)),
    ]


def check_unseen(dt, dev, case):
    mask, lengths, causal, q_offset, seen = unseen_cases(dev)[case]
    q, k, v, do = inputs(2, 150, 170, 2, 2, 40, dt, dev=dev)
    kw = dict(mask=mask, lengths=lengths, causal=causal, q_offset=q_offset)
    hidden = ~seen.transpose(1, 2).to(dev)                      # (B, Lq, H)
    assert hidden.any() and not hidden.all()
    q0, do0 = (t.masked_fill(hidden[..., None], 0) for t in (q, do))
    res = formula(q0, k, v, do0, **kw)
    for bad_q, bad_do in ((float('nan'), float('inf')), (float('-inf'), float('nan')), (float('inf'), torch.finfo(dt).max)):
        q1 = q.masked_fill(hidden[..., None], bad_q).requires_grad_(True)
        do1 = do.masked_fill(hidden[..., None], bad_do)
        k1, v1 = (t.detach().requires_grad_(True) for t in (k, v))
        out = attention(q1, k1, v1, **kw)
        assert (out[hidden] == 0).all()
        close(out, res, 'out')
        grads = torch.autograd.grad(out, (q1, k1, v1), do1)
        assert (grads[0][hidden] == 0).all()
        for n, t in zip(('dq', 'dk', 'dv'), grads):
            close(t, res, n)


@pytest.mark.parametrize('case', range(5))
def test_plain_form_queries_without_keys(case):
    check_unseen(torch.float32, 'cpu', case)


@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
@pytest.mark.parametrize('case', range(5))
def test_queries_without_keys(ext_ops, dt, case):
    check_unseen(DTS[dt], DEV, case)


@pytest.mark.gpu
@pytest.mark.parametrize('bad', ['dout', 'v'])
def test_other_items_keep_their_bits(ext_ops, bad):
    """fp16: an infinity or NaN in one item makes that item's gradients useless, not coarser those of the
    others, whose dout lies far under fp16's range without the backward's common scale: they keep the bits
    that they have beside a finite item (the row in question is zero there, so it decides no scale)."""
    q, k, v, do = inputs(2, 90, 1400, 1, 2, 64, torch.float16)
    do = do * 2.0 ** -12
    row = (do if bad == 'dout' else v)[0, 5, 0]
    row.zero_()

    def gradients():
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(attention(*leaves), leaves, do)
    clean = gradients()
    for n, t in zip(('dq', 'dk', 'dv'), clean):
        close(t[1:], formula(q[1:], k[1:], v[1:], do[1:]), n)
    for value in (float('inf'), float('nan')):
        row[3] = value
        grads = gradients()
        assert not all(torch.isfinite(g[0]).all() for g in grads)
        assert all(torch.equal(a[1], b[1]) for a, b in zip(grads, clean))


@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
@pytest.mark.parametrize('lq', [1, 9, 140])
def test_single_keys_hold_anything(ext_ops, dt, lq):
    """One key: a query's output is that key's value, whatever it is, also infinite (Lk = 1, and an item
    of one key among longer ones).  The key's probability is p = 1 + d, d from the fp32 rounding of the
    exponent (under 2^-18 for scores of this size), and the sum l is p itself.  16-bit types: p rounds to
    1, and v / l lies within 2^-18 of v, relative, under half a step of both types: it rounds to v.  fp32:
    v p (1 / l) has the roundings of the product, the reciprocal (one step, 2 w) and the last product:
    4 w, w = 2^-24."""
    q, k, v, _ = inputs(2, lq, 1, 2, 2, 64, DTS[dt])
    v[0, 0, 0, :3] = torch.tensor([float('inf'), float('-inf'), float('nan')])
    out = attention(q, k, v)
    ref = v.repeat_interleave(2, 2).expand_as(q)
    finite = torch.isfinite(ref)
    assert torch.equal(out[~finite].nan_to_num(7.), ref[~finite].nan_to_num(7.))
    tol = 4 * 2.0 ** -24 if dt == 'fp32' else 0
    assert ((out[finite] - ref[finite]).abs() <= tol * ref[finite].abs()).all()
    long_k, long_v = (torch.full((2, 70, 2, 64), float('nan'), dtype=v.dtype, device=DEV) for _ in range(2))
    long_k[:, :1], long_v[:, :1] = k, v
    one = torch.ones(2, dtype=torch.int32, device=DEV)
    assert torch.equal(attention(q, long_k, long_v, lengths=one).nan_to_num(7.), out.nan_to_num(7.))


def scale_range(dev, impl):
    """Scores are formed in fp32, in units of log 2: a scale outside that range made every hidden place NaN
    (0 * -inf) or every score (infinity * 0)."""
    q, k, v, _ = inputs(1, 3, 40, 1, 1, 32, torch.float32, dev=dev)
    mask = torch.ones(3, 40, dtype=torch.bool, device=dev)
    mask[:, 17:] = False
    for scale in (1e-60, 2.0 ** -151, 3e38, 1e39, 1e300, 5e-324):
        with pytest.raises(ValueError, match='scale'):
            attention(q, k, v, scale=scale, mask=mask, impl=impl)
    # the smallest scales: all scores are 0 to fp32, the seen keys' mean
    for scale in (2.0 ** -149, 1e-40, 2.0 ** -126):
        out = attention(q, k, v, scale=scale, mask=mask, impl=impl)
        mean = v[:, :17].double().mean(1, keepdim=True)
        # sums of 17 terms and a division in fp32
        assert ((out - mean).abs() <= 20 * 2.0 ** -24 * v[:, :17].double().abs().mean(1, keepdim=True)).all()
    # large ones, where q and k are small enough
    out = attention(q * 2.0 ** -50, k * 2.0 ** -50, v, scale=2.0 ** 100, impl=impl)
    res = formula(q, k, v, scale=1.)
    close(out, res, 'out')


def test_plain_form_scales():
    scale_range('cpu', 'torch')


@pytest.mark.gpu
def test_scales(ext_ops):
    scale_range(DEV, 'hip')


@pytest.mark.gpu
def test_first_row_of_a_far_key(ext_ops):
    """Keys far before the queries of a large group: (position - key) * heads passes 2^31.  One query at the
    last position sees all keys that its mask leaves (some heads see none), so causal changes nothing, to
    the bit."""
    heads, lk = 2560, (1 << 20) + 77
    g = torch.Generator(device=DEV).manual_seed(0)
    mk = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    q, k, v, do = mk(1, 1, heads, 8), mk(1, lk, 1, 8), mk(1, lk, 1, 8), mk(1, 1, heads, 8)
    mask = (torch.arange(heads, device=DEV) % 7 != 3)[None, :, None, None]
    grads = []
    for causal in (True, False):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        grads.append(torch.autograd.grad(attention(*leaves, causal=causal, mask=mask), leaves, do))
    for n, a, b in zip(('dq', 'dk', 'dv'), *grads):
        assert torch.equal(a, b), '%s: %d values differ' % (n, (a != b).sum())
    assert (grads[0][2] != 0).any(-1).all()


@pytest.mark.gpu
@pytest.mark.parametrize('lq', [3, 90])
def test_ends_of_lengths_and_offsets(ext_ops, lq):
    """Lengths under 0 and past Lk, offsets at the ends of int32: clamped to what they mean."""
    q, k, v, do = inputs(4, lq, 150, 2, 2, 32, torch.bfloat16)
    big = 2 ** 31 - 1
    lengths = torch.tensor([-big - 1, big, 151, 70], dtype=torch.int32, device=DEV)
    first = torch.tensor([big, -big - 1, big, -1], dtype=torch.int32, device=DEV)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    out = attention(*leaves, causal=True, lengths=lengths, q_offset=first)
    grads = torch.autograd.grad(out, leaves, do)
    res = formula(q, k, v, do, causal=True, lengths=lengths.clamp(0, 150), q_offset=first.clamp(-lq, 150))
    close(out, res, 'out')
    for n, t in zip(('dq', 'dk', 'dv'), grads):
        close(t, res, n)


@pytest.mark.gpu
def test_gradients_of_long_caches(ext_ops):
    """Keys, values and their gradients of more than 2^31 values: all are 0 but five rows at both ends, so a
    row's sum is known: total = sum over the five of exp(s) + the number of others.  Bounds: P and dS rounded
    once to bf16 and the result once more, 2^-8 each, scores of fp32 sums: 2^-6 of the terms' sizes."""
    heads, d, lq = 8, 128, 33
    lk = (1 << 31) // (heads * d) + 777
    g = torch.Generator().manual_seed(4)
    mk = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)  # noqa: E731
    rows = torch.tensor([0, 5, lk - 300, lk - 2, lk - 1])
    other = torch.tensor([1, 1000, lk // 2, lk - 3])
    kv, q, do = (mk(5, heads, d), mk(5, heads, d)), 0.2 * mk(lq, heads, d), mk(lq, heads, d)
    big = [torch.zeros(1, lk, heads, d, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    for t, x in zip(big, kv):
        t[0, rows.to(DEV)] = x.to(DEV)
        t.requires_grad_(True)
    qg = q[None].to(DEV).requires_grad_(True)
    dq, dk, dv = torch.autograd.grad(attention(qg, *big, scale=0.5), (qg, *big), do[None].to(DEV))
    q, do, k, v = (t.double().transpose(0, 1) for t in (q, do, *kv))       # (heads, rows, d)
    s = 0.5 * q @ k.transpose(1, 2)
    top = s.amax(-1, keepdim=True).clamp(min=0)
    total = (s - top).exp().sum(-1, keepdim=True) + (lk - 5) * (-top).exp()
    p, p0 = (s - top).exp() / total, (-top).exp() / total                 # of the five, of any other key
    o = p @ v
    dp, delta = do @ v.transpose(1, 2), (do * o).sum(-1, keepdim=True)
    ds, ds0, size, size0 = p * (dp - delta), -p0 * delta, p * (dp.abs() + delta.abs()), p0 * delta.abs()
    # delta's own bound: the output off by 2^-8 sum P|v|
    more = 2.0 ** -8 * (do.abs() * (p @ v.abs())).sum(-1, keepdim=True)
    size, size0 = size + 64 * p * more, size0 + 64 * p0 * more

    def bound(got, ref, terms):
        assert ((got.cpu().double() - ref).abs() <= 2.0 ** -6 * terms + 1e-30).all()
    take = lambda t, at: t[0, at.to(DEV)].transpose(0, 1)  # noqa: E731
    bound(take(dv, rows), p.transpose(1, 2) @ do, p.transpose(1, 2) @ do.abs())
    bound(take(dv, other), (p0.transpose(1, 2) @ do).expand(-1, 4, -1), (p0.transpose(1, 2) @ do.abs()).expand(-1, 4, -1))
    bound(take(dk, rows), 0.5 * ds.transpose(1, 2) @ q, 0.5 * size.transpose(1, 2) @ q.abs())
    bound(take(dk, other), 0.5 * (ds0.transpose(1, 2) @ q).expand(-1, 4, -1), 0.5 * (size0.transpose(1, 2) @ q.abs()).expand(-1, 4, -1))
    bound(dq[0].transpose(0, 1), 0.5 * ds @ k, 0.5 * size @ k.abs())


@pytest.mark.gpu
def test_gradients_of_many_queries(ext_ops):
    """Queries, outputs and their gradients of more than 2^31 values: the last rows by the formula, and the
    keys' gradients against those of the same rows in two calls, whose sums differ in order only."""
    heads, d, lk = 8, 128, 40
    lq = (1 << 31) // (heads * d) + 99
    g = torch.Generator(device=DEV).manual_seed(4)
    mk = lambda *s: torch.empty(*s, dtype=torch.bfloat16, device=DEV).normal_(generator=g)  # noqa: E731
    q, do, k, v = mk(1, lq, heads, d), mk(1, lq, heads, d), mk(1, lk, heads, d), mk(1, lk, heads, d)

    def grads(part):
        leaves = [t.detach().requires_grad_(True) for t in (q[:, part], k, v)]
        out = attention(*leaves)
        return (out.detach(), *torch.autograd.grad(out, leaves, do[:, part]))
    whole, first, last = (grads(s) for s in (slice(None), slice(0, lq // 2), slice(lq // 2, lq)))
    res = formula(q[:, -50:], k, v, do[:, -50:])
    close(whole[0][:, -50:], res, 'out')
    close(whole[1][:, -50:], res, 'dq')
    for i in (2, 3):
        a, b, c = (t[i].double() for t in (whole, first, last))
        # three results rounded once each, 2^-8 of their values, whose halves are no larger in norm than
        # about the whole; the order of fp32 sums of 2^21 terms of random sign makes some 2^-24 2^10 of it.
        # (A row read or written at a wrong place changes a gradient by about its own size.)
        assert (a - b - c).norm() <= 2.0 ** -6 * a.norm()
