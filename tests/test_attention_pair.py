"""What attention's rounding takes away (the third output of attn_fwd) and the backward's row sums that it
serves: delta_i = sum_d dout_id o_id from the output as a pair of 16-bit values.

Rows where one key takes all: query i is 2 k_t + noise / 4 for a key t among the first 16, so s_it is about
16 and the others' scores N(0, 2): the rest of the row holds some 1e-4.  Key t lies in the first tile of its
row, so its probability relative to the running reference is 1, exact in 16 bits.  With u, w, e as in
test_attention.py, r_j = [j != t] and all sums over j:
  out + lo   u sum r_j P|v| + e sum P|v - o| + w (Lk + 16) sum P|v| + u^2 |o|  (lo <= u |o|, rounded once);
             fp16: + sum min(P, 2^-25)|v| for probabilities under its range, + 2^-25 for lo itself
A lo that is lost or belongs elsewhere leaves errors of up to u |o|.
  dq         dP - delta is some 1e-3 where |dP| and |delta| are about 8, so a delta from the rounded output
             alone is off by about u / 2 * 8 there, and dq by as much times scale |k_t|; with the pair what is
             left are roundings of dS and dq themselves, u of values of 1e-3, and fp32 sums: the errors'
             norms are about a thousand apart in fp16 as in bf16, and more than 8 at any rate.
"""
import math

import pytest
import torch

from test_attention import DEV, DTS

# one pass; one pass with keys split and joined; few rows; few rows split and joined
SIZES = {'pass': (150, 70), 'pass_join': (150, 300), 'few': (20, 70), 'few_join': (20, 300)}


def rows(size, dt, d=64):
    lq, lk = SIZES[size]
    g = torch.Generator().manual_seed(3)
    mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    k, v, do = mk(lk, d), mk(lk, d), mk(lq, d)
    top = torch.randint(0, 16, (lq,), generator=g)
    q = 2 * k[top] + 0.25 * mk(lq, d)
    q, k, v, do = (t.to(dt) for t in (q, k, v, do))
    qq, kk, vv = (t.double() for t in (q, k, v))
    scale = d ** -0.5
    p = torch.softmax(scale * qq @ kk.t(), -1)
    assert (p[torch.arange(lq), top] > 0.99).all()
    return (q, k, v, do), top, p, p @ vv, scale


def forward(ext_ops, q, k, v, scale):
    put = lambda t: t[None, :, None].to(DEV)  # noqa: E731
    return ext_ops.attn_fwd(put(q), put(k), put(v), scale, False, None, None, None, True)


@pytest.mark.gpu
@pytest.mark.parametrize('dt', ['bf16', 'fp16'])
@pytest.mark.parametrize('size', list(SIZES))
def test_pair_of_outputs(ext_ops, dt, size):
    (q, k, v, _), top, p, o, scale = rows(size, DTS[dt])
    out, _, lo = forward(ext_ops, q, k, v, scale)
    out, lo = (t[0, :, 0].cpu().double() for t in (out, lo))
    u, w = torch.finfo(DTS[dt]).eps / 2, 2.0 ** -24
    (lq, lk), d = SIZES[size], q.shape[1]
    va = v.double().abs()
    es = w * (d + 8) * scale * (q.double().abs() @ k.double().abs().t())
    e = 2 * es.max(-1, keepdim=True).values + w * (lk + 16)
    rest = p.clone()
    rest[torch.arange(lq), top] = 0
    spread = (p[:, :, None] * (v.double()[None] - o[:, None]).abs()).sum(1)
    tol = u * rest @ va + e * spread + w * (lk + 16) * (p @ va) + u * u * o.abs()
    if dt == 'fp16':
        tol = tol + p.clamp(max=2.0 ** -25) @ va + 2.0 ** -25
    assert ((out + lo - o).abs() <= 1.01 * tol).all()
    # the bound is far under the rounding that lo holds: it could not hold without lo
    assert ((out - o).abs() > 1.01 * tol).double().mean() > 0.5


@pytest.mark.gpu
@pytest.mark.parametrize('dt', ['bf16', 'fp16'])
@pytest.mark.parametrize('size', list(SIZES))
def test_row_sums_from_the_pair(ext_ops, dt, size):
    (q, k, v, do), _, p, o, scale = rows(size, DTS[dt])
    dp = do.double() @ v.double().t()
    dq = scale * (p * (dp - (do.double() * o).sum(-1, keepdim=True))) @ k.double()
    out, lse, lo = forward(ext_ops, q, k, v, scale)
    put = lambda t: t[None, :, None].to(DEV)  # noqa: E731
    err = []
    for low in (lo, torch.empty(0, dtype=lo.dtype, device=DEV)):
        got = ext_ops.attn_bwd(put(do), put(q), put(k), put(v), out, lse, low, scale, False, None, None, None)[0]
        err.append((got[0, :, 0].cpu().double() - dq).norm().item())
    assert math.isfinite(err[1]) and 8 * err[0] < err[1], err


@pytest.mark.gpu
def test_fp32_needs_no_pair(ext_ops):
    (q, k, v, _), *_, scale = rows('pass', torch.float32)
    assert forward(ext_ops, q, k, v, scale)[2].numel() == 0
