"""Norms and 8-bit products of more than 2^31 elements: the last rows come out as they do by themselves."""
import pytest
import torch

from pytorch_raft_amd.ops.int8 import int8_linear
from pytorch_raft_amd.ops.rms_norm import rms_norm, rms_norm_int8

DEV = 'cuda'


@pytest.mark.gpu
@pytest.mark.parametrize('c', [120, 8200])
def test_norms(ext_ops, c):
    rows = (1 << 31) // c + 300
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.empty(rows, c, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    r, dy = x.flip(0), x.roll(1, 0)
    w = 1 + 0.1 * torch.randn(c, generator=g, device=DEV)
    for t in (x, r, w):
        t.requires_grad_(True)
    y, h = rms_norm(x, w, residual=r)
    dx, dr, dw = torch.autograd.grad((y, h), (x, r, w), (dy, dy))
    q, scale, h8 = rms_norm_int8(x.detach(), w.detach(), residual=r.detach())
    for part in (slice(0, 5), slice(rows - 5, rows)):
        xs, rs = (t.detach()[part].clone().requires_grad_(True) for t in (x, r))
        ys, hs = rms_norm(xs, w, residual=rs)
        dxs, _, _ = torch.autograd.grad((ys, hs), (xs, rs, w), (dy[part], dy[part]))
        qs, ss, _ = rms_norm_int8(xs.detach(), w.detach(), residual=rs.detach())
        assert torch.equal(y[part], ys) and torch.equal(h[part], hs) and torch.equal(h8[part], hs)
        assert torch.equal(dx[part], dxs) and torch.equal(dr[part], dxs)
        assert torch.equal(q[part], qs) and torch.equal(scale[part], ss)
    # dw: sums of `rows` products in fp32 (each off by 2^-24 of the sum of their sizes per addition of a
    # part: at most rows / 1024 in a block and 1024 blocks), against 64-bit sums of a column
    col = c - 1
    rstd = (h.detach().double().square().mean(-1) + 1e-6).rsqrt() if c < 1000 else None
    if rstd is not None:
        terms = dy[:, col].double() * h.detach()[:, col].double() * rstd
        steps = rows / 1024 + 1024 + c
        assert abs(dw[col].double() - terms.sum()) <= steps * 2.0 ** -24 * terms.abs().sum()


@pytest.mark.gpu
@pytest.mark.parametrize('m,n,k', [(66000, 32640, 48), (70000, 50, 30704), (40, 70000, 30704), (70000, 50, 30703)])
def test_products(ext_ops, m, n, k):
    """Outputs, x or w past 2^31 elements."""
    g = torch.Generator(device=DEV).manual_seed(0)
    x, w = (torch.randint(-128, 128, s, generator=g, device=DEV, dtype=torch.int8) for s in ((m, k), (n, k)))
    xs, ws = torch.rand(m, generator=g, device=DEV), torch.rand(n, generator=g, device=DEV)
    out = int8_linear(x, xs, w, ws, out_dtype=torch.float32)
    for rows in (slice(0, 3), slice(m - 3, m)):
        for cols in (slice(0, 3), slice(n - 3, n)):
            ref = (x[rows].cpu().double() @ w[cols].cpu().double().t()) * xs[rows].cpu().double()[:, None] * ws[cols].cpu().double()
            # the integer sum, two scales: three fp32 roundings
            assert ((out[rows, cols].cpu().double() - ref).abs() <= 3.01 * 2.0 ** -24 * ref.abs()).all()
