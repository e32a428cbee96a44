"""Root-mean-square norm (ops/rms_norm.py): plain form, refusals, and the HIP kernels against the
formula in 64 bits.

Tolerances, with u = eps / 2 of the type, w = 2^-24, C channels, for each element:
  h      exact (one fp32 sum of two values, rounded once; a 64-bit sum rounded once can differ only
         where the fp32 sum was itself rounded onto a tie: u |h| covers it)
  y      u |y| + e |y|, e = w (C / 2 + 6): the sum of C squares is off by at most C w relative, its root
         by half of that, and a handful of roundings
  dx     u |dx| + rstd e' (|g| + |h| rstd^2 mean|g h|) + w |dh|, e' = w (2 C + 16)
  dw     (w (rows + 8) + e) sum |dy h rstd|, plus u |dw| in the weight's type
  8 bit  the scale is off by e + w relative; q by the rounding of y * 127 / max: at most 1/2 + 127 (2 e + 4 w)
         from the exact quotient
Results under fp16's least normal value are off by up to 2^-25 more.
"""
import pytest
import torch

from pytorch_raft_amd.ops.rms_norm import rms_norm, rms_norm_int8, torch_rms_norm, torch_rms_norm_int8

DEV = 'cuda'
DTS = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
W = 2.0 ** -24


def inputs(rows, c, dt, dev=DEV, seed=0, wdt=torch.float32):
    g = torch.Generator().manual_seed(seed)
    mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, r, dy, dh = (mk(rows, c).to(dt).to(dev) for _ in range(4))
    return x, r, (1 + 0.3 * mk(c)).to(wdt).to(dev), dy, dh


def half(t):
    return torch.finfo(t).eps / 2


def bound(got, ref, tol, dt, name):
    tol = 1.01 * tol + (2.0 ** -25 if dt == torch.float16 else 0) + 1e-37
    d = (got.detach().cpu().double() - ref).abs()
    assert (d <= tol).all(), '%s: %.3g where %.3g is allowed' % (name, d.flatten()[(d - tol).argmax()], tol.flatten()[(d - tol).argmax()])


def formula(x, r, weight, dy, dh, eps):
    x, weight, dy = (t.detach().cpu().double() for t in (x, weight, dy))
    h = x if r is None else r
    rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    y = h * rstd * weight
    g = dy * weight
    dx = rstd * (g - h * rstd ** 2 * (g * h).mean(-1, keepdim=True))
    size = rstd * (g.abs() + h.abs() * rstd ** 2 * (g * h).abs().mean(-1, keepdim=True))
    if dh is not None:
        dx = dx + dh.cpu().double()
    return y, dx, size, (dy * h * rstd).sum(0), (dy * h * rstd).abs().sum(0)


def check(rows, c, dt, residual, wdt=torch.float32, eps=1e-6):
    x, r, weight, dy, dh = inputs(rows, c, dt, wdt=wdt)
    leaves = [t.requires_grad_(True) for t in ((x, weight, r) if residual else (x, weight))]
    if residual:
        y, h = rms_norm(x, weight, residual=r, eps=eps, impl='hip')
        exact = x.detach().cpu().double() + r.detach().cpu().double()
        bound(h, exact, half(dt) * exact.abs(), dt, 'h')
        assert h.dtype == dt
        grads = torch.autograd.grad((y, h), leaves, (dy, dh))
        assert torch.equal(grads[0], grads[2])
    else:
        y, h, dh = rms_norm(x, weight, eps=eps, impl='hip'), None, None
        grads = torch.autograd.grad(y, leaves, dy)
    ry, rdx, size, rdw, sdw = formula(x, None if h is None else h.detach().cpu().double(), weight, dy, dh, eps)
    e = W * (c / 2 + 6)
    bound(y, ry, (half(dt) + e) * ry.abs(), dt, 'y')
    bound(grads[0], rdx, half(dt) * rdx.abs() + W * (2 * c + 16) * size + (W * dh.cpu().double().abs() if residual else 0), dt, 'dx')
    bound(grads[1], rdw, (W * (rows + 8) + e) * sdw + half(wdt) * rdw.abs(), wdt, 'dw')
    assert y.dtype == dt and grads[0].dtype == dt and grads[1].dtype == wdt


def check8(x, r, weight, eps=1e-6):
    q, scale, h = rms_norm_int8(x, weight, residual=r, eps=eps, impl='hip')
    c = x.shape[-1]
    hh = (x if r is None else h).cpu().double()
    y = hh * (hh.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.cpu().double()
    top = y.abs().amax(-1, keepdim=True)
    e = W * (c / 2 + 6)
    assert q.dtype == torch.int8 and scale.dtype == torch.float32 and scale.shape == x.shape[:-1]
    bound(scale, (top / 127)[..., 0], (e + 2 * W) * (top / 127)[..., 0], torch.float32, 'scale')
    want = torch.where(top == 0, torch.zeros_like(y), y * 127 / top)
    bound(q, want, 0.5 + 127 * (2 * e + 4 * W) + 0 * want, torch.float32, 'q')
    if r is None:
        assert h is None
    else:
        exact = x.cpu().double() + r.cpu().double()
        bound(h, exact, half(x.dtype) * exact.abs(), x.dtype, 'h')


# ------------------------------------------------------------------------------------------- CPU
def test_plain_form_gradients_against_differences():
    x, r, w, _, _ = inputs(3, 7, torch.float64, dev='cpu', wdt=torch.float64)
    for t in (x, r, w):
        t.requires_grad_(True)
    assert torch.autograd.gradcheck(lambda x, r, w: torch_rms_norm(x, w, r), (x, r, w))


def test_plain_8_bit():
    x, r, w, _, _ = inputs(4, 33, torch.bfloat16, dev='cpu')
    x[1] = 0
    q, s, h = torch_rms_norm_int8(x, w)
    assert h is None and (q[1] == 0).all() and s[1] == 0 and q.abs().amax(-1)[[0, 2, 3]].eq(127).all()
    y = torch_rms_norm(x.float(), w)
    assert ((q.float() * s[:, None] - y).abs() <= 0.5001 * s[:, None]).all()


def tiny_rows(dev, impl):
    """Rows whose largest value is under 2^-121, where 127 over it passes fp32's range: a power of two on
    the weight changes no quotient (y stays a normal number where it is compared)."""
    x, _, weight, _, _ = inputs(6, 100, torch.float32, dev=dev)
    x[0, :50] = 0
    weight = weight.sign() * weight.abs().clamp(0.5, 2)
    q, scale, _ = rms_norm_int8(x, weight, impl=impl)
    small, tiny, _ = rms_norm_int8(x, weight * 2.0 ** -123, impl=impl)
    # a value under 2^-126 may lose bits of its own: at most half a step of 2^-149 against a step of
    # max / 127 > 2^-131, so a quotient moves by less than 2^-18 and q by one where it lay that near a tie
    d = (small.int() - q.int()).abs()
    assert d.max() <= 1 and (d != 0).sum() <= 2
    assert (small[0, :50] == 0).all() and small.abs().amax(-1).eq(127).all()
    assert ((tiny.double() * 2.0 ** 123 - scale.double()).abs() <= 2.0 ** -17 * scale.double()).all()


def test_plain_8_bit_of_tiny_rows():
    tiny_rows('cpu', 'torch')


def test_refusals():
    x, r, w, _, _ = inputs(4, 16, torch.float32, dev='cpu')
    for args, kw in (((x, w[:8]), {}), ((x, w), {'residual': r[:3]}), ((x, w), {'residual': r.half()}),
                     ((x, w), {'eps': -1.}), ((x, w), {'eps': float('nan')}), ((x[:, :0], w[:0]), {}),
                     ((torch.zeros(1, 16385), torch.zeros(16385)), {})):
        for f in (rms_norm, rms_norm_int8):
            with pytest.raises(ValueError):
                f(*args, **kw)
    with pytest.raises(TypeError):
        rms_norm(x, w.half())
    with pytest.raises(RuntimeError):
        rms_norm_int8(x.requires_grad_(True), w)


# ------------------------------------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
@pytest.mark.parametrize('c', [1, 3, 8, 100, 127, 128, 129, 256, 271, 512, 1000, 1024, 2048, 2114, 4096, 5000, 8192, 8200, 16384])
@pytest.mark.parametrize('residual', [False, True])
def test_channels(ext_ops, dt, c, residual):
    check(19, c, DTS[dt], residual)
    x, r, w, _, _ = inputs(19, c, DTS[dt])
    check8(x, r if residual else None, w)


@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
@pytest.mark.parametrize('rows', [1, 2, 63, 65, 4000])
@pytest.mark.parametrize('c', [40, 300, 1111])
def test_rows(ext_ops, dt, rows, c):
    check(rows, c, DTS[dt], True, wdt=DTS[dt])
    x, r, w, _, _ = inputs(rows, c, DTS[dt], wdt=DTS[dt])
    check8(x, r, w)


@pytest.mark.gpu
def test_many_rows(ext_ops):
    check(40001, 72, torch.float32, True)
    check(5000, 2050, torch.bfloat16, False)


@pytest.mark.gpu
@pytest.mark.parametrize('dt', list(DTS))
def test_layouts_and_unused_outputs(ext_ops, dt):
    x, r, w, dy, dh = inputs(24, 96, DTS[dt])
    ref, href = rms_norm(x, w, residual=r)
    view = lambda t: t.view(2, 3, 4, 96)  # noqa: E731
    y, h = rms_norm(view(x), w, residual=view(r).transpose(0, 2).contiguous().transpose(0, 2))
    assert torch.equal(y.reshape(24, 96), ref) and torch.equal(h.reshape(24, 96), href) and y.shape == (2, 3, 4, 96)
    wide = torch.zeros(24, 200, dtype=x.dtype, device=DEV)
    wide[:, 7:103] = x
    assert torch.equal(rms_norm(wide[:, 7:103], w, residual=r)[0], ref)
    assert rms_norm(x[:0], w).shape == (0, 96)
    flat = torch.zeros(24 * 96 + 1, dtype=x.dtype, device=DEV)      # off 16 bytes
    flat[1:] = x.flatten()
    assert torch.equal(rms_norm(flat[1:].view(24, 96), w, residual=r)[0], ref)
    for t in (x, r, w):
        t.requires_grad_(True)
    y, h = rms_norm(x, w, residual=r)
    full = torch.autograd.grad((y, h), (x, w), (dy, torch.zeros_like(dh)), retain_graph=True)
    only = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(full, only))
    assert torch.equal(torch.autograd.grad(h, x, dh, retain_graph=True)[0], dh)
    with pytest.raises(RuntimeError, match='second derivative'):
        torch.autograd.grad(y, x, dy, create_graph=True)
    one = rms_norm(x[0], w)                        # a single vector
    assert one.shape == (96,) and torch.equal(one, rms_norm(x, w)[0])
    q, s, none = rms_norm_int8(x[0].detach(), w.detach())
    assert q.shape == (96,) and s.shape == () and none is None


@pytest.mark.gpu
def test_special_rows(ext_ops):
    x, r, w, _, _ = inputs(6, 300, torch.float32)
    x[1] = 0
    x[2] *= 1e-18
    x[3, 5] = float('nan')
    x[4, 5] = float('inf')
    y = rms_norm(x, w)
    assert (y[1] == 0).all() and torch.isnan(y[3]).all() and torch.isnan(y[4, 5])
    q, s, _ = rms_norm_int8(x, w)
    assert s[1] == 0 and (q[1] == 0).all() and torch.isnan(s[3]) and torch.isnan(s[4])
    check8(x[[0, 1, 2, 5]], None, w)


@pytest.mark.gpu
def test_8_bit_of_tiny_rows(ext_ops):
    tiny_rows(DEV, 'hip')


@pytest.mark.gpu
def test_same_bits_and_graph_replays(ext_ops):
    x, r, w, dy, dh = inputs(500, 600, torch.bfloat16)
    for t in (x, r, w):
        t.requires_grad_(True)

    def once():
        y, h = rms_norm(x, w, residual=r)
        q = rms_norm_int8(x.detach(), w.detach(), residual=r.detach())
        return (y, h, *q, *torch.autograd.grad((y, h), (x, r, w), (dy, dh)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = once()
    for step in range(3):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(step)).to(x))
        graph.replay()
        torch.cuda.synchronize()
        ref = once()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(ref, static)), step


@pytest.mark.gpu
def test_gpu_refusals(ext_ops):
    x, r, w, _, _ = inputs(4, 16, torch.float32)
    with pytest.raises(TypeError):
        rms_norm(x.double(), w)
    with pytest.raises(ValueError):
        rms_norm(x, w.cpu())
    with pytest.raises(RuntimeError):
        ext_ops.rms_fwd(x.t(), w, None, 1e-6, False)
    with pytest.raises(RuntimeError):
        ext_ops.rms_fwd(x, w, r[:3], 1e-6, False)
