"""Token operators given tensors that torch keeps lazily: views with a pending negation (the imaginary part
of a conjugate is one), and zeros without memory, which are refused."""
import pytest
import torch

from pytorch_raft_amd.ops.attention import attention
from pytorch_raft_amd.ops.int8 import int8_linear
from pytorch_raft_amd.ops.rms_norm import rms_norm, rms_norm_int8

DEV = 'cuda'


def calls():
    g = torch.Generator().manual_seed(0)
    mk = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    i8 = lambda *s: torch.randint(-9, 9, s, generator=g).to(torch.int8).to(DEV)  # noqa: E731
    ints = torch.tensor([9, 4], dtype=torch.int32, device=DEV)
    yield lambda q, k, v, n, o: attention(q, k, v, causal=True, lengths=n, q_offset=o), \
        (mk(2, 6, 2, 32), mk(2, 9, 2, 32), mk(2, 9, 2, 32), ints, ints - 3), (0, 1, 2)
    yield attention, (mk(2, 6, 2, 13), mk(2, 9, 2, 13), mk(2, 9, 2, 13)), (0, 1, 2)
    yield rms_norm, (mk(5, 16), mk(16)), (0, 1)
    yield lambda x, w, r: rms_norm(x, w, residual=r), (mk(5, 16), mk(16), mk(5, 16)), (0, 1, 2)
    yield lambda x, w, r: rms_norm_int8(x, w, residual=r), (mk(5, 16), mk(16), mk(5, 16)), ()
    yield lambda x, xs, w, ws, b: int8_linear(x, xs, w, ws, bias=b), (i8(5, 32), mk(5), i8(7, 32), mk(7), mk(7)), ()


def outputs(f, args):
    out = f(*args)
    return [t for t in out if t is not None] if isinstance(out, tuple) else [out]


@pytest.mark.gpu
def test_negated_views(ext_ops):
    for f, args, _ in calls():
        ref = outputs(f, args)
        for i, t in enumerate(args):
            lazy = torch._neg_view(-t)
            assert lazy.is_neg()
            got = outputs(f, [lazy if i == j else a for j, a in enumerate(args)])
            assert all(torch.equal(a, b) for a, b in zip(got, ref)), i


@pytest.mark.gpu
def test_negated_views_in_training(ext_ops):
    for f, args, leaves in calls():
        if not leaves:
            continue

        def grads(wrap):
            a = [t.detach().clone().requires_grad_(True) if i in leaves else t for i, t in enumerate(args)]
            out = outputs(f, [wrap(t) if i in leaves else t for i, t in enumerate(a)])
            return torch.autograd.grad(out, [a[i] for i in leaves], [wrap(torch.full_like(t, 0.5)) for t in out])
        for a, b in zip(grads(lambda t: torch._neg_view(-t)), grads(lambda t: t)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_zeros_without_memory_are_refused(ext_ops):
    for f, args, _ in calls():
        for i, t in enumerate(args):
            zeros = torch._efficientzerotensor(t.shape, dtype=t.dtype, device=DEV)
            with pytest.raises(RuntimeError, match='memory'):
                f(*(zeros if i == j else a for j, a in enumerate(args)))
    q = torch.ones(1, 4, 1, 32, device=DEV, requires_grad=True)
    out = attention(q, q, q)
    with pytest.raises(RuntimeError, match='memory'):
        torch.autograd.grad(out, q, torch._efficientzerotensor(out.shape, device=DEV))
