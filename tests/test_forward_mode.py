"""Forward-mode derivatives of the token operators: none in the kernels, so a tangent raises (dropped in
silence it would count as zero); the plain forms of the differentiable ones carry it."""
import pytest
import torch
from torch.autograd import forward_ad

from pytorch_raft_amd.ops.attention import attention
from pytorch_raft_amd.ops.int8 import int8_linear
from pytorch_raft_amd.ops.rms_norm import rms_norm, rms_norm_int8


def calls(dev):
    """(function, its floating arguments, whether it has a gradient)"""
    g = torch.Generator().manual_seed(0)
    mk = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    x, w = (torch.randint(-9, 9, s, generator=g).to(torch.int8).to(dev) for s in ((5, 32), (7, 32)))
    return [(attention, (mk(1, 6, 2, 32), mk(1, 9, 2, 32), mk(1, 9, 2, 32)), True),
            (attention, (mk(1, 6, 2, 13), mk(1, 9, 2, 13), mk(1, 9, 2, 13)), True),
            (rms_norm, (mk(5, 16), mk(16)), True),
            (lambda x, w, r: rms_norm(x, w, residual=r), (mk(5, 16), mk(16), mk(5, 16)), True),
            (lambda x, w, r: rms_norm_int8(x, w, residual=r), (mk(5, 16), mk(16), mk(5, 16)), False),
            (lambda xs, ws, b: int8_linear(x, xs, w, ws, bias=b), (mk(5), mk(7), mk(7)), False)]


def refused(f, args):
    for i in range(len(args)):
        for grad in (True, False):
            with forward_ad.dual_level(), torch.set_grad_enabled(grad):
                dual = [forward_ad.make_dual(t, torch.ones_like(t)) if i == j else t for j, t in enumerate(args)]
                with pytest.raises(RuntimeError, match='forward-mode'):
                    f(*dual)
    with forward_ad.dual_level(), torch.no_grad():
        f(*args)                        # no tangent anywhere: nothing to refuse


def test_plain_forms():
    for f, args, differentiable in calls('cpu'):
        if not differentiable:
            refused(f, args)
            continue
        with forward_ad.dual_level():
            out = f(*(forward_ad.make_dual(t, torch.ones_like(t)) for t in args))
            out = out[0] if isinstance(out, tuple) else out
            assert forward_ad.unpack_dual(out).tangent is not None


@pytest.mark.gpu
def test_kernels_refuse(ext_ops):
    for f, args, differentiable in calls('cuda'):
        refused(f, args)
        if differentiable:              # a tangent on the output's gradient
            leaves = [t.requires_grad_(True) for t in args]
            out = f(*leaves)
            for y in out if isinstance(out, tuple) else (out,):
                with forward_ad.dual_level(), pytest.raises(RuntimeError, match='forward-mode'):
                    torch.autograd.grad(y, leaves[0], forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)),
                                        retain_graph=True)
