"""quantize_weight (ops/int8.py): rows at the edges of fp32's range, and the layout that the product reads."""
import torch

from pytorch_raft_amd.ops.int8 import quantize_weight


def test_tiny_rows():
    """127 over a row's largest value passes fp32's range under 2^-121.  The values are powers of two, down
    to 2^-149, so 127 / top and every quotient are exact in fp32: 127, 63.5 (a tie, to the even 64), 0
    and -31.75, whatever the power of two on the row."""
    row = torch.tensor([1, 0.5, 0, -0.25])
    want = torch.tensor([127, 64, 0, -32], dtype=torch.int8)
    for e in (0, -100, -119, -121, -123, -126, -140, -147, 100, 127):
        q, s = quantize_weight(torch.stack([row * 2.0 ** e, torch.zeros(4), row]))
        assert torch.equal(q[0], want), e
        assert torch.equal(q[2], want) and not q[1].any() and s[1] == 0
        # the scale is rounded to fp32 once, under 2^-126 to a multiple of 2^-149
        assert abs(s[0].double() - 2.0 ** e / 127) <= max(2.0 ** -24 * 2.0 ** e / 127, 2.0 ** -150)


def test_layout():
    """The product reads rows of k: whatever the layout of the weight, no call copies the result again."""
    w = torch.randn(32, 48, generator=torch.Generator().manual_seed(0))
    q, s = quantize_weight(w)
    wide = torch.zeros(32, 96)
    wide[:, ::2] = w
    for other in (w.t().contiguous().t(), wide[:, ::2], w.t().contiguous().double().t()):
        q2, s2 = quantize_weight(other)
        assert q2.is_contiguous() and s2.is_contiguous()
        assert torch.equal(q2, q) and torch.equal(s2, s)
