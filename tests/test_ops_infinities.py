"""Infinite values in the operators of rlfluidcontrol_amd.ops: they reach what the formulas let them reach and nothing else (on
either device)."""
import pytest
import torch

from rlfluidcontrol_amd import ops
from tests.test_ops import conv_case

INF = float("inf")


def conv_weight_grad(c, x):
    w, b = (c[k].clone().requires_grad_() for k in ("weight", "bias"))
    y = ops.causal_conv(x, w, b, False, c["state"], c["lengths"])
    return torch.autograd.grad(y, [w, b], [c["dy"]])


def an_infinite_last_input(device):
    """it enters the filter's gradient through the newest tap only: the positions where the other taps would meet it lie behind the row"""
    for L, W, K, lengths in ((12, 8, 4, [12, 5, 3]), (40, 6, 3, [40, 8, 17]), (40, 9, 2, [33, 16, 1]), (6, 3, 4, [6, 2, 5])):
        c = conv_case(L + W, 3, L, W, K, device=device, lengths=lengths)
        want = conv_weight_grad(c, c["x"])
        for b, n in enumerate(lengths):
            x = c["x"].clone()
            x[b, n - 1, 1] = INF
            got = conv_weight_grad(c, x)
            assert torch.equal(got[0][:, :-1], want[0][:, :-1]) and torch.equal(got[1], want[1]), (L, K, b)
            assert float(got[0][1, -1]) == INF * float(c["dy"][b, n - 1, 1].sign())


def an_infinite_input(device):
    """every tap meets it once, wherever the work is divided"""
    for K in (2, 3, 4):
        c = conv_case(K, 2, 50, 5, K, device=device)
        for p in list(range(20)) + [31, 32, 33, 45]:
            x = c["x"].clone()
            x[1, p, 2] = INF
            dw = conv_weight_grad(c, x)[0]
            assert torch.equal(dw[2].cpu(), torch.stack([INF * c["dy"][1, p + K - 1 - k, 2].sign() for k in range(K)]).cpu()), (K, p)
            assert bool(torch.isfinite(dw[torch.arange(5) != 2]).all())


CHECKS = [an_infinite_last_input, an_infinite_input]


@pytest.mark.parametrize("which", CHECKS)
def test_on_the_cpu(which):
    which("cpu")
