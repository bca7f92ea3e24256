"""Infinite values in the operators of rlfluidcontrol_amd.ops: they reach what the formulas let them reach and nothing else (on
either device)."""
import pytest
import torch

from rlfluidcontrol_amd import ops
from tests import ops_reference as ref
from tests.test_ops import conv_case, scan_case

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


def no_skip(device):
    """without D there is no term D x: what is infinite stays infinite and does not turn to NaN (a state that a kernel fills up to the next
    size has zeros there, so that it may be either)"""
    for N, W in ((16, 20), (64, 6), (4, 37), (8, 70), (3, 8), (5, 70)):
        def is_infinite(t):
            return t == INF if N % 4 == 0 else ~torch.isfinite(t)

        c = scan_case(N, 2, 40, W, N, device=device, D=False, z=False)
        c["B"], c["C"] = c["B"].abs() + 0.1, c["C"].abs() + 0.1
        x = c["x"].clone()
        x[1, 21, 2] = INF
        args = (x, c["dt"], c["A"], c["B"], c["C"])
        y = ops.selective_scan(*args, dt_bias=c["dt_bias"], softplus=True, initial_state=c["state"])
        inf = torch.zeros_like(y, dtype=torch.bool)
        inf[1, 21:, 2] = True
        assert torch.equal(is_infinite(y), inf) and bool(torch.isfinite(y[~inf]).all()), N
        state = c["state"].clone()
        step = ops.selective_scan_step(*(t[:, 21] if t.dim() > 2 else t for t in args), state, dt_bias=c["dt_bias"], softplus=True)
        assert torch.equal(is_infinite(step), inf[:, 21]) and bool(torch.isfinite(step[~inf[:, 21]]).all()), N
        leaf, dy = c["x"].detach().clone().requires_grad_(), c["dy"].clone()
        dy[1, 21, 2] = INF
        y = ops.selective_scan(leaf, *args[1:], dt_bias=c["dt_bias"], softplus=True, initial_state=c["state"])
        dx, = torch.autograd.grad(y, [leaf], [dy])
        inf = torch.zeros_like(inf)
        inf[1, :22, 2] = True
        assert torch.equal(is_infinite(dx), inf) and bool(torch.isfinite(dx[~inf]).all()), N


def no_skip_with_a_gate(device):
    c = scan_case(8, 2, 40, 20, 16, device=device, D=False)
    c["B"], c["C"], c["dy"] = c["B"].abs() + 0.1, c["C"].abs() + 0.1, c["dy"].abs() + 0.1
    c["z"] = c["z"].abs() + 0.1  # the gate's slope is positive
    x, z = c["x"].clone(), c["z"].detach().clone().requires_grad_()
    x[1, 21, 2] = INF
    y = ops.selective_scan(x, c["dt"], c["A"], c["B"], c["C"], z=z, dt_bias=c["dt_bias"], softplus=True)
    dz, = torch.autograd.grad(y, [z], [c["dy"]])
    assert bool((y[1, 21:, 2] == INF).all()) and bool((dz[1, 21:, 2] == INF).all())
    assert int(torch.isfinite(dz).sum()) == dz.numel() - 19


def a_row_that_ends_in_an_infinite_state(device):
    """no position of the row comes after that state, so the rates' gradient does not meet it"""
    for N, W, L, lengths in ((16, 20, 40, [40, 21, 1]), (3, 8, 20, [16, 17, 20]), (64, 6, 300, [299, 33, 32]), (8, 40, 600, [600, 590, 1])):
        c = scan_case(N, 3, L, W, N, device=device, lengths=lengths)
        for dlast in (False, True):
            grads = []
            for last in (1.0, INF):
                x = c["x"].clone()
                for b, n in enumerate(lengths):
                    x[b, n - 1, 1] = last
                A, dt = c["A"].detach().clone().requires_grad_(), c["dt"].detach().clone().requires_grad_()
                y, h = ops.selective_scan(x, dt, A, c["B"], c["C"], c["D"], c["z"], c["dt_bias"], True, c["state"], c["lengths"], return_final_state=True)
                grads.append(torch.autograd.grad([y] + [h] * dlast, [A, dt], [c["dy"]] + [c["dlast"]] * dlast))
            # The same products, summed in another order: either order's additions, one a position, round by u of a sum that the sum of
            # the products' sizes bounds
            size = ref.scan(torch.where(x == INF, 1.0, x), c["dt"], c["A"], c["B"], c["C"], c["D"], c["z"], c["dt_bias"], True, c["state"], c["lengths"], c["dy"],
                            c["dlast"] if dlast else None, magnitude=True)["dA"]
            assert bool(((grads[0][0] - grads[1][0]).abs().cpu() <= 2 * 3 * L * 2.0 ** -24 * size).all()), (N, dlast)
            for b, n in enumerate(lengths):  # and of the step sizes only the last one's does
                assert torch.equal(grads[0][1][b, :n - 1], grads[1][1][b, :n - 1]) and not bool(grads[1][1][b, n:].any())


def an_infinite_adjoint_of_the_final_state(device):
    """it reaches the rates' gradient through the row's own positions: infinite and not NaN, wherever the row ends"""
    for N, W, L, lengths in ((16, 20, 40, [40, 21, 2]), (64, 6, 40, [33, 32, 31]), (8, 40, 600, [600, 590, 3])):
        c = scan_case(N, 3, L, W, N, device=device, lengths=lengths)
        c["state"] = c["state"].abs() + 0.1  # every state in front of a position is positive
        c["B"], c["x"] = c["B"].abs(), c["x"].abs()
        for b in range(3):
            dlast = c["dlast"].clone()
            dlast[b, 1, 2] = INF
            A = c["A"].detach().clone().requires_grad_()
            A.data[1, 2] = -0.001  # (nothing on the way back through a long row is so small that it comes to zero)
            y, h = ops.selective_scan(c["x"], c["dt"], A, c["B"], c["C"], c["D"], c["z"], c["dt_bias"], True, c["state"], c["lengths"], return_final_state=True)
            dA, = torch.autograd.grad([y, h], [A], [c["dy"], dlast])
            want = torch.zeros_like(dA, dtype=torch.bool)
            want[1, 2] = True
            assert torch.equal(dA == INF, want) and bool(torch.isfinite(dA[~want]).all()), (N, b)


def a_rate_without_memory_at_the_smallest_step(device):
    for N, W in ((16, 20), (3, 8), (64, 6)):
        for dtype in (torch.float32, torch.bfloat16):
            x = torch.zeros(2, 3, W, device=device, dtype=dtype)
            B = torch.ones(2, 3, N, device=device, dtype=dtype)
            A = torch.full((W, N), -INF, device=device)
            for delta, left in ((1.01e-36, 0.0), (0.0, 1.0)):  # (1.01: 16 bits round it to above 1e-36)
                dt, h = torch.full_like(x, delta), torch.ones(2, W, N, device=device)
                y, last = ops.selective_scan(x, dt, A, B, B, initial_state=h, return_final_state=True)
                assert bool((last == left).all()) and bool((y == N * left).all()), (N, delta)
                ops.selective_scan_step(x[:, 0], dt[:, 0], A, B[:, 0], B[:, 0], h)
                assert bool((h == left).all()), (N, delta)


CHECKS = [a_rate_without_memory_at_the_smallest_step, an_infinite_adjoint_of_the_final_state, an_infinite_last_input, an_infinite_input, a_row_that_ends_in_an_infinite_state, no_skip, no_skip_with_a_gate]


@pytest.mark.parametrize("which", CHECKS)
def test_on_the_cpu(which):
    which("cpu")
