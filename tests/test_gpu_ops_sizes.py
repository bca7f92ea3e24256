"""The kernels of rlfluidcontrol_amd.ops at sizes whose blocks do not fit one launch (fewer than 2^32 threads along x): the rows of
every slice, and the sums over all of them."""
import pytest
import torch

from rlfluidcontrol_amd import ops
from tests import ops_reference as ref
from tests.test_ops import check_conv, check_scan, conv_case, scan_case

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


@pytest.fixture(autouse=True)
def memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def spread(t, rows, at):
    """zeros but for t's rows at `at`"""
    big = torch.zeros((rows,) + tuple(t.shape[1:]), dtype=t.dtype, device=DEV)
    big[at] = t
    return big


def same_rows(big, small, at, name):
    assert torch.equal(big[at], small), name
    assert int(torch.count_nonzero(big)) == int(torch.count_nonzero(small)), name


def test_scan_of_many_rows():
    """2^24 blocks and more in both directions, 2^32 partial sums of db and dc"""
    rows = (1 << 24) + 3
    at = torch.tensor(list(range(5)) + list(range(rows - 5, rows)), device=DEV)
    c = scan_case(1, 10, 8, 1, 1, 1, F32, DEV, state=False)
    want = check_scan(c, True, dlast=False)
    size = ref.scan(c["x"], c["dt"], c["A"], c["B"], c["C"], c["D"], c["z"], c["dt_bias"], True, None, None, c["dy"], magnitude=True)
    names = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")
    leaves = {n: (spread(c[n], rows, at) if n in ("x", "dt", "B", "C", "z") else c[n].detach().clone()).requires_grad_() for n in names}
    y, last = ops.selective_scan(*leaves.values(), softplus=True, return_final_state=True)
    same_rows(y.detach(), want["y"].detach(), at, "y")
    same_rows(last.detach(), want["last"].detach(), at, "last")
    grads = dict(zip(names, torch.autograd.grad(y, list(leaves.values()), [spread(c["dy"], rows, at)])))
    for n in ("x", "dt", "B", "C", "z"):
        same_rows(grads[n], want["d" + n], at, n)
    for n, r in (("A", "dA"), ("D", "dD"), ("dt_bias", "dbias")):  # the same 80 terms and zeros, in another order
        assert bool(((grads[n] - want[r]).abs().cpu() <= 2 * 80 * U * size[r]).all()) and bool(grads[n].any()), n


@pytest.mark.parametrize("N", [1, 4])
def test_scan_step_of_many_rows(N):
    rows = (1 << 26) + 5
    at = torch.tensor(list(range(7)) + list(range(rows - 7, rows)), device=DEV)
    c = scan_case(N, 14, 1, 1, N, 1, F32, DEV)
    one = {n: c[n][:, 0].contiguous() for n in ("x", "dt", "B", "C", "z")}
    state = c["state"].clone()
    want = ops.selective_scan_step(one["x"], one["dt"], c["A"], one["B"], one["C"], state, c["D"], one["z"], c["dt_bias"], True)
    big = {n: spread(t, rows, at) for n, t in one.items()}
    h = spread(c["state"], rows, at)
    y = ops.selective_scan_step(big["x"], big["dt"], c["A"], big["B"], big["C"], h, c["D"], big["z"], c["dt_bias"], True)
    same_rows(y, want, at, "y")
    same_rows(h, state, at, "state")


def test_conv_of_many_rows():
    rows = (1 << 24) + 3
    at = torch.tensor(list(range(5)) + list(range(rows - 5, rows)), device=DEV)
    c = conv_case(1, 10, 2, 1, 3, F32, DEV, bias=False)
    want = check_conv(c, True)
    size = ref.conv(c["x"], c["weight"], None, True, c["state"], None, c["dy"], c["dlast"], magnitude=True)["dweight"]
    leaves = [spread(c["x"], rows, at).requires_grad_(), c["weight"].clone().requires_grad_(), spread(c["state"], rows, at).requires_grad_()]
    y, last = ops.causal_conv(leaves[0], leaves[1], None, True, leaves[2], return_final_state=True)
    dx, dw, ds = torch.autograd.grad([y, last], leaves, [spread(c["dy"], rows, at), spread(c["dlast"], rows, at)])
    for got, n in ((y, "y"), (last, "last"), (dx, "dx"), (ds, "dstate")):
        same_rows(got.detach(), want[n].detach(), at, n)
    assert bool(((dw - want["dweight"]).abs().cpu() <= 2 * 20 * U * size).all())  # the same 20 terms and zeros, in another order


def test_conv_of_many_channels():
    """2^22 blocks and more for the sums of the filter's gradient"""
    W = 1 << 26
    x, dy = (torch.randn(1, 1, W, device=DEV) for _ in range(2))
    w = torch.randn(W, 4, device=DEV, requires_grad=True)
    y = ops.causal_conv(x, w)
    assert torch.equal(y[0, 0], (x[0, 0] * w[:, 3]).detach())  # one product each, and zeros
    dw, = torch.autograd.grad(y, [w], [dy])
    assert torch.equal(dw[:, 3], (x * dy)[0, 0]) and not bool(dw[:, :3].any())


def test_conv_step_of_many_rows():
    W = 5
    rows = (1 << 32) // W + 100
    x = torch.empty(rows, W, device=DEV, dtype=BF16).normal_()
    state = torch.empty(rows, 1, W, device=DEV, dtype=BF16).normal_()
    w = torch.randn(W, 2, device=DEV)
    half = rows // 2
    states = [state[:half].clone(), state[half:].clone()]  # two calls of one launch each
    want = [ops.causal_conv_step(x[:half], states[0], w), ops.causal_conv_step(x[half:], states[1], w)]
    y = ops.causal_conv_step(x, state, w)
    assert torch.equal(y[:half], want[0]) and torch.equal(y[half:], want[1]) and torch.equal(state[:, 0], x)
    assert torch.equal(states[0][:, 0], x[:half])
