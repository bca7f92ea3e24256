"""How the operators of rlfluidcontrol_amd.ops may be called: what the torch binding refuses, before it asks for a GPU where it can."""
import pytest
import torch

from rlfluidcontrol_amd import build, ops
from tests.test_ops import calls_of_the_binding, conv_case


@pytest.fixture(scope="module", autouse=True)
def built():
    build.build_ops()


def tracing_is_refused(device):
    from torch.fx.experimental.proxy_tensor import make_fx
    for name, names, values, call in calls_of_the_binding(device):
        n = names[0]
        with torch.no_grad():
            with pytest.raises(RuntimeError, match="traced"):
                torch.jit.trace(lambda t: call(dict(values, **{n: t})), (values[n],))
            for kw in (dict(), dict(pre_dispatch=True), dict(tracing_mode="fake")):
                with pytest.raises(RuntimeError, match="traced"):
                    make_fx(lambda t: call(dict(values, **{n: t})), **kw)(values[n])


def test_tracing_is_refused():
    tracing_is_refused("cpu")


def test_the_plain_path_is_traced():
    c = conv_case(3, 2, 5, 4, 3)
    f = torch.jit.trace(lambda x: ops.causal_conv(x, c["weight"], c["bias"], True), (c["x"],))
    assert torch.equal(f(c["dy"]), ops.causal_conv(c["dy"], c["weight"], c["bias"], True))


def negated(t):
    """the values of t, as a view of memory that holds their negatives"""
    v = torch._neg_view(-t)
    assert v.is_neg() and torch.equal(v, t)
    return v


# what a kernel reads or updates where it lies (the other operands are copied where they have to be)
IN_PLACE = {"causal_conv": ("x",), "causal_conv_step": ("x", "state"), "selective_scan": ("x", "dt", "B", "C", "z"),
            "selective_scan_step": ("x", "dt", "B", "C", "z", "state"), "clip": ("g", "h", "out"), "norm": ("g",)}


def negated_views_are_refused(device):
    for name, names, values, call in calls_of_the_binding(device):
        for n in set(names) & set(IN_PLACE[name]):
            with torch.no_grad(), pytest.raises(ValueError, match="resolve_neg"):
                call(dict(values, **{n: negated(values[n])}))


def test_negated_views_are_refused():
    negated_views_are_refused("cpu")


def test_launches_that_could_not_be_made_are_refused():
    """made-up pointers: the checks come before any device, and before the first launch of a call"""
    import ctypes as C
    from tests import ops_abi as abi
    from tests.test_ops import fake_conv, fake_scan
    lib = abi.load()

    def many(f, p):
        assert f(C.byref(p), None) == -1 and b"too many blocks" in lib.afc_ops_last_error()

    rows = (1 << 30) - 1
    many(lib.afc_scan, fake_scan(batch=rows, length=1, groups=4))  # a block for each row and group
    many(lib.afc_scan_step, fake_scan(batch=rows, length=1, state=3, width=1 << 12, groups=1, initial_state=4096, final_state=4096))
    many(lib.afc_conv, fake_conv(batch=rows, length=1, width=1 << 12))
    many(lib.afc_conv_grad, fake_conv(batch=rows, length=1, width=1 << 12))
    many(lib.afc_scan_grad, fake_scan(batch=1 << 20, length=1 << 20, width=1, groups=1, state=64))  # 2^40 x 128 partial sums
    p = abi.ClipArgs()
    p.count, p.inp, p.numel, p.in_dtype = 1 << 23, 4096, 4096, 4096
    assert lib.afc_clip_workspace(C.byref(p), C.byref(C.c_uint64())) == -1 and b"count" in lib.afc_ops_last_error()
