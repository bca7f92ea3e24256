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
