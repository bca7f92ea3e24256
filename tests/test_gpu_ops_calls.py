"""The kernels of rlfluidcontrol_amd.ops called in other ways than in a plain program."""
import pytest
import torch

from rlfluidcontrol_amd import ops
from tests.test_ops import conv_case
from tests.test_ops_calls import tracing_is_refused

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_tracing_is_refused():
    tracing_is_refused(DEV)


def test_a_compiled_caller_runs_them_as_they_are():
    c = conv_case(3, 2, 5, 8, 3, device=DEV)
    f = torch.compile(lambda x: ops.causal_conv(x + 1, c["weight"], c["bias"], True) * 2, backend="eager")
    with torch.no_grad():
        assert torch.equal(f(c["x"]), ops.causal_conv(c["x"] + 1, c["weight"], c["bias"], True) * 2)
