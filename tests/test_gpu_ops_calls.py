"""The kernels of rlfluidcontrol_amd.ops called in other ways than in a plain program."""
import pytest
import torch

from rlfluidcontrol_amd import ops
from tests.test_ops import calls_of_the_binding, conv_case, scan_case
from tests import test_ops_infinities as infinities
from tests.test_ops_calls import IN_PLACE, negated, negated_views_are_refused, tracing_is_refused

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_tracing_is_refused():
    tracing_is_refused(DEV)


def test_a_compiled_caller_runs_them_as_they_are():
    c = conv_case(3, 2, 5, 8, 3, device=DEV)
    f = torch.compile(lambda x: ops.causal_conv(x + 1, c["weight"], c["bias"], True) * 2, backend="eager")
    with torch.no_grad():
        assert torch.equal(f(c["x"]), ops.causal_conv(c["x"] + 1, c["weight"], c["bias"], True) * 2)


def test_negated_views_are_refused():
    negated_views_are_refused(DEV)


def test_negated_parameters():
    for name, names, values, call in calls_of_the_binding(DEV):
        for n in set(names) - set(IN_PLACE[name]):
            with torch.no_grad():
                fresh = lambda: {k: v.clone() if v is not None else None for k, v in values.items()}  # noqa: E731  (a step moves its state)
                assert torch.equal(call(dict(fresh(), **{n: negated(values[n])})), call(fresh())), (name, n)


def test_negated_adjoints():
    c, s = conv_case(4, 2, 9, 8, 3, device=DEV), scan_case(4, 2, 9, 8, 4, device=DEV)
    for case, call, names in ((c, lambda a: ops.causal_conv(a["x"], a["weight"], initial_state=a["state"], return_final_state=True), ("x", "weight", "state")),
                              (s, lambda a: ops.selective_scan(a["x"], a["dt"], a["A"], a["B"], a["C"], initial_state=a["state"], return_final_state=True), ("x", "dt", "A", "B", "C", "state"))):
        leaves = {n: case[n].detach().clone().requires_grad_() for n in names}
        outs = call(leaves)
        want = torch.autograd.grad(outs, list(leaves.values()), [case["dy"], case["dlast"]], retain_graph=True)
        got = torch.autograd.grad(outs, list(leaves.values()), [negated(case["dy"]), negated(case["dlast"])])
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("which", infinities.CHECKS)
def test_infinities(which):
    which(DEV)
