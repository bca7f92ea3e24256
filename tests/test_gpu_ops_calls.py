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


def all_grads(case, call, names):
    leaves = {n: case[n].detach().clone().requires_grad_() for n in names}
    return torch.autograd.grad(call(leaves), list(leaves.values()), [case["dy"], case["dlast"]])


def both_operators():
    c, s = conv_case(4, 2, 40, 24, 3, device=DEV, lengths=[40, 17]), scan_case(4, 2, 40, 24, 16, device=DEV, lengths=[40, 17])
    return ((c, lambda a: ops.causal_conv(a["x"], a["weight"], a["bias"], True, a["state"], c["lengths"], return_final_state=True), ("x", "weight", "bias", "state")),
            (s, lambda a: ops.selective_scan(a["x"], a["dt"], a["A"], a["B"], a["C"], a["D"], a["z"], a["dt_bias"], True, a["state"], s["lengths"], return_final_state=True),
             ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state")))


def test_saved_tensors_that_travel():
    """recomputed activations, and saved tensors that wait in host memory"""
    from torch.utils.checkpoint import checkpoint
    for case, call, names in both_operators():
        want = all_grads(case, call, names)
        again = all_grads(case, lambda a: checkpoint(lambda: call(a), use_reentrant=False), names)
        assert all(torch.equal(p, q) for p, q in zip(want, again))
        with torch.autograd.graph.save_on_cpu():
            leaves = {n: case[n].detach().clone().requires_grad_() for n in names}
            outs = call(leaves)
        assert all(torch.equal(p, q) for p, q in zip(want, torch.autograd.grad(outs, list(leaves.values()), [case["dy"], case["dlast"]])))


@pytest.mark.parametrize("change", [lambda t: t.bfloat16() if t.dtype == torch.float32 else t, lambda t: t.cpu(), lambda t: t[..., :-1].contiguous(), lambda t: t[:1]])
def test_saved_tensors_that_come_back_as_others_are_refused(change):
    for case, call, names in both_operators():
        for which in range(12):
            seen = []

            def pack(t):
                seen.append(t)
                return t, len(seen) - 1

            def unpack(p):
                return change(p[0]) if p[1] == which else p[0]

            with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
                leaves = {n: case[n].detach().clone().requires_grad_() for n in names}
                outs = call(leaves)
            if which >= len(seen):
                break
            t = seen[which]
            if change(t).shape == t.shape and change(t).dtype == t.dtype and change(t).device == t.device:
                continue
            with pytest.raises((ValueError, RuntimeError)):
                torch.autograd.grad(outs, list(leaves.values()), [case["dy"], case["dlast"]])
