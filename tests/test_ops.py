"""rlfluidcontrol_amd.ops on the CPU: the formulas against differences, the plain path against the formulas, refusals, and the
C ABI's own checks (which refuse before any device is touched)."""
import ctypes as C
import os
import re
import shutil

import pytest
import torch

from rlfluidcontrol_amd import build, codeobj, ops
from tests import ops_abi as abi
from tests import ops_reference as ref
from tests.conftest import ROOT


def conv_case(seed, B, L, W, K, dtype=torch.float32, device="cpu", lengths=None, state=True, bias=True):
    g = torch.Generator().manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g)

    return dict(x=r(B, L, W).to(dtype).to(device), weight=(0.5 * r(W, K)).to(device), bias=(0.3 * r(W)).to(device) if bias else None,
                state=r(B, K - 1, W).to(dtype).to(device) if state else None, dy=r(B, L, W).to(dtype).to(device), dlast=r(B, K - 1, W).to(dtype).to(device),
                lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=device))


def scan_case(seed, B, L, W, N, G=1, dtype=torch.float32, device="cpu", lengths=None, D=True, z=True, bias=True, state=True):
    g = torch.Generator().manual_seed(seed)

    def r(*s):
        return torch.randn(*s, generator=g)

    def to(t, on=True):
        return t.to(dtype).to(device) if on else None

    return dict(x=to(r(B, L, W)), dt=to(0.5 * r(B, L, W) - 2), A=(-torch.rand(W, N, generator=g) * 4 - 0.1).to(device), B=to(r(B, L, G, N)), C=to(r(B, L, G, N)),
                D=(1 + 0.3 * r(W)).to(device) if D else None, z=to(r(B, L, W), z), dt_bias=(0.3 * r(W) - 1).to(device) if bias else None,
                state=r(B, W, N).to(device) if state else None, dy=to(r(B, L, W)), dlast=r(B, W, N).to(device),
                lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=device))


def check_conv(c, silu, dy=True, dlast=True):
    """forward and backward of ops.causal_conv against the reference"""
    leaves = {k: c[k].detach().clone().requires_grad_() for k in ("x", "weight", "bias", "state") if c[k] is not None}
    y, last = ops.causal_conv(leaves["x"], leaves["weight"], leaves.get("bias"), silu, leaves.get("state"), c["lengths"], return_final_state=True)
    outs = [(y, c["dy"])] * dy + [(last, c["dlast"])] * dlast
    got = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs], allow_unused=True)
    args = (c["x"], c["weight"], c["bias"], silu, c["state"], c["lengths"], c["dy"] if dy else torch.zeros_like(c["dy"]), c["dlast"] if dlast else None)
    r, m = ref.conv(*args), ref.conv(*args, magnitude=True)
    k = ref.conv_bounds(m, c["x"].dtype, c["x"], c["weight"].shape[1], silu)
    res = dict(y=y, last=last, **{"d" + n: t for n, t in zip(leaves, got)})
    for name, t in res.items():
        t = torch.zeros_like(leaves[name[1:]]) if t is None else t
        assert ref.off(t, r[name], m[name], k[name], t.dtype) <= 1, name
    return res


def check_scan(c, softplus, dy=True, dlast=True):
    names = [n for n in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state") if c[n] is not None]
    leaves = {n: c[n].detach().requires_grad_() for n in names}
    y, last = ops.selective_scan(leaves["x"], leaves["dt"], leaves["A"], leaves["B"], leaves["C"], leaves.get("D"), leaves.get("z"), leaves.get("dt_bias"),
                                 softplus, leaves.get("state"), c["lengths"], return_final_state=True)
    outs = [(y, c["dy"])] * dy + [(last, c["dlast"])] * dlast
    got = torch.autograd.grad([o for o, _ in outs], list(leaves.values()), [g for _, g in outs], allow_unused=True)
    args = (c["x"], c["dt"], c["A"], c["B"], c["C"], c["D"], c["z"], c["dt_bias"], softplus, c["state"], c["lengths"],
            c["dy"] if dy else torch.zeros_like(c["dy"]), c["dlast"] if dlast else None)
    r, m = ref.scan(*args), ref.scan(*args, magnitude=True)
    k = ref.scan_bounds(r, c["x"], c["A"].shape[1], c["B"].shape[2])
    res = dict(y=y, last=last, **{"d" + ("bias" if n == "dt_bias" else "dt" if n == "dt" else n): t for n, t in zip(leaves, got)})
    for name, t in res.items():
        t = torch.zeros_like(leaves[name[1:]]) if t is None else t
        assert ref.off(t, r[name], m[name], k[name], t.dtype) <= 1, name
    # without gradients the same values come back (another kernel may have made them)
    with torch.no_grad():
        y2, last2 = ops.selective_scan(c["x"], c["dt"], c["A"], c["B"], c["C"], c["D"], c["z"], c["dt_bias"], softplus, c["state"], c["lengths"],
                                       return_final_state=True)
    assert ref.off(y2, r["y"], m["y"], k["y"], y2.dtype) <= 1 and ref.off(last2, r["last"], m["last"], k["last"], last2.dtype) <= 1
    return res


# ---- the reference's gradients against differences ----

def test_scan_gradients_against_differences():
    c = scan_case(1, 2, 5, 4, 3, G=2, lengths=[5, 3])
    c = {k: v.double() if v is not None and v.is_floating_point() else v for k, v in c.items()}

    def loss(**kw):
        a = dict(c, **kw)
        r = ref.scan(a["x"], a["dt"], a["A"], a["B"], a["C"], a["D"], a["z"], a["dt_bias"], True, a["state"], a["lengths"])
        return float((r["y"] * c["dy"]).sum() + (r["last"] * c["dlast"]).sum())

    r = ref.scan(c["x"], c["dt"], c["A"], c["B"], c["C"], c["D"], c["z"], c["dt_bias"], True, c["state"], c["lengths"], c["dy"], c["dlast"])
    g = torch.Generator().manual_seed(2)
    for name, grad in (("x", "dx"), ("dt", "ddt"), ("A", "dA"), ("B", "dB"), ("C", "dC"), ("D", "dD"), ("z", "dz"), ("dt_bias", "dbias"), ("state", "dstate")):
        way = torch.randn(c[name].shape, generator=g, dtype=torch.float64)
        eps = 1e-5  # central differences: off by eps^2 f'''/6 (some 1e-9) and 2^-53 |loss| / eps (some 1e-10)
        diff = (loss(**{name: c[name] + eps * way}) - loss(**{name: c[name] - eps * way})) / (2 * eps)
        assert abs(diff - float((r[grad] * way).sum())) < 1e-6 * (1 + abs(diff)), name


def test_conv_gradients_against_differences():
    c = conv_case(1, 3, 5, 4, 3, lengths=[5, 0, 2])
    c = {k: v.double() if v is not None and v.is_floating_point() else v for k, v in c.items()}

    def loss(**kw):
        a = dict(c, **kw)
        r = ref.conv(a["x"], a["weight"], a["bias"], True, a["state"], a["lengths"])
        return float((r["y"] * c["dy"]).sum() + (r["last"] * c["dlast"]).sum())

    r = ref.conv(c["x"], c["weight"], c["bias"], True, c["state"], c["lengths"], c["dy"], c["dlast"])
    g = torch.Generator().manual_seed(2)
    for name in ("x", "weight", "bias", "state"):
        way = torch.randn(c[name].shape, generator=g, dtype=torch.float64)
        eps = 1e-5
        diff = (loss(**{name: c[name] + eps * way}) - loss(**{name: c[name] - eps * way})) / (2 * eps)
        assert abs(diff - float((r["d" + name] * way).sum())) < 1e-6 * (1 + abs(diff)), name


# ---- the plain path ----

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lengths", [None, [7, 0, 3]])
def test_plain_path_follows_the_formulas(dtype, lengths):
    check_conv(conv_case(3, 3, 7, 6, 4, dtype=dtype, lengths=lengths), True)
    check_scan(scan_case(4, 3, 7, 6, 5, G=2, dtype=dtype, lengths=lengths), True)


def test_plain_steps_continue_a_sequence():
    with torch.no_grad():
        c = conv_case(5, 2, 6, 4, 4)
        y, last = ops.causal_conv(c["x"], c["weight"], c["bias"], True, c["state"], return_final_state=True)
        s = c["state"].clone()
        steps = torch.stack([ops.causal_conv_step(c["x"][:, l], s, c["weight"], c["bias"], True) for l in range(6)], 1)
        assert torch.equal(s, last) and torch.allclose(steps, y, atol=1e-6)
        c = scan_case(6, 2, 6, 4, 5, G=2)
        y, last = ops.selective_scan(c["x"], c["dt"], c["A"], c["B"], c["C"], c["D"], c["z"], c["dt_bias"], True, c["state"], return_final_state=True)
        s = c["state"].clone()
        steps = torch.stack([ops.selective_scan_step(c["x"][:, l], c["dt"][:, l], c["A"], c["B"][:, l], c["C"][:, l], s, c["D"], c["z"][:, l], c["dt_bias"], True)
                             for l in range(6)], 1)
        assert torch.allclose(s, last, atol=1e-6) and torch.allclose(steps, y, atol=1e-6)


def test_plain_clip():
    grads = [torch.tensor([3.0, 0.0]), None, torch.tensor([[4.0]]).bfloat16()]
    assert float(ops.grad_norm(grads)) == 5.0
    assert float(ops.clip_grad_norm(grads, 10.0)) == 5.0 and grads[0].tolist() == [3.0, 0.0]
    out = [torch.empty(2), None, torch.empty(1, 1)]
    assert float(ops.clip_grad_norm(grads, 2.5, out=out)) == 5.0
    assert torch.allclose(out[0], torch.tensor([1.5, 0.0]), atol=1e-6) and abs(float(out[2]) - 2.0) < 1e-6
    assert float(ops.clip_grad_norm([], 1.0)) == 0.0


# ---- refusals ----

def refused(f, *a, error=ValueError, **kw):
    with pytest.raises(error):
        f(*a, **kw)


def refusals_of_conv(dev):
    x, w = torch.randn(2, 5, 4, device=dev), torch.randn(4, 3, device=dev)
    refused(ops.causal_conv, x[0], w)
    refused(ops.causal_conv, x.double(), w)
    refused(ops.causal_conv, x, torch.randn(4, 5, device=dev))
    refused(ops.causal_conv, x, torch.randn(4, 1, device=dev))
    refused(ops.causal_conv, x, torch.randn(5, 3, device=dev))
    refused(ops.causal_conv, x, w.bfloat16())
    refused(ops.causal_conv, x, w, torch.randn(3, device=dev))
    refused(ops.causal_conv, x, w, initial_state=torch.randn(2, 3, 4, device=dev))
    refused(ops.causal_conv, x, w, lengths=torch.tensor([1, 2], device=dev))
    refused(ops.causal_conv, x.transpose(1, 2).contiguous().transpose(1, 2), w)
    refused(ops.causal_conv, x.tolist(), w, error=TypeError)
    refused(ops.causal_conv, x, None, error=TypeError)
    refused(ops.causal_conv_step, x[:, 0], torch.randn(2, 2, 4, device=dev).transpose(0, 1).contiguous().transpose(0, 1), w)
    refused(ops.causal_conv_step, x[:, 0], torch.randn(2, 3, 4, device=dev), w)
    refused(ops.causal_conv_step, x[:, 0], torch.randn(2, 2, 4, device=dev), w.clone().requires_grad_())


def refusals_of_scan(dev):
    c = scan_case(1, 2, 5, 6, 4, G=2, device=dev)
    ok = dict(x=c["x"], dt=c["dt"], A=c["A"], B=c["B"], C=c["C"])
    ops.selective_scan(**ok)
    for bad in (dict(x=c["x"][0]), dict(dt=c["dt"][:, :4]), dict(dt=c["dt"].bfloat16()), dict(A=c["A"].double()), dict(A=torch.randn(6, 65, device=dev)), dict(A=torch.randn(6, 0, device=dev)),
                dict(B=torch.randn(2, 5, 4, 4, device=dev), C=torch.randn(2, 5, 4, 4, device=dev)), dict(C=c["C"][:, :, :1]), dict(B=torch.randn(2, 5, device=dev)), dict(z=c["z"][:, :1]),
                dict(D=torch.randn(5, device=dev)), dict(dt_bias=torch.randn(6, 1, device=dev)), dict(initial_state=torch.randn(2, 6, 5, device=dev)), dict(initial_state=torch.randn(2, 6, 4, device=dev).half()),
                dict(lengths=torch.ones(3, dtype=torch.int32, device=dev)), dict(lengths=torch.ones(2, device=dev))):
        refused(ops.selective_scan, **{**ok, **bad})
    refused(ops.selective_scan, **{**ok, "A": 1.0}, error=TypeError)
    step = dict(x=c["x"][:, 0], dt=c["dt"][:, 0], A=c["A"], B=c["B"][:, 0], C=c["C"][:, 0], state=c["state"])
    ops.selective_scan_step(**step)
    refused(ops.selective_scan_step, **{**step, "state": c["state"].transpose(1, 2).contiguous().transpose(1, 2)})
    refused(ops.selective_scan_step, **{**step, "state": c["state"][:1]})
    refused(ops.selective_scan_step, **{**step, "x": step["x"].clone().requires_grad_()})


def refusals_of_clip(dev):
    g = torch.randn(4, 4, device=dev)
    refused(ops.clip_grad_norm, [g], -1.0)
    refused(ops.clip_grad_norm, [g], float("nan"))
    refused(ops.clip_grad_norm, g, 1.0, error=TypeError)
    refused(ops.clip_grad_norm, [g.double()], 1.0)
    refused(ops.clip_grad_norm, [g[:, ::2]], 1.0)
    refused(ops.clip_grad_norm, [g[:1].expand(4, 4)], 1.0)
    refused(ops.clip_grad_norm, [g], 1.0, out=[])
    refused(ops.clip_grad_norm, [g], 1.0, out=[g.t().contiguous().t()])
    refused(ops.clip_grad_norm, [g, None], 1.0, out=[None, g])
    refused(ops.clip_grad_norm, [g, "x"], 1.0, error=TypeError)
    refused(ops.clip_grad_norm, [g.clone().requires_grad_()], 1.0)
    assert ops._without_gaps(g.t()) and ops._without_gaps(torch.randn(2, 3, 4, 5, device=dev).permute(3, 0, 2, 1)) and not ops._without_gaps(g[:, :3])


@pytest.mark.parametrize("which", [refusals_of_conv, refusals_of_scan, refusals_of_clip])
def test_refusals(which):
    which("cpu")


# ---- the C ABI ----

@pytest.fixture(scope="module")
def lib():
    build.build_ops()
    return abi.load()


def test_header_symbols_exported(lib):
    txt = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "afc_ops.h")).read(), flags=re.S)
    decl = sorted(set(re.findall(r"\b(afc_[a-z0-9_]+)\s*\(", txt)))
    assert sorted(abi.SYMBOLS) == decl
    for name in decl:
        assert hasattr(lib, name), name


def test_struct_layouts_follow_the_header(tmp_path):
    import subprocess
    src = tmp_path / "sizes.c"
    fields = [("afc_seq", abi.Seq), ("afc_conv_args", abi.ConvArgs), ("afc_scan_args", abi.ScanArgs), ("afc_clip_args", abi.ClipArgs)]
    lines = []
    for name, t in fields:
        lines.append('printf("%%zu\\n", sizeof(%s));' % name)
        for f, _ in t._fields_:
            lines.append('printf("%%zu\\n", offsetof(%s, %s));' % (name, "in" if f == "inp" else f))
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "afc_ops.h"\nint main(void) {%s return 0;}' % "\n".join(lines))
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "sizes")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "sizes")], text=True).split()]
    want = []
    for _, t in fields:
        want.append(C.sizeof(t))
        want += [getattr(t, f).offset for f, _ in t._fields_]
    assert got == want


def fake_conv(**kw):
    p = abi.ConvArgs()
    p.taps, p.batch, p.length, p.width, p.weight = 3, 2, 5, 4, 4096
    p.x = p.y = p.dy = p.dx = abi.Seq(4096, 20, 4, 0)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def fake_scan(**kw):
    p = abi.ScanArgs()
    p.state, p.batch, p.length, p.width, p.groups, p.a, p.checkpoints = 4, 2, 5, 4, 2, 4096, 4096
    for k in ("x", "dt", "b", "c", "y", "dy", "dx", "ddt", "db", "dc"):
        setattr(p, k, abi.Seq(4096, 20, 4, 4))
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_c_abi_refuses_bad_arguments(lib):
    """pointers here are made up: every one of these calls is turned down on the host"""
    def bad(f, p):
        assert f(p if p is None else C.byref(p), None) == -1
        assert lib.afc_ops_last_error()

    big = 1 << 62
    for f in (lib.afc_conv, lib.afc_conv_grad, lib.afc_conv_step, lib.afc_scan, lib.afc_scan_grad, lib.afc_scan_step, lib.afc_clip):
        bad(f, None)
    for kw in (dict(dtype=3), dict(dtype=-1), dict(taps=1), dict(taps=5), dict(batch=-1), dict(length=-1), dict(width=0), dict(weight=0), dict(length=1 << 31),
               dict(x=abi.Seq(0, 20, 4, 0)), dict(x=abi.Seq(4096, -20, 4, 0)), dict(y=abi.Seq(4096, big, 4, 0)), dict(y=abi.Seq(0, 20, 4, 0))):
        bad(lib.afc_conv, fake_conv(**kw))
    for kw in (dict(dx=abi.Seq()), dict(dy=abi.Seq())):
        bad(lib.afc_conv_grad, fake_conv(**kw))
    for kw in (dict(length=2), dict(length=1), dict(length=1, initial_state=4096, final_state=8192), dict(length=1, initial_state=4096, final_state=4096, lengths=4096)):
        bad(lib.afc_conv_step, fake_conv(**kw))
    for kw in (dict(dtype=3), dict(state=0), dict(state=65), dict(groups=0), dict(groups=3), dict(width=0), dict(a=0), dict(batch=-1), dict(length=-1),
               dict(x=abi.Seq()), dict(dt=abi.Seq()), dict(b=abi.Seq()), dict(c=abi.Seq(4096, 1, 1, big)), dict(z=abi.Seq(4096, 1, -1, 0)), dict(y=abi.Seq())):
        bad(lib.afc_scan, fake_scan(**kw))
    for kw in (dict(dx=abi.Seq()), dict(ddt=abi.Seq()), dict(db=abi.Seq()), dict(dc=abi.Seq()), dict(checkpoints=0), dict(dz=abi.Seq(4096, 20, 4, 0)),
               dict()):  # the last: no workspace
        bad(lib.afc_scan_grad, fake_scan(**kw))
    bad(lib.afc_scan_step, fake_scan(length=1))

    def clip(ins, numel, outs=None, in_dtype=None, out_dtype=None, max_norm=1.0, norm=4096, ws=1 << 30, size=1 << 30, count=None):
        n = len(ins)
        keep = [(C.c_void_p * n)(*ins), (C.c_int64 * n)(*numel), (C.c_int32 * n)(*(in_dtype or [0] * n)), (C.c_void_p * n)(*(outs or [0] * n)),
                (C.c_int32 * n)(*(out_dtype or [0] * n))]
        p = abi.ClipArgs()
        p.count, p.norm, p.workspace, p.workspace_bytes, p.max_norm = n if count is None else count, norm, ws, size, max_norm
        p.inp, p.numel, p.in_dtype, p.out_dtype = (C.addressof(keep[k]) for k in (0, 1, 2, 4))
        p.out = C.addressof(keep[3]) if outs else None
        p.keep = keep
        return p

    a, b = 1 << 20, 1 << 21
    for p in (clip([a], [4], norm=0), clip([a], [4], count=-1), clip([a], [-1]), clip([0], [4]), clip([a], [4], in_dtype=[3]), clip([a], [4], ws=0),
              clip([a], [4], size=8), clip([a], [4], ws=(1 << 30) + 8), clip([a], [4], outs=[0]), clip([a], [4], outs=[b], out_dtype=[7]),
              clip([a], [4], outs=[a], max_norm=-1.0), clip([a], [4], outs=[a], max_norm=float("nan")), clip([a], [4], outs=[a], out_dtype=[1]),
              clip([a, a], [4, 4], outs=[a, a]), clip([a, a + 8], [4, 4], outs=[a, a + 8]), clip([a], [4], outs=[a + 4]), clip([a, b], [4, 4], outs=[b, a]),
              clip([a, b], [4, 4], outs=[b + 64, b + 68])):
        bad(lib.afc_clip, p)


def test_workspaces_need_sizes_only(lib):
    p = abi.ConvArgs()
    p.taps, p.batch, p.length, p.width = 4, 2, 100, 24
    n = (C.c_uint64 * 3)()
    at = [C.cast(C.byref(n, 8 * k), C.POINTER(C.c_uint64)) for k in range(3)]
    assert lib.afc_conv_workspace(C.byref(p), at[0]) == 0 and n[0] >= 5 * 24 * 4
    q = abi.ScanArgs()
    q.state, q.batch, q.length, q.width, q.groups = 16, 2, 100, 24, 2
    assert lib.afc_scan_workspace(C.byref(q), *at) == 0 and n[0] >= 2 * 7 * 24 * 16 * 4 and n[2] > 0
    q.length = 0
    assert lib.afc_scan_workspace(C.byref(q), *at) == 0
    assert lib.afc_scan_workspace(C.byref(q), None, at[0], at[1]) == -1 and lib.afc_conv_workspace(C.byref(p), None) == -1


@pytest.mark.skipif(not os.path.exists(os.path.join(codeobj.LLVM, "clang-offload-bundler")) or shutil.which("objcopy") is None, reason="ROCm LLVM tools not available")
def test_kernels_use_scalar_float_arithmetic_and_no_scratch(lib):
    path = build.build_ops()
    assert not re.search(r"v_pk_(add|mul|fma)_f32", codeobj.disassembly(path))
    for name, r in codeobj.kernel_resources(path).items():
        assert r["private_segment_fixed_size"] == 0, name


def test_no_cpu_fallback_of_the_library(lib):
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    assert lib.afc_conv(C.byref(fake_conv()), None) == -2 and b"no HIP device" in lib.afc_ops_last_error()
    assert lib.afc_scan(C.byref(fake_scan()), None) == -2


def test_overlaps_are_found_among_any_tensors(lib):
    """the library's check of a few random ranges against every pair; an accepted call goes on to look for a device"""
    import random
    rng = random.Random(3)
    seen = set()
    for _ in range(400):
        n = rng.randint(1, 4)
        numel = [rng.randint(0, 6) for _ in range(n)]
        ins = [4096 + 4 * rng.randint(0, 40) for _ in range(n)]
        outs = [a if rng.random() < 0.4 else 4096 + 4 * rng.randint(0, 40) for a in ins]
        spans = [(o, o + 4 * k, i, True) for i, (o, k) in enumerate(zip(outs, numel)) if k]
        spans += [(a, a + 4 * k, i, False) for i, (a, o, k) in enumerate(zip(ins, outs, numel)) if k and a != o]
        bad = any(p[0] < q[1] and q[0] < p[1] and (p[3] or q[3]) for x, p in enumerate(spans) for q in spans[:x])
        keep = [(C.c_void_p * n)(*ins), (C.c_int64 * n)(*numel), (C.c_int32 * n)(), (C.c_void_p * n)(*outs)]
        p = abi.ClipArgs()
        p.device, p.count, p.norm, p.workspace, p.workspace_bytes, p.max_norm = 1 << 20, n, 4096, 1 << 30, 1 << 30, 1.0  # (no such device)
        p.inp, p.numel, p.in_dtype, p.out, p.out_dtype = (C.addressof(keep[k]) for k in (0, 1, 2, 3, 2))
        assert lib.afc_clip(C.byref(p), None) != 0
        assert (b"overlap" in lib.afc_ops_last_error()) == bad, (ins, outs, numel)
        seen.add(bad)
    assert seen == {True, False}


def test_more_elements_than_can_be_laid_out(lib):
    n = C.c_uint64()
    for axes, ok in (((1 << 29, 1 << 10, 1 << 9), False), ((1 << 20, 1 << 10, 1 << 18), False), ((1 << 29, 0, 1 << 20), False), ((1 << 10, 1 << 18, 1 << 10), True)):
        a = abi.ConvArgs()
        a.taps, a.batch, a.length, a.width = (4,) + axes
        assert (lib.afc_conv_workspace(C.byref(a), C.byref(n)) == 0) == ok, axes
    keep = [(C.c_void_p * 9)(*[4096] * 9), (C.c_int64 * 9)(*[(1 << 45) - 1] * 9), (C.c_int32 * 9)()]
    for count, ok in ((8, True), (9, False)):
        a = abi.ClipArgs()
        a.count, a.inp, a.numel, a.in_dtype = (count,) + tuple(C.addressof(k) for k in keep)
        assert (lib.afc_clip_workspace(C.byref(a), C.byref(n)) == 0) == ok, count


# ---- what shares memory, what is infinite (on either device) ----

def scan_results(c, softplus=True):
    names = [n for n in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state") if c[n] is not None]
    leaves = {n: c[n].detach().clone().requires_grad_() for n in names}
    args = [leaves.get(n) for n in ("x", "dt", "A", "B", "C", "D", "z", "dt_bias")]
    y, last = ops.selective_scan(*args, softplus=softplus, initial_state=leaves.get("state"), lengths=c["lengths"], return_final_state=True)
    grads = torch.autograd.grad([y, last], [leaves[n] for n in names], [c["dy"], c["dlast"]])
    return dict(y=y.detach(), last=last.detach(), **{"d" + n: g for n, g in zip(names, grads)})


def rates_without_memory(device):
    """a rate of -inf is one so large that no step size leaves anything; behind a row's end the step size is zero, and the state stays"""
    for N, W, L in ((16, 40, 37), (3, 8, 20), (64, 20, 300)):
        c = scan_case(N, 3, L, W, N, device=device, lengths=[L, L - 5, 0])
        big, inf = c["A"].clone(), c["A"].clone()
        big[::3, ::2], inf[::3, ::2] = -1e30, float("-inf")
        want, got = scan_results(dict(c, A=big)), scan_results(dict(c, A=inf))
        for k in want:
            assert bool(torch.isfinite(got[k]).all()) and torch.equal(want[k], got[k]), k
        tokens = [c[k][:, 0] if c[k] is not None else None for k in ("x", "dt", "B", "C", "z")]
        tokens[1] = torch.where(torch.arange(W, device=device) % 2 == 0, -1000.0, tokens[1])  # step sizes of zero
        outs = []
        for A in (big, inf):
            h = c["state"].clone()
            x, dt, B, Cm, z = tokens
            outs.append((ops.selective_scan_step(x, dt, A, B, Cm, h, c["D"], z, c["dt_bias"], True), h))
        assert all(bool(torch.isfinite(b).all()) and torch.equal(a, b) for a, b in zip(*outs))


def infinite_adjoints(device):
    c = scan_case(5, 2, 21, 16, 16, device=device, lengths=[4, 18])
    c["dlast"][:, 0] = float("inf")
    c["state"][0, 0, 0] = float("inf")
    got = scan_results(c)
    for k in ("dx", "ddt", "dB", "dC", "dz"):
        for b, n in enumerate((4, 18)):
            assert not bool(got[k][b, n:].any()) and not bool(got[k][b, n:].isnan().any()), k


def states_of_their_own(device):
    x, w = torch.randn(2, 8, device=device), torch.randn(8, 4, device=device)
    memory = torch.randn(2, 3, 8, device=device)
    keep = memory.clone()
    for bad in (memory[:, 0], memory[:, 2], memory.view(-1)[1:17].view(2, 8)):
        with pytest.raises(ValueError, match="state shares memory with x"):
            ops.causal_conv_step(bad, memory, w)
    with pytest.raises(ValueError, match="state shares memory with bias"):
        ops.causal_conv_step(x, memory, w, memory.view(-1)[:8])
    flat = torch.randn(200, device=device)
    h, B = flat[:64].view(2, 8, 4), flat[64:72].view(2, 4)
    A = -torch.rand(8, 4, device=device)
    for kw, name in ((dict(B=flat[60:68].view(2, 4)), "B"), (dict(C=flat[:8].view(2, 4)), "C"), (dict(x=flat[:16].view(2, 8)), "x"), (dict(A=flat[32:64].view(8, 4)), "A"),
                     (dict(D=flat[8:16]), "D"), (dict(z=flat[1:17].view(2, 8)), "z")):
        with pytest.raises(ValueError, match="state shares memory with %s" % name):
            ops.selective_scan_step(**{**dict(x=x, dt=x, A=A, B=B, C=B, state=h), **kw})
    ops.causal_conv_step(x[:0], x.view(-1)[5:5].view(0, 3, 8), w)  # nothing is shared where there is nothing
    ops.selective_scan_step(x, x, A, B, B, h)  # neighbours in one buffer are no neighbours' memory
    assert torch.equal(memory, keep)


def updates_in_place(device):
    x, w = torch.randn(2, 8, device=device), torch.randn(8, 4, device=device)
    scale = torch.ones((), device=device, requires_grad=True)
    token = torch.randn(2, 4, device=device)
    for state, update in ((torch.randn(2, 3, 8, device=device), lambda s: ops.causal_conv_step(x, s, w)),
                          (torch.randn(2, 8, 4, device=device), lambda s: ops.selective_scan_step(x, x, -w.abs(), token, token, s)),
                          (torch.randn(50, device=device), lambda s: ops.clip_grad_norm([s], 0.1))):
        saved = (state * scale).sum()  # the backward pass needs the state as it is
        with torch.no_grad():
            update(state)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            saved.backward()
    with torch.inference_mode():
        state = torch.zeros(2, 3, 8, device=device)
        ops.causal_conv_step(x, state, w)
        assert torch.equal(state[:, -1], x)


def steps_of_no_rows(device):
    w, A = torch.randn(8, 4, device=device), -torch.rand(8, 4, device=device)

    def none(*axes):
        return torch.empty(0, *axes, device=device)

    assert ops.causal_conv_step(none(8), none(3, 8), w).shape == (0, 8)
    assert ops.selective_scan_step(none(8), none(8), A, none(4), none(4), none(8, 4), torch.ones(8, device=device), none(8)).shape == (0, 8)
    assert float(ops.clip_grad_norm([none(3), none(2, 2)], 1.0)) == 0 and ops.grad_norm([]) == 0


@pytest.mark.parametrize("which", [rates_without_memory, infinite_adjoints, states_of_their_own, updates_in_place, steps_of_no_rows])
def test_on_the_cpu(which):
    which("cpu")


def test_plain_clip_refuses_tensors_that_overlap():
    a = torch.ones(100)
    for grads, out in (([a, a], None), ([a[:60], a[50:]], None), ([a[:50]], [a[25:75]])):
        with pytest.raises(ops.OpsError, match="overlap"):
            ops.clip_grad_norm(grads, 1.0, out=out)
    assert torch.equal(a, torch.ones(100))
    ops.clip_grad_norm([a[50:], a[:50], a[50:50]], 1.0)
    assert abs(float(a.norm()) - 1) < 1e-5 and abs(float(ops.grad_norm([a, a])) - 2 ** 0.5) < 1e-5


# ---- what the binding refuses before it asks for a GPU ----

def calls_of_the_binding(device="cpu"):
    """every call of the binding as (name, call, its floating-point tensors); a call takes one of them replaced"""
    c, v = scan_case(1, 2, 5, 6, 4, device=device), conv_case(1, 2, 5, 6, 3, device=device)
    m = ops._gpu()
    one = {k: c[k][:, 0].contiguous() for k in ("x", "dt", "B", "C", "z")}
    cases = [
        ("causal_conv", ("x", "weight", "bias", "state"), v, lambda a: m.causal_conv(a["x"], a["weight"], a["bias"], True, a["state"], None, True)[0]),
        ("causal_conv_step", ("x", "state", "weight", "bias"), dict(v, x=v["x"][:, 0]), lambda a: m.causal_conv_step(a["x"], a["state"], a["weight"], a["bias"], True)),
        ("selective_scan", ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state"), c,
         lambda a: m.selective_scan(a["x"], a["dt"], a["A"], a["B"], a["C"], a["D"], a["z"], a["dt_bias"], True, a["state"], None, True)[0]),
        ("selective_scan_step", ("x", "dt", "A", "B", "C", "state", "D", "z", "dt_bias"), dict(c, **one),
         lambda a: m.selective_scan_step(a["x"], a["dt"], a["A"], a["B"], a["C"], a["state"], a["D"], a["z"], a["dt_bias"], True)),
        ("clip", ("g", "h"), dict(g=torch.randn(4, device=device), h=torch.randn(3, device=device)), lambda a: m.clip([a["g"], a["h"]], 1.0, None)),
        ("clip", ("out",), dict(g=torch.randn(4, device=device), out=torch.randn(4, device=device)), lambda a: m.clip([a["g"]], 1.0, [a["out"]])),
        ("norm", ("g",), dict(g=torch.randn(4, device=device)), lambda a: m.clip([a["g"]], -1.0, None)),
    ]
    return [(name, names, values, call) for name, names, values, call in cases]


def tangents_are_refused(device):
    import torch.autograd.forward_ad as fwd
    for name, names, values, call in calls_of_the_binding(device):
        for n in names:
            for leaf in (False, True):
                with fwd.dual_level(), torch.set_grad_enabled(leaf and name in ("causal_conv", "selective_scan")):
                    t = values[n].clone().requires_grad_(torch.is_grad_enabled())
                    with pytest.raises(NotImplementedError, match="tangent"):
                        call(dict(values, **{n: fwd.make_dual(t, torch.ones_like(t))}))


def test_the_binding_refuses_tangents(lib):
    tangents_are_refused("cpu")


def test_tangents_on_the_cpu():
    import torch.autograd.forward_ad as fwd
    c = conv_case(3, 2, 5, 4, 3)
    with fwd.dual_level():
        y = fwd.unpack_dual(ops.causal_conv(fwd.make_dual(c["x"], c["dy"]), c["weight"], None, True))
    eps = 1e-3
    a, b = (ops.causal_conv(c["x"] + s * c["dy"], c["weight"], None, True) for s in (eps, -eps))
    # central differences in 32 bits: values of up to 8 are off by 8 u a few times, over 2 eps; the third derivative by eps^2
    assert float(((a - b) / (2 * eps) - y.tangent).abs().max()) < 16 * 8 * 2.0 ** -24 / (2 * eps) + 100 * eps ** 2
