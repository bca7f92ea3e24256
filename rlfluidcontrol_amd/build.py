"""Builds libafc_env.so (the environment: HIP kernels + C ABI) and libafc_ops.so (the learner's sequence and gradient
operators) with its torch binding _ops_torch.so in-tree for gfx950.

    python -m rlfluidcontrol_amd.build [--force] [--ops]     (--ops: only libafc_ops.so and its binding)

hipcc cross-compiles without a GPU.  -ffp-contract=off: the reference (Java) never fuses
multiply-add, and parity with the oracle is checked at the bit level wherever the
reference's operation order is kept.
"""
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libafc_env.so")
# translation units, compiled in parallel: the C ABI + small kernels, the three instantiations of the step kernels
# (shipped / diagnostics compiled in / perf mode / few envs per CU: step_kernels.h), the host geometry
SOURCES = ["afc_env.hip", "step_prod.hip", "step_diag.hip", "step_perf.hip", "step_lat.hip", "geometry.cpp"]

def _deps():
    d = [os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".h", ".hip", ".cpp"))]
    d.append(os.path.join(HERE, "..", "include", "afc_env.h"))
    return d

# -fno-slp-vectorize: left to itself the SLP vectoriser pairs scalar float operations into v_pk_*_f32 and pays for it
# in register moves (every phase here is bound by VALU issue); packed arithmetic is written out where it pays
# (the QUICK faces of advdif_v2).  Measured +2 % on the whole step.
FLAGS = (os.environ.get("AFC_EXTRA_FLAGS", "").split()) + ["-O3", "-std=c++17", "-fPIC", "--offload-arch=gfx950", "-ffp-contract=off",
         "-fno-fast-math", "-fno-slp-vectorize", "-Wall", "-Wno-unused-function"]


STAMP = os.path.join(HERE, "build", "flags.stamp")

# libafc_ops.so (include/afc_ops.h).  Scalar float arithmetic only: its kernels fuse multiply-adds where the source says so
# (__builtin_fmaf), and the packed forms, which the compiler would make of them by itself, are switched off.
OPS_LIB = os.path.join(HERE, "libafc_ops.so")
OPS_CSRC = os.path.join(CSRC, "ops")
OPS_SOURCES = ["conv.hip", "scan.hip", "clip.hip"]
OPS_STAMP = os.path.join(HERE, "build", "ops_flags.stamp")
OPS_FLAGS = FLAGS + ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
BINDING = os.path.join(HERE, "_ops_torch.so")
BINDING_STAMP = os.path.join(HERE, "build", "binding_flags.stamp")


def _ops_deps():
    d = [os.path.join(OPS_CSRC, f) for f in os.listdir(OPS_CSRC)]
    return d + [os.path.join(HERE, "..", "include", f) for f in ("afc_ops.h", "afc_env.h")]


def _binding_flags():
    """(compile, link) flags of _ops_torch.so: host code only, against the torch that imports it; None where there is nothing to
    build it against (no torch, one without a GPU's runtime, no headers of torch or Python)"""
    import sysconfig
    try:
        import torch
    except ImportError:
        return None
    inc, lib = os.path.join(os.path.dirname(torch.__file__), "include"), os.path.join(os.path.dirname(torch.__file__), "lib")
    python = sysconfig.get_paths()["include"]
    headers = (os.path.join(inc, "torch", "extension.h"), os.path.join(python, "Python.h"))
    if torch.version.hip is None or not all(map(os.path.exists, headers)):
        return None
    compile_ = ["-O2", "-std=c++17", "-fPIC", "-x", "c++", "-Wall", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1", "-DTORCH_EXTENSION_NAME=_ops_torch",
                "-D_GLIBCXX_USE_CXX11_ABI=%d" % torch._C._GLIBCXX_USE_CXX11_ABI,
                "-DAFC_BUILT_FOR_TORCH=" + torch.__version__]  # (read by nothing but flag_string(): another torch in the same place is another build)
    for d in (inc, os.path.join(inc, "torch", "csrc", "api", "include"), "/opt/rocm/include", python):
        compile_ += ["-isystem", d]
    return compile_, ["-L" + HERE, "-lafc_ops", "-Wl,-rpath,$ORIGIN", "-L" + lib, "-ltorch", "-ltorch_cpu", "-ltorch_hip", "-ltorch_python", "-lc10", "-lc10_hip"]


class _Library:
    def __init__(self, path, csrc, sources, deps, flags, stamp, link=()):
        self.path, self.csrc, self.sources, self.deps, self.flags, self.stamp, self.link = path, csrc, sources, deps, flags, stamp, list(link)

    def flag_string(self):
        """the effective compile + link flags: a library built with other flags (AFC_EXTRA_FLAGS) is not reused silently"""
        return " ".join(self.flags + self.link) + " | HIPCC=" + os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")

    def needs_build(self):
        if not os.path.exists(self.path):
            return True
        t = os.path.getmtime(self.path)
        if any(os.path.getmtime(d) > t for d in self.deps()):
            return True
        if os.environ.get("AFC_EXTRA_FLAGS") or os.path.exists(self.stamp):
            # a stamp exists only next to a library this module built: compare the flags it was built with
            try:
                return open(self.stamp).read() != self.flag_string()
            except OSError:
                return True
        return False


ENV = _Library(LIB, CSRC, SOURCES, _deps, FLAGS, STAMP)
OPS = _Library(OPS_LIB, OPS_CSRC, OPS_SOURCES, _ops_deps, OPS_FLAGS, OPS_STAMP, ["-Wl,-soname,libafc_ops.so"])


def needs_build():
    return ENV.needs_build()


def build(force=False, verbose=False):
    """Everything, the environment's library (returned) first: it needs neither torch nor what is built after it."""
    path = _build(ENV, force, verbose)
    build_ops(force, verbose)
    return path


def build_ops(force=False, verbose=False):
    """libafc_ops.so (returned) and, where there is a torch to build it against, its binding"""
    path = _build(OPS, force, verbose)
    flags = _binding_flags()
    if flags is not None:
        _build(_Library(BINDING, OPS_CSRC, ["binding.cpp"], _ops_deps, flags[0], BINDING_STAMP, flags[1]), force, verbose)
    return path


def _build(lib, force, verbose):
    if not force and not lib.needs_build():
        return lib.path
    import fcntl
    # several ranks of one node may get here together (torchrun): serialise, re-check, build to a
    # temporary name and rename so that nobody ever loads a half-written library
    with open(os.path.join(HERE, ".build.lock"), "w") as lk:
        fcntl.flock(lk, fcntl.LOCK_EX)
        try:
            if force or lib.needs_build():
                hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
                tmp = lib.path + ".tmp.%d" % os.getpid()
                objdir = os.path.join(HERE, "build")
                os.makedirs(objdir, exist_ok=True)
                jobs = []
                try:
                    for src in lib.sources:
                        obj = os.path.join(objdir, os.path.splitext(src)[0] + ".%d.o" % os.getpid())
                        cmd = [hipcc] + lib.flags + ["-c", "-o", obj, os.path.join(lib.csrc, src)]
                        if verbose:
                            print(" ".join(cmd))
                        jobs.append((obj, cmd, subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)))
                    failed = []
                    for obj, cmd, pr in jobs:
                        out = pr.communicate()[0].decode(errors="replace")
                        if pr.returncode != 0:
                            failed.append((cmd, out))
                        elif verbose and out.strip():
                            print(out)
                    if failed:
                        for cmd, out in failed:
                            sys.stderr.write(" ".join(cmd) + "\n" + out + "\n")
                        raise subprocess.CalledProcessError(1, failed[0][0])
                    # the extra flags reach the link step too (a CPU-side -fsanitize needs its runtime there)
                    extra = os.environ.get("AFC_EXTRA_FLAGS", "").split()
                    subprocess.check_call([hipcc] + extra + ["-shared", "-fPIC", "--offload-arch=gfx950", "-o", tmp] +
                                          [j[0] for j in jobs] + lib.link)
                    os.replace(tmp, lib.path)
                    with open(lib.stamp, "w") as f:
                        f.write(lib.flag_string())
                finally:  # object files never outlive the call, whether a translation unit failed or not
                    for obj, _, pr in jobs:
                        if pr.poll() is None:
                            pr.wait()
                        if os.path.exists(obj):
                            os.remove(obj)
                    if os.path.exists(tmp):
                        os.remove(tmp)
        finally:
            fcntl.flock(lk, fcntl.LOCK_UN)
    return lib.path


if __name__ == "__main__":
    print((build_ops if "--ops" in sys.argv else build)(force="--force" in sys.argv, verbose=True))
