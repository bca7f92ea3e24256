"""Times of the learner's operators (rlfluidcontrol_amd.ops) on the GPU: profiles/ops_times.txt.

    python tools/ops_times.py                       rates of the card, then the cases of perf/operators.py (plain torch operations and
                                                    kernels in turn, whole calls as a program makes them) and some more of the kernels alone
    python tools/ops_times.py --run CASE --passes N only N passes of one case's kernels (for rocprofv3: ops_counters.sh)
"""
import argparse
import importlib.util
import math
import os
import statistics
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
cases = importlib.util.module_from_spec(spec)
spec.loader.exec_module(cases)

# other types, states and sizes than the listed cases have
MORE = [
    dict(name="conv_long_f32", op="conv", dtype="f32", batch=3, length=8191, width=4096, taps=4, train=True, ragged=False),
    dict(name="conv_long_f16", op="conv", dtype="f16", batch=3, length=8191, width=4096, taps=4, train=True, ragged=False),
    dict(name="scan_train_f32", op="scan", dtype="f32", batch=8, length=2048, width=2048, state=16, groups=1, train=True, ragged=False),
    dict(name="scan_train_f16", op="scan", dtype="f16", batch=8, length=2048, width=2048, state=16, groups=1, train=True, ragged=False),
    dict(name="scan_train_state64", op="scan", dtype="bf16", batch=8, length=2048, width=512, state=64, groups=1, train=True, ragged=False),
    dict(name="scan_step_state13", op="scan_step", dtype="f32", batch=1024, width=256, state=13, groups=1),
    dict(name="scan_step_state1", op="scan_step", dtype="bf16", batch=1024, width=4096, state=1, groups=1),
]


def seconds(f, passes, groups):
    for _ in range(3):
        f()
    torch.cuda.synchronize()
    t = []
    for _ in range(groups):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(passes):
            f()
        b.record()
        torch.cuda.synchronize()
        t.append(a.elapsed_time(b) * 1e-3 / passes)
    return statistics.median(t)


def rates():
    x = torch.empty(1 << 30, dtype=torch.uint8, device="cuda")
    y = torch.empty_like(x)
    print("copy of 1 GiB: %.0f GB/s" % (2 * x.numel() / seconds(lambda: y.copy_(x), 20, 5) / 1e9))
    x = torch.empty(1 << 26, dtype=torch.float32, device="cuda")
    print("sum of 256 MiB: %.0f GB/s" % (4 * x.numel() / seconds(lambda: x.sum(), 20, 5) / 1e9))
    a, b = (torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    print("bf16 product of 8192^3: %.0f TFLOP/s" % (2 * 8192 ** 3 / seconds(lambda: a @ b, 20, 5) / 1e12))
    z = torch.zeros(64, device="cuda")
    print("smallest kernel, back to back: %.2f us" % (seconds(lambda: z.add_(1), 200, 5) * 1e6), flush=True)


def time_case(case, plain):
    state = cases.prepare(case, 1)
    us = {}
    for turn in range(2):
        for own in ([False] if plain else []) + [True]:
            cases.own = own
            once = seconds(lambda: cases.run(state), 1, 3)
            us.setdefault(own, []).append(1e6 * seconds(lambda: cases.run(state), max(1, min(50, int(0.02 / once))), 9))
    work = cases.work(case)
    own = min(us[True])
    line = "%-20s kernels %9.1f us  %6.0f GB/s  %6.2f TFLOP/s" % (case["name"], own, work["bytes"] / own / 1e3, work["flops"] / own / 1e6)
    ratio = None
    if plain:
        ratio = min(us[False]) / own
        line += "   plain %10.1f us  %6.1fx" % (min(us[False]), ratio)
    print(line, flush=True)
    return ratio


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--run", help="case to run (kernels only)")
    ap.add_argument("--passes", type=int, default=20)
    a = ap.parse_args()
    if a.run:
        case = next(c for c in cases.listed() + MORE if c["name"] == a.run)
        cases.own = True
        state = cases.prepare(case, 1)
        for _ in range(a.passes):
            cases.run(state)
        torch.cuda.synchronize()
        print("done", flush=True)
        return
    rates()
    ratios = [time_case(c, True) for c in cases.listed()]
    print("geometric mean of the ratios: %.1f" % math.exp(statistics.mean(math.log(r) for r in ratios)))
    for c in MORE:
        time_case(c, False)


if __name__ == "__main__":
    main()
