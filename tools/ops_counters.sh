#!/bin/bash
# ops_counters.sh out_dir case ...: kernel times and SQ counters of cases of tools/ops_times.py, one line a kernel, into
# out_dir/ops_kernels.txt and out_dir/ops_counters.txt (kernel trace and counters in runs of their own)
root=$(cd "$(dirname "$0")/.." && pwd)
out=$(cd "$1" && pwd); shift
cd /tmp && export TMPDIR=/tmp
: > "$out/ops_kernels.txt"; : > "$out/ops_counters.txt"
for c in "$@"; do
  timeout -s KILL 120 rocprofv3 --kernel-trace --stats --output-format csv -d "$out/trace" -- python3 "$root/tools/ops_times.py" --run "$c" --passes 20 > "$out/trace.log" 2>&1 || exit 1
  echo "$c" >> "$out/ops_kernels.txt"
  python3 - "$out" >> "$out/ops_kernels.txt" <<'PY'
import csv, glob, re, sys
for f in glob.glob(sys.argv[1] + "/trace/**/*kernel_stats.csv", recursive=True):
    for r in sorted(csv.DictReader(open(f)), key=lambda r: -float(r["TotalDurationNs"])):
        m = re.search(r"afc_ops::(k_\w+(<.*>)?)\(", r["Name"])
        if m:
            print("   %-40s calls %5s  mean %8.2f us  min %8.2f us" % (m.group(1).replace("afc_ops::", ""), r["Calls"], float(r["AverageNs"]) / 1e3, float(r["MinNs"]) / 1e3))
PY
  rm -r "$out/trace"
  tail -1 "$out/ops_kernels.txt"
  for pass in "SQ_WAVES SQ_WAVE_CYCLES SQ_BUSY_CU_CYCLES SQ_INSTS_VALU SQ_ACTIVE_INST_VALU SQ_INSTS_LDS SQ_ACTIVE_INST_LDS SQ_LDS_BANK_CONFLICT" "GRBM_GUI_ACTIVE"; do
    timeout -s KILL 60 rocprofv3 --pmc $pass --output-format csv -d "$out/pmc" -- python3 "$root/tools/ops_times.py" --run "$c" --passes 3 > "$out/pmc.log" 2>&1 || exit 1
    python3 - "$out" "$c" >> "$out/ops_counters.txt" <<'PY'
import collections, csv, glob, re, sys
sums, calls = collections.defaultdict(lambda: collections.defaultdict(float)), collections.Counter()
for f in glob.glob(sys.argv[1] + "/pmc/**/*counter_collection.csv", recursive=True):
    for r in csv.DictReader(open(f)):
        m = re.search(r"afc_ops::(k_\w+(<.*>)?)\(", r["Kernel_Name"])
        if m:
            k = m.group(1).replace("afc_ops::", "")
            sums[k][r["Counter_Name"]] += float(r["Counter_Value"])
            calls[k, r["Counter_Name"]] += 1
for k in sums:
    print("%-20s %-32s %s" % (sys.argv[2], k, " ".join("%s=%.4g" % (c, v / calls[k, c]) for c, v in sorted(sums[k].items()))))
PY
    rm -r "$out/pmc"
  done
done
rm -f "$out/trace.log" "$out/pmc.log"
