#!/usr/bin/env python3
"""Runs every listed case of perf/operators.py a dozen times over three sets of inputs, for a kernel trace or counters:
  rocprofv3 --kernel-trace --output-format csv -d DIR -o t -- python3 profiles/diag/lowbit_kernels.py [case,case]
and, with `--sum FILE.csv`, prints the median of each low-bit kernel in such a trace (or each counter's, in a counter file)."""
import collections
import csv
import importlib.util
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def run(names):
    sys.path.insert(0, ROOT)
    import torch

    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    ops.own = True
    for case in ops.listed():
        if names and case["name"] not in names:
            continue
        sets = [ops.prepare(case, k) for k in range(3)]
        torch.cuda.synchronize()
        for k in range(12):
            ops.run(sets[k % 3])
        torch.cuda.synchronize()
        print(case["name"], flush=True)
        del sets
        torch.cuda.empty_cache()


def summary(path):
    times = collections.OrderedDict()
    for r in csv.DictReader(open(path)):
        name = r["Kernel_Name"]
        if "mx_" not in name and "act_" not in name:
            continue
        if "Counter_Name" in r:
            key, value = (name, r["Grid_Size"], r["Counter_Name"]), float(r["Counter_Value"])
        else:
            key = (name, "x".join(r[f"Grid_Size_{c}"] for c in "XYZ"), f"{r['VGPR_Count']}+{r['Accum_VGPR_Count']} registers",
                   f"{r['LDS_Block_Size']} B LDS", f"{r['Scratch_Size']} B scratch")
            value = (int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3
        times.setdefault(key, []).append(value)
    for key, v in times.items():
        v.sort()
        print(f"{v[len(v) // 2]:12.2f} (least {v[0]:.2f}, {len(v)} launches)  " + "  ".join(key))


if __name__ == "__main__":
    if len(sys.argv) > 2 and sys.argv[1] == "--sum":
        summary(sys.argv[2])
    else:
        run(sys.argv[1].split(",") if len(sys.argv) > 1 else None)
