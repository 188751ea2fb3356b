#!/usr/bin/env python3
"""Runs every listed case of perf/operators.py, and the forms of the operators that none of them has (`FORMS`), a dozen times
over three sets of inputs, for a kernel trace or counters:
  rocprofv3 --kernel-trace --output-format csv -d DIR -o t -- python3 profiles/diag/lowbit_kernels.py [case,case]
and, with `--sum FILE.csv [case,case]`, prints the median of each low-bit kernel of each case in such a trace (or each counter's, in
a counter file)."""
import collections
import csv
import importlib.util
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


# (name, rows, columns, outputs, type of the rows and results or of the gradient): what a rollout step computes between its layers,
# products of long rows, and weight gradients of other types and sizes, with a mask and the cut gradient ("kept"), with a mask alone
# ("cut") and without
FORMS = [
    ("acting_131072x202x512_to_mxfp4", 131072, 202, 512, "float32", "mxfp4"),
    ("acting_131072x512x256_from_mxfp4", 131072, 512, 256, "mxfp4", "float32"),
    ("between_131072x512x256_from_and_to_mxfp4", 131072, 512, 256, "mxfp4", "mxfp4"),
    ("acting_32x202x512_to_mxfp4", 32, 202, 512, "float32", "mxfp4"),
    ("acting_32x512x256_from_mxfp4", 32, 512, 256, "mxfp4", "float32"),
    ("linear_131072x202x512_bf16", 131072, 202, 512, "bfloat16", "bfloat16"),
    ("linear_131072x512x256_bf16", 131072, 512, 256, "bfloat16", "bfloat16"),
    ("linear_4096x4096x4096_from_mxfp4", 4096, 4096, 4096, "mxfp4", "float32"),
    ("grad_kept_131072x512x202", 131072, 202, 512, "float32", "kept"),
    ("grad_cut_131072x512x202", 131072, 202, 512, "float32", "cut"),
    ("grad_kept_bf16_131072x256x512", 131072, 512, 256, "bfloat16", "kept"),
    ("grad_bf16_131072x256x512", 131072, 512, 256, "bfloat16", "plain"),
    ("grad_kept_f16_131072x256x512", 131072, 512, 256, "float16", "kept"),
    ("grad_131072x20x512", 131072, 512, 20, "float32", "plain"),
    ("grad_kept_131072x512x40", 131072, 40, 512, "float32", "kept"),
    ("grad_1048576x8x256", 1048576, 256, 8, "float32", "plain"),
    ("grad_131072x1024x1024", 131072, 1024, 1024, "float32", "plain"),
    ("grad_131072x2048x2048", 131072, 2048, 2048, "float32", "plain"),
    ("sums_2048x512", 2048, 512, 0, "float32", "plain"),
    ("sums_131072x512", 131072, 512, 0, "float32", "plain"),
]


def form(name, rows, cols, out, kind, what):
    import torch
    from marl_amd import act8, mxfp4

    calls = []
    for k in range(3):
        g = torch.Generator(device="cuda").manual_seed(k)
        rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
        if name.startswith("sums"):
            calls.append(lambda x=rand(rows, cols): act8.column_sums(x))
        elif name.startswith("grad"):
            act, grad = act8.compress(torch.relu(rand(rows, cols)), nonnegative=True), rand(rows, out).to(getattr(torch, kind))
            mask = None if what == "plain" else act8.compress(torch.relu(rand(rows, out)), nonnegative=True)
            calls.append(lambda a=act, g=grad, m=mask: act8.weight_grad(g, a, m, want_masked=what == "kept"))
        else:
            x = torch.relu(rand(rows, cols))
            x = mxfp4.quantize(x) if kind == "mxfp4" else x.to(getattr(torch, kind))
            w = mxfp4.quantize(rand(out, cols) * 0.06)
            calls.append(lambda x=x, w=w, b=rand(out): mxfp4.linear(x, w, b, relu=True, out_dtype=what if what == "mxfp4" else getattr(torch, what)))
    return calls


def cases(names):
    """(name, function that prepares three calls)"""
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    ops.own = True
    both = [(c["name"], lambda c=c: [lambda s=ops.prepare(c, k): ops.run(s) for k in range(3)]) for c in ops.listed()]
    both += [(f[0], lambda f=f: form(*f)) for f in FORMS]
    return [c for c in both if not names or c[0] in names]


def run(names):
    sys.path.insert(0, ROOT)
    import torch

    for name, prepare in cases(names):
        calls = prepare()
        torch.cuda._sleep(1)  # in a trace, what lies between two of its kernels is one case's
        for k in range(12):
            calls[k % 3]()
        torch.cuda.synchronize()
        torch.cuda._sleep(1)
        torch.cuda.synchronize()
        print(name, flush=True)
        del calls
        torch.cuda.empty_cache()


def summary(path, names):
    times, marks, names = collections.OrderedDict(), [], [c[0] for c in cases(names)]
    rows = list(csv.DictReader(open(path)))
    for r in sorted(rows, key=lambda r: int(r["Dispatch_Id"])):
        name = r["Kernel_Name"]
        if "spin_kernel" in name and r["Dispatch_Id"] not in marks:  # a counter file has a line for each counter
            marks.append(r["Dispatch_Id"])
        if len(marks) % 2 == 0 or not any(k in name for k in ("mx_", "act_", "column_sums")):
            continue
        case, name = names[len(marks) // 2], name.split("(")[0].replace("void ", "")
        if "Counter_Name" in r:
            key, value = (case, name, r["Counter_Name"]), float(r["Counter_Value"])
        else:
            key = (case, name, "x".join(r[f"Grid_Size_{c}"] for c in "XYZ"), f"{r['VGPR_Count']}+{r['Accum_VGPR_Count']} registers",
                   f"{r['LDS_Block_Size']} B LDS", f"{r['Scratch_Size']} B scratch")
            value = (int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3
        times.setdefault(key, []).append(value)
    for key, v in times.items():
        v.sort()
        print(f"{v[len(v) // 2]:12.2f} (least {v[0]:.2f}, {len(v)} launches)  " + "  ".join(key))


if __name__ == "__main__":
    if len(sys.argv) > 2 and sys.argv[1] == "--sum":
        summary(sys.argv[2], sys.argv[3].split(",") if len(sys.argv) > 3 else None)
    else:
        run(sys.argv[1].split(",") if len(sys.argv) > 1 else None)
