"""Kernels of the class evidence and of the MXFP4 operators: one case per run, three inputs in turn.

  python scratch/operators_kernels.py names              # the cases
  python scratch/operators_kernels.py run CASE           # 240 passes (scratch/operators_kernels.sh profiles these)
  python scratch/operators_kernels.py calls              # time per call back to back from Python: median of 25 blocks of 20
  python scratch/operators_kernels.py table CASE DIR     # rows for profiles/operators/kernels.csv from a kernel trace in DIR
"""
import collections
import csv
import glob
import os
import re
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)

LABELS = {
    "evidence_image": "300 rows x 80 classes fp16 top 5", "evidence_batch": "64 x 300 rows x 80 classes fp32 top 5",
    "bins_batch": "64 x 4 x 8400 x 16 planes fp16 top 2", "vocabulary_rows": "511 x 32001 bf16 top 10",
    "vocabulary_long": "2 x 200001 fp32 top 20", "quantize_weights": "640 x 2560 fp32", "quantize_features": "409600 x 320 fp16 to fp32",
    "linear_row": "1 x 1280 -> 1000 bf16", "linear_wide": "8192 x 2560 -> 2560 quantised bf16", "conv_image": "640 -> 640 on 20 x 20 fp16",
    "conv_odd": "3 x 400 -> 75 on 37 x 53 fp32", "conv_batch": "64 x 1280 -> 320 on 80 x 80 fp16",
}


def _rows(name, rows, classes, top):
    return {"name": name, "op": "rows", "rows": rows, "classes": classes, "top": top, "activation": "softmax", "dtype": "bf16", "masked": 0.0}


def _linear(name, k, packed):
    return {"name": name, "op": "linear", "m": 8192, "k": k, "n": 2560, "bias": True, "act": "", "dtype": "bf16", "packed": packed}


def _conv(name, k, n, h, layout="planes"):
    return {"name": name, "op": "pointwise", "batch": 64, "k": k, "n": n, "h": h, "w": h, "act": "silu", "dtype": "f16", "layout": layout}


MORE = [_rows("16384 x 32001 bf16 top 10", 16384, 32001, 10), _rows("102400 x 80 rows bf16 top 5", 102400, 80, 5),
        _linear("8192 x 10240 -> 2560 quantised bf16", 10240, True), _linear("8192 x 2560 -> 2560 bf16 rows", 2560, False),
        _conv("64 x 320 -> 320 on 80 x 80 fp16", 320, 320, 80), _conv("64 x 320 -> 320 on 80 x 80 fp16 channels-last", 320, 320, 80, "channels_last"),
        _conv("64 x 1280 -> 320 on 80 x 80 fp16 channels-last", 1280, 320, 80, "channels_last"), _conv("64 x 64 -> 32 on 160 x 160 fp16", 64, 32, 160)]


def cases():
    from perf import operators as P
    P.own = True
    return P, {**{LABELS[c["name"]]: c for c in P.listed()}, **{c["name"]: c for c in MORE}}


def states(P, case):
    import torch
    sts = [P.prepare(case, seed) for seed in range(3)]
    if case.get("layout") == "channels_last":
        for st in sts:
            st["x"] = st["x"].contiguous(memory_format=torch.channels_last)
    return sts


def main():
    mode = sys.argv[1]
    if mode == "names":
        print("\n".join(cases()[1]))
    elif mode == "run":
        import torch
        P, all_cases = cases()
        sts = states(P, all_cases[sys.argv[2]])
        with torch.inference_mode():
            for i in range(240):
                P.run(sts[i % 3])
        torch.cuda.synchronize()
        print("done")
    elif mode == "calls":
        import torch
        P, all_cases = cases()
        for name, case in all_cases.items():
            sts, times = states(P, case), []
            with torch.inference_mode():
                for i in range(60):
                    P.run(sts[i % 3])
                for _ in range(25):
                    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                    torch.cuda.synchronize()
                    a.record()
                    for i in range(20):
                        P.run(sts[i % 3])
                    b.record()
                    torch.cuda.synchronize()
                    times.append(a.elapsed_time(b) / 20 * 1e3)
            print(f"{name}: {sorted(times)[len(times) // 2]:.1f} us per call", flush=True)
            del sts
            torch.cuda.empty_cache()
    elif mode == "table":
        case, where = sys.argv[2:]
        times = collections.defaultdict(list)
        for row in csv.DictReader(open(glob.glob(os.path.join(where, "**", "*kernel_trace.csv"), recursive=True)[0])):
            name = row["Kernel_Name"]
            if re.search(r"(evidence|mx)_[a-z_]+?_kernel", name):
                times[name].append((int(row["Start_Timestamp"]), (int(row["End_Timestamp"]) - int(row["Start_Timestamp"])) / 1e3))
        for name, t in times.items():
            if len(t) < 200:      # weights, and rows that come quantised: once per input
                continue
            t = sorted(v for _, v in sorted(t)[len(t) // 4:])
            short = re.search(r"(evidence|mx)_[a-z_]+?_kernel", name).group()
            print(f'{case},{short},{len(t)},{t[len(t) // 2]:.1f},{t[0]:.1f}')


main()
