"""Runs cases of perf/more_operators.py under a profiler, and sums up what it wrote.

    python3 profiles/train_operators.py run CASE [PASSES]     three sets of inputs in turn; CASE is a listed name, its values changed by ,key=value
    python3 profiles/train_operators.py times FOLDER          median and least time of each kernel in a --kernel-trace run
    python3 profiles/train_operators.py counters FOLDER       mean of each counter per dispatch of each kernel in a --pmc run
"""
import collections
import csv
import glob
import importlib
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LAST = 20   # dispatches of a kernel that count (the first ones load it)
OWN = ("spread_kernel", "collect_kernel", "checkpoint_kernel", "backward_kernel", "ragged_k", "lay_rows")


def run(case, passes=LAST):
    os.chdir(ROOT)
    sys.path.insert(0, ROOT)
    import torch
    operators = importlib.import_module("perf.more_operators")
    operators.own = True
    name, *changes = case.split(",")
    case = next(c for c in operators.listed() if c["name"] == name)
    for change in changes:
        key, value = change.split("=")
        case[key] = type(case[key])(value)
    states = [operators.prepare(case, seed) for seed in range(3)]
    for i in range(3 + int(passes)):
        operators.run(states[i % 3])
    torch.cuda.synchronize()
    print("done:", case, flush=True)


def rows(folder, kind):
    """Rows of the profiler's tables of a kind, in the order of the dispatches, of these operators' kernels."""
    for path in sorted(glob.glob(os.path.join(folder, "**", f"*{kind}.csv"), recursive=True)):
        with open(path) as f:
            yield from sorted((r for r in csv.DictReader(f) if any(n in r["Kernel_Name"] for n in OWN) and "at::" not in r["Kernel_Name"]),
                              key=lambda r: int(r["Dispatch_Id"]))


def short(name):
    return name.replace("void ", "").replace("(anonymous namespace)::", "").split("(")[0]


def times(folder):
    found = collections.defaultdict(list)
    for r in rows(folder, "kernel_trace"):
        found[short(r["Kernel_Name"])].append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
    for name, v in found.items():
        if len(v) >= LAST:
            v = sorted(v[-LAST:])
            print(f"{v[len(v) // 2]:10.2f} us  (least {v[0]:8.2f})  {name}")


def counters(folder):
    found = collections.defaultdict(lambda: collections.defaultdict(list))
    for r in rows(folder, "counter_collection"):
        found[short(r["Kernel_Name"])][r["Counter_Name"]].append(float(r["Counter_Value"]))
    for name, by in found.items():
        if max(map(len, by.values())) >= LAST:
            print("  " + name + "\n    " + "  ".join(f"{c} {sum(v[-LAST:]) / len(v[-LAST:]):,.0f}" for c, v in sorted(by.items())))


if __name__ == "__main__":
    {"run": run, "times": times, "counters": counters}[sys.argv[1]](*sys.argv[2:])
