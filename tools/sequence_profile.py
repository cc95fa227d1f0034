"""Kernel times and counters of the operators along time, for profiles/sequence_operators.txt:

    rocprofv3 --kernel-trace --stats -f csv -d DIR -o p -- python3 tools/sequence_profile.py run [NAME,NAME]
    rocprofv3 --pmc SQ_WAVES SQ_INSTS_VALU SQ_INSTS_LDS SQ_LDS_BANK_CONFLICT GRBM_GUI_ACTIVE -f csv -d DIR2 -o p -- python3 tools/sequence_profile.py run
    python3 tools/sequence_profile.py table DIR [DIR2]

`run` takes the listed cases of perf/operators.py (those whose name starts with one of NAME), 24 passes each on two sets of arrays in
turn; `table` prints the median and minimum of every kernel and launch size, and from the counters its vector issue (SQ_INSTS_VALU /
1024 SIMDs x 4 cycles / (GRBM_GUI_ACTIVE / 8 XCDs)) and LDS bank conflict cycles an LDS instruction."""
import collections
import csv
import glob
import os
import re
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def run(names):
    sys.path.insert(0, ROOT)
    import torch
    from perf import operators
    operators.own = True
    for case in operators.listed():
        if names and not case["name"].startswith(tuple(names)):
            continue
        states = [operators.prepare(case, seed) for seed in (1, 2)]
        for k in range(24):
            operators.run(states[k % 2])
        torch.cuda.synchronize()
        print(case["name"], flush=True)


def rows(folder, kind):
    out = []
    for f in glob.glob(os.path.join(folder, "**", f"*{kind}.csv"), recursive=True):
        with open(f) as h:
            out += [r for r in csv.DictReader(h) if "mfcc" in r["Kernel_Name"]]
    return sorted(out, key=lambda r: int(r["Start_Timestamp"]))


def name(r):
    """The kernel, and the types in its name that the profiler leaves mangled or garbles where they are 16 bits wide"""
    return re.search(r"[a-z][a-z_]*_kernel", r["Kernel_Name"]).group(), r["Kernel_Name"]


def median(v):
    return sorted(v)[len(v) // 2]


def table(trace, counters=None):
    times = collections.OrderedDict()
    for r in rows(trace, "kernel_trace"):
        size = int(r["Grid_Size_X"]) * int(r["Grid_Size_Y"])
        times.setdefault((name(r), size), []).append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
    found = collections.defaultdict(lambda: collections.defaultdict(list))
    for r in rows(counters, "counter_collection") if counters else []:
        found[name(r), int(r["Grid_Size"])][r["Counter_Name"]].append(float(r["Counter_Value"]))
    for key, v in times.items():
        line = f"{key[0][0]:26s} threads {key[1]:9d}  launches {len(v):3d}  median {median(v):7.1f} us  min {min(v):7.1f}"
        c = {n: median(w) for n, w in found[key].items()}
        if c:
            line += f"  vector issue {c['SQ_INSTS_VALU'] / 1024 * 4 / (c['GRBM_GUI_ACTIVE'] / 8):.2f}"
            line += f"  conflicts {c['SQ_LDS_BANK_CONFLICT'] / max(c['SQ_INSTS_LDS'], 1):.2f}"
        print(line)


if __name__ == "__main__":
    if sys.argv[1] == "run":
        run(sys.argv[2].split(",") if len(sys.argv) > 2 else None)
    else:
        table(*sys.argv[2:4])
