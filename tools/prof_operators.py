"""Time, bytes and counters of the operators' kernels, case by case.

Without an argument: eight passes of each case of perf/operators.py (and six
copies of 1 GB), each between two marker kernels. Run it under rocprofv3 four
times, each into a folder of its own under one DIR:

    --kernel-trace --stats -d DIR/trace       --pmc FETCH_SIZE -d DIR/fetch
    --pmc WRITE_SIZE -d DIR/write
    --pmc SQ_ACTIVE_INST_VALU SQ_BUSY_CU_CYCLES SQ_WAVE_CYCLES SQ_WAIT_ANY
        -d DIR/waves

with --output-format csv. With DIR as its argument: prints the table from
what they left (profiles/operators_kernels.txt).
"""

import csv
import glob
import os
import re
import sys

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
COPY = "copy 1 GB"
PASSES, COPIES = 8, 6


def cases():
    sys.path.insert(0, REPO)
    from perf import operators
    operators.own = True
    return operators


def run():
    import torch
    operators = cases()
    flag = torch.ones(1, dtype=torch.int32, device="cuda")

    def marked(f, times):
        torch.bitwise_not(flag)
        for k in range(times):
            f(k)
        torch.bitwise_not(flag)
        torch.cuda.synchronize()

    a = torch.empty(1 << 30, dtype=torch.uint8, device="cuda")
    b = torch.empty_like(a)
    marked(lambda k: b.copy_(a), COPIES)
    del a, b
    for case in operators.listed():
        states = [operators.prepare(case, seed) for seed in range(2)]
        for s in states:
            operators.run(s)
        marked(lambda k: operators.run(states[k % 2]), PASSES)
        print(case["name"], flush=True)
        del states, s


def sections(rows, names):
    """{case: {kernel: its rows}} of rows in the order of their launches."""
    out, at, inside = {}, -1, False
    for row in rows:
        if "bitwise_not" in row["Kernel_Name"]:
            inside = not inside
            at += inside
            continue
        kernel = re.search(r"(glr|adamw)_\w+?_kernel|[cC]opy",
                           row["Kernel_Name"])
        if inside and kernel and (names[at] == COPY) == (
                kernel.group(1) is None):
            name = kernel.group(0) if kernel.group(1) else "copy"
            out.setdefault(names[at], {}).setdefault(name, []).append(row)
    return out


def read(folder, kind):
    (path,) = glob.glob(os.path.join(folder, "**", f"*{kind}.csv"),
                        recursive=True)
    with open(path) as f:
        return list(csv.DictReader(f))


def counters(folder, names):
    launches = {}
    for row in read(folder, "counter_collection"):
        one = launches.setdefault(int(row["Dispatch_Id"]),
                                  {"Kernel_Name": row["Kernel_Name"]})
        one[row["Counter_Name"]] = float(row["Counter_Value"])
    return sections([launches[k] for k in sorted(launches)], names)


def middle(rows, value):
    return sorted(map(value, rows))[len(rows) // 2]


def table(folder):
    names = [COPY] + [case["name"] for case in cases().listed()]
    trace = sections(sorted(read(os.path.join(folder, "trace"),
                                 "kernel_trace"),
                            key=lambda r: int(r["Start_Timestamp"])), names)
    fetch, write, waves = (counters(os.path.join(folder, k), names)
                           for k in ("fetch", "write", "waves"))
    fetched = lambda r: r["FETCH_SIZE"]  # noqa: E731
    written = lambda r: r["WRITE_SIZE"]  # noqa: E731
    per_read = (1 << 30) / middle(fetch[COPY]["copy"], fetched)
    per_write = (1 << 30) / middle(write[COPY]["copy"], written)
    for case, kernels in trace.items():
        for kernel, rows in kernels.items():
            us = middle(rows, lambda r: (int(r["End_Timestamp"]) - int(
                r["Start_Timestamp"])) / 1e3)
            mb = [middle(fetch[case][kernel], fetched) * per_read / 1e6,
                  middle(write[case][kernel], written) * per_write / 1e6]
            w = waves[case][kernel]
            busy = middle(w, lambda r: r["SQ_ACTIVE_INST_VALU"]
                          / max(1, r["SQ_BUSY_CU_CYCLES"]))
            wait = middle(w, lambda r: r["SQ_WAIT_ANY"]
                          / max(1, r["SQ_WAVE_CYCLES"]))
            times = len(rows) // (COPIES if case == COPY else PASSES)
            print(f"{case:18} {kernel:20} x{times} {us:9.1f} us  "
                  f"read {mb[0]:8.1f} MB  written {mb[1]:8.1f} MB  "
                  f"{sum(mb) / us:5.2f} TB/s  VALU {100 * busy:2.0f} % of "
                  f"CU-busy, waves wait {100 * wait:2.0f} %")


if __name__ == "__main__":
    table(sys.argv[1]) if len(sys.argv) > 1 else run()
