"""Times the workloads of perf/operators.py: their plain forms and the kernels.

    python perf/time_operators.py [--only NAME ...] [--kernels] [--gbs 6539.5]

For each case, both forms on inputs of the same seed, one after the other: 3
passes of warm-up, then 7 blocks of passes between CUDA events on the current
stream, each block at least 20 ms (2 to 400 passes).  Printed is a pass's time
in the median block and, in brackets, in the fastest and the slowest.  Passes
follow one another on one set of inputs, so cases below 126 MB run out of L2, as
they do inside a step.  The floor is the case's bytes at --gbs.  --kernels lists
the kernels of a pass with their device times (torch.profiler, a run of its own).
"""

from __future__ import annotations

import argparse
import os
import statistics
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "perf")]
import operators  # noqa: E402


def block(state, passes: int) -> float:
    """Microseconds of a pass."""
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    torch.cuda.synchronize()
    start.record()
    for _ in range(passes):
        operators.run(state)
    end.record()
    torch.cuda.synchronize()
    return start.elapsed_time(end) * 1e3 / passes


def timed(case: dict, own: bool, seed: int = 1) -> list[float]:
    operators.own = own
    state = operators.prepare(case, seed)
    block(state, 3)
    passes = max(2, min(400, int(20e3 / block(state, 2)) + 1))
    return sorted(block(state, passes) for _ in range(7))


def kernels(case: dict, seed: int = 1, passes: int = 5) -> list[tuple[float, str]]:
    """(microseconds a pass, name) of the kernels of a pass, longest first."""
    from torch.profiler import ProfilerActivity, profile

    operators.own = True
    state = operators.prepare(case, seed)
    block(state, 3)
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        block(state, passes)
    return sorted(((e.self_device_time_total / passes, e.key) for e in p.key_averages()
                   if e.self_device_time_total > 0), reverse=True)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--only", nargs="*", help="names of cases (default: all)")
    ap.add_argument("--kernels", action="store_true")
    ap.add_argument("--gbs", type=float, default=6539.5, help="memory rate of the floor, GB/s")
    args = ap.parse_args()
    for case in operators.listed():
        if args.only and case["name"] not in args.only:
            continue
        cells = []
        for own in (False, True):
            t = timed(case, own)
            cells.append(f"{statistics.median(t):9.1f} [{t[0]:.1f}, {t[-1]:.1f}]")
            torch.cuda.empty_cache()
        floor = operators.work(case)["bytes"] / args.gbs / 1e3
        print(f"{case['name']:26s} floor {floor:7.1f}   plain {cells[0]:30s} here {cells[1]}",
              flush=True)
        for us, name in kernels(case) if args.kernels else ():
            print(f"    {us:9.1f}  {name[:120]}")
        torch.cuda.empty_cache()


if __name__ == "__main__":
    main()
