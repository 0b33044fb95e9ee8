"""Times residual_norm, residual_norm_bwd, grad_norm and clip_grads on the cases of perf/operators.py (one GPU): microseconds of a
call from Python and, for comparison, the share of a large copy's rate that its least traffic makes of that.

    python tools/train_ops_bench.py [--match SUBSTRING] [--iters N]
    rocprofv3 --kernel-trace --stats -- python3 tools/train_ops_bench.py --iters 20
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf"))
import operators  # noqa: E402

COPY = 5.4e12        # bytes/s that a 512 MB device copy reaches, read and written


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--match", default="")
    ap.add_argument("--iters", type=int, default=100)
    args = ap.parse_args()
    operators.own = True
    for case in operators.listed():
        if args.match not in case["name"]:
            continue
        state = operators.prepare(case, 0)
        for _ in range(5):
            operators.run(state)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(args.iters):
            operators.run(state)
        b.record()
        b.synchronize()
        us = a.elapsed_time(b) / args.iters * 1e3
        floor = operators.work(case)["bytes"] / COPY * 1e6
        print("%-28s %9.2f us   least traffic %8.2f us   %5.1f %%" % (case["name"], us, floor, 100 * floor / us), flush=True)
        del state
        torch.cuda.empty_cache()


if __name__ == "__main__":
    main()
