"""The calls of paged_step_kernel_trace.md: each case of perf/more_operators.py and some
that it does not list, 21 times (three sets of inputs in turn) through the public
entry points.  From the repository's root:

    rocprofv3 --kernel-trace -f csv -d DIR -- python3 profiles/paged_step_calls.py
    rocprofv3 --pmc FETCH_SIZE -f csv -d DIR -- python3 profiles/paged_step_calls.py 6

and, without the profiler, `--time` for the time of a replayed graph of the calls."""
import os
import sys

import torch

sys.path.insert(0, os.getcwd())
from perf import more_operators as ops  # noqa: E402

HEADS = {"heads": 32, "kv": 8, "D": 128}
MORE = [
    {"name": "norms, 126 of 128 columns rotated", "op": "rope", "T": 8192, **HEADS, "pairs": 63, "inter": False, "norm": True, "x": "bf16"},
    {"name": "norms, 126 columns, all rotated", "op": "rope", "T": 8192, "heads": 32, "kv": 8, "D": 126, "pairs": 63, "inter": False,
     "norm": True, "x": "bf16"},
    {"name": "append and read 32768 tokens, fp32 and int8", "op": "store", "B": 1, "T": 32768, "kv": 8, "D": 128, "page": 64, "max": 32784,
     "one": True, "new": "f32", "cache": "i8", "ragged": False},
    {"name": "512 tokens over 8192, bf16", "op": "attend", "B": 1, "T": 512, **HEADS, "page": 64, "max": 8192, "window": 0, "q": "bf16",
     "cache": "bf16"},
    {"name": "512 tokens over 8192, e4m3", "op": "attend", "B": 1, "T": 512, **HEADS, "page": 64, "max": 8192, "window": 0, "q": "bf16",
     "cache": "f8"},
    {"name": "256 sequences up to 8192, e4m3", "op": "attend", "B": 256, "T": 1, **HEADS, "page": 64, "max": 8192, "window": 0, "q": "bf16",
     "cache": "f8"},
]


def replayed(states):
    """us of a call among others, in a replayed graph."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.run(states[0])
    torch.cuda.synchronize()
    graph, best = torch.cuda.CUDAGraph(), float("inf")
    with torch.cuda.graph(graph):
        for i in range(12):
            ops.run(states[i % 3])
    for _ in range(8):
        start, end = torch.cuda.Event(True), torch.cuda.Event(True)
        start.record()
        graph.replay()
        end.record()
        torch.cuda.synchronize()
        best = min(best, start.elapsed_time(end) / 12 * 1e3)
    return best


def main():
    ops.own = True
    calls = int(sys.argv[1]) if len(sys.argv) > 1 and sys.argv[1].isdigit() else 21
    for case in ops.listed() + MORE:
        states = [ops.prepare(case, seed) for seed in (1, 2, 3)]
        if "--time" in sys.argv:
            print(f"{case['name']}: {replayed(states):.1f} us", flush=True)
            continue
        for i in range(calls):
            ops.run(states[i % 3])
        torch.cuda.synchronize()
        print(case["name"], flush=True)
        del states


if __name__ == "__main__":
    main()
