"""The paged key-value cache's operators and the verification of drafted tokens at the cases of perf/operators.py: microseconds a call (three
sets of inputs in turn, so that nothing small stays in the caches by itself), bytes they cannot do without and the rate that makes.
`--plain` times the plain torch forms instead; names of cases as arguments pick some.  Under `rocprofv3 --kernel-trace` with `--few`."""
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch  # noqa: E402

from perf import operators as P  # noqa: E402


def main():
    flags = {a for a in sys.argv[1:] if a.startswith("--")}
    names = [a for a in sys.argv[1:] if not a.startswith("--")]
    P.own = "--plain" not in flags
    for case in P.listed():
        if names and case["name"] not in names:
            continue
        sets = [P.prepare(case, 1 + k) for k in range(3)]
        for s in sets:
            P.run(s)
        torch.cuda.synchronize()
        best = float("inf")
        for _ in range(1 if "--few" in flags else 6):
            torch.cuda.synchronize()
            t = time.perf_counter()
            for k in range(9 if "--few" in flags else 30):
                P.run(sets[k % 3])
            torch.cuda.synchronize()
            best = min(best, (time.perf_counter() - t) / (9 if "--few" in flags else 30))
        b = P.work(case)["bytes"]
        print(f"{case['name']:<20s} {best * 1e6:9.2f} us  {b / 1e6:9.2f} MB  {b / best / 1e9:7.0f} GB/s", flush=True)
        del sets
        torch.cuda.empty_cache()


if __name__ == "__main__":
    main()
