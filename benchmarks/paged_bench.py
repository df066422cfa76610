"""The paged key-value cache's operators and the verification of drafted tokens at the cases of perf/operators.py: microseconds a call (three
sets of inputs in turn, so that nothing small stays in the caches by itself), bytes they cannot do without and the rate that makes.
`--plain` times the plain torch forms instead; names of cases as arguments pick some.  Under `rocprofv3 --kernel-trace` with `--few`.
`--decode`: tokens a second of generate() over the dense and the paged cache, bounded, and of speculative_generate with the passes it took (bf16, the
nocat shape, 80 tokens, random weights: the distributions are flat, so that a small random model's drafts are mostly accepted as well)."""
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch  # noqa: E402

from perf import operators as P  # noqa: E402


def decode():
    import multimodal_amd as mm
    from bench import CONFIGS, build_model, synth_batch
    from multimodal_amd import generate as G
    dev, c, steps = torch.device("cuda:0"), CONFIGS["local_config_nocat"], 80
    m, small = build_model(c, dev).eval(), build_model(dict(c, L=1, E=256), dev, seed=1).eval()
    passes, target_run = [0], G._PagedDecoder.run

    def counted(self, ids):
        passes[0] += 1
        return target_run(self, ids)
    G._PagedDecoder.run = counted
    for B in (1, 32, 1024):
        ir, nmr, _ = synth_batch(c, B, dev, 4321)
        gen = torch.Generator(device=dev).manual_seed(1)
        spec = lambda d, t: G.speculative_generate(m, d, nmr, ir, max_len=steps, eos_id=-7, n_draft=4, temperature=t, generator=gen)
        forms = {"dense": lambda: m.generate(nmr, ir, max_len=steps, early_stop=False),
                 "page_size=16": lambda: m.generate(nmr, ir, max_len=steps, early_stop=False, page_size=16),
                 "kv_budget=128, kv_recent=16": lambda: m.generate(nmr, ir, max_len=steps, early_stop=False, kv_budget=128, kv_recent=16),
                 "drafted, own weights": lambda: spec(m, 0), "drafted, one layer of 256": lambda: spec(small, 1.0)}
        for name, run in forms.items():
            with mm.compute_dtype(torch.bfloat16):
                run()
                best = float("inf")
                for _ in range(3):
                    torch.cuda.synchronize()
                    passes[0], t = 0, time.perf_counter()
                    run()
                    torch.cuda.synchronize()
                    best = min(best, time.perf_counter() - t)
            print(f"B {B:<5d} {name:<28s} {B * steps / best:10.0f} tokens/s  {best * 1e3:9.1f} ms" + (f"  {passes[0]} passes" if passes[0] else ""), flush=True)


def main():
    flags = {a for a in sys.argv[1:] if a.startswith("--")}
    names = [a for a in sys.argv[1:] if not a.startswith("--")]
    if "--decode" in flags:
        return decode()
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
