"""Times page_plan, rope_pages, attention_pages and logits_pick on one B200, over the cases of perf/operators.py.

    python profiles/paged_operators.py [--plain] [--draw N --seed S] [--more] [--only START ...]
    python profiles/paged_operators.py --only NAME --once

A case's inputs are made several times over (seeds 1, 2, ...), 300 MB of them or 24 sets, and passes take the sets in
turn, so that what is larger than L2 together is not found there. `graph` is a pass of a captured run over all sets (the
median of 9 replays), `called` a pass among others as a program enqueues them, launches and the stream's lookup included,
`plain` the same of the plain forms (torch operators). `--draw` adds cases drawn from a seed, `--more` those that comments
beside the kernels quote, `--only` takes those whose names begin so, `--once` runs three passes of one set and times nothing. One line a case: microseconds, and
the bytes that a pass cannot do without over the graph's time.
"""

import argparse
import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parent.parent


def operators():
    sys.path.insert(0, str(ROOT))
    spec = importlib.util.spec_from_file_location("operators", ROOT / "perf" / "operators.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def more():
    """Cases beside the listed ones."""
    out = []
    wide = dict(op="attention_pages", chunk=1, heads=32, kv_heads=8, head_dim=128, page=16, pad=0, type="bf16")
    slim = dict(op="attention_pages", chunk=1, heads=16, kv_heads=2, head_dim=64, page=64, pad=0, type="bf16")
    for rows in (64, 128, 256):
        out.append(dict(wide, name=f"own pages alone, {rows} rows to 1024, 32/8 heads of 128", rows=rows, first=0, ownlen=1024))
    for rows in (64, 128):
        out.append(dict(slim, name=f"own pages alone, {rows} rows to 1024, 16/2 heads of 64", rows=rows, first=0, ownlen=1024))
    for first in (4096, 16384):
        for rows in (1, 32, 64, 128):
            out.append(dict(wide, name=f"prefix of {first}, {rows} rows of one own position, 32/8 heads of 128", rows=rows, first=first, ownlen=1))
    out.append(dict(slim, name="prefix of 8191, 128 rows of one own position, 16/2 heads of 64", rows=128, first=8191, ownlen=1))
    out.append(dict(slim, name="f32, 128 rows of one own position behind 4096, 16/2 heads of 64", rows=128, first=4096, ownlen=1, type="f32"))
    out.append(dict(wide, name="f32, 64 rows of one own position behind 4096, 32/8 heads of 128", rows=64, first=4096, ownlen=1, type="f32"))
    out.append(dict(wide, name="64 requests of 4 rows, own pages to 1024, 32/8 heads of 128", rows=256, chunk=4, first=0, ownlen=1024))
    rope = dict(op="rope_pages", rows=2047, heads=32, kv_heads=8, head_dim=128, inter=True, page=48, positions=32768, pad=9, type="bf16", c="bf16")
    out += [dict(rope, name="rope, 100 of 128 turned, pairs", rot=100), dict(rope, name="rope, 100 of 128 turned, halves", rot=100, inter=False)]
    pick = dict(op="logits_pick", vocab=128000, gap=0, seen=1, biases=0, masks=0, type="f32")
    for rows in (1, 32, 64, 128):
        out.append(dict(pick, name=f"logits, {rows} rows of 128000, no controls but one token", rows=rows))
    out.append(dict(pick, name="logits, 128 rows of 128000 in bf16, histories to 4096", rows=128, seen=4096, biases=64, masks=16, type="bf16"))
    for seen in (4000, 20000):
        out.append(dict(pick, name=f"logits, 64 rows of 128000, histories to {seen}", rows=64, seen=seen))
    return out


def tensors(state):
    return sum(t.numel() * t.element_size() for t in state.values() if isinstance(t, torch.Tensor))


def timed(go, passes, repeats=9):
    """The median time of a pass, in microseconds."""
    times = []
    for _ in range(3):
        go()
    for _ in range(repeats):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        torch.cuda.synchronize()
        a.record()
        go()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 1e3 / passes)
    return sorted(times)[repeats // 2]


def measure(ops, case, plain):
    first = ops.prepare(case, 1)
    sets = min(24, max(2, math.ceil(300e6 / tensors(first))))
    states = [first] + [ops.prepare(case, seed) for seed in range(2, sets + 1)]
    passes = sets * math.ceil(24 / sets)

    def go():
        for i in range(passes):
            ops.run(states[i % sets])

    if plain:
        return timed(go, passes, 5), None
    called = timed(go, passes)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    out = called, timed(graph.replay, passes)
    del graph
    return out


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--plain", action="store_true")
    ap.add_argument("--more", action="store_true")
    ap.add_argument("--draw", type=int, default=0)
    ap.add_argument("--seed", type=int, default=1)
    ap.add_argument("--only", nargs="+", default=[""])
    ap.add_argument("--once", action="store_true")
    args = ap.parse_args()
    ops = operators()
    rng = random.Random(args.seed)
    cases = ops.listed() + [dict(ops.draw(rng), name=f"drawn {i}") for i in range(args.draw)] + (more() if args.more else [])
    cases = [case for case in cases if case["name"].startswith(tuple(args.only))]
    ops.own = True
    if args.once:
        for case in cases:
            state = ops.prepare(case, 1)
            for _ in range(3):
                ops.run(state)
            torch.cuda.synchronize()
        return
    ratios = []
    for case in cases:
        ops.own = True
        called, graph = measure(ops, case, False)
        line = f"{case['name']:70s} graph {graph:8.2f}  called {called:8.2f}  {ops.work(case)['bytes'] / graph / 1e3:7.0f} GB/s"
        if args.plain:
            ops.own = False
            plain, _ = measure(ops, case, True)
            ratios.append(plain / called)
            line += f"  plain {plain:9.1f}"
        print(line, flush=True)
    if ratios:
        print(f"plain over called, geometric mean of {len(ratios)}: {math.exp(sum(map(math.log, ratios)) / len(ratios)):.1f}")


if __name__ == "__main__":
    main()
