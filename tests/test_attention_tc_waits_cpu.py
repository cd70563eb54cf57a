"""Waits of the tcgen05 attention kernel (cuda-fp8-ampere_b200/csrc/kv_attention_tc.cu), checked on the CPU: a model
of its warps, in which every order of their steps is gone through. An mbarrier's waiter names a phase by its parity
only, so the phase that it waits for must be the present one or the one just ended whenever it looks: one phase
further and it waits for ever, one phase earlier and it goes on too soon.

The model's threads: two of the load warps, the one that issues products, two of each softmax group, and the tensor
core, which finishes products in the order of their issue. Barrier counts and the places of K's barriers are read
from the source."""
import os
import re

import pytest

from conftest import PKG

SRC = os.path.join(PKG, "csrc", "kv_attention_tc.cu")


def k_barriers():
    """(barriers of K, log2 of them) as declared; all uses take barrier `tile mod n`, phase `tile div n`."""
    text = open(SRC).read()
    n = int(re.search(r"\bs_k_full\[(\d+)\]", text).group(1))
    log = n.bit_length() - 1
    at = "g" if n == 2 else "idx & %d" % (n - 1)
    assert len(re.findall(r"wait\(&s_k_full\[%s\], idx >> %d\)" % (at, log), text)) == 2
    assert len(re.findall(r"mbar_arrive\(&s_k_full\[%s\]\)" % at, text)) == 1
    assert len(re.findall(r"s_k_full", text)) == 5
    return n, log


def programs(segments, n_k, loads, softs):
    """The threads' steps: ("wait", barrier, phase), ("arrive", barrier), ("block", barrier, phase)."""
    log_k = n_k.bit_length() - 1
    k_bar = lambda i: "k%d" % (i % n_k)  # noqa: E731
    size = {"q": 2 * softs, "o": 2 * softs, "named": 2 * softs}
    load, mma, tensor = [], [], []
    soft = ([], [])
    idx = named = done_segments = 0

    def join(g):
        soft[g].extend([("arrive", "named"), ("block", "named", named)])

    for tiles in segments:
        if tiles:
            for g in (0, 1):
                soft[g].append(("arrive", "q"))
                join(g)
            named += 1
        last = [None, None]
        for t in range(tiles):
            i = idx + t
            g = i & 1
            if i > 0:
                load.append(("wait", "s%d" % (g ^ 1), (i - 1) >> 1))
            load.append(("arrive", k_bar(i)))
            if i > 1:
                load.append(("wait", "pv%d" % g, (i >> 1) - 1))
            load.append(("arrive", "v%d" % g))
            soft[g].extend([("wait", "s%d" % g, i >> 1), ("wait", k_bar(i), i >> log_k), ("wait", "v%d" % g, i >> 1), ("arrive", "p%d" % g)])
            last[g] = i

        def product(i, first):
            g = i & 1
            mma.extend([("wait", "v%d" % g, i >> 1), ("wait", "p%d" % g, i >> 1)])
            if first and done_segments > 0:
                mma.append(("wait", "o", done_segments - 1))
            mma.append(("arrive", "issued"))
            tensor.extend([("block", "issued", len(tensor) // 2), ("arrive", "pv%d" % g)])

        for t in range(tiles):
            i = idx + t
            mma.append(("wait", k_bar(i), i >> log_k))
            if t == 0:
                mma.append(("wait", "q", done_segments))
            mma.append(("arrive", "issued"))
            tensor.extend([("block", "issued", len(tensor) // 2), ("arrive", "s%d" % (i & 1))])
            if t > 0:
                product(i - 1, t <= 2)
        if tiles:
            product(idx + tiles - 1, tiles <= 2)
        for g in (0, 1):
            if last[g] is not None:
                soft[g].append(("wait", "pv%d" % g, last[g] >> 1))
            join(g)
            if tiles:
                soft[g].append(("arrive", "o"))
        named += 1
        for g in (0, 1):
            join(g)
        named += 1
        idx += tiles
        done_segments += tiles > 0
    for g in (0, 1):
        size.update({"s%d" % g: 1, "pv%d" % g: 1, "v%d" % g: loads, "p%d" % g: softs})
    size.update({"k%d" % i: loads for i in range(n_k)})
    size["issued"] = 1
    return [load] * loads + [mma, tensor] + [soft[0]] * softs + [soft[1]] * softs, size


def explore(threads, size):
    """Goes through every order of the threads' steps; the first wait that can go wrong, or None."""
    names = sorted(size)
    at = {b: k for k, b in enumerate(names)}
    before = []  # arrivals of a thread before its step i
    for prog in threads:
        rows = [[0] * len(names)]
        for op in prog:
            rows.append(list(rows[-1]))
            if op[0] == "arrive":
                rows[-1][at[op[1]]] += 1
        before.append(rows)
    start = tuple(0 for _ in threads)
    seen, todo = {start}, [start]
    while todo:
        state = todo.pop()
        phase = [sum(before[t][i][k] for t, i in enumerate(state)) // size[b] for k, b in enumerate(names)]
        moved = False
        for t, i in enumerate(state):
            if i == len(threads[t]):
                continue
            op = threads[t][i]
            if op[0] != "arrive":
                ended = phase[at[op[1]]]
                if op[0] == "wait" and not op[2] <= ended <= op[2] + 1:
                    return "step %d of thread %d, %s: the barrier has ended %d phases" % (i, t, op, ended)
                if ended <= op[2]:
                    continue
            moved = True
            new = state[:t] + (i + 1,) + state[t + 1:]
            if new not in seen:
                seen.add(new)
                todo.append(new)
        if not moved and any(i < len(threads[t]) for t, i in enumerate(state)):
            return "every thread waits: %s" % (state,)
    return None


@pytest.mark.parametrize("segments, loads, softs", [
    ([10], 1, 1), ([5], 2, 2), ([1, 3, 2, 4], 1, 1), ([3, 0, 1, 1, 2], 1, 1), ([2, 2], 2, 2), ([6], 2, 1), ([6], 1, 2)])
def test_no_wait_is_overtaken(segments, loads, softs):
    n, _ = k_barriers()
    assert explore(*programs(segments, n, loads, softs)) is None


def test_the_model_sees_an_overtaken_wait():
    """With two barriers for K the loads of a tile may end before a softmax warp has looked for those two tiles earlier."""
    assert "k0" in explore(*programs([6], 2, 1, 1)) or "k1" in explore(*programs([6], 2, 1, 1))
