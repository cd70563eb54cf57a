"""The row sums of residual_norm (cuda-fp8-ampere_b200/csrc/residual_norm.cu), checked on the CPU: a model of a team's
warps, in which every order of their steps is gone through. A sum is a write of the warp's part, a barrier, and a read
of all warps' parts; no part may be written anew before every warp has read it.

Which place a sum takes is read from the source."""
import os
import re

import pytest

from conftest import PKG

SRC = os.path.join(PKG, "csrc", "residual_norm.cu")


def places(post, pre, rounds):
    """The places (of two) that the sums of `rounds` rounds take in the kernel whose CTAs go through many rows."""
    text = open(SRC).read()
    body = text[text.index("residual_norm_vec_kernel("):text.index("residual_norm_kernel(")]
    calls = list(re.finditer(r"team_sum\(s, s_sum\[(\w+)\], p\.team, warp\);\s*(turn \^= 1;)?", body))
    assert len(calls) == 2  # after y's norm, before the next one's
    assert "if (a.post_weight)" in body[:calls[0].start()] and "if (!a.pre_weight) continue;" in body[calls[0].end():calls[1].start()]
    out, turn = [], 0
    for _ in range(rounds):
        for call, on in zip(calls, (post, pre)):
            if on:
                at, flip = call.groups()
                out.append(turn if at == "turn" else int(at))
                turn ^= flip is not None
    return out


def explore(order, warps, barrier_a_round=False):
    """The first write that can meet a read still to come, or None. order: the places of a team's sums, one after another."""
    prog = []
    for k, p in enumerate(order):
        if barrier_a_round:
            prog.append(("bar", None))
        prog += [("write", p, k), ("bar", None)] + [("read", p, k, w) for w in range(warps)]
    passed = [sum(op[0] == "bar" for op in prog[:i]) for i in range(len(prog) + 1)]  # barriers before a step
    start = (0,) * warps
    seen, todo = {start}, [start]
    while todo:
        state = todo.pop()
        for w, i in enumerate(state):
            if i == len(prog):
                continue
            op = prog[i]
            if op[0] == "bar" and any(passed[j] < passed[i] or (passed[j] == passed[i] and prog[j][0] != "bar") for j in state):
                continue  # others have still to come
            if op[0] == "read":
                # the sum whose part that warp wrote last at this place
                last = [o[2] for o in prog[:state[op[3]]] if o[0] == "write" and o[1] == op[1]]
                if not last or last[-1] != op[2]:
                    return "warp %d reads sum %d from warp %d, which holds %s" % (w, op[2], op[3], last[-1:] or "none")
            new = state[:w] + (i + 1,) + state[w + 1:]
            if new not in seen:
                seen.add(new)
                todo.append(new)
    return None


@pytest.mark.parametrize("post, pre", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("warps, rounds", [(2, 4), (3, 3)])
def test_no_sum_is_overwritten_before_it_is_read(post, pre, warps, rounds):
    assert explore(places(post, pre, rounds), warps) is None


def test_the_model_sees_a_place_taken_twice():
    assert explore([1, 1], 2) is not None
    assert explore([0, 1, 0], 2) is None
    assert explore([1, 1], 2, barrier_a_round=True) is None
