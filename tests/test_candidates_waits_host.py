"""The barriers between the roles of tree attention's tensor-core kernel for head
sizes above 128: in every order in which the roles' steps may follow one another,
each wait ends.

A wait asks whether the phase of one parity is complete, so a barrier that
completes two phases while a role has not asked yet holds that role for good (in
the kernel: until the bounded wait runs out).  The roles are modelled as lists of
waits, arrivals and commits in the kernel's order; which barrier the products of
an output half wait for, and whether that half's lane arrives on it, are read from
the source.
"""
import re
from pathlib import Path

import pytest

SOURCE = (Path(__file__).resolve().parents[1] / "gncx_b200" / "csrc" / "tree_tc.cu").read_text()


def kernel_order():
    waits_for = re.search(r"wait_all3\(&pfull\[([^\]]*)\], phase\(t\)", SOURCE).group(1)
    assert waits_for in ("x", "WIDE ? 0 : x")
    arrives = re.search(r"\n *(if \(writes\) )?mbar_arrive\(&pfull\[x\]\);", SOURCE)
    return waits_for == "x", arrives.group(1) is None


def roles(n_tiles, own_weights, both_arrive):
    products = [("wait", "k0", 0), ("commit", "s0"), ("commit", "k0 free")]
    outputs = 0
    for t in range(n_tiles):
        b = t & 1
        for half in range(2):
            products += [("wait", f"p{half if own_weights else 0}", t & 1), ("wait", f"v{b}", (t >> 1) & 1),
                         ("wait", "o free", (outputs - 1) & 1), ("commit", f"o{half}")]
            outputs += 1
            if half == 1:
                products.append(("commit", f"v{b} free"))
            elif t + 1 < n_tiles:
                products += [("wait", f"k{1 - b}", ((t + 1) >> 1) & 1), ("commit", f"s{1 - b}"), ("commit", f"k{1 - b} free")]
    loads = []
    for t in range(n_tiles):
        for kind in "kv":
            if t >= 2:
                loads.append(("wait", f"{kind}{t & 1} free", ((t >> 1) - 1) & 1))
            loads.append(("arrive", f"{kind}{t & 1}"))
    lanes = [[], []]
    for x, lane in enumerate(lanes):
        for t in range(n_tiles):
            lane += [("wait", f"s{t & 1}", (t >> 1) & 1), ("wait", f"v{t & 1}", (t >> 1) & 1)]
            if x == 0 or both_arrive:
                lane.append(("arrive", f"p{x}"))
            lane += [("wait", f"o{x}", t & 1), ("arrive", "o free")]
    return [products, loads, *lanes]


def held(n_tiles, own_weights, both_arrive):
    """States in which no role can go on and not all have ended, over all orders."""
    todo_of = roles(n_tiles, own_weights, both_arrive)
    names = sorted({step[1] for role in todo_of for step in role})
    at = {name: i for i, name in enumerate(names)}
    start = ((0,) * len(todo_of), (0,) * len(names), ())  # steps done, phases completed, commits under way
    seen, todo, stuck = {start}, [start], []

    def completed(phases, name):
        return tuple(p + (i == at[name]) for i, p in enumerate(phases))

    while todo:
        done, phases, commits = todo.pop()
        after = [(done, completed(phases, commits[0]), commits[1:])] if commits else []
        for r, role in enumerate(todo_of):
            if done[r] == len(role):
                continue
            step, further = role[done[r]], done[:r] + (done[r] + 1,) + done[r + 1:]
            if step[0] == "commit":
                after.append((further, phases, commits + (step[1],)))
            elif step[0] == "arrive":
                after.append((further, completed(phases, step[1]), commits))
            elif phases[at[step[1]]] & 1 != step[2]:
                after.append((further, phases, commits))
        if not after and any(d < len(role) for d, role in zip(done, todo_of)):
            stuck.append(done)
        for state in after:
            if state not in seen:
                seen.add(state)
                todo.append(state)
    return stuck


@pytest.mark.parametrize("n_tiles", [1, 2, 3, 6, 7])
def test_no_order_of_the_roles_holds_one(n_tiles):
    assert held(n_tiles, *kernel_order()) == []


def test_the_model_sees_an_overtaken_wait():
    assert held(6, False, False) != []
