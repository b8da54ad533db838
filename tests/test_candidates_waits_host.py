"""The barriers between the roles of tree attention's tensor-core kernel: in every
order in which the roles' steps may follow one another, each wait ends.

A wait asks whether the phase of one parity is complete, so a barrier that
completes two phases while a role has not asked yet holds that role for good (in
the kernel: until the bounded wait runs out).  The roles are modelled as lists of
waits, arrivals and commits in the kernel's order; for head sizes above 128, which
barrier the products of an output half wait for, and whether that half's lane
arrives on it, are read from the source.
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


def roles(form, n_tiles, sized, own_weights=True, both_arrive=True):
    """The roles' steps, and how many arrivals complete a barrier's phase (1 if not given).  Each lane has two warps,
    one with query rows and one without; `sized`: the tiles whose rows of V get scales of their own."""
    alternating, wide = form == "alternating lanes", form == "columns above 128"
    shared = alternating or wide
    halves = 2 if wide or form == "two lanes" else 1
    ahead = 2 if alternating else 1
    of_lane = (lambda t: (t >> 1) & 1) if alternating else (lambda t: t & 1)
    of_scores = (lambda t: (t >> 1) & 1) if shared else (lambda t: t & 1)
    products = []
    for t in range(min(ahead, n_tiles)):
        products.append(("wait", f"k{t} sized", 0))
        products += [("commit", f"s{t if shared else x}") for x in range(1 if shared else halves)]
        products.append(("commit", f"k{t} free"))
    outputs = 0
    for t in range(n_tiles):
        for i in range(halves):
            x = t & 1 if alternating else i
            products += [("wait", f"p{x if own_weights else 0}", of_lane(t)), ("wait", f"v{t & 1} sized", (t >> 1) & 1),
                         ("wait", "o free", (outputs - 1) & 1), ("commit", f"o{x}")]
            outputs += 1
            if i == halves - 1:
                products.append(("commit", f"v{t & 1} free"))
            then = t + ahead
            if then < n_tiles and not (wide and i == 1):
                if i == 0:
                    products.append(("wait", f"k{then & 1} sized", (then >> 1) & 1))
                products.append(("commit", f"s{then & 1 if wide else x}"))
                if wide or i == halves - 1:
                    products.append(("commit", f"k{then & 1} free"))
    loads, sizes = [], {"k": [], "v": []}
    for t in range(n_tiles):
        for kind in "kv":
            if t >= 2:
                loads.append(("wait", f"{kind}{t & 1} free", ((t >> 1) - 1) & 1))
            loads.append(("arrive", f"{kind}{t & 1}"))
            sizes[kind] += [("wait", f"{kind}{t & 1}", (t >> 1) & 1), ("arrive", f"{kind}{t & 1} sized")]
    lanes = []
    for x in range(2 if shared or halves == 2 else 1):
        for has_rows in (True, False):
            lane = []
            for t in range(x if alternating else 0, n_tiles, 2 if alternating else 1):
                lane.append(("wait", f"s{t & 1 if wide else x}", of_scores(t)))
                if has_rows:
                    lane.append(("wait", f"v{t & 1}", (t >> 1) & 1))
                    if t in sized:
                        lane.append(("wait", f"v{t & 1} sized", (t >> 1) & 1))
                if x == 0 or both_arrive:
                    lane.append(("arrive", f"p{x}"))
                lane += [("wait", f"o{x}", of_lane(t)), ("arrive", "o free")]
            lanes.append(lane)
    return [products, loads, *sizes.values(), *lanes], {"p0": 2, "p1": 2, "o free": 2}


def held(model):
    """States in which no role can go on and not all have ended, over all orders."""
    todo_of, arrivals = model
    names = sorted({step[1] for role in todo_of for step in role})
    at, needs = {name: i for i, name in enumerate(names)}, [arrivals.get(name, 1) for name in names]
    start = ((0,) * len(todo_of), (0,) * len(names), ())  # steps done, arrivals, commits under way
    seen, todo, stuck = {start}, [start], []

    def arrived(counts, name):
        i = at[name]
        return counts[:i] + (counts[i] + 1,) + counts[i + 1:]

    while todo:
        done, counts, commits = todo.pop()
        after = [(done, arrived(counts, commits[0]), commits[1:])] if commits else []
        for r, role in enumerate(todo_of):
            if done[r] == len(role):
                continue
            kind, name, *parity = role[done[r]]
            further = done[:r] + (done[r] + 1,) + done[r + 1:]
            if kind == "commit":
                after.append((further, counts, commits + (name,)))
            elif kind == "arrive":
                after.append((further, arrived(counts, name), commits))
            elif (counts[at[name]] // needs[at[name]]) & 1 != parity[0]:
                after.append((further, counts, commits))
        if not after and any(d < len(role) for d, role in zip(done, todo_of)):
            stuck.append(done)
        for state in after:
            if state not in seen:
                seen.add(state)
                todo.append(state)
    return stuck


@pytest.mark.parametrize("form", ["one lane", "two lanes", "alternating lanes", "columns above 128"])
@pytest.mark.parametrize("n_tiles,sized", [(1, ()), (2, (1,)), (4, (0, 1, 2, 3)), (4, (1, 2))])
def test_no_order_of_the_roles_holds_one(form, n_tiles, sized):
    assert held(roles(form, n_tiles, sized, *kernel_order())) == []


def test_the_model_sees_an_overtaken_wait():
    assert held(roles("columns above 128", 4, (), False, False)) != []
