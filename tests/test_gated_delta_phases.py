"""The barriers of the gated delta rule's kernels, as a model on the CPU: which warps arrive and wait where, and every order in which they can run.

A wait on an mbarrier knows the parity of a phase, not its number.  A warp that comes to its wait for phase n when phase n + 1 is complete too sees the parity of phase n
again, waits for a phase that does not come, and gives up: so nobody may complete the phase behind the one that somebody still has to see.  The search goes through
all interleavings of two compute warps (of each kind), the warp that issues the products and the one that has the loads, over a few chunks."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kda_b200", "csrc")


def search(counts, warps):
    """counts: arrivals per phase of each barrier; warps: lists of ("a", barrier) and ("w", barrier, phase).  What goes wrong in some order, or None."""
    names = sorted(counts)
    at = {b: i for i, b in enumerate(names)}
    start = (tuple(0 for _ in warps), tuple((0, 0) for _ in names))      # of each barrier: complete phases, arrivals of the open one
    seen, todo = {start}, [start]
    while todo:
        pcs, bars = todo.pop()
        moved = False
        for i, warp in enumerate(warps):
            if pcs[i] == len(warp):
                continue
            op = warp[pcs[i]]
            done, here = bars[at[op[1]]]
            if op[0] == "w":
                if done > op[2] + 1:
                    return f"warp {i} missed phase {op[2]} of {op[1]}"
                if done <= op[2]:
                    continue
                new = bars
            else:
                here += 1
                done, here = (done + 1, 0) if here == counts[op[1]] else (done, here)
                new = bars[:at[op[1]]] + ((done, here),) + bars[at[op[1]] + 1:]
            moved = True
            state = (pcs[:i] + (pcs[i] + 1,) + pcs[i + 1:], new)
            if state not in seen:
                seen.add(state)
                todo.append(state)
        if not moved and any(pc != len(w) for pc, w in zip(pcs, warps)):
            return "nobody can go on"
    return None


FIRST = ["bwd_scan", "scan_t"]      # walks whose loading warp waits for oReady in front of the chunk's last load; in the others it takes part in that barrier


def walk(kind, chunks, closed):
    """The four walks; `closed`: the warp with the loads takes part in the phases of oReady that it waits for."""
    A = lambda b: ("a", b)      # noqa: E731
    W = lambda b, n: ("w", b, n)      # noqa: E731
    full, free = (lambda i: W(f"fullA{i & 1}", i >> 1)), (lambda i: W(f"freeA{i & 1}", i >> 1))
    krow, orow, issue, loads = [], [], [], []
    for i in range(chunks):
        if kind == "scan":
            krow += [full(i), A("hReady"), W("fullB", i), W("m1", i), A("rReady"), W("m2", i), A("uReady"), W("m3", i)]
            orow += [full(i), A("hReady"), W("m1", i), W("m2", i), A("oReady"), W("m3", i)]
        elif kind == "scan_t":
            krow += [full(i), A("hReady"), W("m1", i), A("rReady"), W("m2", i), A("uReady"), A("oReady"), W("m3", i)]
        else:
            krow += [full(i), A("hReady")] + ([W("fullB", i)] if kind == "bwd_scan" else []) + [A("dReady"), W("m1", i), A("xReady"), W("m2", i), A("yReady"), A("oReady"), W("m3", i)]
        second = [W("rReady", i)] if "bwd" not in kind else [W("dReady", i), W("xReady", i)]
        issue += [full(i), W("hReady", i), A("m1"), W("fullB", i), *second, A("m2"), A("freeB"), W("uReady" if "bwd" not in kind else "yReady", i), A("m3"), A(f"freeA{i & 1}")]
    loads += [A("oReady")] * closed + [A("fullA0"), A("fullB")] + [A("fullA1")] * (chunks > 1)
    for i in range(chunks):
        seen = [W("oReady", i)] + [A("oReady")] * closed
        more_b = [W("freeB", i), A("fullB")] if i + 1 < chunks else []
        if kind == "scan":
            loads += [W("uReady", i)]
        loads += (seen + more_b if kind in FIRST else more_b + seen) + ([free(i), A(f"fullA{i & 1}")] if i + 2 < chunks else [])
    compute = [krow, krow] + ([orow, orow] if kind == "scan" else [])
    counts = {op[1]: 1 for w in (issue, loads, *compute) for op in w}
    for b in counts:
        per = sum(any(op == ("a", b) for op in w) for w in compute)
        counts[b] = max(1, per) + (closed if b == "oReady" else 0)
    return counts, [*compute, issue, loads]


def gradients(tiles, norm, closed):
    A, W = (lambda b: ("a", b)), (lambda b, n: ("w", b, n))      # noqa: E731
    full = lambda n: W(f"fullA{n & 1}", n >> 1)      # noqa: E731
    compute, issue, loads = [], [], [A("ready"), A("done")] * closed + [A("fullA0"), A("fullB")]
    for n in range(tiles):
        compute += [full(n), W("fullB", n), A("ready"), A("used"), W("mS", n), A("eReady"), W("mY", n), W("mD", n), A("done")] + ([W("done", n)] if norm else [])
        issue += [full(n), W("fullB", n), W("ready", n), A("mS"), A("mY"), W("eReady", n), A("mD")]
        loads += [W("ready", n)] + [A("ready")] * closed + ([A(f"fullA{n + 1 & 1}"), W("mY", n), W("used", n), A("fullB")] if n + 1 < tiles else []) + [W("done", n)] + [A("done")] * closed
    compute += [A("ready")]
    loads += [W("ready", tiles)]
    counts = {op[1]: 2 if op[1] in ("ready", "used", "eReady", "done") else 1 for w in (compute, issue, loads) for op in w}
    counts["ready"] += closed
    counts["done"] += closed
    return counts, [compute, compute, issue, loads]


@pytest.mark.parametrize("chunks", [1, 2, 3, 5])
@pytest.mark.parametrize("kind", ["scan", "scan_t", "bwd_scan", "bwd_scan_t"])
def test_walks(kind, chunks):
    assert search(*walk(kind, chunks, closed=kind not in FIRST)) is None


@pytest.mark.parametrize("tiles", [1, 2, 3, 5])
@pytest.mark.parametrize("norm", [False, True])
def test_gradients(tiles, norm):
    assert search(*gradients(tiles, norm, closed=True)) is None


def test_the_model_finds_a_missed_phase():
    """Without the loading warp's part: the chunk behind needs nothing of it but the load that it asked for before its wait."""
    for kind in ("scan", "bwd_scan_t"):
        assert "missed" in search(*walk(kind, 3, closed=False))
    assert "missed" in search(*gradients(3, False, closed=False))


def source(file):
    with open(os.path.join(CSRC, file)) as f:
        return f.read()


@pytest.mark.parametrize("file,barrier,count", [("delta_scan.cu", "oReady", "BULK ? 5 : 4"), ("delta_bwd_scan_t.cu", "oReady", "CW + 1"), ("delta_bwd_main.cu", "ready", "CW + 1"),
                                                ("delta_bwd_main.cu", "done", "CW + 1")])
def test_the_kernels_take_part(file, barrier, count):
    text = source(file)
    assert f"mbar_init(&s.{barrier}, {count});" in text
    assert len(re.findall(rf"mbar_arrive\(&s\.{barrier}\);", text)) == 2      # in front of the loop, and behind the wait


@pytest.mark.parametrize("kind", FIRST)
def test_the_kernels_wait_first(kind):
    text = source(f"delta_{kind}.cu")
    assert text.index("mbar_wait(&s.oReady, i & 1)") < text.index("loadB(i + 1);")
