"""The prompt attention kernels' ring of direct-to-LDS loads, in the built code:
its barriers found without looking at the waits before them, so that a wait that
is missing shows as well as one that waits for too little.

A kernel has one reduction over the workgroup (whether a block holds values that
are not finite), the only place that writes LDS by ds_or: the barriers around it
publish no load. Every other barrier does. At such a barrier the 16-bit kernels
may have what was requested since the one before outstanding, the f32 kernels,
whose ring has two blocks, nothing; and no load may outlive the wavefront."""
import re

import pytest

from test_direct_lds_waits import VM
from test_serving_built import tile_kernels  # noqa: F401 (a fixture)


def ring(code):
    """The code without the reduction's barriers, and the number of those that are left."""
    at = [i for i, ins in enumerate(code) if ins[1].startswith("ds_or_")]
    assert len(at) == 1
    barriers = [i for i, ins in enumerate(code) if ins[1] == "s_barrier"]
    inside = {max(i for i in barriers if i < at[0]), *[i for i in barriers if i > at[0]][:2]}
    kept = [(ins[0], "s_nop", "0", None) if i in inside else ins for i, ins in enumerate(code)]
    return kept, len(barriers) - len(inside)


def outstanding(code, slack):
    """Addresses of the barriers that some path reaches with a load into LDS
    outstanding that has passed `slack` barriers already, and of the ends it
    reaches with any."""
    index = {ins[0]: i for i, ins in enumerate(code)}
    bad, seen, todo = set(), set(), [(0, "")]
    while todo:
        i, queue = todo.pop()  # queue, oldest first: the barriers a load into LDS has passed, w another access
        while i < len(code) and (i, queue) not in seen:
            seen.add((i, queue))
            address, op, operands, target = code[i]
            if "load_lds" in op:
                queue += "0"
            elif VM.match(op):
                queue += "w"
            elif op == "s_waitcnt" and (n := re.search(r"vmcnt\((\d+)\)", operands)):
                queue = queue[max(0, len(queue) - int(n[1])):]
            elif op == "s_barrier":
                if any(q != "w" and int(q) >= slack for q in queue):
                    bad.add(address)
                queue = queue.replace("1", "2").replace("0", "1")
            elif op == "s_endpgm":
                if queue.strip("w"):
                    bad.add(address)
                break
            queue = queue[-64:]  # vmcnt counts no further
            if target is not None:
                if op == "s_branch":
                    i = index[target]
                    continue
                todo.append((index[target], queue))
            i += 1
    return bad


def is_f32(name):
    return "attention_tiles_kernelIf" in name


def slack_of(name):
    return 0 if is_f32(name) else 1


def test_no_ring_load_passes_its_barrier(tile_kernels):  # noqa: F811
    for name, code in tile_kernels.items():
        kept, left = ring(code)
        # one behind the zeros, before the loop (16 bits only), in it, behind it
        assert left == (3 if is_f32(name) else 4), name
        assert sum("load_lds" in ins[1] for ins in kept) > 0, name
        assert outstanding(kept, slack_of(name)) == set(), name


def test_a_ring_without_one_of_its_waits_is_found(tile_kernels):  # noqa: F811
    """Each wait for vector memory right before a barrier, left out or one short, in
    a copy of the listing. (The kernels that look every row's page up wait for these
    lookups before each load, which may cover the loop's own wait: that one alone
    need not be missed there.)"""
    for name, code in tile_kernels.items():
        kept, left = ring(code)
        waits = [i for i, ins in enumerate(kept)
                 if ins[1] == "s_waitcnt" and "vmcnt" in ins[2] and kept[i + 1][1] == "s_barrier"]
        assert len(waits) == left - 1, name  # (not behind the zeros)
        unseen = set()
        for i in waits:
            count = int(re.search(r"vmcnt\((\d+)\)", kept[i][2])[1])
            for text in ("lgkmcnt(0)", f"vmcnt({count + 1}) lgkmcnt(0)"):
                less = kept[:i] + [(kept[i][0], "s_waitcnt", text, None)] + kept[i + 1:]
                if not outstanding(less, slack_of(name)):
                    unseen.add(hex(kept[i][0]))
        by_page = "ELb0EEE" in name
        assert len(unseen) <= by_page, (name, unseen)


@pytest.mark.parametrize("slack", [0, 1])
def test_the_walk_counts_barriers_and_ends(slack):
    load, barrier, end = ("global_load_lds_dwordx4", ""), ("s_barrier", ""), ("s_endpgm", "")

    def stream(*ops):
        return [(4 * i, o[0], o[1], o[2] if len(o) > 2 else None) for i, o in enumerate(ops)]

    wait = lambda n: ("s_waitcnt", f"vmcnt({n}) lgkmcnt(0)")
    assert outstanding(stream(load, wait(0), barrier, end), slack) == set()
    assert outstanding(stream(load, barrier, wait(0), end), slack) == (set() if slack else {4})
    assert outstanding(stream(load, barrier, barrier, wait(0), end), slack) == ({8} if slack else {4, 8})
    assert outstanding(stream(load, end), slack) == {4}
    assert outstanding(stream(load, barrier, load, wait(1), barrier, wait(0), end), slack) == (set() if slack else {4, 16})
    # round a loop: what the first round requested reaches the second and third round's barrier
    assert outstanding(stream(barrier, load, ("s_cbranch_scc1", "", 0), wait(0), end), slack) == {0}
