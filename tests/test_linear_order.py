"""CPU: no wait of the linear attention's tensor-core kernel rests on timing (test_barrier_order.py has the method), and its roles cannot wait for one another in a ring.

Parts of several lengths, one of them without tokens, go through a block one after the other; ``states`` is the kernel that finds what parts make of nothing."""
import os
import re

import pytest

from tests.test_barrier_order import CSRC, Roles

PARTS = (3, 1, 0, 2, 1)      # stretches of 128 tokens in each


def linear_kernel(states, fp32=False, half=False):
    text = open(os.path.join(CSRC, "linear_tc.cu")).read()
    ring = int(re.search(r"SLOTS = (\d+)", text)[1])
    members = re.search(r"struct Shared \{(.*?)\n\};", text, re.S)[1]
    found = {n: ring if d == "SLOTS" else int(d or 1) for line in re.findall(r"uint64_t ([^;]*);", members) for n, d in re.findall(r"(\w+)(?:\[(\w+)\])?", line)}
    r = Roles(found)
    r.count.update(dict.fromkeys(("p_ready", "f_ready", "s_ready", "o_scaled", "o_free", "o_staged", "e_ready"), 2))      # of the eight warps two, one of which may be late
    per, stretches = (2 if states else 3), [(p, t, c) for p, c in enumerate(PARTS) for t in range(c)]
    load = r.agent("load")
    for tile in range(per * len(stretches)):
        if tile >= ring:
            load[0]("empty", tile - ring)
        load[1]("full", tile)
    wait, arrive = r.agent("products")
    for n in range(len(stretches)):
        a, b, c = n * per, n * per + per - 2, n * per + per - 1
        if not states:
            wait("full", a)
        wait("full", b)
        if not states:
            arrive("p0_done", n)
        wait("s_ready", n)
        for q in range(4):
            wait("f_ready", 4 * n + q)
            arrive("f_free", 4 * n + q)
            if q == 1 and not states:
                if n:
                    wait("o_free", n - 1)
                arrive("in_done", n)
                arrive("empty", a)
        arrive("x_done", n)
        if states:
            arrive("empty", b)
        if not states:
            wait("p_ready", n)
            wait("o_scaled", n)
            wait("full", c)
            arrive("o_done", n)
        if not fp32:
            arrive("empty", c)
    wait("empty", len(stretches) * per - 1)
    if not states:
        wait, arrive = r.agent("store")
        for n in range(len(stretches)):
            wait("o_staged", n)
            arrive("empty", n * per + 1)
            if fp32:                                   # rows of the output lie in the place of c, too
                arrive("empty", n * per + 2)
    for w in range(2):
        if not states:
            wait, arrive = r.agent(f"rows {w}")
            for n in range(len(stretches)):
                if half:
                    wait("e_ready", n)
                wait("p0_done", n)
                arrive("p_ready", n)
                wait("in_done", n)
                arrive("o_scaled", n)
                wait("o_done", n)
                arrive("o_free", n)
                arrive("o_staged", n)
        wait, arrive = r.agent(f"factors {w}")
        for n, (_, t, chunks) in enumerate(stretches):
            wait("full", n * per + per - 1)
            if t == chunks - 1:                        # a short stretch
                wait("full", n * per + per - 2)
            if half and not states:                    # the largest magnitudes of all three tiles
                wait("full", n * per + 1)
                wait("full", n * per)
                arrive("e_ready", n)
            for q in range(4):
                if 4 * n + q >= found["f_free"]:
                    wait("f_free", 4 * n + q - found["f_free"])
                arrive("f_ready", 4 * n + q)
        wait, arrive = r.agent(f"state {w}")
        n = 0
        for chunks in PARTS:
            for t in range(chunks):
                if t:
                    wait("x_done", n - 1)
                arrive("s_ready", n)
                n += 1
            if chunks:
                wait("x_done", n - 1)
    return r


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("states,fp32", [(False, False), (False, True), (True, False)])
def test_waits_of_the_linear_kernel(states, fp32, half):
    assert not linear_kernel(states, fp32, half).late_waits()
