"""CPU: no product of the linear attention's tensor-core kernel rests on another one's being over by the time it runs.

Products of one thread are ordered among themselves only where they share an accumulator.  Everywhere else what a product writes (its accumulator) must not be what an earlier one still
reads or writes, and what it reads must not be what an earlier one still writes, unless a wait in front of it says that the earlier one is over: on the barrier of a commit behind it, or on one
of another role that itself has waited for such a barrier.  The thread's waits, products and commits are read from the source, in order, and played over several stretches."""
import os
import re

from tests.test_barrier_order import CSRC

STRETCHES = 6
#: what the other roles have waited for in front of an arrival: (barrier, of how many uses ago)
BEHIND = {"s_ready": ("x_done", 1), "f_ready": ("f_free", 2), "o_free": ("o_done", 0), "p_ready": ("p0_done", 0), "o_scaled": ("in_done", 0)}


def issued():
    """Waits, products and commits of the thread that issues products, as they stand in the source."""
    text = open(os.path.join(CSRC, "linear_tc.cu")).read()
    text = re.search(r"warp == WARP_MMA\)(.*?)warp == WARP_STORE\)", text, re.S)[1]
    found = []
    for wait, commit, to, left in re.findall(r"(?:wait_mma|mbar_wait)\(&sh\.(\w+)|commit\(&sh\.(\w+)|mma_bf16\w*\(tmem \+ (\w), (\w+)", text):
        found.append(("wait", wait) if wait else ("commit", commit) if commit else ("product", to, left))
    return found


def test_the_source_is_what_is_played():
    assert issued() == [
        ("wait", "full"), ("wait", "full"), ("wait", "o_done"), ("product", "P", "ad"), ("commit", "p0_done"), ("wait", "s_ready"),
        ("wait", "o_free"), ("product", "O", "ad"), ("product", "O", "ad"), ("commit", "in_done"), ("commit", "empty"),      # once, between the second and third part of X
        ("wait", "f_ready"), ("product", "X", "at"), ("product", "X", "at"), ("product", "X", "at"), ("commit", "f_free"),
        ("commit", "x_done"), ("commit", "empty"), ("wait", "p_ready"), ("wait", "o_scaled"), ("wait", "full"), ("product", "O", "at"), ("product", "O", "at"), ("commit", "o_done"), ("commit", "empty"),
        ("wait", "empty")]


def played():
    """(what, reads, writes) of products, waits and commits over the stretches; operands in tensor memory and what warps write into shared memory.  Tiles of the ring are fetched
    behind a commit of all that reads them."""
    ops, has_wait = [], ("wait", "o_done") in issued()
    for n in range(STRETCHES):
        if n and has_wait:
            ops.append(("wait", "o_done", n - 1))
        ops += [("product", "P0", (), "P"), ("commit", "p0_done", n), ("wait", "s_ready", n)]
        for q in range(4):
            if q == 2:
                if n:
                    ops.append(("wait", "o_free", n - 1))
                ops += [("product", "in", ("state",), "O"), ("commit", "in_done", n)]
            ops += [("wait", "f_ready", 4 * n + q), ("product", "X", ("F%d" % (q & 1),), "X"), ("commit", "f_free", 4 * n + q)]
        ops += [("commit", "x_done", n), ("wait", "p_ready", n), ("wait", "o_scaled", n), ("product", "Pc", ("P",), "O"), ("commit", "o_done", n)]
    return ops


def test_products_of_different_accumulators_wait_for_one_another():
    committed, open_, seen = {}, [], 0      # barrier and use -> products in front of the commit; (index, name, reads, writes) of products that may still run
    for op in played():
        if op[0] == "commit":
            committed[op[1:]] = seen
        elif op[0] == "wait":
            bar, k = op[1:]
            if bar in BEHIND:
                bar, k = BEHIND[bar][0], k - BEHIND[bar][1]
            if k >= 0:
                open_ = [p for p in open_ if p[0] >= committed[bar, k]]
        else:
            _, name, reads, writes = op
            for _, other, r, w in open_:
                assert w == writes or not (writes in r or w in reads), (other, name)
            open_.append((seen, name, reads, writes))
            seen += 1
