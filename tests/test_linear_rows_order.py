"""CPU: the waits of the linear attention's tensor-core kernel that stand beside those of test_linear_order.py: pairs of a stretch wait for the product that reads the last stretch's, and in
fp16 the eight warps of the rows wait for one another's largest values in front of a row's scale.  Nobody else has a part in the latter."""
import os
import re

import pytest

from tests.test_barrier_order import CSRC
from tests.test_linear_order import linear_kernel


def with_waits(fp32, half):
    r = linear_kernel(False, fp32, False)
    for name, ops in r.agents.items():
        new = []
        for op in ops:
            if name == "products" and op[0] == "arrive" and op[1][0] == "p0_done":
                n = sum(o[0] == "arrive" and o[1][0] == "p0_done" for o in new)
                if n:
                    new.append(("wait", *r.at("o_done", n - 1)))
            new.append(op)
            if half and name.startswith("rows") and op[0] == "wait" and op[1][0] == "p0_done":
                n = sum(o[0] == "wait" and o[1][0] == "p0_done" for o in new) - 1
                new += [("arrive", r.at("e_ready", n)[0], None), ("wait", *r.at("e_ready", n))]
        ops[:] = new
    return r


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("fp32", [False, True])
def test_waits_with_rows_that_wait_for_one_another(fp32, half):
    assert not with_waits(fp32, half).late_waits()


def test_only_rows_arrive_for_their_scales():
    text = open(os.path.join(CSRC, "linear_tc.cu")).read()
    rows = re.search(r"pairs and output: row i(.*?)f c, transposed", text, re.S)[1]
    kernel = text[text.index("linear_tc_kernel(const"):]
    assert len(re.findall(r"sh\.e_ready\[n", rows)) == len(re.findall(r"sh\.e_ready\[n", kernel)) == 2
