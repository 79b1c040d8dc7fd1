"""GPU: the operators around the layer with each option by itself, and scans whose sequences are cut into parts in one direction only or differently in both; against the
definitions in 64 bits, with the tolerances of test_block_gpu.py."""
import pytest
import torch

import mogankda_b200 as mk
from tests.test_block_gpu import DTYPES, conv_reference, differentiate, near, rand, scan_leaves, scan_reference

pytestmark = pytest.mark.gpu
SCAN_ARGS = ("x", "dt", "A", "B", "C", "D", "z", "bias")


def against_scan_reference(lv, ups, softplus, cu=None, last=True):
    mine = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}
    wide = {n: t.double().requires_grad_(True) for n, t in lv.items()}
    cu_t = None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")
    outs, grads = differentiate(lambda: mk.selective_scan(*(mine.get(n) for n in SCAN_ARGS), dt_softplus=softplus, initial_state=mine.get("h0"), output_final_state=last,
                                                          cu_seqlens=cu_t), mine, [u.cuda() for u in ups], list(lv))
    routs, rgrads = differentiate(lambda: scan_reference(*(wide.get(n) for n in SCAN_ARGS), softplus, wide.get("h0"), cu, last), wide, [u.double() for u in ups], list(lv))
    for n, a, b in zip(["y", "last"][:len(outs)] + ["d" + n for n in lv], outs + grads, routs + rgrads):
        near(n, a.cpu(), b)


# ---- options, each by itself -------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("option", ["bias", "silu", "state", "last"])
def test_conv_options(option, dtype):
    gen = torch.Generator().manual_seed(55)
    T, D, cu = 61, 72, (0, 2, 2, 40, 58)
    lv = dict(x=rand(gen, 1, T, D).to(dtype), w=rand(gen, D, 4) * 0.5)
    if option == "bias":
        lv["bias"] = rand(gen, D)
    if option == "state":
        lv["state"] = rand(gen, 4, 3, D).to(dtype)
    ups, last = [rand(gen, 1, T, D).to(dtype), rand(gen, 4, 3, D).to(dtype)], option == "last"
    mine = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}
    wide = {n: t.double().requires_grad_(True) for n, t in lv.items()}
    outs, grads = differentiate(lambda: mk.causal_conv1d(mine["x"], mine["w"], mine.get("bias"), activation="silu" if option == "silu" else None, initial_state=mine.get("state"),
                                                         output_final_state=last, cu_seqlens=torch.tensor(cu, device="cuda")), mine, [u.cuda() for u in ups], list(lv))
    routs, rgrads = differentiate(lambda: conv_reference(wide["x"], wide["w"], wide.get("bias"), option == "silu", wide.get("state"), cu, last), wide,
                                  [u.double() for u in ups], list(lv))
    for n, a, b in zip((["y", "last"] if last else ["y"]) + ["d" + n for n in lv], outs + grads, routs + rgrads):
        near(n, a.cpu(), b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("option", ["D", "z", "bias", "softplus", "h0", "last", "D z", "bias softplus", "z h0"])
def test_scan_options(option, dtype):
    gen = torch.Generator().manual_seed(56)
    T, D, N, cu = 75, 40, 16, (0, 20, 20, 53, 70)
    full = scan_leaves(gen, 1, T, D, N, 2, cu, dtype, True)
    lv = {n: t for n, t in full.items() if n in ("x", "A", "B", "C") or n in option.split()}
    softplus = "softplus" in option
    if "bias" in lv and not softplus:
        lv["bias"] = lv["bias"].exp()                      # time passes forwards: d = dt + bias > 0
    lv["dt"] = full["dt"] if softplus else scan_leaves(gen, 1, T, D, N, 2, cu, dtype, False)["dt"]
    if softplus and "bias" not in lv:
        lv["dt"] = lv["dt"] - 3
    against_scan_reference(lv, [rand(gen, 1, T, D).to(dtype), rand(gen, 4, D, N)], softplus, cu, last=option == "last")


# ---- parts -------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [
    (1, 450, 2500, 16, 1, None),                           # 79 blocks: whole forward, three parts backward
    (1, 700, 512, 64, 2, (0, 650, 700)),                   # 64 blocks: whole and four parts
    (1, 1300, 512, 30, 1, (0, 1200, 1300)),                # parts of 320 and 192 tokens
    (1, 1500, 512, 16, 1, (0, 1200, 1206, 1206, 1499)),    # parts of 192 and 128 tokens
], ids=str)
def test_scan_with_other_parts_in_each_direction(shape, dtype):
    B, T, D, N, G, cu = shape
    gen = torch.Generator().manual_seed(57)
    lv = scan_leaves(gen, B, T, D, N, G, cu, dtype, True)
    seqs = B if cu is None else len(cu) - 1
    against_scan_reference(lv, [rand(gen, B, T, D).to(dtype), rand(gen, seqs, D, N)], True, cu)
