"""GPU: the operators around the layer at the far ends of their arguments' values, with each option by itself, and where sequences are cut into parts in one direction
only or differently in both; against the definitions in 64 bits, with the tolerances of test_block_gpu.py."""
import pytest
import torch

import mogankda_b200 as mk
from tests.test_block_gpu import DTYPES, call_scan, conv_reference, differentiate, near, rand, scan_leaves, scan_reference

pytestmark = pytest.mark.gpu
SCAN_ARGS = ("x", "dt", "A", "B", "C", "D", "z", "bias")


def against_scan_reference(lv, ups, softplus, cu=None, last=True, only=None):
    """Results and gradients, all of them or those named."""
    mine = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}
    wide = {n: t.double().requires_grad_(True) for n, t in lv.items()}
    cu_t = None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")
    outs, grads = differentiate(lambda: mk.selective_scan(*(mine.get(n) for n in SCAN_ARGS), dt_softplus=softplus, initial_state=mine.get("h0"), output_final_state=last,
                                                          cu_seqlens=cu_t), mine, [u.cuda() for u in ups], list(lv))
    routs, rgrads = differentiate(lambda: scan_reference(*(wide.get(n) for n in SCAN_ARGS), softplus, wide.get("h0"), cu, last), wide, [u.double() for u in ups], list(lv))
    for n, a, b in zip(["y", "last"][:len(outs)] + ["d" + n for n in lv], outs + grads, routs + rgrads):
        if only is None or n in only:
            near(n, a.cpu(), b)


# ---- values ------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("T,D,N", [(33, 40, 16), (64, 24, 5), (70, 9, 64), (900, 8, 16)])
def test_scan_with_a_decay_rate_at_the_end_of_its_range(T, D, N):
    """A = -3e38 times log2 e is no fp32 number.  It leaves nothing of a state, and the tokens behind a sequence's end, for which no time passes, leave the state alone."""
    gen = torch.Generator().manual_seed(51)
    lv = scan_leaves(gen, 2, T, D, N, 1, None, torch.float32, True)
    lv["A"][3], lv["A"][5, 0] = -3e38, torch.finfo(torch.float32).min
    against_scan_reference(lv, [rand(gen, 2, T, D), rand(gen, 2, D, N)], True)


@pytest.mark.parametrize("T", [1, 33, 900])
def test_scan_with_an_infinite_decay_rate(T):
    """exp(-inf) = 0: the state is what the last token brought."""
    gen = torch.Generator().manual_seed(52)
    lv = scan_leaves(gen, 2, T, 12, 16, 1, None, torch.float32, True)
    lv["A"][2] = -float("inf")
    with torch.no_grad():
        y, end = call_scan({n: t.cuda() for n, t in lv.items()}, None, True)
        ry, rend = scan_reference(*(lv[n].double() for n in SCAN_ARGS), True, lv["h0"].double(), None, True)
        state = lv["h0"].cuda()
        sy = mk.selective_scan_step(lv["x"][:, 0].cuda(), lv["dt"][:, 0].cuda(), lv["A"].cuda(), lv["B"][:, 0].cuda(), lv["C"][:, 0].cuda(), state, lv["D"].cuda(),
                                    lv["z"][:, 0].cuda(), lv["bias"].cuda(), dt_softplus=True)
    near("y", y.cpu(), ry)
    near("end", end.cpu(), rend)
    near("step", sy.cpu(), ry[:, 0])


def alike(name, got, want):
    """The same places are NaN, the same infinite with the same sign, and the others are near."""
    got, want = got.cpu(), want.float()
    assert torch.equal(got.isnan(), want.isnan()), f"{name}: NaN in other places"
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()]), f"{name}: infinities"
    ok = torch.isfinite(want)
    near(name, got[ok], want[ok].double())


@pytest.mark.parametrize("N", [1, 5, 12, 16, 20, 50])
@pytest.mark.parametrize("what", ["x", "dt"])
def test_scan_of_infinite_values(N, what):
    """An infinite x (or dt) makes y infinite, not NaN, whatever the number of states: the states that fill up a channel's lanes have no part in it."""
    gen = torch.Generator().manual_seed(53)
    T, D = 37, 20
    lv = scan_leaves(gen, 1, T, D, N, 1, None, torch.float32, False)
    lv["x"], lv["B"], lv["C"] = lv["x"].abs() + 0.1, lv["B"].abs() + 0.1, lv["C"].abs() + 0.1
    lv[what][0, 20, 7] = float("inf")
    with torch.no_grad():
        y, end = mk.selective_scan(*(lv[n].cuda() for n in SCAN_ARGS[:5]), output_final_state=True)
        ry, rend = scan_reference(*(lv[n].double() for n in SCAN_ARGS[:5]), last=True)
        before = torch.rand(8, D, N, generator=gen)
        rows = slice(14, 22)                               # a token of each of eight sequences: four of them a thread or one
        ref = scan_reference(*(lv[n][0, rows, None].double() if n in ("x", "dt", "B", "C") else lv[n].double() for n in SCAN_ARGS[:5]), h0=before.double(), last=True)
        for copies in (1, 2000):
            state = before.repeat(copies, 1, 1).cuda()
            args = [lv[n][0, rows].repeat(copies, *(1,) * (lv[n].dim() - 2)).cuda() if n in ("x", "dt", "B", "C") else lv[n].cuda() for n in SCAN_ARGS[:5]]
            sy = mk.selective_scan_step(*args, state)
            alike("step", sy[-8:], ref[0][:, 0])
            alike("state", state[-8:], ref[1])
    assert ry.isinf().any()
    alike("y", y, ry)
    alike("end", end, rend)


@pytest.mark.parametrize("N", [5, 16, 50])
def test_gradients_of_a_scan_that_ends_in_infinite_values(N):
    """An infinite x in a sequence's last token: the gradients that the definition does not form from it stay finite, those behind the end of the tile's tokens included."""
    gen = torch.Generator().manual_seed(54)
    T, D = 37, 12
    lv = scan_leaves(gen, 1, T, D, N, 1, None, torch.float32, False)
    lv["x"][0, -1, 4] = float("inf")
    against_scan_reference(lv, [rand(gen, 1, T, D), rand(gen, 1, D, N)], False, last=False, only=("dx", "dA"))


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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_scan_of_a_long_document_beside_many_short_ones(dtype):
    gen = torch.Generator().manual_seed(58)
    cu = [0, 5]
    for i in range(300):
        cu.append(cu[-1] + (1500 if i == 150 else i % 9))
    T = cu[-1] + 3
    lv = scan_leaves(gen, 1, T, 24, 16, 1, cu, dtype, True)
    against_scan_reference(lv, [rand(gen, 1, T, 24).to(dtype), rand(gen, len(cu) - 1, 24, 16)], True, tuple(cu))
