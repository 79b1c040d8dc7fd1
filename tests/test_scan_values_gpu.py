"""GPU: the selective scan at the far ends of its arguments' values, against its definition in 64 bits: what is finite there is near it (tolerances of test_block_gpu.py),
what is infinite there is infinite with the same sign, and nothing else is NaN."""
import pytest
import torch

import mogankda_b200 as mk
from tests.test_block_gpu import near, rand, scan_leaves, scan_reference

pytestmark = pytest.mark.gpu
INF = float("inf")


def alike(name, got, want):
    got, want = got.cpu(), want.float()
    assert torch.equal(got.isnan(), want.isnan()), f"{name}: NaN in other places"
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()]), f"{name}: infinities"
    ok = torch.isfinite(want)
    near(name, got[ok], want[ok].double())


def both(lv, ups=None, softplus=False):
    """(results and gradients of the operator, of the definition), as dicts; gradients of all leaves where ``ups`` holds incoming ones of y and of the final state."""
    sides = []
    for cast, run in ((lambda t: t.cuda(), lambda m: mk.selective_scan(*(m.get(n) for n in ("x", "dt", "A", "B", "C", "D", "z", "bias")), dt_softplus=softplus,
                                                                      initial_state=m.get("h0"), output_final_state=True)),
                      (lambda t: t.double(), lambda m: scan_reference(*(m.get(n) for n in ("x", "dt", "A", "B", "C", "D", "z", "bias")), softplus, m.get("h0"), None, True))):
        m = {n: cast(t).requires_grad_(ups is not None) for n, t in lv.items()}
        y, end = run(m)
        got = dict(y=y, end=end)
        if ups is not None:
            got.update(zip(("d" + n for n in m), torch.autograd.grad((y, end), list(m.values()), [cast(u) for u in ups])))
        sides.append({n: t.detach() for n, t in got.items()})
    return sides


def positive(gen, T, D, N, more=()):
    """Leaves without a sum of terms of both signs."""
    lv = scan_leaves(gen, 1, T, D, N, 1, None, torch.float32, False)
    lv.update((n, scan_leaves(gen, 1, T, D, N, 1, None, torch.float32, True)[n]) for n in more)
    return {n: t if n in ("A", "dt") else t.abs() + 0.1 for n, t in lv.items()}


def step_like(lv, rows, before, copies):
    """One token of each of as many sequences as there are ``rows``, on states ``before``; ``copies`` of them in one call."""
    tok = {n: lv[n][0, rows] for n in ("x", "dt", "B", "C")}
    ref = scan_reference(*(tok[n][:, None].double() if n in tok else lv[n].double() for n in ("x", "dt", "A", "B", "C")), h0=before.double(), last=True)
    state = before.repeat(copies, 1, 1).cuda()
    with torch.no_grad():
        args = [tok[n].repeat(copies, *(1,) * (tok[n].dim() - 1)).cuda() if n in tok else lv[n].cuda() for n in ("x", "dt", "A", "B", "C")]
        y = mk.selective_scan_step(*args, state)
    n = before.shape[0]
    alike("y of a step", y[-n:], ref[0][:, 0])
    alike("state of a step", state[-n:], ref[1])


def test_infinite_values_without_a_skip():
    """Without D there is no term D x, also where x is infinite, nor one D dy in its gradient."""
    gen = torch.Generator().manual_seed(53)
    T, D, N = 32, 20, 16
    lv = positive(gen, T, D, N, more=("z",))
    ups = [rand(gen, 1, T, D).abs() + 0.1, torch.zeros(1, D, N)]
    lv["x"][0, 20, 7] = INF
    got, want = both(lv, ups)
    assert want["y"].isinf().any() and want["dz"].isinf().any()
    for n in ("y", "end", "dz", "dx"):
        alike(n, got[n], want[n])
    before = torch.rand(8, D, N, generator=gen)
    for copies in (1, 2000):
        step_like(lv, slice(14, 22), before, copies)
    lv["x"][0, 20, 7] = 1.0
    ups[0][0, 9, 3] = INF
    got, want = both(lv, ups)
    assert want["dx"].isinf().any()
    alike("dx of an infinite gradient", got["dx"], want["dx"])


@pytest.mark.parametrize("T,D,N", [(33, 40, 16), (64, 24, 5), (70, 9, 64), (900, 8, 16)])
def test_a_decay_rate_at_the_end_of_its_range(T, D, N):
    """A = -3e38 times log2 e is no fp32 number.  It leaves nothing of a state, and the tokens behind a sequence's end, for which no time passes, leave the state alone."""
    gen = torch.Generator().manual_seed(51)
    lv = scan_leaves(gen, 2, T, D, N, 1, None, torch.float32, True)
    lv["A"][3], lv["A"][5, 0] = -3e38, torch.finfo(torch.float32).min
    got, want = both(lv, [rand(gen, 2, T, D), rand(gen, 2, D, N)], True)
    for n in want:
        near(n, got[n].cpu(), want[n])


@pytest.mark.parametrize("T", [1, 33, 900])
def test_an_infinite_decay_rate(T):
    """exp(-inf) = 0: the state is what the last token brought."""
    gen = torch.Generator().manual_seed(52)
    lv = scan_leaves(gen, 2, T, 12, 16, 1, None, torch.float32, True)
    lv["A"][2] = -INF
    got, want = both(lv, softplus=True)
    state = lv["h0"].cuda()
    with torch.no_grad():
        step = mk.selective_scan_step(lv["x"][:, 0].cuda(), lv["dt"][:, 0].cuda(), lv["A"].cuda(), lv["B"][:, 0].cuda(), lv["C"][:, 0].cuda(), state, lv["D"].cuda(),
                                      lv["z"][:, 0].cuda(), lv["bias"].cuda(), dt_softplus=True)
    for n in want:
        near(n, got[n].cpu(), want[n])
    near("step", step.cpu(), want["y"][:, 0])


@pytest.mark.parametrize("N", [1, 5, 12, 16, 20, 50])
@pytest.mark.parametrize("what", ["x", "dt"])
@pytest.mark.parametrize("T", [37, 700])
def test_infinite_values_beside_any_number_of_states(N, what, T):
    """An infinite x (or dt) makes y infinite, not NaN: the states that fill up a channel's lanes have no part in it.  700: cut into parts."""
    gen = torch.Generator().manual_seed(53)
    D = 20
    lv = positive(gen, T, D, N)
    lv[what][0, T - 17, 7] = INF
    got, want = both(lv)
    assert want["y"].isinf().any() and not want["y"].isnan().any()
    for n in want:
        alike(n, got[n], want[n])
    before = torch.rand(8, D, N, generator=gen)
    for copies in (1, 2000):
        step_like(lv, slice(T - 20, T - 12), before, copies)


@pytest.mark.parametrize("N", [5, 16, 50])
@pytest.mark.parametrize("T", [37, 700])
def test_gradients_where_only_the_last_state_is_infinite(N, T):
    """The rates' gradient has no term of the state behind the last token, nor of the tokens that fill up its tile."""
    gen = torch.Generator().manual_seed(54)
    D = 12
    lv = scan_leaves(gen, 1, T, D, N, 1, None, torch.float32, False)
    lv["x"][0, -1, 4] = INF
    got, want = both(lv, [rand(gen, 1, T, D), rand(gen, 1, D, N)])
    for n in ("dx", "dA"):
        near(n, got[n].cpu(), want[n])


@pytest.mark.parametrize("N", [3, 7, 11, 15, 31, 47])
@pytest.mark.parametrize("T", [37, 700])
def test_infinite_values_beside_all_states_of_a_lane_but_one(N, T):
    """One state fills up the last lane that has any, or none of the others of its lanes: the upper half of a pair of numbers."""
    gen = torch.Generator().manual_seed(55)
    lv = positive(gen, T, 9, N)
    lv["x"][0, T // 2, 4] = INF
    got, want = both(lv)
    for n in want:
        alike(n, got[n], want[n])


@pytest.mark.parametrize("N", [16, 47])
def test_infinite_states_cross_parts(N):
    """An infinite state stays infinite over every token, also where the decay over a whole part of the sequence is 0 in fp32."""
    gen = torch.Generator().manual_seed(56)
    T, D = 1500, 9
    lv = positive(gen, T, D, N)
    lv["A"][:], lv["dt"] = -50.0, lv["dt"] + 0.05
    lv["x"][0, 300, 4] = INF
    got, want = both(lv)
    assert want["end"].isinf().any()
    for n in want:
        alike(n, got[n], want[n])
