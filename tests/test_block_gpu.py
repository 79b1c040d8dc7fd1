"""GPU: the operators around the layer against their definitions in 64 bits.

Tolerances.  A result is compared in the 2-norm, ``|a - b| <= tol |b|``, and element by element against the size of its terms.  Results in 16 bits are rounded
once: at most half a step, ``finfo.eps / 2``, relative to the value, and no more in any norm.  The arithmetic in front of that rounding, and results in 32
bits: every operation is off by 2^-24, an exponential or a quotient of the special function unit by 2^-22; a chain of a few dozen of them, and sums of random
signs whose terms are larger than the sum, stay below 2^-17 = 8e-6 of the 2-norm (128 roundings of 2^-24 in a row, or 30 of 2^-22)."""
import math

import pytest
import torch

import mogankda_b200 as mk

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ARITHMETIC = 2.0 ** -17


def tolerance(dtype):
    return ARITHMETIC + (0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)


def near(name, got, ref, terms=0.0):
    """``terms``: the 2-norm of the terms that the result is the difference of, where they may cancel: the arithmetic is that exact relative to them."""
    assert got is not None and got.shape == ref.shape, f"{name}: {None if got is None else got.shape} {ref.shape}"
    a, b = got.double(), ref.double()
    assert torch.isfinite(a).all(), f"{name}: not finite"
    off, norm = (a - b).norm().item(), b.norm().item()
    assert off <= tolerance(got.dtype) * norm + ARITHMETIC * terms + 1e-30, f"{name}: {off / norm if norm else off:.3e} (tolerance {tolerance(got.dtype):.1e})"
    if b.numel():          # one element: 16 times the tolerance of the larger of its value and the root mean square
        rms = norm / math.sqrt(b.numel())
        worst = ((a - b).abs() / b.abs().clamp_min(rms + 1e-30)).max().item()
        assert worst <= 16 * (tolerance(got.dtype) + ARITHMETIC * terms / (norm + 1e-30)), f"{name}: one element is off by {worst:.3e}"


def rand(gen, *shape):
    return torch.randn(*shape, generator=gen)


def spans(B, T, cu):
    return [(b, 0, T) for b in range(B)] if cu is None else [(0, p, q) for p, q in zip(cu[:-1], cu[1:])]


def differentiate(fn, leaves, ups, names):
    outs = fn()
    outs = [o for o in outs if o is not None]
    some = [(o, u) for o, u in zip(outs, ups) if o.requires_grad]
    grads = torch.autograd.grad([o for o, _ in some], [leaves[n] for n in names], [u for _, u in some], allow_unused=True) if some else [None] * len(names)
    return outs, [torch.zeros_like(leaves[n]) if g is None else g for n, g in zip(names, grads)]


# ---- convolution -----------------------------------------------------------------------------------------------------------------------------
def conv_reference(x, w, bias, act, state, cu, last):
    B, T, D = x.shape
    W = w.shape[1]
    y, ends = x * 0, []
    for i, (b, p, q) in enumerate(spans(B, T, cu)):
        head = state[i] if state is not None else x.new_zeros(W - 1, D)
        seq = torch.cat([head, x[b, p:q]])
        pre = sum(w[:, j] * seq[j:j + q - p] for j in range(W)) + (bias if bias is not None else 0)
        y = y.clone()
        y[b, p:q] = pre * torch.sigmoid(pre) if act else pre
        ends.append(seq[q - p:])
    return y, (torch.stack(ends) if ends else x.new_zeros(0, W - 1, D)) if last else None


CONV = [  # B, T, D, W, cu
    (1, 1, 8, 4, None), (2, 3, 16, 4, None), (3, 37, 64, 3, None), (1, 130, 1001, 2, None), (2, 200, 520, 4, None), (1, 77, 1, 4, None),
    (1, 100, 40, 4, (0, 1, 3, 3, 20, 100)), (1, 70, 24, 3, (0, 0, 2, 64, 66)), (1, 9, 36, 4, (0, 2, 4, 5, 9)), (1, 300, 136, 4, (0, 0, 0, 299, 300, 300)),
    (1, 5, 16, 2, (0,)), (2, 1500, 2056, 4, None), (1, 4099, 1032, 3, (0, 1000, 1003, 1004, 4000)),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", CONV, ids=str)
@pytest.mark.parametrize("option", ["plain", "all"])
def test_conv(shape, dtype, option):
    B, T, D, W, cu = shape
    gen = torch.Generator().manual_seed(B * 1000 + T + D)
    N = B if cu is None else len(cu) - 1
    full = option == "all"
    lv = dict(x=rand(gen, B, T, D).to(dtype), w=rand(gen, D, W) * W ** -0.5)
    if full:
        lv.update(bias=rand(gen, D), state=rand(gen, N, W - 1, D).to(dtype))
    ups = [rand(gen, B, T, D).to(dtype), rand(gen, N, W - 1, D).to(dtype)]
    mine = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}
    wide = {n: t.double().requires_grad_(True) for n, t in lv.items()}
    cu_t = None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")
    act = "silu" if full else None
    outs, grads = differentiate(lambda: mk.causal_conv1d(mine["x"], mine["w"], mine.get("bias"), activation=act, initial_state=mine.get("state"),
                                                         output_final_state=full, cu_seqlens=cu_t), mine, [u.cuda() for u in ups], list(lv))
    routs, rgrads = differentiate(lambda: conv_reference(wide["x"], wide["w"], wide.get("bias"), full, wide.get("state"), cu, full), wide,
                                  [u.double() for u in ups], list(lv))
    for n, a, b in zip(["y", "last"] + ["d" + n for n in lv], outs + grads, routs + rgrads):
        near(n, a.cpu(), b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_conv_steps_continue_a_prompt(dtype):
    gen = torch.Generator().manual_seed(1)
    x, w, b = rand(gen, 3, 40, 264).to(dtype).cuda(), rand(gen, 264, 4).cuda(), rand(gen, 264).cuda()
    with torch.no_grad():
        whole, end = mk.causal_conv1d(x, w, b, activation="silu", output_final_state=True)
        y, state = mk.causal_conv1d(x[:, :33], w, b, activation="silu", output_final_state=True)
        parts = [y]
        for t in range(33, 40):
            before = state._version
            parts.append(mk.causal_conv1d_step(x[:, t], state, w, b, activation="silu")[:, None])
            assert state._version == before + 1
    assert torch.equal(torch.cat(parts, 1), whole) and torch.equal(state, end)


def test_conv_halo_of_a_slice():
    """A sequence in two slices: the second takes the last tokens of the first as its state; gradients flow back through them."""
    gen = torch.Generator().manual_seed(2)
    x, w = rand(gen, 1, 50, 48).cuda().requires_grad_(True), rand(gen, 48, 4).cuda().requires_grad_(True)
    up = rand(gen, 1, 50, 48).cuda()
    whole, _ = mk.causal_conv1d(x, w, activation="silu")
    want = torch.autograd.grad(whole, (x, w), up)
    a, _ = mk.causal_conv1d(x[:, :20], w, activation="silu")
    b, _ = mk.causal_conv1d(x[:, 20:], w, activation="silu", initial_state=x[:, 17:20])
    got = torch.autograd.grad((a, b), (x, w), (up[:, :20], up[:, 20:]))
    assert torch.equal(torch.cat([a, b], 1), whole)
    for g, r in zip(got, want):
        near("gradient", g, r.double())


# ---- scan ------------------------------------------------------------------------------------------------------------------------------------
def scan_reference(x, dt, A, B, C, D=None, z=None, bias=None, softplus=False, h0=None, cu=None, last=False):
    Bs, T, W = x.shape
    N = A.shape[1]
    if B.dim() == 3:
        B, C = B[:, :, None], C[:, :, None]
    per = W // B.shape[2]
    d = dt + bias if bias is not None else dt
    d = torch.nn.functional.softplus(d, threshold=1000) if softplus else d
    rows, ends = {}, []
    for i, (b, p, q) in enumerate(spans(Bs, T, cu)):
        h = h0[i] if h0 is not None else x.new_zeros(W, N)
        for t in range(p, q):
            Bt, Ct = B[b, t].repeat_interleave(per, 0), C[b, t].repeat_interleave(per, 0)
            h = torch.exp(d[b, t][:, None] * A) * h + (d[b, t] * x[b, t])[:, None] * Bt
            y = (h * Ct).sum(-1)
            y = y + D * x[b, t] if D is not None else y
            rows[b, t] = y * z[b, t] * torch.sigmoid(z[b, t]) if z is not None else y
        ends.append(h)
    zero = x.new_zeros(W)
    y = torch.stack([torch.stack([rows.get((b, t), zero) for t in range(T)]) if T else x.new_zeros(0, W) for b in range(Bs)])
    return y, (torch.stack(ends) if ends else x.new_zeros(0, W, N)) if last else None


def scan_leaves(gen, B, T, W, N, G, cu, dtype, full, squeeze=False):
    seqs = B if cu is None else len(cu) - 1
    step = torch.exp(torch.rand(W, generator=gen) * math.log(100.0) + math.log(1e-3))
    lv = dict(x=rand(gen, B, T, W).to(dtype))
    lv["dt"] = (rand(gen, B, T, W) * 0.5).to(dtype) if full else (step * torch.exp(0.5 * rand(gen, B, T, W))).to(dtype)
    lv["A"] = -torch.rand(W, N, generator=gen) * N - 0.1
    bc = (B, T, N) if squeeze else (B, T, G, N)
    lv["B"], lv["C"] = rand(gen, *bc).to(dtype), rand(gen, *bc).to(dtype)
    if full:
        lv.update(D=rand(gen, W), z=rand(gen, B, T, W).to(dtype), bias=step + torch.log(-torch.expm1(-step)), h0=rand(gen, seqs, W, N))
    return lv


def call_scan(lv, cu, full):
    get = lv.get
    return mk.selective_scan(lv["x"], lv["dt"], lv["A"], lv["B"], lv["C"], get("D"), get("z"), get("bias"), dt_softplus=full, initial_state=get("h0"),
                             output_final_state=full, cu_seqlens=cu)


SCAN = [  # B, T, D, states, groups, cu
    (1, 1, 8, 16, 1, None), (2, 5, 32, 16, 1, None), (1, 33, 64, 16, 2, None), (3, 64, 40, 16, 1, None), (1, 50, 33, 16, 1, None), (2, 17, 130, 16, 2, None),
    (1, 40, 200, 8, 1, None), (1, 35, 24, 1, 1, None), (1, 35, 24, 5, 3, None), (2, 20, 48, 32, 2, None), (1, 37, 17, 64, 1, None), (1, 18, 20, 50, 1, None),
    (1, 1, 1, 16, 1, None), (1, 100, 48, 16, 1, (0, 1, 17, 17, 33, 100)), (1, 60, 40, 16, 2, (0, 0, 16, 48, 50)), (1, 90, 16, 12, 1, (0, 32, 64, 90, 90)),
    (1, 5, 16, 16, 1, (0,)), (1, 70, 300, 16, 1, (0, 3, 70)),
    (1, 257, 40, 16, 1, None), (2, 700, 33, 16, 1, None), (1, 300, 16, 8, 1, None), (1, 900, 24, 30, 1, (0, 290, 300, 899)), (1, 270, 9, 64, 1, None),
    (1, 200, 4100, 16, 2, tuple(range(0, 196, 5)) + (197, 200)),
    # few channels and long sequences: cut into parts that run side by side, in both directions or (600 tokens) only backward
    (1, 1300, 17, 16, 1, None), (2, 600, 40, 16, 2, None), (1, 1025, 70, 5, 1, None), (1, 900, 10, 64, 2, None), (1, 1500, 20, 16, 1, (0, 3, 3, 1400, 1410, 1450)),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SCAN, ids=str)
@pytest.mark.parametrize("full", [False, True], ids=["plain", "all"])
def test_scan(shape, dtype, full):
    B, T, W, N, G, cu = shape
    gen = torch.Generator().manual_seed(T * 7 + W + N)
    lv = scan_leaves(gen, B, T, W, N, G, cu, dtype, full, squeeze=G == 1 and T % 2 == 1)
    seqs = B if cu is None else len(cu) - 1
    ups = [rand(gen, B, T, W).to(dtype), rand(gen, seqs, W, N)]
    mine = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}
    wide = {n: t.double().requires_grad_(True) for n, t in lv.items()}
    cu_t = None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")
    outs, grads = differentiate(lambda: call_scan(mine, cu_t, full), mine, [u.cuda() for u in ups], list(lv))
    routs, rgrads = differentiate(lambda: scan_reference(wide["x"], wide["dt"], wide["A"], wide["B"], wide["C"], wide.get("D"), wide.get("z"), wide.get("bias"),
                                                         full, wide.get("h0"), cu, full), wide, [u.double() for u in ups], list(lv))
    for n, a, b in zip((["y", "last"] if full else ["y"]) + ["d" + n for n in lv], outs + grads, routs + rgrads):
        near(n, a.cpu(), b)
    with torch.no_grad():          # the same without what a backward pass needs
        again = call_scan(mine, cu_t, full)
    assert torch.equal(again[0], outs[0])


def test_scan_gradients_against_differences():
    """Central differences of a weighted sum of the results along random directions; fp32, so that the steps may be small: the truncation is of the order of
    step^2 = 1e-4 of the derivative, the rounding 2^-17 / step."""
    gen = torch.Generator().manual_seed(5)
    lv = {n: t.cuda() for n, t in scan_leaves(gen, 1, 40, 16, 16, 1, None, torch.float32, True).items()}
    ups = [rand(gen, 1, 40, 16).cuda(), rand(gen, 1, 16, 16).cuda()]
    leaves = {n: t.clone().requires_grad_(True) for n, t in lv.items()}
    outs = call_scan(leaves, None, True)
    grads = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), ups)))

    def value(moved):
        with torch.no_grad():
            return sum((o.double() * u.double()).sum() for o, u in zip(call_scan(moved, None, True), ups)).item()

    size = sum((o.double() * u.double()).norm().item() for o, u in zip(outs, ups))
    for n in lv:
        way = rand(gen, *lv[n].shape).cuda()
        step = 1e-2 * lv[n].norm().item() / way.norm().item()
        diff = (value(dict(lv, **{n: lv[n] + step * way})) - value(dict(lv, **{n: lv[n] - step * way}))) / (2 * step)
        told = (grads[n].double() * way.double()).sum().item()
        assert abs(diff - told) <= 2e-3 * grads[n].norm().item() * way.norm().item() / math.sqrt(way.numel()) + 2.0 ** -17 * size / step, n


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N,G,W", [(16, 1, 264), (16, 3, 33), (7, 1, 20), (64, 2, 24)])
def test_scan_steps_continue_a_prompt(dtype, N, G, W):
    gen = torch.Generator().manual_seed(N)
    lv = {n: t.cuda() for n, t in scan_leaves(gen, 3, 24, W, N, G, None, dtype, True).items()}
    with torch.no_grad():
        whole, end = call_scan(lv, None, True)
        cut = {n: t[:, :17] if n in ("x", "dt", "B", "C", "z") else t for n, t in lv.items()}
        y, state = call_scan(cut, None, True)
        parts = [y]
        for t in range(17, 24):
            before = state._version
            parts.append(mk.selective_scan_step(lv["x"][:, t], lv["dt"][:, t], lv["A"], lv["B"][:, t], lv["C"][:, t], state, lv["D"], lv["z"][:, t], lv["bias"],
                                                dt_softplus=True)[:, None])
            assert state._version == before + 1
    near("y", torch.cat(parts, 1), whole.double())
    near("state", state, end.double())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [3, 8, 16, 30, 64])
def test_scan_steps_of_many_sequences(dtype, N):
    """Four sequences a thread give each what it gets in a call of its own."""
    gen = torch.Generator().manual_seed(N)
    rows, W, G = 203, {3: 3002, 8: 3002, 16: 1502, 30: 752, 64: 402}[N], 2
    lv = {n: t.cuda() for n, t in scan_leaves(gen, rows, 1, W, N, G, None, dtype, True).items()}
    tok = {n: lv[n][:, 0] for n in ("x", "dt", "B", "C", "z")}

    def step(a, b, state):
        return mk.selective_scan_step(tok["x"][a:b], tok["dt"][a:b], lv["A"], tok["B"][a:b], tok["C"][a:b], state, lv["D"], tok["z"][a:b], lv["bias"], dt_softplus=True)

    with torch.no_grad():
        state, parts = lv["h0"].clone(), [lv["h0"][i:i + 2].clone() for i in range(0, rows, 2)]
        y = step(0, rows, state)
        ys = [step(2 * i, min(2 * i + 2, rows), s) for i, s in enumerate(parts)]
        whole, end = call_scan(lv, None, True)
    near("y", torch.cat(ys), y.double())
    near("state", torch.cat(parts), state.double())
    near("y of a prompt", whole[:, 0], y.double())
    near("state of a prompt", end, state.double())


def test_scan_of_any_decay():
    """No decay at all, decays that leave nothing (the exponential underflows), and softplus at both ends of its range."""
    gen = torch.Generator().manual_seed(9)
    lv = scan_leaves(gen, 1, 40, 32, 16, 1, None, torch.float32, True)
    lv["A"][:8] = 0.0
    lv["A"][8:16] = -1e4
    lv["dt"][:, 10:20] = -30.0
    lv["dt"][:, 20:22] = 60.0
    ups = [rand(gen, 1, 40, 32), rand(gen, 1, 32, 16)]
    mine = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}
    wide = {n: t.double().requires_grad_(True) for n, t in lv.items()}
    outs, grads = differentiate(lambda: call_scan(mine, None, True), mine, [u.cuda() for u in ups], list(lv))
    routs, rgrads = differentiate(lambda: scan_reference(*(wide[n] for n in ("x", "dt", "A", "B", "C", "D", "z", "bias")), True, wide["h0"], None, True), wide,
                                  [u.double() for u in ups], list(lv))
    for n, a, b in zip(["y", "last"] + ["d" + n for n in lv], outs + grads, routs + rgrads):
        near(n, a.cpu(), b)


def test_scan_without_time_passing_keeps_its_state():
    """dt = 0: exp(0) is 1 exactly, whatever A and x are; also what the tokens behind a sequence's last one inside a tile rely on."""
    gen = torch.Generator().manual_seed(31)
    for T, W in ((1, 40), (33, 40), (500, 8)):
        lv = {n: t.cuda() for n, t in scan_leaves(gen, 2, T, W, 16, 1, None, torch.bfloat16, True).items()}
        zero = torch.zeros_like(lv["x"])
        _, h = mk.selective_scan(lv["x"], zero, 100 * lv["A"], lv["B"], lv["C"], initial_state=lv["h0"], output_final_state=True)
        assert torch.equal(h, lv["h0"])
        state = lv["h0"].clone()
        mk.selective_scan_step(lv["x"][:, 0], zero[:, 0], lv["A"], lv["B"][:, 0], lv["C"][:, 0], state)
        assert torch.equal(state, lv["h0"])


def test_scan_of_growing_states_behind_zeros():
    """A > 0 and a long stretch of zeros: nothing grows into nothing, also where the growth of a part of the sequence is past the largest number."""
    gen = torch.Generator().manual_seed(21)
    T, D, N, few = 1500, 8, 16, 10
    x, up = torch.zeros(1, T, D), torch.zeros(1, T, D)
    x[:, -few:], up[:, :few] = rand(gen, 1, few, D), rand(gen, 1, few, D)
    lv = {"x": x, "dt": torch.ones(1, T, D), "A": torch.full((D, N), 2.0), "B": rand(gen, 1, T, N), "C": rand(gen, 1, T, N)}
    mine = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}
    wide = {n: t.double().requires_grad_(True) for n, t in lv.items()}
    outs, grads = differentiate(lambda: mk.selective_scan(*mine.values()), mine, [up.cuda()], list(lv))
    routs, rgrads = differentiate(lambda: scan_reference(*wide.values()), wide, [up.double()], list(lv))
    for n, a, b in zip(["y"] + ["d" + n for n in lv], outs + grads, routs + rgrads):
        near(n, a.cpu(), b)


def test_scan_of_states_that_leave_the_range_of_a_decay():
    """What a part of a sequence lets through may be below the smallest number where what comes out of it is not: 2^90 by 2^-185 (a part of 128 tokens)."""
    T, D, N = 512, 8, 16
    gen = torch.Generator().manual_seed(22)
    lv = {"x": torch.zeros(1, T, D), "dt": torch.ones(1, T, D), "A": torch.full((D, N), -1.0), "B": rand(gen, 1, T, N), "C": rand(gen, 1, T, N)}
    h0 = (1 + rand(gen, 1, D, N).abs()) * 2.0 ** 90
    with torch.no_grad():
        y, _ = mk.selective_scan(*(t.cuda() for t in lv.values()), initial_state=h0.cuda())
        ref, _ = scan_reference(*(t.double() for t in lv.values()), h0=h0.double())
    # 140 tokens are 140 factors off by 2^-22 each and as many roundings of 2^-24: 140 (2^-22 + 2^-24) = 4.2e-5 of the value, of each term of the sum over the states
    got, ref = y[0, :140].double().cpu(), ref[0, :140]
    size = torch.einsum("tn,dn->td", lv["C"][0, :140].double().abs(), h0[0].double()) * torch.exp(-torch.arange(1, 141).double())[:, None]
    assert ((got - ref).abs() <= 4.2e-5 * size).all()


# ---- norm ------------------------------------------------------------------------------------------------------------------------------------
def norm_reference(x, w, res, eps, res_dtype):
    s = x
    if res is not None:
        s = x + res
        s = s + (s.detach().to(res_dtype).double() - s.detach())
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return (y * w if w is not None else y), (s if res is not None else None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,H", [(1, 1), (5, 7), (3, 128), (9, 256), (4, 264), (33, 1000), (2, 1024), (7, 2048), (3, 4096), (2, 5000), (2, 8192), (1, 16384), (1, 32768), (700, 96), (600, 4096)])
@pytest.mark.parametrize("residual", [None, "same", "fp32"])
def test_norm(rows, H, dtype, residual):
    gen = torch.Generator().manual_seed(rows * 31 + H)
    rdt = torch.float32 if residual == "fp32" else dtype
    lv = dict(x=rand(gen, rows, H).to(dtype))
    if H % 3:
        lv["w"] = (1 + 0.2 * rand(gen, H)).to(torch.float32 if residual else dtype)
    if residual:
        lv["res"] = (2 * rand(gen, rows, H)).to(rdt)
    ups = [rand(gen, rows, H).to(dtype), rand(gen, rows, H).to(rdt)]
    mine = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}
    wide = {n: t.double().requires_grad_(True) for n, t in lv.items()}

    def own():
        got = mk.rms_norm(mine["x"], mine.get("w"), residual=mine.get("res"), eps=1e-5)
        return got if residual else (got,)

    outs, grads = differentiate(own, mine, [u.cuda() for u in ups], list(lv))
    routs, rgrads = differentiate(lambda: norm_reference(wide["x"], wide.get("w"), wide.get("res"), 1e-5, rdt), wide, [u.double() for u in ups], list(lv))
    # ds = r dn - r s (r^2 mean(dn s)): two terms of the norm of r dn at most (the second is a projection of the first), each off by a few 2^-22 of itself.  A row of one
    # channel is 1e-5 / s^2 of them; from a few channels on they do not cancel
    s = wide["x"].detach() + (wide["res"].detach() if residual else 0)
    terms = (ups[0].double() * wide.get("w", torch.ones(())).detach() / torch.sqrt((s * s).mean(-1, keepdim=True) + 1e-5)).norm().item()
    for n, a, b in zip((["y", "s"] if residual else ["y"]) + ["d" + n for n in lv], outs + grads, routs + rgrads):
        near(n, a.cpu(), b, terms if n in ("dx", "dres") else 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,H,group", [(1, 128, 128), (5, 384, 128), (3, 4096, 128), (2, 8192, 128), (4, 100, None), (3, 2048, None), (700, 640, 128), (1300, 264, None), (1, 32768, None), (6, 1001, None)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_in_8_bits(rows, H, group, dtype, residual):
    """e4m3 has three bits of mantissa: half a step is 2^-4 of a normal value, 2^-10 of a subnormal one; the scale brings the largest to 448."""
    gen = torch.Generator().manual_seed(rows + H)
    x, w = rand(gen, rows, H).to(dtype), 1 + 0.2 * rand(gen, H)
    x[0, :min(H, 128)] = 0                                  # a group of zeros (a whole row of them where that is all there is)
    res = rand(gen, rows, H).to(dtype) if residual else None
    if residual:
        res[0, :min(H, 128)] = 0
    with torch.no_grad():
        got = mk.rms_norm(x.cuda(), w.cuda(), residual=None if res is None else res.cuda(), out_dtype=torch.float8_e4m3fn, scale_group=group)
    q, scale = got[0], got[1]
    y, s = norm_reference(x.double(), w.double(), None if res is None else res.double(), 1e-6, dtype)
    if residual:
        assert torch.equal(got[2].cpu(), s.to(dtype))
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape
    parts = y.view(rows, -1, group or H)
    top = parts.abs().amax(-1)
    assert scale.shape == top.shape
    want = (top / 448).clamp_min(2.0 ** -126)
    assert ((scale.cpu().double() - want).abs() <= ARITHMETIC * want).all()
    held = q.cpu().float().double().view_as(parts)
    exact = parts / want[..., None]
    assert ((held - exact).abs() <= (2.0 ** -4 + ARITHMETIC) * exact.abs() + 2.0 ** -10).all()
    assert (held.abs().amax(-1)[top > 0] == 448).all()


def test_norm_of_rows_that_are_not_finite():
    x = torch.randn(4, 512, device="cuda")
    x[0, 3], x[1, 5] = float("nan"), float("inf")
    with torch.no_grad():
        y = mk.rms_norm(x)
        q, scale = mk.rms_norm(x, out_dtype=torch.float8_e4m3fn)
    assert y[0].isnan().all() and y[1, 5].isnan() and (y[1, :5] == 0).all() and torch.isfinite(y[2:]).all()
    assert scale[0].isnan() and scale[1].isnan() and torch.isfinite(scale[2:]).all() and q.float()[0].isnan().all()


# ---- together ----------------------------------------------------------------------------------------------------------------------------------
def test_strided_and_unaligned_activations():
    """Slices of one projection, at places that are not multiples of 16 bytes: read where they lie, with the gradients of the slices."""
    gen = torch.Generator().manual_seed(3)
    for dtype, off in ((torch.bfloat16, 3), (torch.float32, 1), (torch.float16, 8)):
        W, N, T = 40, 16, 37
        proj = rand(gen, 2, T, off + 3 * W + 2 * N + 5).to(dtype).cuda()
        A = -torch.rand(W, N, generator=gen).cuda()
        up = rand(gen, 2, T, W).to(dtype).cuda()

        def split(p):
            return (p[..., off:off + W], p[..., off + W:off + 2 * W], p[..., off + 2 * W:off + 3 * W], p[..., off + 3 * W:off + 3 * W + N],
                    p[..., off + 3 * W + N:off + 3 * W + 2 * N])

        def run(p, copy):
            x, dt, z, B, C = (v.contiguous() if copy else v for v in split(p))
            x, _ = mk.causal_conv1d(x, wc, activation="silu")
            y, _ = mk.selective_scan(x, dt, A, B, C, z=z, dt_softplus=True)
            return mk.rms_norm(y, residual=z)

        wc = rand(gen, W, 4).cuda()
        got = []
        for copy in (False, True):
            p = proj.clone().requires_grad_(True)
            o, s = run(p, copy)
            got.append((o, s, torch.autograd.grad((o, s), p, (up, up))[0]))
        for a, b in zip(*got):
            near("slices", a, b.double())


def block(h, p, state=None, cu=None):
    """A block of a model: norm -> projection -> convolution -> scan -> projection, with the residual stream beside it."""
    n, stream = mk.rms_norm(h, p["norm"], residual=p["stream"])
    W, N = p["A"].shape
    xz = n @ p["inp"]
    conv, ssm = state or (None, None)
    x, conv = mk.causal_conv1d(xz[..., :W], p["conv"], p["cbias"], activation="silu", initial_state=conv, output_final_state=True, cu_seqlens=cu)
    dbc = x @ p["dbc"]
    y, ssm = mk.selective_scan(x, dbc[..., :W], p["A"], dbc[..., W:W + N], dbc[..., W + N:], p["D"], xz[..., W:], p["dtb"], dt_softplus=True,
                               initial_state=ssm, output_final_state=True, cu_seqlens=cu)
    return y @ p["out"], stream, (conv, ssm)


def block_params(gen, dtype, B, T, H=64, W=96, N=16):
    p = dict(norm=1 + 0.1 * rand(gen, H), inp=(rand(gen, H, 2 * W) * H ** -0.5).to(dtype), conv=rand(gen, W, 4) * 0.5, cbias=0.1 * rand(gen, W),
             dbc=(rand(gen, W, W + 2 * N) * W ** -0.5).to(dtype), A=-torch.rand(W, N, generator=gen) * 4, D=rand(gen, W), dtb=rand(gen, W) - 3,
             out=(rand(gen, W, H) * W ** -0.5).to(dtype), stream=rand(gen, B, T, H))
    return {n: t.cuda() for n, t in p.items()}, rand(gen, B, T, H).to(dtype).cuda()


def test_block_prompt_then_tokens():
    gen = torch.Generator().manual_seed(4)
    p, h = block_params(gen, torch.float32, 2, 30)
    W, N = p["A"].shape
    with torch.no_grad():
        whole, _, (conv_end, ssm_end) = block(h, p)
        y, _, (conv, ssm) = block(h[:, :25], dict(p, stream=p["stream"][:, :25]))
        for t in range(25, 30):
            n, _ = mk.rms_norm(h[:, t], p["norm"], residual=p["stream"][:, t])
            xz = n @ p["inp"]
            x = mk.causal_conv1d_step(xz[:, :W], conv, p["conv"], p["cbias"], activation="silu")
            dbc = x @ p["dbc"]
            o = mk.selective_scan_step(x, dbc[:, :W], p["A"], dbc[:, W:W + N], dbc[:, W + N:], ssm, p["D"], xz[:, W:], p["dtb"], dt_softplus=True)
            y = torch.cat([y, (o @ p["out"])[:, None]], 1)
    # the library's products of 25, 30 and 1 rows round differently: each fp32 product of at most 96 terms is off by less than 96 x 2^-24 of its terms
    for a, b in ((y, whole), (conv, conv_end), (ssm, ssm_end)):
        assert (a - b).norm() <= 4 * (ARITHMETIC + 96 * 2.0 ** -24) * b.norm()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_block_trains_packed_like_apart(dtype):
    """Packed documents give each what it gives alone, gradients of the parameters included (sums over documents, in another order)."""
    gen = torch.Generator().manual_seed(6)
    cu = [0, 7, 8, 40]
    p, h = block_params(gen, dtype, 1, 40)
    names = list(p)
    up = rand(gen, 1, 40, 64).to(dtype).cuda()

    def grads(parts):
        leaves = {n: t.clone().requires_grad_(True) for n, t in p.items()}
        x = h.clone().requires_grad_(True)
        ys, ss = [], []
        for a, b, c in parts:
            y, s, _ = block(x[:, a:b], dict(leaves, stream=leaves["stream"][:, a:b]), cu=c)
            ys.append(y)
            ss.append(s)
        return torch.cat(ys, 1), torch.autograd.grad((torch.cat(ys, 1), torch.cat(ss, 1)), [x] + [leaves[n] for n in names], (up, up.float()))

    y0, g0 = grads([(0, 40, torch.tensor(cu, dtype=torch.int64, device="cuda"))])
    y1, g1 = grads([(a, b, None) for a, b in zip(cu[:-1], cu[1:])])
    step = 2.0 ** -17 if dtype == torch.float32 else 4 * 2.0 ** -8      # a handful of 16-bit stores between the ends, each half a step, partly in other places
    for n, a, b in zip(["y", "dh"] + names, (y0, *g0), (y1, *g1)):
        assert (a.double() - b.double()).norm() <= step * b.double().norm(), n


def test_side_streams_graphs_and_repeated_runs():
    """The same bits on another stream, out of a replayed graph (forward and backward), and every time."""
    gen = torch.Generator().manual_seed(8)
    p, h = block_params(gen, torch.bfloat16, 2, 70)
    leaves = {n: t.clone().requires_grad_(True) for n, t in p.items()}
    x = h.clone().requires_grad_(True)
    up = rand(gen, 2, 70, 64).to(torch.bfloat16).cuda()

    def step():
        y, s, _ = block(x, leaves)
        return [y, s, *torch.autograd.grad((y, s), [x, *leaves.values()], (up, up.float()))]

    first = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            second = [t.detach().clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(2):
        graph.replay()
    for a, b, c in zip(first, second, captured):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_a_captured_call_keeps_the_boundaries_of_its_sequences():
    """The table of the boundaries is the framework's own: a replay reads it however many other calls came in between."""
    from mogankda_b200 import index
    gen = torch.Generator().manual_seed(23)
    x = rand(gen, 1, 90, 64).to(torch.bfloat16).cuda().requires_grad_(True)
    bc, A, w, up = rand(gen, 1, 90, 16).to(torch.bfloat16).cuda(), -torch.ones(64, 16, device="cuda"), rand(gen, 64, 4).cuda(), torch.ones(1, 90, 64, device="cuda", dtype=torch.bfloat16)
    cu = torch.tensor([0, 20, 21, 90], device="cuda")

    def step():
        y, _ = mk.causal_conv1d(x, w, cu_seqlens=cu)
        z, _ = mk.selective_scan(y, y, A, bc, bc, dt_softplus=True, cu_seqlens=cu)
        return z.detach(), *torch.autograd.grad(z, x, up)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.detach().clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    index._cache.clear()
    torch.cuda.synchronize()
    others = [torch.zeros(10, dtype=torch.int32, device="cuda") for _ in range(512)]      # boundaries of nothing, in the memory that a lost table would have left
    graph.replay()
    torch.cuda.synchronize()
    assert len(others) == 512 and all(torch.equal(a, b) for a, b in zip(want, out))


@pytest.mark.parametrize("T", [200, 1700])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_what_is_not_finite_stays_in_its_sequence(T, what):
    """Sequences next to one that is not finite, and in front of a tail that no sequence covers, have the bits that they have beside finite ones (1700: cut into parts)."""
    gen = torch.Generator().manual_seed(24)
    D, N = 40, 16
    cu, bad = [0, 5, 37, 38, T - 90, T - 20], [1, 3]                # sequences that are spoiled
    lv = {n: rand(gen, 1, T, m).to(torch.bfloat16) for n, m in (("x", D), ("dt", D), ("z", D), ("B", N), ("C", N))}
    h0, w, A = rand(gen, 5, D, N), rand(gen, D, 4), -torch.rand(D, N, generator=gen)
    up = rand(gen, 1, T, D).to(torch.bfloat16)
    keep = torch.zeros(T, dtype=torch.bool)
    for i, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        keep[a:b] = i not in bad
    table = torch.tensor(cu, device="cuda")

    def run(spoil):
        def at(t):
            t = t.clone()
            if spoil:
                t[:, ~keep] = what
            return t.cuda()
        m = {n: at(t).requires_grad_(True) for n, t in lv.items()}
        s = h0.clone()
        if spoil:
            s[bad] = what
        s, u = s.cuda().requires_grad_(True), at(up)
        c, last = mk.causal_conv1d(m["x"], w.cuda(), cu_seqlens=table, activation="silu", output_final_state=True)
        y, end = mk.selective_scan(m["x"], m["dt"], A.cuda(), m["B"], m["C"], z=m["z"], dt_softplus=True, initial_state=s, output_final_state=True, cu_seqlens=table)
        g = torch.autograd.grad((c, y), [*m.values(), s], (u, u))
        good = [i for i in range(5) if i not in bad]
        return [t[:, keep.cuda()] for t in (c, y, *g[:-1])] + [t[good] for t in (last, end, g[-1])], [t[:, cu[-1]:] for t in (c, y, *g[:-1])]

    (want, tails), (got, spoiled) = run(False), run(True)
    for a, b in zip(want, got):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    for t in tails + spoiled:
        assert (t == 0).all()


@pytest.mark.parametrize("how", ["stride", "size"])
def test_offsets_past_32_bits(how):
    """Rows whose offsets do not fit into 32 bits, by the stride of a wide projection or by the size of the tensors themselves: the last tokens are those of a short call
    that continues from the states in front of them, bit for bit."""
    T, W, tail = 70001, 40 if how == "stride" else 32768, 70
    store = torch.empty(1, T, 65536 if how == "stride" else W, dtype=torch.bfloat16, device="cuda")
    x = store[..., -W:]
    x[:, :tail].normal_()
    for a in range(tail, T, 10000):          # cheap to fill: the same rows again and again
        x[:, a:a + 10000] = x[:, :tail].repeat(1, 143, 1)[:, :min(10000, T - a)]
    assert x[0, -1, 0].data_ptr() - x.data_ptr() > 2 ** 32
    w, A = torch.randn(W, 4, device="cuda"), -torch.rand(W, 4, device="cuda")
    bc = torch.randn(1, T, 4, dtype=torch.bfloat16, device="cuda")
    with torch.no_grad():
        y, last = mk.causal_conv1d(x, w, output_final_state=True)
        short, end = mk.causal_conv1d(x[:, -tail:].contiguous(), w, initial_state=x[:, -tail - 3:-tail].contiguous(), output_final_state=True)
        assert torch.equal(y[:, -tail:], short) and torch.equal(last, end)
        del y
        n, s = mk.rms_norm(x, residual=x)
        a, b = mk.rms_norm(x[:, -tail:].contiguous(), residual=x[:, -tail:].contiguous())
        assert torch.equal(n[:, -tail:], a) and torch.equal(s[:, -tail:], b)
        del n, s
        if how == "size":                                  # many channels: not cut, so that the state in front of the tail is the long call's own
            cut = T - 64 * 2
            _, state = mk.selective_scan(x[:, :cut], x[:, :cut], A, bc[:, :cut], bc[:, :cut], dt_softplus=True, output_final_state=True)
            y, last = mk.selective_scan(x, x, A, bc, bc, dt_softplus=True, output_final_state=True)
            short, end = mk.selective_scan(x[:, cut:].contiguous(), x[:, cut:].contiguous(), A, bc[:, cut:], bc[:, cut:], dt_softplus=True, initial_state=state, output_final_state=True)
            assert torch.equal(y[:, cut:], short) and torch.equal(last, end)
        else:
            y, last = mk.selective_scan(x, x, A, bc, bc, dt_softplus=True, output_final_state=True)
            near("y", y[:, -tail:], mk.selective_scan(x.contiguous(), x.contiguous(), A, bc, bc, dt_softplus=True)[0][:, -tail:].double())
    if how == "stride":
        leaf = x.detach().requires_grad_(True)
        up = torch.ones(1, T, W, dtype=torch.bfloat16, device="cuda")
        dense = x.detach().contiguous().requires_grad_(True)
        for call in (lambda v: mk.causal_conv1d(v, w, activation="silu")[0], lambda v: mk.rms_norm(v), lambda v: mk.selective_scan(v, v, A, bc, bc, dt_softplus=True)[0]):
            g, = torch.autograd.grad(call(leaf), leaf, up)
            h, = torch.autograd.grad(call(dense), dense, up)
            assert torch.equal(g, h)


def test_more_sequences_than_a_grid_has_rows():
    gen = torch.Generator().manual_seed(21)
    B, W, N = 70000, 8, 4
    x, bc, A = rand(gen, B, 1, W).cuda().requires_grad_(True), rand(gen, B, 1, N).cuda(), -torch.rand(W, N, generator=gen).cuda()
    h0, w, s0 = rand(gen, B, W, N).cuda().requires_grad_(True), rand(gen, W, 3).cuda(), rand(gen, B, 2, W).cuda()

    def run(a, b, cu=None):
        shape = (lambda t: t[a:b]) if cu is None else (lambda t: t[a:b].reshape(1, b - a, *t.shape[2:]))
        y, h = mk.selective_scan(shape(x), shape(x), A, shape(bc), shape(bc), initial_state=h0[a:b], output_final_state=True, dt_softplus=True, cu_seqlens=cu)
        c, s = mk.causal_conv1d(shape(x), w, initial_state=s0[a:b], output_final_state=True, cu_seqlens=cu)
        g = torch.autograd.grad((y, h, c), (x, h0), (torch.ones_like(y), torch.ones_like(h), torch.ones_like(c)))
        return y.reshape(-1, W), h, c.reshape(-1, W), s, g[0][a:b], g[1][a:b]

    whole, packed = run(0, B), run(0, B, torch.arange(B + 1, device="cuda"))
    for a, b in ((0, 3), (65534, 65537), (B - 2, B)):
        for t, p, r in zip(whole, packed, run(a, b)):
            assert torch.equal(t[a:b], r) and torch.equal(p[a:b], r)


def test_capture_while_an_eager_graph_of_the_same_leaves_lives():
    """What torch's own operators do there: the capture fails with an error that the program can catch, or succeeds; the process goes on."""
    code = """
import torch, mogankda_b200 as mk
x = torch.randn(1, 40, 32, device="cuda", requires_grad=True)
w = torch.randn(32, 4, device="cuda", requires_grad=True)
A, bc = -torch.rand(32, 16, device="cuda"), torch.randn(1, 40, 16, device="cuda")
def step():
    y, _ = mk.causal_conv1d(mk.rms_norm(x, w[:, 0]), w, activation="silu")
    return mk.selective_scan(y, x, A, bc, bc, D=w[:, 1], dt_softplus=True)[0]
alive = step()
graph = torch.cuda.CUDAGraph()
try:
    with torch.cuda.graph(graph):
        step().backward(torch.ones_like(x))
except RuntimeError as e:
    print("raised", type(e).__name__)
torch.cuda.synchronize()
torch.autograd.grad(alive, (x, w), torch.ones_like(x))
torch.cuda.synchronize()
print("alive")
"""
    import os
    import subprocess
    import sys
    run = subprocess.run([sys.executable, "-W", "ignore", "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "alive" in run.stdout, run.stderr[-2000:]


def test_two_graphs_and_two_streams_at_once():
    """Nothing is shared between calls: two captured steps replayed side by side, and eager calls beside them, give the bits of each alone."""
    gen = torch.Generator().manual_seed(11)
    steps = []
    for T in (70, 300):
        p, h = block_params(gen, torch.bfloat16, 1, T)
        leaves = {n: t.clone().requires_grad_(True) for n, t in p.items()}
        up = torch.ones(1, T, 64, dtype=torch.bfloat16, device="cuda")

        def step(h=h, leaves=leaves, up=up):
            y, s, _ = block(h, leaves)
            return [y, s, *torch.autograd.grad((y, s), list(leaves.values()), (up, up.float()))]

        steps.append(step)
    alone = [[t.detach().clone() for t in step()] for step in steps]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for step, stream in zip(steps, streams):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(step())
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(3):
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
        eager = steps[0]()
        torch.cuda.synchronize()
        for got, want in zip((*outs, eager), (*alone, alone[0])):
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_inference_mode_and_saved_tensor_hooks():
    gen = torch.Generator().manual_seed(12)
    p, h = block_params(gen, torch.bfloat16, 1, 50)
    cu = [0, 20, 50]
    want = block(h, p, cu=torch.tensor(cu, device="cuda"))[0]
    with torch.inference_mode():
        t = torch.tensor(cu, device="cuda")
        assert torch.equal(block(h, p, cu=t)[0], want)
        t[1] = 30                                          # no version counter tells
        assert not torch.equal(block(h, p, cu=t)[0], want)
        state = torch.zeros(2, 3, 16, device="cuda")
        mk.causal_conv1d_step(torch.ones(2, 16, device="cuda"), state, torch.ones(16, 4, device="cuda"))
        assert (state[:, 2] == 1).all()
    leaves = {n: t.clone().requires_grad_(True) for n, t in p.items()}
    plain = torch.autograd.grad(block(h, leaves)[0].sum(), list(leaves.values()), allow_unused=True)
    with torch.autograd.graph.save_on_cpu():
        y = block(h, leaves)[0]
    for a, b in zip(plain, torch.autograd.grad(y.sum(), list(leaves.values()), allow_unused=True)):
        assert (a is None and b is None) or torch.equal(a, b)


def test_autograd_of_the_block_operators():
    """In-place changes, a second backward pass, a second differentiation, forward-mode AD, checkpointing."""
    from torch.utils.checkpoint import checkpoint
    w = torch.randn(16, 4, device="cuda", requires_grad=True)
    x = torch.randn(1, 9, 16, device="cuda", requires_grad=True)
    y, _ = mk.causal_conv1d(x, w)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    y = mk.rms_norm(x, residual=x.detach())[0]
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    assert not g.requires_grad or pytest.raises(RuntimeError, lambda: torch.autograd.grad(g.sum(), x))
    up = torch.ones_like(y).requires_grad_(True)
    y, _ = mk.causal_conv1d(x, w)
    g, = torch.autograd.grad(y, x, up, create_graph=True)
    with pytest.raises(RuntimeError, match="double backward"):
        g.sum().backward()
    leaf = torch.randn(1, 9, 16, device="cuda")
    scaled = (x * 2)
    y, _ = mk.causal_conv1d(scaled, w)
    with torch.no_grad():
        scaled.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(leaf, torch.ones_like(leaf))
        with pytest.raises(NotImplementedError):
            mk.causal_conv1d(dual, w)
    gen = torch.Generator().manual_seed(1)
    p, h = block_params(gen, torch.float32, 1, 20)
    h = h.requires_grad_(True)
    a, = torch.autograd.grad(block(h, p)[0].sum(), h)
    b, = torch.autograd.grad(checkpoint(lambda v: block(v, p)[0], h, use_reentrant=False).sum(), h)
    assert torch.equal(a, b)


@pytest.mark.parametrize("op", ["conv", "scan", "norm"])
def test_nothing_at_all(op):
    """No rows, no tokens."""
    for B, T in ((0, 5), (2, 0), (0, 0)):
        x = torch.randn(B, T, 24, device="cuda", requires_grad=True)
        if op == "conv":
            w, s0 = torch.randn(24, 4, device="cuda", requires_grad=True), torch.randn(B, 3, 24, device="cuda", requires_grad=True)
            y, last = mk.causal_conv1d(x, w, initial_state=s0, output_final_state=True)
        elif op == "scan":
            w, s0 = -torch.rand(24, 16, device="cuda").requires_grad_(True), torch.randn(B, 24, 16, device="cuda", requires_grad=True)
            bc = torch.randn(B, T, 16, device="cuda", requires_grad=True)
            y, last = mk.selective_scan(x, x, w, bc, bc, initial_state=s0, output_final_state=True)
        else:
            w, s0 = torch.randn(24, device="cuda", requires_grad=True), torch.randn(B, T, 24, device="cuda", requires_grad=True)
            y, last = mk.rms_norm(x, w, residual=s0)
        assert y.shape == x.shape and last.shape == s0.shape and torch.equal(last, s0)
        up = torch.randn_like(last)
        gw, gs = torch.autograd.grad((y, last), (w, s0), (torch.ones_like(y), up))
        assert (gw == 0).all() and torch.equal(gs, up)


def test_refusals_on_the_gpu():
    x, w = torch.randn(2, 6, 16, device="cuda"), torch.randn(16, 4, device="cuda")
    A, bc = -torch.rand(16, 8, device="cuda"), torch.randn(2, 6, 8, device="cuda")
    cu = torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    cases = [
        (AssertionError, lambda: mk.causal_conv1d(x, w[:, :1])), (AssertionError, lambda: mk.causal_conv1d(x, torch.randn(16, 5, device="cuda"))),
        (AssertionError, lambda: mk.causal_conv1d(x, w[:8])), (AssertionError, lambda: mk.causal_conv1d(x[0], w)), (AssertionError, lambda: mk.causal_conv1d(x.double(), w)),
        (AssertionError, lambda: mk.causal_conv1d(x, w, w[:8, 0])), (ValueError, lambda: mk.causal_conv1d(x, w, activation="relu")),
        (ValueError, lambda: mk.causal_conv1d(x, w, cu_seqlens=cu)), (ValueError, lambda: mk.causal_conv1d(x[:1], w, cu_seqlens=cu + 1)),
        (ValueError, lambda: mk.causal_conv1d(x[:1], w, cu_seqlens=cu.float())), (ValueError, lambda: mk.causal_conv1d(x[:1], w, cu_seqlens=cu * 2)),
        (ValueError, lambda: mk.causal_conv1d(x, w, initial_state=torch.zeros(3, 3, 16, device="cuda"))),
        (AssertionError, lambda: mk.causal_conv1d(x, w, initial_state=torch.zeros(2, 4, 16, device="cuda"))),
        (AssertionError, lambda: mk.causal_conv1d(x, w, initial_state=torch.zeros(2, 3, 16, device="cuda", dtype=torch.bfloat16))),
        (RuntimeError, lambda: mk.causal_conv1d(x, w.cpu())),
        (AssertionError, lambda: mk.causal_conv1d_step(x[:, 0], torch.zeros(2, 16, 3, device="cuda").transpose(1, 2), w)),
        (AssertionError, lambda: mk.causal_conv1d_step(x[:, 0], torch.zeros(1, 3, 16, device="cuda").expand(2, 3, 16), w)),
        (AssertionError, lambda: mk.causal_conv1d_step(x[:, 0], torch.zeros(3, 3, 16, device="cuda"), w)),
        (RuntimeError, lambda: mk.causal_conv1d_step(x[:, 0], torch.zeros(2, 3, 16, device="cuda"), w.clone().requires_grad_(True))),
        (AssertionError, lambda: mk.selective_scan(x, x, A[:8], bc, bc)), (AssertionError, lambda: mk.selective_scan(x, x, A, bc[..., :4], bc[..., :4])),
        (AssertionError, lambda: mk.selective_scan(x, x.bfloat16(), A, bc, bc)), (AssertionError, lambda: mk.selective_scan(x, x[:, :5], A, bc, bc)),
        (AssertionError, lambda: mk.selective_scan(x, x, -torch.rand(16, 65, device="cuda"), torch.randn(2, 6, 65, device="cuda"), torch.randn(2, 6, 65, device="cuda"))),
        (AssertionError, lambda: mk.selective_scan(x, x, A, torch.randn(2, 6, 3, 8, device="cuda"), torch.randn(2, 6, 3, 8, device="cuda"))),
        (AssertionError, lambda: mk.selective_scan(x, x, A, bc[:1], bc[:1])), (AssertionError, lambda: mk.selective_scan(x, x, A, bc, bc, D=torch.ones(8, device="cuda"))),
        (ValueError, lambda: mk.selective_scan(x, x, A, bc, bc, initial_state=torch.zeros(3, 16, 8, device="cuda"))),
        (AssertionError, lambda: mk.selective_scan(x, x, A, bc, bc, initial_state=torch.zeros(2, 16, 8, device="cuda").bfloat16())),
        (TypeError, lambda: mk.selective_scan(x, None, A, bc, bc)), (TypeError, lambda: mk.selective_scan_step(x[:, 0], x[:, 0], A, bc[:, 0], bc[:, 0], None)),
        (AssertionError, lambda: mk.selective_scan_step(x[:, 0], x[:, 0], A, bc[:, 0], bc[:, 0], torch.zeros(2, 16, 8, device="cuda").bfloat16())),
        (AssertionError, lambda: mk.rms_norm(x, w)), (AssertionError, lambda: mk.rms_norm(x, residual=x[:1])), (AssertionError, lambda: mk.rms_norm(x, residual=x.bfloat16())),
        (AssertionError, lambda: mk.rms_norm(x.half(), residual=x.bfloat16())), (ValueError, lambda: mk.rms_norm(x, out_dtype=torch.float16)),
        (ValueError, lambda: mk.rms_norm(x, scale_group=128)), (AssertionError, lambda: mk.rms_norm(x, out_dtype=torch.float8_e4m3fn, scale_group=128)),
        (ValueError, lambda: mk.rms_norm(x, out_dtype=torch.float8_e4m3fn, scale_group=64)), (AssertionError, lambda: mk.rms_norm(torch.zeros(1, 32769, device="cuda"))),
        (RuntimeError, lambda: mk.rms_norm(x.clone().requires_grad_(True), out_dtype=torch.float8_e4m3fn)),
    ]
    for error, call in cases:
        with pytest.raises(error):
            call()
    torch.cuda.synchronize()
