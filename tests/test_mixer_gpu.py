"""GPU: the linear attention with a decay for each head, the rotary positions and the layer norm against their definitions in 64 bits.

Tolerances are those of test_block_gpu.py (``near``): results in 16 bits are rounded once, half a step relative to the value; the arithmetic in front of that, and results in 32
bits, stay below 2^-17 of the 2-norm.  For the linear attention that is: products of 16-bit inputs are exact, and sums of up to 128 of them in 32 bits; pair weights and states
that meet another product as two 16-bit halves are off by at most 2^-16 each of the value, 2^-17.2 in the root mean square of one (uniformly distributed) and less in a sum's 2-norm
relative to its own; what goes into the state has three parts, 2^-24.  fp16 inputs: two parts of 11 bits each, of values scaled by powers of two, 2^-22.  Rotary: an angle is off by 2 pi 2^-26 = 2^-23.3 at most, a sine by 2^-22."""
import math

import pytest
import torch

import mogankda_b200 as mk
from tests.test_block_gpu import ARITHMETIC, DTYPES, differentiate, near, rand, spans

pytestmark = pytest.mark.gpu


# ---- linear attention ------------------------------------------------------------------------------------------------------------------------
def linear_reference(q, k, v, d, scale, h0=None, cu=None, last=False):
    """Token by token."""
    B, T, HK, K = q.shape
    H, V = v.shape[2:]
    lam = torch.exp(d)[:, None, None]
    rows, ends = {}, []
    q, k = q.repeat_interleave(H // HK, 2), k.repeat_interleave(H // HK, 2)
    for i, (b, p, e) in enumerate(spans(B, T, cu)):
        s = h0[i] if h0 is not None else v.new_zeros(H, K, V)
        for t in range(p, e):
            s = lam * s + k[b, t][:, :, None] * v[b, t][:, None]
            rows[b, t] = scale * (q[b, t][:, :, None] * s).sum(1)
        ends.append(s)
    zero = v.new_zeros(H, V)
    o = torch.stack([torch.stack([rows.get((b, t), zero) for t in range(T)]) if T else v.new_zeros(0, H, V) for b in range(B)])
    return o, (torch.stack(ends) if ends else v.new_zeros(0, H, K, V)) if last else None


LINEAR = [  # B, T, HK, HV, K, V, cu
    (1, 1, 1, 1, 8, 8, None), (2, 3, 1, 2, 16, 16, None), (1, 33, 2, 2, 128, 128, None), (1, 130, 2, 4, 64, 128, None), (2, 257, 1, 1, 128, 64, None), (1, 100, 3, 3, 40, 24, None),
    (1, 50, 1, 3, 1, 5, None), (1, 77, 2, 2, 17, 33, None), (1, 128, 1, 1, 128, 128, None), (1, 129, 1, 2, 128, 128, None), (3, 64, 2, 2, 32, 128, None),
    (1, 100, 1, 2, 64, 64, (0, 1, 3, 3, 20, 100)), (1, 60, 2, 2, 128, 128, (0, 0, 16, 48, 50)), (1, 300, 1, 1, 128, 128, (0, 128, 256, 257, 299)), (1, 5, 1, 2, 16, 16, (0,)),
    (1, 9, 2, 2, 128, 72, (0, 0, 0, 9, 9)),
    # long sequences of few heads: cut into parts that run side by side
    (1, 300, 2, 2, 128, 128, None), (1, 330, 1, 2, 17, 33, (0, 64, 64, 321, 329)), (3, 257, 1, 1, 64, 24, None), (1, 1300, 1, 1, 64, 64, None), (2, 700, 1, 2, 32, 64, None), (1, 1024, 1, 1, 128, 128, None), (1, 1500, 1, 1, 40, 128, (0, 3, 3, 1400, 1410, 1450)), (1, 900, 1, 1, 24, 24, (0, 257, 899)),
]


def linear_leaves(gen, shape, dtype, full):
    B, T, HK, H, K, V, cu = shape
    n = B if cu is None else len(cu) - 1
    lv = dict(q=rand(gen, B, T, HK, K).to(dtype), k=rand(gen, B, T, HK, K).to(dtype), v=rand(gen, B, T, H, V).to(dtype))
    if full:
        lv["h0"] = rand(gen, n, H, K, V)
    d = -torch.exp(-6 * torch.rand(H, generator=gen))      # memories of 1 to 400 tokens
    return lv, d, [rand(gen, B, T, H, V).to(dtype), rand(gen, n, H, K, V)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", LINEAR, ids=str)
@pytest.mark.parametrize("full", [False, True], ids=["plain", "all"])
def test_linear(shape, dtype, full):
    cu = shape[-1]
    gen = torch.Generator().manual_seed(sum(shape[:-1]))
    lv, d, ups = linear_leaves(gen, shape, dtype, full)
    scale = 0.3 if full else None
    mine = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}
    wide = {n: t.double().requires_grad_(True) for n, t in lv.items()}
    cu_t = None if cu is None else torch.tensor(cu, dtype=torch.int32, device="cuda")

    def call():
        return mk.linear_attention(mine["q"], mine["k"], mine["v"], d.cuda(), scale=scale, initial_state=mine.get("h0"), output_final_state=full, cu_seqlens=cu_t)

    outs, grads = differentiate(call, mine, [u.cuda() for u in ups], list(lv))
    routs, rgrads = differentiate(lambda: linear_reference(wide["q"], wide["k"], wide["v"], d.double(), scale or shape[4] ** -0.5, wide.get("h0"), cu, full), wide,
                                  [u.double() for u in ups], list(lv))
    for n, a, b in zip((["o", "last"] if full else ["o"]) + ["d" + n for n in lv], outs + grads, routs + rgrads):
        near(n, a.cpu(), b)
    with torch.no_grad():          # the same without a backward pass, and twice the same
        again = call()
    assert torch.equal(again[0], outs[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_gradients_against_differences(dtype):
    """The results are linear in each of q, k, v and the state: a difference of two calls is the derivative, to the rounding of the results (half a step each, and the inputs' own where
    they are moved: steps of the size of the values, by powers of two of a random sign, are exact)."""
    gen = torch.Generator().manual_seed(3)
    lv, d, ups = linear_leaves(gen, (1, 200, 1, 2, 64, 64, None), dtype, True)
    mine = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}
    ups = [u.cuda() for u in ups]

    def call(x):
        return mk.linear_attention(x["q"], x["k"], x["v"], d.cuda(), initial_state=x["h0"], output_final_state=True)

    grads = dict(zip(lv, torch.autograd.grad(call(mine), list(mine.values()), ups)))
    for n in lv:
        way = torch.where(torch.rand(lv[n].shape, generator=gen) < 0.5, -1.0, 1.0).cuda().to(lv[n].dtype)
        with torch.no_grad():
            moved = [call(dict(mine, **{n: w})) for w in (way, torch.zeros_like(way))]
        diff = sum(((a.double() - b.double()) * u.double()).sum() for a, b, u in zip(*moved, ups)).item()
        told = (grads[n].double() * way.double()).sum().item()
        eps = ARITHMETIC + (0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2)
        size = sum((torch.cat([a.double().flatten(), b.double().flatten()]).norm() * u.double().abs().max()).item() for a, b, u in zip(*moved, ups)) + grads[n].double().norm().item()
        # errors of random signs add up as their squares do: three (a sum's root mean square, four times over) times the rounding of all that is summed
        assert abs(diff - told) <= 4 * eps * size, (n, diff, told)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(3, 40, 2, 2, 128, 128), (2, 24, 1, 3, 17, 33), (5, 30, 2, 4, 64, 128)], ids=str)
def test_linear_steps_continue_a_prompt(dtype, shape):
    gen = torch.Generator().manual_seed(4)
    lv, d, _ = linear_leaves(gen, (*shape, None), dtype, True)
    lv, d, T = {n: t.cuda() for n, t in lv.items()}, d.cuda(), shape[1]
    with torch.no_grad():
        whole, end = mk.linear_attention(lv["q"], lv["k"], lv["v"], d, initial_state=lv["h0"], output_final_state=True)
        cut = T - 7
        o, state = mk.linear_attention(lv["q"][:, :cut], lv["k"][:, :cut], lv["v"][:, :cut], d, initial_state=lv["h0"], output_final_state=True)
        parts = [o]
        for t in range(cut, T):
            before = state._version
            parts.append(mk.linear_attention_step(lv["q"][:, t], lv["k"][:, t], lv["v"][:, t], d, state)[:, None])
            assert state._version == before + 1
    # both sides are rounded
    step = 0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    got = torch.cat(parts, 1).double()
    assert (got - whole.double()).norm() <= 2 * (ARITHMETIC + step) * whole.double().norm()
    near("state", state, end.double())


def test_linear_of_any_decay():
    """No decay at all, hardly any, strong ones whose powers underflow, and one that leaves nothing."""
    gen = torch.Generator().manual_seed(5)
    for dtype in DTYPES:
        shape = (1, 300, 3, 6, 64, 64, None)
        lv, _, ups = linear_leaves(gen, shape, dtype, True)
        d = torch.tensor([0.0, -1e-6, -1.0, -20.0, -1000.0, -math.inf])
        mine = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}
        wide = {n: t.double().requires_grad_(True) for n, t in lv.items()}
        outs, grads = differentiate(lambda: mk.linear_attention(mine["q"], mine["k"], mine["v"], d.cuda(), initial_state=mine["h0"], output_final_state=True), mine, [u.cuda() for u in ups], list(lv))
        routs, rgrads = differentiate(lambda: linear_reference(wide["q"], wide["k"], wide["v"], d.double(), 64 ** -0.5, wide["h0"], None, True), wide, [u.double() for u in ups], list(lv))
        for n, a, b in zip(["o", "last"] + ["d" + n for n in lv], outs + grads, routs + rgrads):
            near(n, a.cpu(), b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes", [(-10, -10, 8), (6, 6, -6), (-4, 12, -12), (0, 0, -14), (7, -7, 4)], ids=str)
def test_linear_of_any_size(dtype, sizes):
    """q, k and v of very different sizes (powers of two), whose products leave fp16's range where results do not; rows of a stretch, too, differ by 2^8."""
    gen = torch.Generator().manual_seed(17)
    shape = (1, 300, 1, 2, 128, 128, None)
    lv, d, ups = linear_leaves(gen, shape, torch.float32, True)
    by = torch.exp2(torch.randint(-8, 1, (1, 300, 1, 1), generator=gen).float())
    for n, e in zip("qkv", sizes):
        lv[n] = (lv[n] * 2.0 ** e * (by if n != "q" else 1.0)).to(dtype)
    lv["h0"] = lv["h0"] * 2.0 ** (sizes[1] + sizes[2])
    ups = [ups[0].to(dtype), ups[1]]
    mine = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}
    wide = {n: t.double().requires_grad_(True) for n, t in lv.items()}
    scale = 2.0 ** -(sizes[0] + sizes[1] + sizes[2]) / 16 if abs(sum(sizes)) > 4 else 1 / 16
    outs, grads = differentiate(lambda: mk.linear_attention(mine["q"], mine["k"], mine["v"], d.cuda(), scale=scale, initial_state=mine["h0"], output_final_state=True), mine, [u.cuda() for u in ups], list(lv))
    routs, rgrads = differentiate(lambda: linear_reference(wide["q"], wide["k"], wide["v"], d.double(), scale, wide["h0"], None, True), wide, [u.double() for u in ups], list(lv))
    for n, a, b in zip(["o", "last"] + ["d" + n for n in lv], outs + grads, routs + rgrads):
        if dtype == torch.float16 and (b.abs().max() > 60000 or b.abs().median() < 2.0 ** -12):
            continue                                       # not a result that fp16 holds to half a step
        near(n, a.cpu(), b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_reads_slices_of_a_projection(dtype):
    gen = torch.Generator().manual_seed(6)
    B, T, HK, H, D = 2, 140, 2, 4, 64
    wide = rand(gen, B, T, (2 * HK + H) * D + 8).to(dtype).cuda()
    ups = rand(gen, B, T, H, D).to(dtype).cuda()
    d = -torch.rand(H, generator=gen).cuda()

    def call(w, copy):
        q, k, v = w[..., :HK * D], w[..., HK * D:2 * HK * D], w[..., 2 * HK * D:(2 * HK + H) * D]
        q, k, v = (x.unflatten(-1, (-1, D)) for x in (q, k, v))
        if copy:
            q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        return mk.linear_attention(q, k, v, d)[0]

    got = []
    for w, copy in ((wide, False), (wide, True), (torch.cat([wide[..., :1], wide], -1)[..., 1:], False)):      # and from an odd address
        w = w.detach().requires_grad_(True) if w.is_contiguous() else w
        leaf = w if w.requires_grad else w.requires_grad_(True)
        o = call(leaf, copy)
        got.append((o, *torch.autograd.grad(o, leaf, ups)))
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


def test_linear_of_broadcast_inputs():
    """Heads and tokens that are one in memory."""
    gen = torch.Generator().manual_seed(7)
    q, k, v = (rand(gen, 1, 90, 1, 32).cuda().requires_grad_(True) for _ in range(3))
    d = -torch.rand(3, generator=gen).cuda()
    up = rand(gen, 1, 90, 3, 32).cuda()
    a = torch.autograd.grad(mk.linear_attention(q.expand(1, 90, 3, 32), k.expand(1, 90, 3, 32), v.expand(1, 90, 3, 32), d)[0], (q, k, v), up)
    b = torch.autograd.grad(mk.linear_attention(q, k, v.expand(1, 90, 3, 32).contiguous(), d)[0], (q, k, v), up)
    for x, y in zip(a, b):
        near("gradient", x, y.double())


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_of_one_token_over_and_over(dtype):
    """All tokens are one in memory (a stride of 0), or half of one overlaps the next."""
    gen = torch.Generator().manual_seed(14)
    d = -torch.rand(2, generator=gen).cuda()
    one = rand(gen, 1, 1, 2, 32).cuda().to(dtype)
    flat = rand(gen, 32 * 150 + 64).cuda().to(dtype)
    lap = flat.as_strided((1, 150, 2, 32), (0, 32, 32, 1))
    for x in (one.expand(1, 150, 2, 32), lap):
        with torch.no_grad():
            a, b = mk.linear_attention(x, x, x, d), mk.linear_attention(*(x.contiguous() for _ in range(3)), d)
        assert torch.equal(a[0], b[0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,cu", [(0, 7, None), (2, 0, None), (1, 0, (0, 0, 0)), (1, 40, (0, 0, 40, 40)), (1, 40, (0, 0, 0))], ids=str)
def test_linear_of_nothing(dtype, B, T, cu):
    """No sequence, no token, sequences without tokens: states pass through, and so do their gradients."""
    n = B if cu is None else len(cu) - 1
    gen = torch.Generator().manual_seed(15)
    lv = dict(q=rand(gen, B, T, 1, 64).to(dtype), k=rand(gen, B, T, 1, 64).to(dtype), v=rand(gen, B, T, 2, 64).to(dtype), h0=rand(gen, n, 2, 64, 64))
    mine = {m: t.cuda().requires_grad_(True) for m, t in lv.items()}
    d = -torch.rand(2, generator=gen)
    o, last = mk.linear_attention(mine["q"], mine["k"], mine["v"], d.cuda(), initial_state=mine["h0"], output_final_state=True, cu_seqlens=None if cu is None else torch.tensor(cu, dtype=torch.int32).cuda())
    up = rand(gen, n, 2, 64, 64).cuda()
    grads = torch.autograd.grad(last, list(mine.values()), up)          # nothing comes back through o
    assert o.shape == lv["v"].shape and all(g.shape == t.shape for g, t in zip(grads, lv.values()))
    for i in range(n):
        if cu is None or cu[i] == cu[i + 1]:
            assert torch.equal(last[i], mine["h0"][i]) and torch.equal(grads[3][i], up[i])
    if cu and cu[-1] == 0:
        assert (o == 0).all() and all((g == 0).all() for g in grads[:3])


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_of_many_sequences_beside_a_long_one(dtype):
    """Sequences of a few tokens, more than a wave of blocks has places, and one that is cut by itself."""
    gen = torch.Generator().manual_seed(16)
    few, long = 500, 3000
    lens = [int(x) for x in torch.randint(0, 9, (few,), generator=gen)]
    cu = [0]
    for n in lens[:250] + [long] + lens[250:]:
        cu.append(cu[-1] + n)
    q, k, v = (rand(gen, 1, cu[-1], 1, 64).to(dtype).cuda() for _ in range(3))
    d = torch.tensor([-0.02]).cuda()
    with torch.no_grad():
        o, last = mk.linear_attention(q, k, v, d, cu_seqlens=torch.tensor(cu, dtype=torch.int32).cuda(), output_final_state=True)
        for i in (0, 100, 249, 250, 251, 400, 500):
            s = slice(cu[i], cu[i + 1])
            a, b = mk.linear_attention(q[:, s], k[:, s], v[:, s], d, output_final_state=True)
            near("state", last[i:i + 1], b.double())
            if a.numel():          # both are rounded
                step = 0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
                assert (a.double() - o[:, s].double()).norm() <= 2 * (ARITHMETIC + step) * a.double().norm()


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_leaves_tokens_of_no_sequence_alone(dtype):
    """Behind the last boundary nothing is read and results are zero; what is not finite stays in its sequence."""
    gen = torch.Generator().manual_seed(8)
    lv, d, ups = linear_leaves(gen, (1, 400, 1, 2, 128, 128, None), dtype, False)
    cu = torch.tensor([0, 70, 200, 290], dtype=torch.int32).cuda()
    got = []
    for bad in (0.0, math.nan, math.inf):
        x = {n: t.clone() for n, t in lv.items()}
        up = ups[0].clone()
        for t in (*x.values(), up):
            t[:, 290:] = bad
            if bad != 0:
                t[:, 70:200] = bad                         # a sequence in the middle, too
        x = {n: t.cuda().requires_grad_(True) for n, t in x.items()}
        o, last = mk.linear_attention(x["q"], x["k"], x["v"], d.cuda(), cu_seqlens=cu, output_final_state=True)
        g = torch.autograd.grad((o, last), list(x.values()), (up.cuda(), torch.ones_like(last)))
        got.append([t[:, s] for t in (o, *g) for s in (slice(0, 70), slice(200, 400))] + [last[0], last[2]])
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))
    assert all(torch.isfinite(t).all() for t in got[0]) and got[0][1][:, 90:].abs().max() == 0


NOT_FINITE = [  # K, V, tokens, the token and the channel
    (128, 128, 300, 200, 70), (64, 40, 128, 0, 3), (64, 64, 130, 129, 63), (17, 33, 150, 70, 16), (128, 64, 1200, 640, 5),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", NOT_FINITE, ids=str)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan], ids=str)
def test_linear_of_what_is_not_finite(shape, dtype, bad):
    """One element of q, k, v or the gradient from above: what it has no part in stays as it is.  Those results are compared with the ones beside a finite value; both are rounded."""
    K, V, T, at, ch = shape
    gen = torch.Generator().manual_seed(17)
    lv, d, ups = linear_leaves(gen, (1, T, 2, 2, K, V, None), dtype, False)
    up, dev = ups[0], torch.device("cuda")
    step = 0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2

    def run(name, value):
        x = {n: t.clone() for n, t in (*lv.items(), ("up", up))}
        x[name][0, at, 1, ch if name in ("v", "up") else ch % K] = value
        x = {n: t.to(dev) for n, t in x.items()}
        rows = [x[n].requires_grad_(True) for n in "qkv"]
        o, last = mk.linear_attention(*rows, d.to(dev), output_final_state=True)
        return dict(zip(("o", "last", "dq", "dk", "dv"), (t.detach().cpu().double() for t in (o, last, *torch.autograd.grad(o, rows, x["up"])))))

    front, behind, one, other = slice(0, at), slice(at + 1, T), [t for t in range(T) if t != at], [c for c in range(V) if c != ch]
    # result: the tokens that the element has no part in
    clean = {"q": dict(o=one, dq=slice(0, T), dk=behind, dv=behind), "k": dict(o=front, dq=front, dk=slice(0, T), dv=one), "v": dict(o=front, dq=front, dk=one, dv=slice(0, T)),
             "up": dict(o=slice(0, T), dq=one, dk=behind, dv=behind)}
    hit = {"q": ("o", "dk", "dv"), "k": ("o", "dq", "dv"), "v": ("o", "dq", "dk"), "up": ("dq", "dk", "dv")}
    for name in clean:
        got, want = run(name, bad), run(name, 0.5)
        for n, tokens in clean[name].items():
            a, b = got[n][0, tokens], want[n][0, tokens]
            assert torch.isfinite(a).all(), (name, n)
            assert (a - b).norm() <= 2 * (ARITHMETIC + step) * b.norm(), (name, n)
            assert torch.isfinite(got[n][0, :, 0]).all(), (name, n)          # the other head
        for n in hit[name]:
            assert not torch.isfinite(got[n][0, at, 1]).all(), (name, n)
        if name == "v":          # a channel of v is one of o and of the state
            for n in ("o", "last"):
                assert torch.isfinite(got[n][..., other]).all() and not torch.isfinite(got[n][0, 1 if n == "last" else at, ..., ch]).all()
                assert (got[n][..., other] - want[n][..., other]).norm() <= 2 * (ARITHMETIC + step) * want[n][..., other].norm()
            assert not torch.isfinite(got["o"][0, at:at + 20, 1, ch]).any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_of_a_state_that_is_not_finite(dtype):
    """A column of the state is one of the results; the others stay as they are."""
    gen = torch.Generator().manual_seed(18)
    lv, d, ups = linear_leaves(gen, (1, 140, 1, 1, 64, 64, None), dtype, True)
    step = 0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    got, other = [], [c for c in range(64) if c != 9]
    for value in (0.5, math.inf, math.nan):
        lv["h0"][0, 0, 3, 9] = value
        o, last = mk.linear_attention(*(lv[n].cuda() for n in "qkv"), d.cuda(), initial_state=lv["h0"].cuda(), output_final_state=True)
        got.append([t.cpu().double() for t in (o, last)])
    for case in got[1:]:
        for a, b in zip(got[0], case):
            assert (a[..., other] - b[..., other]).norm() <= 2 * (ARITHMETIC + step) * a[..., other].norm() and not torch.isfinite(b[..., 9]).all()


def test_linear_does_not_depend_on_its_neighbours():
    """The same sequence in a batch, packed and by itself (short sequences: none of the calls is cut)."""
    gen = torch.Generator().manual_seed(9)
    lv, d, _ = linear_leaves(gen, (4, 200, 2, 2, 128, 128, None), torch.bfloat16, False)
    lv, d = {n: t.cuda() for n, t in lv.items()}, d.cuda()
    with torch.no_grad():
        batch, last = mk.linear_attention(*lv.values(), d, output_final_state=True)
        packed, plast = mk.linear_attention(*(t.reshape(1, -1, *t.shape[2:]) for t in lv.values()), d, output_final_state=True, cu_seqlens=torch.arange(5, dtype=torch.int32).cuda() * 200)
        for i in range(4):
            one, olast = mk.linear_attention(*(t[i:i + 1] for t in lv.values()), d, output_final_state=True)
            assert torch.equal(one[0], batch[i]) and torch.equal(olast[0], last[i]) and torch.equal(packed[0, 200 * i:200 * i + 200], batch[i]) and torch.equal(plast[i], last[i])


def test_linear_from_a_new_thread():
    """A thread that has called nothing of CUDA yet, and memory that the allocator has at hand."""
    import threading
    q = torch.randn(1, 200, 2, 128, device="cuda", dtype=torch.bfloat16)
    d = -torch.rand(2, device="cuda")
    with torch.no_grad():
        want, _ = mk.linear_attention(q, q, q, d)
        spare = torch.empty_like(want)
        del spare
        got = []
        run = threading.Thread(target=lambda: got.append(mk.linear_attention(q, q, q, d)[0]))
        run.start()
        run.join()
    assert len(got) == 1 and torch.equal(got[0], want)


def test_linear_backward_as_the_first_call_of_its_thread():
    """In a process of its own: the thread that torch runs backward passes in has called nothing of CUDA yet."""
    import os
    import subprocess
    import sys
    code = """
import torch
import mogankda_b200 as mk
q, k, v = (torch.randn(1, 200, 2, 128, device="cuda", dtype=torch.bfloat16) for _ in range(3))
d, up = -torch.rand(2, device="cuda"), torch.randn_like(v)
spare = [torch.empty_like(v) for _ in range(8)]
del spare
for x in (q, k, v):
    x.requires_grad_(True)
o, _ = mk.linear_attention(q, k, v, d)
g = torch.autograd.grad(o, (q, k, v), up)
assert all(torch.isfinite(x).all() for x in g) and mk.device_status() == 0
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=root, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]


def test_linear_refuses():
    q, v, d = torch.randn(1, 5, 2, 16).cuda(), torch.randn(1, 5, 4, 16).cuda(), -torch.rand(4).cuda()
    for bad in (lambda: mk.linear_attention(q, q, v[:, :, :3], d[:3]), lambda: mk.linear_attention(q, q.bfloat16(), v, d), lambda: mk.linear_attention(q, q[..., :8], v, d),
                lambda: mk.linear_attention(q, q, v, d[:2]), lambda: mk.linear_attention(q, q, v[:, :4], d), lambda: mk.linear_attention(q.double(), q.double(), v.double(), d),
                lambda: mk.linear_attention(q, q, v, d, initial_state=torch.zeros(1, 4, 16, 16).cuda().bfloat16()), lambda: mk.linear_attention(q, q, v, d, initial_state=torch.zeros(1, 4, 16, 8).cuda()),
                lambda: mk.linear_attention(torch.randn(1, 5, 2, 129).cuda(), torch.randn(1, 5, 2, 129).cuda(), v, d), lambda: mk.linear_attention_step(q[0], q[0], v[0], d, torch.zeros(5, 4, 16, 8).cuda()),
                lambda: mk.linear_attention_step(q[0], q[0], v[0], d, torch.zeros(5, 4, 16, 16).cuda().transpose(2, 3))):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(ValueError):
        mk.linear_attention(q, q, v, d, initial_state=torch.zeros(2, 4, 16, 16).cuda())
    with pytest.raises(ValueError):
        mk.linear_attention(q.expand(2, 5, 2, 16), q.expand(2, 5, 2, 16), v.expand(2, 5, 4, 16), d, cu_seqlens=torch.tensor([0, 5]).cuda())
    with pytest.raises(RuntimeError, match="log_decay"):
        mk.linear_attention(q, q, v, d.clone().requires_grad_(True))
    with pytest.raises(RuntimeError, match="no_grad"):
        mk.linear_attention_step(q[0], q[0], v[0].requires_grad_(True), d, torch.zeros(5, 4, 16, 16).cuda())
    x = torch.randn(1, 5, 2, 16).cuda().requires_grad_(True)
    o, _ = mk.linear_attention(x, x, v.detach(), d)
    (g,) = torch.autograd.grad(o.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="double backward"):
        g.sum().backward()


def test_linear_past_32_bits():
    """More than 2^31 elements in each tensor: the last heads of the last tokens against a call of their own."""
    T, H, D = 135000, 128, 128
    assert T * H * D > 2 ** 31
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(1, T, H, D, generator=gen, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    d = torch.full((H,), -0.5, device="cuda")              # a thousand tokens are all that it remembers
    with torch.no_grad():
        o, last = mk.linear_attention(q, k, v, d, output_final_state=True)
        part, plast = mk.linear_attention(*(t[:, -2000:, -2:].contiguous() for t in (q, k, v)), d[-2:], output_final_state=True)
    near("o", o[:, -1000:, -2:].float(), part[:, -1000:].double(), terms=torch.finfo(torch.bfloat16).eps / ARITHMETIC * part[:, -1000:].double().norm().item())
    near("last", last[:, -2:], plast.double())


# ---- rotary positions ------------------------------------------------------------------------------------------------------------------------
def rotary_reference(x, angle, interleaved):
    n = angle.shape[-1]
    z = x[..., :2 * n]
    a, b = (z[..., 0::2], z[..., 1::2]) if interleaved else (z[..., :n], z[..., n:])
    c, s = torch.cos(angle)[..., None, :], torch.sin(angle)[..., None, :]
    a, b = a * c - b * s, a * s + b * c
    return torch.cat([torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1), x[..., 2 * n:]], -1)


ROTARY = [  # lead, HQ, HK, D, F, axes
    ((1, 1), 1, 1, 2, 1, 0), ((3,), 4, 0, 128, 64, 0), ((2, 37), 5, 2, 64, 32, 3), ((1, 100), 3, 1, 96, 24, 2), ((2, 3, 7), 2, 2, 50, 25, 3), ((9,), 1, 1, 7, 2, 0), ((40,), 40, 8, 128, 64, 3),
    ((5,), 2, 1, 512, 256, 4), ((4,), 3, 1, 16, 0, 0), ((0, 5), 2, 1, 16, 8, 0), ((), 2, 1, 16, 8, 0), ((1, 4000), 2, 1, 24, 8, 0), ((33,), 2, 3, 72, 35, 1),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", ROTARY, ids=str)
@pytest.mark.parametrize("interleaved", [False, True], ids=["halves", "neighbours"])
def test_rotary(shape, dtype, interleaved):
    lead, HQ, HK, D, F, axes = shape
    gen = torch.Generator().manual_seed(D + F)
    lv = dict(q=rand(gen, *lead, HQ, D).to(dtype))
    if HK:
        lv["k"] = rand(gen, *lead, HK, D).to(dtype)
    freq = (10000.0 ** (-torch.arange(F) / max(F, 1))).float()
    most = 2 ** 31 - 1 if D % 4 else 100000                # far positions: 64-bit angles of 2^31 turns are exact to 2^-21
    pos = torch.randint(-5, most, ((axes, *lead) if axes else lead), generator=gen, dtype=torch.int64)
    pos = pos.to(torch.int32) if D % 3 else pos
    of = [int(i) for i in torch.randint(0, axes, (F,), generator=gen)] if axes else None
    at = pos[of] if axes else pos[None].expand(F, *lead)
    angle = at.double().movedim(0, -1) * freq.double()
    ups = [rand(gen, *t.shape).to(dtype) for t in lv.values()]
    mine = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}
    wide = {n: t.double().requires_grad_(True) for n, t in lv.items()}

    def call():
        got = mk.rotary(mine["q"], mine.get("k"), pos.cuda(), freq.cuda(), axes=of, interleaved=interleaved)
        return got if HK else (got,)

    outs, grads = differentiate(call, mine, [u.cuda() for u in ups], list(lv))
    routs, rgrads = differentiate(lambda: [rotary_reference(t, angle, interleaved) for t in wide.values()], wide, [u.double() for u in ups], list(lv))
    for n, a, b in zip([n for n in lv] + ["d" + n for n in lv], outs + grads, routs + rgrads):
        near(n, a.cpu(), b)
        if F == 0:
            assert torch.equal(a.cpu().double(), b)


def test_rotary_of_slices_and_one_gradient():
    gen = torch.Generator().manual_seed(2)
    w = rand(gen, 2, 30, 6 * 64 + 8).cuda().bfloat16().requires_grad_(True)
    pos, freq = torch.arange(30).expand(2, 30).cuda(), torch.rand(32, generator=gen).cuda()
    up = rand(gen, 2, 30, 4, 64).cuda().bfloat16()
    got = []
    for copy in (False, True):
        q, k = w[..., :256].unflatten(-1, (4, 64)), w[..., 256:384].unflatten(-1, (2, 64))
        if copy:
            q, k = q.contiguous(), k.contiguous()
        a, b = mk.rotary(q, k, pos, freq)
        got.append((a, b, *torch.autograd.grad(a, w, up)))           # nothing comes back through k
    assert all(torch.equal(x, y) for x, y in zip(*got)) and got[0][2][..., 256:].abs().max() == 0
    with torch.no_grad():                                             # halves of a head turned in place of their order
        odd = mk.rotary(torch.cat([w[..., :1], w], -1)[..., 1:257].unflatten(-1, (4, 64)), None, pos, freq)
    assert torch.equal(odd, got[0][0])


def test_rotary_refuses():
    q, pos, freq = torch.randn(2, 5, 4, 16).cuda(), torch.zeros(2, 5, dtype=torch.long).cuda(), torch.ones(8).cuda()
    for bad in (lambda: mk.rotary(q, q.bfloat16(), pos, freq), lambda: mk.rotary(q, None, pos.float(), freq), lambda: mk.rotary(q, None, pos[:, :4], freq), lambda: mk.rotary(q, None, pos, freq.double()),
                lambda: mk.rotary(q, None, pos, torch.ones(9).cuda()), lambda: mk.rotary(q, None, pos, freq, axes=[0] * 8), lambda: mk.rotary(q, None, pos[None], freq),
                lambda: mk.rotary(q, None, pos[None], freq, axes=[0] * 7), lambda: mk.rotary(q, None, pos[None], freq, axes=[0] * 7 + [1]), lambda: mk.rotary(q, None, pos[None], freq, axes=[-1] * 8),
                lambda: mk.rotary(q, q[:1], pos, freq), lambda: mk.rotary(torch.randn(2, 5, 1, 514).cuda(), None, pos, freq)):
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(TypeError):
        mk.rotary(q, None, pos[None], freq, axes=[0.5] * 8)
    with pytest.raises(RuntimeError, match="inv_freq"):
        mk.rotary(q, None, pos, freq.clone().requires_grad_(True))


def test_rotary_gradients_are_linear():
    """A gradient of q is no function of q: a penalty on it has nothing to come back through, one on the incoming gradient raises."""
    q, pos, freq = torch.randn(5, 4, 16).cuda().requires_grad_(True), torch.arange(5).cuda(), torch.ones(8).cuda()
    (g,) = torch.autograd.grad(mk.rotary(q, None, pos, freq).sum(), q, create_graph=True)
    assert not g.requires_grad
    (g,) = torch.autograd.grad(mk.rotary(q, None, pos, freq).square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="double backward"):
        g.sum().backward()


def test_rotary_past_32_bits():
    T, H, D = 70000, 256, 128
    q = torch.zeros(T, H, D, dtype=torch.bfloat16, device="cuda")
    q[-3:] = torch.randn(3, H, D, device="cuda").bfloat16()
    pos, freq = torch.arange(T).cuda(), torch.rand(64).cuda()
    assert q.numel() > 2 ** 31
    with torch.no_grad():
        assert torch.equal(mk.rotary(q, None, pos, freq)[-3:], mk.rotary(q[-3:].clone(), None, pos[-3:], freq))


# ---- layer norm ------------------------------------------------------------------------------------------------------------------------------
def layer_norm_reference(x, w, b, res, groups, held):
    s = x
    if res is not None:
        s = x + res
        s = s + (s.detach().to(held).double() - s.detach())      # rounded; its derivative is one
    g = s.unflatten(-1, (groups, -1))
    d = g - g.mean(-1, keepdim=True)
    y = (d / torch.sqrt(d.square().mean(-1, keepdim=True) + 1e-5)).flatten(-2)
    y = y * w if w is not None else y
    return (y + b if b is not None else y), s if res is not None else None


NORM = [  # lead, width, groups
    ((1,), 1, 1), ((3,), 8, 1), ((2, 5), 33, 1), ((7,), 256, 1), ((4,), 257, 1), ((5,), 1000, 1), ((3,), 1025, 1), ((2,), 2048, 1), ((3,), 2056, 1), ((2,), 4096, 1), ((2,), 8192, 1),
    ((2,), 8200, 1), ((2,), 20000, 1), ((1,), 32768, 1), ((0,), 64, 1), ((), 64, 1), ((700,), 64, 1), ((9,), 1024, 8), ((3,), 35, 5), ((5,), 4096, 4), ((2, 3), 66, 33), ((1500,), 256, 2), ((2,), 65536, 2),
    ((2,), 2100, 2), ((600,), 520, 1),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", NORM, ids=str)
@pytest.mark.parametrize("option", ["plain", "all", "wide", "bias"])
def test_layer_norm(shape, dtype, option):
    lead, W, groups = shape
    gen = torch.Generator().manual_seed(W + groups)
    x = rand(gen, *lead, W) + 0.5
    lv = dict(x=x.to(dtype))
    held = torch.float32 if option == "wide" else dtype
    if option in ("all", "wide"):
        lv.update(w=1 + 0.1 * rand(gen, W).to(torch.bfloat16 if option == "wide" else torch.float32), b=rand(gen, W), res=(2 * rand(gen, *lead, W)).to(held))
    elif option == "bias":
        lv.update(b=rand(gen, W).to(dtype))
    ups = [rand(gen, *lead, W).to(dtype), rand(gen, *lead, W).to(held)]
    mine = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}
    wide = {n: t.double().requires_grad_(True) for n, t in lv.items()}

    def call():
        got = mk.layer_norm(mine["x"], mine.get("w"), mine.get("b"), residual=mine.get("res"), groups=groups)
        return got if "res" in lv else (got,)

    outs, grads = differentiate(call, mine, [u.cuda() for u in ups], list(lv))
    routs, rgrads = differentiate(lambda: layer_norm_reference(wide["x"], wide.get("w"), wide.get("b"), wide.get("res"), groups, held), wide, [u.double() for u in ups], list(lv))
    ups0 = ups[0].double().norm().item()
    for n, a, b in zip((["y", "s"] if "res" in lv else ["y"]) + ["d" + n for n in lv], outs + grads, routs + rgrads):
        # few channels to a part: what is left of the incoming gradient may be little of it; times at most 1 / sqrt(var + eps), of the smallest of the parts
        terms = 0.0
        if n in ("dx", "dres") and a.numel():
            s = (wide["x"] + (wide["res"] if "res" in lv else 0)).detach().unflatten(-1, (groups, -1))
            terms = ups0 * (s.var(-1, correction=0).min().item() + 1e-5) ** -0.5
        near(n, a.cpu(), b, terms)


def test_layer_norm_of_far_means_and_outliers():
    """A mean a thousand times the deviation, and one channel a thousand times the others: sums of differences to the mean in 32 bits.  The inputs are what 32 bits hold; the
    difference to the mean loses 2^-24 of the mean, 2^-14 of the deviation."""
    gen = torch.Generator().manual_seed(1)
    x = rand(gen, 6, 4096)
    x[:3] += 1000.0
    x[3:, 7] = 1000.0
    y = mk.layer_norm(x.cuda()).cpu().double()
    ref, _ = layer_norm_reference(x.double(), None, None, None, 1, None)
    assert (y - ref).abs().max() <= 2.0 ** -14 * (1 + ref[:3].abs().max()) and (y - ref)[3:].norm() <= ARITHMETIC * ref[3:].norm()


def test_layer_norm_of_what_is_not_finite():
    """Stays in its row, or its part of one."""
    x = torch.randn(5, 64).cuda()
    clean = mk.layer_norm(x, groups=4)
    x[2, 20], x[3, 0] = math.inf, math.nan
    y = mk.layer_norm(x, groups=4)
    assert torch.isnan(y[2, 16:32]).all() and torch.isnan(y[3, :16]).all()
    y[2, 16:32], y[3, :16] = clean[2, 16:32], clean[3, :16]
    assert torch.equal(y, clean)


def test_layer_norm_reads_slices():
    gen = torch.Generator().manual_seed(3)
    wide = rand(gen, 40, 3 * 264 + 8).cuda().bfloat16()
    w, b = rand(gen, 264).cuda(), rand(gen, 264).cuda()
    for start in (0, 8, 264, 3):
        x = wide[:, start:start + 264]
        leaf = x.detach().clone().requires_grad_(True)
        up = rand(gen, 40, 264).cuda().bfloat16()
        y = mk.layer_norm(leaf, w, b, groups=3)
        (want,) = torch.autograd.grad(y, leaf, up)
        whole = wide.clone().requires_grad_(True)
        z = mk.layer_norm(whole[:, start:start + 264], w, b, groups=3)
        (got,) = torch.autograd.grad(z, whole, up)
        assert torch.equal(y, z) and torch.equal(got[:, start:start + 264], want)


def test_layer_norm_refuses():
    x = torch.randn(4, 64).cuda()
    for bad in (lambda: mk.layer_norm(x, torch.ones(63).cuda()), lambda: mk.layer_norm(x, None, torch.ones(1, 64).cuda()), lambda: mk.layer_norm(x, groups=3), lambda: mk.layer_norm(x, groups=0),
                lambda: mk.layer_norm(x, residual=x[:2]), lambda: mk.layer_norm(x, residual=x.bfloat16()), lambda: mk.layer_norm(x.double()), lambda: mk.layer_norm(torch.randn(2, 32769).cuda())):
        with pytest.raises(AssertionError):
            bad()
    leaf = torch.randn(4, 64).cuda().requires_grad_(True)
    (g,) = torch.autograd.grad(mk.layer_norm(leaf).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="double backward"):
        g.sum().backward()


def test_layer_norm_past_32_bits():
    x = torch.zeros(70000, 32768, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn(3, 32768, device="cuda").bfloat16()
    assert x.numel() > 2 ** 31
    with torch.no_grad():
        for groups in (1, 256):
            assert torch.equal(mk.layer_norm(x, groups=groups)[-3:], mk.layer_norm(x[-3:].clone(), groups=groups))


# ---- together --------------------------------------------------------------------------------------------------------------------------------
def mixer(mine, x, w, pos, freq, d, nw, cu, reference=False):
    """A token mixer of heads with decays: projections, rotary positions, the linear attention, the norm of each head, and the residual's norm behind it."""
    H, D = 4, 64
    q, k, v = (x @ w).unflatten(-1, (3 * H, D)).split(H, -2)
    if reference:
        angle = pos[..., None].double() * freq.double()
        q, k = (rotary_reference(t, angle, False) for t in (q, k))
        o, _ = linear_reference(q, k, v, d.double(), D ** -0.5, None, cu)
        y, _ = layer_norm_reference(o.flatten(-2), nw, None, None, H, None)
        return layer_norm_reference(y, None, None, x, 1, torch.float64)
    q, k = mine.rotary(q, k, pos, freq)
    o, _ = mine.linear_attention(q, k, v, d, cu_seqlens=cu)
    y = mine.layer_norm(o.flatten(-2), nw, groups=H)
    return mine.layer_norm(y, residual=x)


def mixer_inputs(gen):
    x, w, nw = rand(gen, 1, 150, 256), rand(gen, 256, 3 * 256) / 16, 1 + 0.1 * rand(gen, 256)
    pos, freq, d = torch.cat([torch.arange(60), torch.arange(90)])[None], (100.0 ** (-torch.arange(32) / 32)).float(), -torch.rand(4, generator=gen)
    return x, w, nw, pos, freq, d, [rand(gen, 1, 150, 256) for _ in range(2)]


def test_a_block_of_them():
    """fp32, forward and backward; four operators in a row, each within 2^-17 of its input's error, and the products in front of them in 32 bits: within 2^-14."""
    gen = torch.Generator().manual_seed(11)
    x, w, nw, pos, freq, d, ups = mixer_inputs(gen)
    cu = (0, 60, 150)
    mine = {n: t.cuda().requires_grad_(True) for n, t in dict(x=x, w=w, nw=nw).items()}
    wide = {n: t.double().requires_grad_(True) for n, t in dict(x=x, w=w, nw=nw).items()}
    outs = mixer(mk, mine["x"], mine["w"], pos.cuda(), freq.cuda(), d.cuda(), mine["nw"], torch.tensor(cu, dtype=torch.int32).cuda())
    routs = mixer(mk, wide["x"], wide["w"], pos, freq, d, wide["nw"], cu, True)
    grads = torch.autograd.grad(outs, list(mine.values()), [u.cuda() for u in ups])
    rgrads = torch.autograd.grad(routs, list(wide.values()), [u.double() for u in ups])
    for a, b in zip((*outs, *grads), (*routs, *rgrads)):
        assert (a.cpu().double() - b).norm() <= 2.0 ** -14 * b.norm()


def test_a_block_of_them_in_a_graph_on_another_stream():
    """Captured and replayed on new inputs, twice over (two graphs), beside calls on another stream."""
    gen = torch.Generator().manual_seed(12)
    x, w, nw, pos, freq, d, ups = [t.cuda() if torch.is_tensor(t) else [u.cuda() for u in t] for t in mixer_inputs(gen)]
    cu = torch.tensor((0, 60, 150), dtype=torch.int32).cuda()

    def step(leaf):
        outs = mixer(mk, leaf, w, pos, freq, d, nw, cu)
        return (*outs, *torch.autograd.grad(outs, leaf, ups))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        step(x.clone().requires_grad_(True))
        for _ in range(2):
            static = x.clone().requires_grad_(True)
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs = step(static)
            graphs.append((graph, static, outs))
    torch.cuda.current_stream().wait_stream(side)
    for i in range(3):
        for j, (graph, static, _) in enumerate(graphs):
            with torch.no_grad():
                static.copy_(torch.roll(x, i + j, 1))
            graph.replay()
        with torch.cuda.stream(side):
            other = step(torch.roll(x, 7, 1).requires_grad_(True))
        for j, (_, _, outs) in enumerate(graphs):
            want = step(torch.roll(x, i + j, 1).requires_grad_(True))
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
    torch.cuda.synchronize()
    assert all(torch.isfinite(t).all() for t in other)


def test_single_tokens_in_a_graph():
    gen = torch.Generator().manual_seed(13)
    N, H, D = 3, 2, 128
    q, k, v = (rand(gen, N, H, D).cuda().bfloat16() for _ in range(3))
    d, pos, freq, state = -torch.rand(H, generator=gen).cuda(), torch.zeros(N, dtype=torch.int32).cuda(), torch.rand(64, generator=gen).cuda(), torch.zeros(N, H, D, D).cuda()
    keep = state.clone()

    def step(s):
        a, b = mk.rotary(q, k, pos, freq)
        return mk.layer_norm(mk.linear_attention_step(a, b, v, d, s).flatten(-2), groups=H)

    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        step(keep.clone())
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            y = step(state)
        for t in range(4):
            pos.fill_(t)
            graph.replay()
            want = step(keep)
            assert torch.equal(y, want) and torch.equal(state, keep)


def test_gradients_that_arrive_broadcast_or_alone():
    """A sum's gradient is one number for all elements; a result that nobody uses has none.  The definition's gradients are taken of the other results alone."""
    gen = torch.Generator().manual_seed(23)
    for dtype in (torch.float32, torch.bfloat16):
        lv, d, ups = linear_leaves(gen, (1, 140, 1, 2, 64, 64, None), dtype, True)
        x = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}
        for decay in (d, d.to(dtype)):
            o, last = mk.linear_attention(x["q"], x["k"], x["v"], decay.cuda(), initial_state=x["h0"], output_final_state=True)
            wide = torch.autograd.grad(o.float().sum() + last.sum(), list(x.values()), retain_graph=True)
            full = torch.autograd.grad((o, last), list(x.values()), (torch.ones_like(o), torch.ones_like(last)), retain_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(wide, full))
            alone = torch.autograd.grad(last, list(x.values()), ups[1].cuda())
            r = {n: t.double().requires_grad_(True) for n, t in lv.items()}
            _, rlast = linear_reference(r["q"], r["k"], r["v"], decay.double(), 0.125, r["h0"], None, True)
            want = torch.autograd.grad(rlast, [r[n] for n in ("k", "v", "h0")], ups[1].double())
            assert alone[0].abs().max() == 0
            for n, a, b in zip(("dk", "dv", "dh0"), alone[1:], want):
                near(n, a.cpu(), b)
        s = rand(gen, 7, 96).to(dtype).cuda().requires_grad_(True)
        w = rand(gen, 96).cuda().requires_grad_(True)
        y, total = mk.layer_norm(s, w, residual=s, groups=3)
        both = torch.autograd.grad(y.sum() + total.sum(), (s, w), retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(both, torch.autograd.grad((y, total), (s, w), (torch.ones_like(y), torch.ones_like(total)), retain_graph=True)))
        ds, dw = torch.autograd.grad(total.sum(), (s, w))          # the stream alone: 1 from each of the two that are one tensor
        assert torch.equal(ds, torch.full_like(ds, 2)) and dw.abs().max() == 0
        q = rand(gen, 5, 2, 16).to(dtype).cuda().requires_grad_(True)
        args = torch.arange(5).cuda(), torch.tensor([1.0, 0.5, 0.25]).cuda()
        a, b = mk.rotary(q, q, *args)
        assert torch.equal(a, b)
        both = torch.autograd.grad(a.sum() + b.sum(), q, retain_graph=True)[0]
        one = torch.autograd.grad(a, q, torch.ones_like(a))[0]
        assert torch.equal(both, 2 * one)
