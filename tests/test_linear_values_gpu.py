"""GPU: values of the linear attention where tokens, channels and decays differ by much, against its definition in 64 bits.

Tolerances are those of test_block_gpu.py (``near``).  They hold for the tokens and channels that a large one has no part in by themselves: those are compared apart."""
import math

import pytest
import torch

import mogankda_b200 as mk
from tests.test_block_gpu import ARITHMETIC, DTYPES, near, rand
from tests.test_mixer_gpu import linear_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(300, 128, 128, 200, 0.0625, 2.0 ** 10), (300, 128, 128, 130, 0.0625, 2.0 ** 13), (140, 64, 40, 70, 2.0 ** -6, 2.0 ** 12), (1300, 128, 64, 700, 0.0625, 2.0 ** 11)], ids=str)
@pytest.mark.parametrize("rate", [0.02, 3.0], ids=str)
def test_one_large_token(shape, dtype, rate):
    """One token's q, k, v and gradient from above are far larger than all others'.  In front of it (in the gradients of k and v: behind it) it has no part in anything; with a strong
    decay nothing is left of it twenty tokens further on."""
    T, K, V, at, small, large = shape
    gen = torch.Generator().manual_seed(T + at)
    size = dict(q=small, k=small, v=1.0, up=1.0)
    x = {n: (rand(gen, 1, T, 2, K if n in "qk" else V) * size[n]).to(dtype) for n in size}
    for n in x:
        x[n][0, at, :, 3] = large * (1 if n in "qk" else 4)
    d = torch.tensor([-rate, -2 * rate])
    mine = [x[n].cuda().requires_grad_(True) for n in "qkv"]
    wide = [x[n].double().requires_grad_(True) for n in "qkv"]
    o, _ = mk.linear_attention(*mine, d.cuda(), scale=1.0)
    ro, _ = linear_reference(*wide, d.double(), 1.0)
    got = dict(zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, mine, x["up"].cuda()))))
    ref = dict(zip(("o", "dq", "dk", "dv"), (ro, *torch.autograd.grad(ro, wide, x["up"].double()))))
    for n in got:
        near(n, got[n][:, slice(0, at) if n in ("o", "dq") else slice(at + 1, T)].detach().cpu(), ref[n][:, slice(0, at) if n in ("o", "dq") else slice(at + 1, T)].detach())
        if rate > 1:          # on its other side: exp(-3 x 30) of it, 2^-130
            far = slice(at + 31, T) if n in ("o", "dq") else slice(0, max(at - 30, 0))
            near(n, got[n][:, far].detach().cpu(), ref[n][:, far].detach())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(300, 128, 128), (900, 64, 64)], ids=str)
def test_one_large_channel(shape, dtype):
    """A channel of v is one of the results and of the states; each by itself is as exact as the others."""
    T, K, V = shape
    gen = torch.Generator().manual_seed(T)
    size = torch.full((V,), 2.0 ** -10)
    size[5] = 2.0 ** 13
    q, k, v = rand(gen, 1, T, 2, K).to(dtype), rand(gen, 1, T, 2, K).to(dtype), (rand(gen, 1, T, 2, V) * size).to(dtype)
    d = torch.tensor([-0.02, -0.5])
    with torch.no_grad():
        o, last = mk.linear_attention(q.cuda(), k.cuda(), v.cuda(), d.cuda(), scale=2.0 ** -7, output_final_state=True)
    ro, rlast = linear_reference(q.double(), k.double(), v.double(), d.double(), 2.0 ** -7, last=True)
    for c in (0, 4, 5, 6, V - 1):
        near("last", last[..., c].cpu(), rlast[..., c])
        if dtype != torch.float16 or c == 5:      # the others' results are too small for fp16
            near("o", o[..., c].cpu(), ro[..., c])


def test_the_final_state_leaves_results_as_exact():
    """What goes into a state has three parts where one leaves, else two (2^-16 off at most, 2^-17 in the root mean square): both calls' results round the same number but for that, and
    those that come out as neighbours, 2^-8 apart at least, are as many as 4 x 2^-17 / 2^-8 of them, four times over for the small ones among them."""
    gen = torch.Generator().manual_seed(2)
    q, k, v = (rand(gen, 1, 3000, 4, 128).bfloat16().cuda() for _ in range(3))
    d = -torch.tensor([1e-3, 1e-2, 0.1, 1.0]).cuda()
    with torch.no_grad():
        a, b = mk.linear_attention(q, k, v, d)[0].double(), mk.linear_attention(q, k, v, d, output_final_state=True)[0].double()
    assert (a - b).norm() <= 2 * (ARITHMETIC + 2.0 ** -8) * a.norm()
    assert (a != b).double().mean() <= 4 * 4 * ARITHMETIC / 2.0 ** -8


@pytest.mark.parametrize("dtype", DTYPES)
def test_later_tokens_leave_no_trace(dtype):
    """Not a bit of a result depends on tokens behind it (of a gradient of k or v: in front of it), however large these are, in a call that is not cut."""
    gen = torch.Generator().manual_seed(7)
    x = {n: rand(gen, 1, 300, 2, 64).to(dtype) for n in ("q", "k", "v", "up")}
    d = torch.tensor([-0.01, -0.3]).cuda()
    got = []
    for size in (1.0, 30000.0):
        for side in (slice(171, 300), slice(0, 171)):
            y = {n: t.clone() for n, t in x.items()}
            for t in y.values():
                t[:, side] *= size / 5
            leaves = [y[n].cuda().requires_grad_(True) for n in "qkv"]
            o, _ = mk.linear_attention(*leaves, d)
            g = torch.autograd.grad(o, leaves, y["up"].cuda())
            other = slice(0, 171) if side.start else slice(171, 300)
            got.append([t[:, other] for t in ((o, g[0]) if side.start else g[1:])])
    for a, b in ((got[0], got[2]), (got[1], got[3])):
        assert all(torch.isfinite(s).all() and torch.equal(s, t) for s, t in zip(a, b))


WEAK = [-1e-6, -3e-7, -1e-7, -1e-4, -0.03, -1.0, -20.0, 0.0]


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_steps_of_weak_decays(dtype):
    """4096 single tokens of memories that reach much further.  A step rounds its state twice, half a step each: 90 of 2^-24 / sqrt(3) in the root mean square, 3.1e-6, below 2^-17;
    a decay that is off by 2^-25 in each would be off by 1.2e-4 behind them.  That is for k v of 32 bits, whose last places make the roundings fall either way.  k v of 16-bit inputs has
    16 bits (fp16 22) and is mostly a whole multiple of the state's last place: there is nothing but the decay's own share to round, and all 4096 roundings, 2^-24 at most each, may fall the
    same way: 2^-12, which is 32 x 2^-17."""
    n, K, H = 4096, 16, len(WEAK)
    gen = torch.Generator().manual_seed(3)
    q, k, v = (rand(gen, n, 1, H, K).to(dtype).cuda() for _ in range(3))
    start = 64 * rand(gen, 1, H, K, K).cuda()
    d = torch.tensor(WEAK, dtype=torch.float32).cuda()
    state = start.clone()
    for t in range(n):
        o = mk.linear_attention_step(q[t], k[t], v[t], d, state)
    left = torch.exp(d.double()[:, None] * torch.arange(n - 1, -1, -1, device="cuda"))
    want = torch.exp(n * d.double())[:, None, None] * start[0].double() + torch.einsum("ht,thk,thv->hkv", left, k[:, 0].double(), v[:, 0].double())
    same_way = 0 if dtype == torch.float32 else 32
    for h in range(H):
        near(f"state of {WEAK[h]}", state[0, h], want[h], terms=same_way * want[h].norm().item())
    ref = K ** -0.5 * torch.einsum("hk,hkv->hv", q[-1, 0].double(), want)
    near("o", o[0], ref, terms=same_way * (K ** -0.5 * q[-1, 0].double().norm(dim=-1) * want.flatten(1).norm(dim=-1)).norm().item())


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_step_of_weak_decays(dtype):
    """The state behind a step is lam S + k v rounded once, 2^-24 of it, but for what is rounded in front of that: k v, 2^-24 of it, and its sum with the small part of lam S, which is
    2^-25 S at most: 2^-24 of both."""
    gen = torch.Generator().manual_seed(6)
    H, K = len(WEAK), 64
    q, k, v = (rand(gen, 3, H, K).to(dtype).cuda() for _ in range(3))
    start = 64 * rand(gen, 3, H, K, K).cuda()
    d = torch.tensor(WEAK, dtype=torch.float32).cuda()
    state = start.clone()
    mk.linear_attention_step(q, k, v, d, state)
    kv = k.double()[..., None] * v.double()[..., None, :]
    want = torch.exp(d.double())[:, None, None] * start.double() + kv
    assert ((state.double() - want).abs() <= 2.0 ** -24 * (want.abs() + 2 * kv.abs() + 2.0 ** -23 * start.double().abs())).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_prompts_of_weak_decays(dtype):
    """131072 tokens of more heads than there are SMs, so that no sequence is cut, with memories that reach further than that.  A state is multiplied once for 128 tokens, 1024 times: a
    decay rounded to 32 bits, off by up to 2^-25 with one sign for a head, would be off by 3e-5 behind them; sums of 1024 terms, rounded half a step each, are off by 32 x 2^-24."""
    T, H, K = 131072, 160, 8
    gen = torch.Generator(device="cuda").manual_seed(4)
    q, k, v = (torch.randn(1, T, H, K, generator=gen, device="cuda").to(dtype) for _ in range(3))
    d = -1e-6 * torch.rand(H, generator=gen, device="cuda")
    start = torch.randn(1, H, K, K, generator=gen, device="cuda") * 256
    with torch.no_grad():
        _, last = mk.linear_attention(q, k, v, d, initial_state=start, output_final_state=True)
    at = torch.arange(T - 1, -1, -1, device="cuda")
    for h in range(0, H, 5):
        r = d[h].double()
        want = torch.exp(T * r) * start[0, h].double() + (k[0, :, h].double() * torch.exp(r * at)[:, None]).t() @ v[0, :, h].double()
        near(f"state of {d[h].item()}", last[0, h], want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_steps_of_states_that_are_not_finite(dtype):
    """An infinity stays one where something is left of it, NaN stays NaN, and neither reaches another column."""
    state = torch.ones(1, 3, 8, 8, device="cuda")
    state[0, :, 2, 3], state[0, :, 4, 5] = math.inf, math.nan
    one = torch.ones(1, 3, 8, device="cuda").to(dtype)
    o = mk.linear_attention_step(one, one, one, torch.tensor([0.0, -1e-7, -1.0]).cuda(), state)
    assert (state[0, :, 2, 3] == math.inf).all() and torch.isnan(state[0, :, 4, 5]).all()
    assert (o[0, :, 3].float() == math.inf).all() and torch.isnan(o[0, :, 5]).all()
    rest = [c for c in range(8) if c not in (3, 5)]
    assert torch.isfinite(state[..., rest]).all() and torch.isfinite(o[..., rest]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_sums_of_shared_heads_leave_tokens_in_front_of_the_first_sequence_alone(dtype):
    """The C entry point takes boundaries that begin behind the first token; rows of no sequence are written by nobody."""
    from mogankda_b200 import _lib
    lib, S = _lib.load(), _lib.STRUCTS
    gen = torch.Generator().manual_seed(5)
    TT, HK, HV, K, first, end = 40, 1, 2, 16, 8, 30
    x = {n: rand(gen, TT, h, K).to(dtype).cuda() for n, h in (("q", HK), ("k", HK), ("v", HV), ("d_o", HV))}
    cu, d = torch.tensor([first, end], dtype=torch.int32).cuda(), torch.tensor([-0.1, -0.2]).cuda()
    got = {n: torch.full_like(x[m], 7.0) for n, m in (("dq", "q"), ("dk", "k"), ("dv", "v"))}
    part = {n: torch.full((TT, HV, K), 3.0).cuda() for n in ("part_q", "part_k")}
    p = S["MkdaLinearBwd"]()
    f = p.f
    f.S.N, f.S.T, f.S.TT, f.S.cu = 1, TT, TT, cu.data_ptr()
    f.HK, f.HV, f.K, f.V, f.scale, f.dtype = HK, HV, K, K, 0.25, {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype]
    f.q, f.k, f.v, f.log_decay = (t.data_ptr() for t in (x["q"], x["k"], x["v"], d))
    f.q_stride, f.k_stride, f.v_stride = HK * K, HK * K, HV * K
    p.d_o, p.end = x["d_o"].data_ptr(), end
    for n, t in (*got.items(), *part.items()):
        setattr(p, n, t.data_ptr())
    import ctypes
    torch.cuda.synchronize()
    assert lib.mkda_linear_bwd(ctypes.byref(p), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    leaves = [x[n][None, first:end].double().cpu().requires_grad_(True) for n in "qkv"]
    o, _ = linear_reference(*leaves, d.double().cpu(), 0.25)
    for n, r in zip(got, torch.autograd.grad(o, leaves, x["d_o"][None, first:end].double().cpu())):
        near(n, got[n][first:end].cpu(), r[0])
        assert (got[n][:first] == 7).all() and (got[n][end:] == 7).all(), n
