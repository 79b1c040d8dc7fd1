"""GPU: values of the linear attention where tokens, channels and decays differ by much, against its definition in 64 bits.

Tolerances are those of test_block_gpu.py (``near``).  They hold for the tokens and channels that a large one has no part in by themselves: those are compared apart."""

import pytest
import torch

import mogankda_b200 as mk
from tests.test_block_gpu import DTYPES, near, rand
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
