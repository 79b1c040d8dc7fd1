"""GPU: the short convolution over thousands of packed sequences of which some are empty: these hand their state and its gradient through, whichever block of the kernel has
them, and the others are what they are in a batch of their own."""
import pytest
import torch

import mogankda_b200 as mk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("every,L,D", [(7, 3, 40), (2, 1, 33), (4000, 2, 136), (1, 5, 16)])
def test_empty_sequences_hand_their_state_through(every, L, D, dtype):
    """every = 1: all of them are empty, and the tokens belong to none."""
    gen = torch.Generator().manual_seed(every)
    n, W = 5000, 4
    empty = torch.zeros(n, dtype=torch.bool)
    empty[every // 2::every] = True
    lens = torch.where(empty, 0, L)
    x = torch.randn(1, max(int(lens.sum()), 3), D, generator=gen).to(dtype).cuda().requires_grad_(True)
    w = torch.randn(D, W, generator=gen).cuda()
    state = torch.randn(n, W - 1, D, generator=gen).to(dtype).cuda().requires_grad_(True)
    up, ups = torch.randn(x.shape, generator=gen).to(dtype).cuda(), torch.randn(state.shape, generator=gen).to(dtype).cuda()
    cu = torch.cat([torch.zeros(1, dtype=torch.long), lens.cumsum(0)]).cuda()
    y, last = mk.causal_conv1d(x, w, activation="silu", initial_state=state, output_final_state=True, cu_seqlens=cu)
    dx, ds = torch.autograd.grad((y, last), (x, state), (up, ups))
    e, there = empty.cuda(), int(lens.sum())
    assert torch.equal(last[e], state[e]) and torch.equal(ds[e], ups[e])
    assert (y[:, there:] == 0).all() and (dx[:, there:] == 0).all()
    if there:
        xb = x.detach()[:, :there].reshape(-1, L, D).requires_grad_(True)
        sb = state.detach()[~e].requires_grad_(True)
        yb, lb = mk.causal_conv1d(xb, w, activation="silu", initial_state=sb, output_final_state=True)
        gb, gs = torch.autograd.grad((yb, lb), (xb, sb), (up[:, :there].reshape(-1, L, D), ups[~e]))
        for a, b in ((y[:, :there].reshape(-1, L, D), yb), (last[~e], lb), (dx[:, :there].reshape(-1, L, D), gb), (ds[~e], gs)):
            assert torch.equal(a, b)
