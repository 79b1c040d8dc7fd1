"""GPU: gradients of the gradients of the layer and of the operators around it are not provided: a program that needs them gets an error, never a sum with a term
missing; one whose gradients do not depend on what it differentiates by gets its result."""
import pytest
import torch

import mogankda_b200 as mk

pytestmark = pytest.mark.gpu


def leaves(*shapes):
    gen = torch.Generator().manual_seed(3)
    return [torch.randn(*s, generator=gen).cuda().requires_grad_(True) for s in shapes]


def operators():
    """name -> (function of its leaves, the leaves)"""
    x, res, w, z = leaves((1, 40, 32), (1, 40, 32), (32, 4), (1, 40, 32))
    dt, bc = leaves((1, 40, 32), (1, 40, 16))
    A = (-torch.rand(32, 16, device="cuda")).requires_grad_(True)
    q, v = leaves((1, 40, 1, 128), (1, 40, 2, 128))
    g = (-torch.rand(1, 40, 2, 128, device="cuda")).requires_grad_(True)
    beta = torch.rand(1, 40, 2, device="cuda").requires_grad_(True)
    return {
        "norm": (lambda x, w: mk.rms_norm(x, w[:, 0]), (x, w)),
        "norm of a sum": (lambda x, res: mk.rms_norm(x, residual=res)[0], (x, res)),
        "stream of a norm": (lambda x, res: (lambda y, s: y * s)(*mk.rms_norm(x, residual=res)), (x, res)),
        "convolution": (lambda x, w: mk.causal_conv1d(x, w)[0], (x, w)),
        "convolution with SiLU": (lambda x: mk.causal_conv1d(x, w.detach(), activation="silu")[0], (x,)),
        "scan": (lambda x, dt, A, bc: mk.selective_scan(x, dt, A, bc, bc, dt_softplus=True)[0], (x, dt, A, bc)),
        "gated scan by its gate": (lambda z: mk.selective_scan(x.detach(), dt.detach(), A.detach(), bc.detach(), bc.detach(), z=z)[0], (z,)),
        "layer": (lambda q, v, g, beta: mk.chunk_kda(q, q, v, g, beta)[0], (q, v, g, beta)),
        "layer by its keys": (lambda k: mk.chunk_kda(q.detach(), k, v.detach(), g.detach(), beta.detach(), use_qk_l2norm_in_kernel=True)[0], (q,)),
    }


NAMES = ["norm", "norm of a sum", "stream of a norm", "convolution", "convolution with SiLU", "scan", "gated scan by its gate", "layer", "layer by its keys"]


@pytest.mark.parametrize("name", NAMES)
def test_a_penalty_on_a_gradient_is_refused(name):
    """The incoming gradient is a constant here: what the penalty depends on are the saved inputs."""
    fn, lv = operators()[name]
    y = fn(*lv)
    got = torch.autograd.grad(y.sum(), lv, create_graph=True)
    total = y.sum() + sum(g.square().sum() for g in got)
    with pytest.raises(RuntimeError, match="double backward"):
        torch.autograd.grad(total, lv, retain_graph=True)
    with pytest.raises(RuntimeError, match="double backward"):
        torch.autograd.grad(got[0].sum(), lv, allow_unused=True, retain_graph=True)
    with pytest.raises(RuntimeError, match="double backward"):
        total.backward()


@pytest.mark.parametrize("name", NAMES)
def test_a_gradient_that_nobody_differentiates_is_the_same(name):
    fn, lv = operators()[name]
    y = fn(*lv)
    got = torch.autograd.grad(y.sum(), lv, create_graph=True)
    y.sum().backward(create_graph=True)
    for a, b, t in zip(got, torch.autograd.grad(fn(*lv).sum(), lv), lv):
        assert torch.equal(a, b) and torch.equal(t.grad, b)
        t.grad = None


def test_an_incoming_gradient_is_reached_too():
    for name, (fn, lv) in operators().items():
        up = torch.ones_like(fn(*lv)).requires_grad_(True)
        got = torch.autograd.grad(fn(*lv), lv, up, create_graph=True)
        with pytest.raises(RuntimeError, match="double backward"):
            torch.autograd.grad(sum(g.sum() for g in got), up)


def test_gradients_that_depend_on_nothing_stay_usable():
    """Operators that are linear in the only argument that wants a gradient: that gradient is a constant, and a penalty on it adds nothing."""
    x, w, s, v, h0, q = leaves((1, 40, 32), (32, 4), (1, 3, 32), (1, 40, 2, 128), (1, 2, 128, 128), (1, 40, 2, 128))
    A, bc, one = -torch.rand(32, 16, device="cuda"), torch.randn(1, 40, 16, device="cuda"), torch.ones(1, 40, 32, device="cuda")
    g, beta, k = -torch.rand(1, 40, 2, 128, device="cuda"), torch.rand(1, 40, 2, device="cuda"), torch.randn(1, 40, 2, 128, device="cuda") * 0.1
    const = torch.randn(1, 40, 2, 128, device="cuda")
    for fn, lv in (
        (lambda x, s: mk.causal_conv1d(x, w.detach(), initial_state=s)[0], (x, s)), (lambda w: mk.causal_conv1d(x.detach(), w)[0], (w,)),
        (lambda w: mk.rms_norm(x.detach(), w[:, 0]), (w,)), (lambda x: mk.selective_scan(x, one, A, bc, bc)[0], (x,)),
        (lambda c: mk.selective_scan(x.detach(), one, A, bc, c.mT, w[:, 0].detach())[0], (torch.randn(1, 16, 40, device="cuda").requires_grad_(True),)),
        (lambda D: mk.selective_scan(x.detach(), one, A, bc, bc, D[:, 0])[0], (w,)),
        (lambda v, h0: mk.chunk_kda(const, k, v, g, beta, initial_state=h0)[0], (v, h0)), (lambda q: mk.chunk_kda(q, k, const, g, beta)[0], (q,)),
    ):
        y = fn(*lv)
        want = torch.autograd.grad(y.sum(), lv, retain_graph=True)
        got = torch.autograd.grad(y.sum(), lv, create_graph=True)
        total = torch.autograd.grad(y.sum() + sum(g.square().sum() for g in got), lv)
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, total))


def test_gradients_of_a_stream_or_a_state_alone_stay_usable():
    """The sum in front of a norm and the tokens that a convolution keeps are linear in what they come from, whatever the other output is."""
    x, res, w, s = leaves((1, 2, 32), (1, 2, 32), (32, 4), (1, 3, 32))
    for fn, lv in ((lambda x, res: mk.rms_norm(x, w[:, 0], residual=res)[1], (x, res)),
                   (lambda x, s: mk.causal_conv1d(x, w, activation="silu", initial_state=s, output_final_state=True)[1], (x, s))):
        y = fn(*lv)
        want = torch.autograd.grad(y.sum(), lv, retain_graph=True)
        got = torch.autograd.grad(y.sum(), lv, create_graph=True)
        for a, b, c in zip(want, got, torch.autograd.grad(y.sum() + sum(g.square().sum() for g in got), lv)):
            assert torch.equal(a, b) and torch.equal(a, c)
        with pytest.raises(RuntimeError, match="double backward"):
            up = torch.ones_like(y).requires_grad_(True)
            torch.autograd.grad(torch.autograd.grad(fn(*lv), lv, up, create_graph=True)[0].sum(), up)
