"""GPU: scans of packed sequences of very different lengths, whole or cut into parts that run side by side (csrc/block.cpp: cut)."""
import pytest
import torch

import mogankda_b200 as mk
from tests.test_block_gpu import differentiate, near, rand, scan_leaves, scan_reference

pytestmark = pytest.mark.gpu


def workspace(docs, D, N=16):
    """Bytes that a forward call and its backward pass need beside what they return and keep for one another."""
    T = sum(docs)
    x = torch.randn(1, T, D, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    bc, A = torch.randn(1, T, N, device="cuda", dtype=torch.bfloat16), -torch.rand(D, N, device="cuda")
    cu = torch.tensor([0, *docs], device="cuda").cumsum(0)
    peaks = []
    for call in (lambda: mk.selective_scan(x.detach(), x.detach(), A, bc, bc, dt_softplus=True, cu_seqlens=cu)[0],
                 lambda: torch.autograd.grad(y, x, torch.ones_like(y))):
        if peaks:
            y = mk.selective_scan(x, x, A, bc, bc, dt_softplus=True, cu_seqlens=cu)[0]
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        call()
        peaks.append(torch.cuda.max_memory_allocated() - before)
    return peaks


def test_a_long_document_beside_many_short_ones_is_left_whole():
    """Every document would have a row of blocks for each part of the longest one, and a state of workspace: 513 x 16 rows here, 545 us where the whole document takes 140."""
    D, N, T = 128, 16, 8192
    forward, backward = workspace([4096] + [8] * 512, D, N)
    assert forward < 2 * T * D * 2 + (1 << 20)             # y, and no states of parts (513 x 16 of them are 67 MB)
    blocks = D // 32
    assert backward < 4 * T * D * 2 + 2 * blocks * T * N * 4 + 592 * D * N * 4 + (4 << 20)
    forward, _ = workspace([4096, 8, 8], D, N)
    assert forward > 4112 * D * 2 + 3 * 16 * D * N * 4      # few documents: parts of 256 tokens or less


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("short", [80, 300])
def test_scan_of_a_long_document_beside_short_ones(short, dtype):
    """80: cut in both directions, 300: backward only."""
    gen = torch.Generator().manual_seed(58)
    cu = [0, 5]
    for i in range(short):
        cu.append(cu[-1] + (1500 if i == short // 2 else i % 9))
    T = cu[-1] + 3
    lv = scan_leaves(gen, 1, T, 24, 16, 1, cu, dtype, True)
    ups = [rand(gen, 1, T, 24).to(dtype), rand(gen, len(cu) - 1, 24, 16)]
    args = ("x", "dt", "A", "B", "C", "D", "z", "bias")
    mine, wide = {n: t.cuda().requires_grad_(True) for n, t in lv.items()}, {n: t.double().requires_grad_(True) for n, t in lv.items()}
    outs, grads = differentiate(lambda: mk.selective_scan(*(mine[n] for n in args), dt_softplus=True, initial_state=mine["h0"], output_final_state=True,
                                                          cu_seqlens=torch.tensor(cu, device="cuda")), mine, [u.cuda() for u in ups], list(lv))
    routs, rgrads = differentiate(lambda: scan_reference(*(wide[n] for n in args), True, wide["h0"], cu, True), wide, [u.double() for u in ups], list(lv))
    for n, a, b in zip(["y", "last"] + ["d" + n for n in lv], outs + grads, routs + rgrads):
        near(n, a.cpu(), b)


@pytest.mark.parametrize("G", [1, 2])
def test_workspace_of_many_blocks_of_channels(G):
    """dB and dC are left per block of channels, 8 bytes per token, state and block: 512 blocks of 8 channels here.  More than 1 GiB of them are formed by ranges of blocks, whose
    sums are added up in between; all else has the bits of calls on fewer channels."""
    T, D, N, end = 6000, 4096, 64, 5990
    g = torch.Generator(device="cuda").manual_seed(61)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, dt, up = r(1, T, D), 0.1 * torch.rand(1, T, D, generator=g, device="cuda"), r(1, T, D)
    A, B, C, skip, h0, uph = -N * torch.rand(D, N, generator=g, device="cuda"), r(1, T, G, N), r(1, T, G, N), r(D), r(2, D, N), r(2, D, N)
    cu = torch.tensor([0, 5000, end], device="cuda")

    def gradients(ch, gr):
        leaves = [t.contiguous().requires_grad_(True) for t in (x[..., ch], dt[..., ch], A[ch], B[:, :, gr], C[:, :, gr], skip[ch], h0[:, ch])]
        y, end = mk.selective_scan(*leaves[:6], initial_state=leaves[6], output_final_state=True, cu_seqlens=cu)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got = torch.autograd.grad((y, end), leaves, (up[..., ch].contiguous(), uph[:, ch].contiguous()))
        return torch.cuda.max_memory_allocated() - before, got

    halves = [(slice(0, D // 2), slice(0, G // 2 or 1)), (slice(D // 2, D), slice(G // 2, G))]
    (_, a), (_, b) = (gradients(*h) for h in halves)
    peak, got = gradients(slice(0, D), slice(0, G))
    blocks = 512
    assert peak < 0.8 * 8 * blocks * T * N + 4 * 4 * T * D
    for i, dim in ((0, 2), (1, 2), (2, 0), (5, 0), (6, 1)):
        assert torch.equal(got[i], torch.cat([a[i], b[i]], dim))
    for i in (3, 4):
        assert (got[i][:, end:] == 0).all()
        near("dB, dC", got[i], torch.cat([a[i], b[i]], 2).double() if G > 1 else a[i].double() + b[i].double())
