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
