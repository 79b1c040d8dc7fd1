"""CPU: the entry points of the linear attention, the rotary positions and the layer norm refuse what they cannot take before anything is launched."""
import pytest
import torch

import mogankda_b200 as mk
from tests.test_block import _filled, _refused


@pytest.fixture(scope="module")
def lib():
    from mogankda_b200 import _lib, build
    build.build()
    return _lib.load()


def test_cpu_tensors_are_refused(lib):
    q, v, d = torch.randn(1, 5, 2, 16), torch.randn(1, 5, 4, 16), -torch.rand(4)
    pos, freq = torch.arange(5)[None], torch.ones(8)
    for call in (lambda: mk.linear_attention(q, q, v, d), lambda: mk.linear_attention(q, q, v, d, cu_seqlens=torch.tensor([0, 5])),
                 lambda: mk.linear_attention_step(q[0], q[0], v[0], d, torch.zeros(5, 4, 16, 16)), lambda: mk.rotary(q, q, pos, freq), lambda: mk.rotary(q, None, pos, freq),
                 lambda: mk.layer_norm(q), lambda: mk.layer_norm(q, torch.ones(16), torch.zeros(16), residual=q, groups=2)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    for call in (lambda: mk.linear_attention(None, q, v, d), lambda: mk.linear_attention_step(q[0], q[0], v[0], d, None), lambda: mk.rotary(q, q, None, freq), lambda: mk.layer_norm(None)):
        with pytest.raises(TypeError):
            call()


def test_entry_points_refuse_without_launching(lib):
    """Fake addresses: every call has to come back from the checks."""
    from mogankda_b200 import _lib
    S = _lib.STRUCTS
    numbers = dict(HK=2, HV=4, K=16, V=8, dtype=1, q_stride=32, k_stride=32, v_stride=32)
    bad = [("HK", 0), ("HK", 3), ("HV", 0), ("HV", 65536), ("K", 0), ("K", 129), ("V", 0), ("V", 129), ("dtype", 3), ("dtype", -1), ("log_decay", 0), ("q", 0), ("k", 0), ("v", 0)]
    seqs = [("S.N", 3), ("S.N", -1), ("S.N", 65536), ("S.T", -1), ("S.TT", 2 ** 31 - 1), ("S.seg", 64), ("S.seg", 128), ("S.seg", -128), ("h0", 0x30004), ("ht", 0x30008)]
    f = _filled(S["MkdaLinearFwd"](), ("q", "k", "v", "log_decay", "o"), **numbers)
    f.S.TT, f.S.N, f.S.T = 4, 2, 2
    _refused(lib, "mkda_linear_fwd", f, bad + seqs + [("o", 0), ("o", 0x30002), ("seg_h", 0x30004)])
    b = _filled(S["MkdaLinearBwd"](), ("d_o", "dq", "dk", "dv", "part_q", "part_k"), end=4)
    b.f = f
    _refused(lib, "mkda_linear_bwd", b, [("f." + n, v) for n, v in bad + seqs] + [(n, 0) for n in ("d_o", "dq", "dk", "dv", "part_q", "part_k")] + [("dht", 0x30004), ("dh0", 0x30004), ("dq", 0x30002),
                                        ("end", 5), ("end", -1)])
    f.S.seg, f.S.segs, f.seg_h = 128, 1, 0x30000
    b.f = f
    _refused(lib, "mkda_linear_bwd", b, [("seg_g", 0), ("f.S.segs", 0), ("f.S.T", 129)])
    p = _filled(S["MkdaLinearStep"](), ("q", "k", "v", "log_decay", "state", "o"), N=2, **numbers)
    _refused(lib, "mkda_linear_step", p, bad[:3] + bad[4:] + [("state", 0), ("state", 0x30008), ("o", 0), ("N", 65536), ("N", -1)])
    p = _filled(S["MkdaRotary"](), ("q", "k", "q_out", "k_out", "positions", "inv_freq"), tokens=3, heads_q=2, heads_k=1, dim=16, freqs=8, axes=2, dtype=1, q_stride=32, k_stride=16)
    p.axis_of[1] = 1 << 24
    _refused(lib, "mkda_rotary", p, [("tokens", -1), ("heads_q", -1), ("heads_k", 65537), ("dim", 0), ("dim", 513), ("dim", 14), ("freqs", -1), ("freqs", 9), ("axes", 0), ("axes", 1), ("axes", 256),
                                     ("dtype", 3), ("q", 0), ("k", 0), ("q_out", 0), ("k_out", 0), ("positions", 0), ("inv_freq", 0)])
    p = _filled(S["MkdaLayerNormFwd"](), ("x", "y"), rows=2, width=64, groups=4, dtype=1, x_stride=64)
    _refused(lib, "mkda_layer_norm_fwd", p, [("x", 0), ("y", 0), ("residual", 0x30000), ("width", 0), ("width", 62), ("width", 4 * 32769), ("groups", 0), ("groups", 65536), ("rows", -1), ("dtype", 9),
                                             ("stats", 0x30004)])
    p.weight, p.weight_dtype = 0x30000, 5
    _refused(lib, "mkda_layer_norm_fwd", p, [("rows", 3)])
    p = _filled(S["MkdaLayerNormBwd"](), ("s", "dy", "dx", "stats"), rows=2, width=64, groups=4, dtype=1, s_dtype=1, s_stride=64)
    _refused(lib, "mkda_layer_norm_bwd", p, [("s", 0), ("dy", 0), ("dx", 0), ("stats", 0), ("stats", 0x30004), ("width", 0), ("groups", 3), ("dtype", 9), ("s_dtype", -1), ("s_dtype", 2), ("part", 0x30000)])
    assert lib.mkda_layer_norm_bwd_part_rows(2, 64, 3) == 0 and lib.mkda_layer_norm_bwd_part_rows(2, 64, 4) == 1
