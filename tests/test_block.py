"""CPU: the entry points of the operators around the layer refuse what they cannot take before anything is launched, and the tables of packed sequences."""
import ctypes

import pytest
import torch

import mogankda_b200 as mk
from mogankda_b200.index import bounds_table


@pytest.fixture(scope="module")
def lib():
    from mogankda_b200 import _lib, build
    build.build()
    return _lib.load()


def test_block_structs_match_their_header(lib):
    from mogankda_b200 import _lib
    n = len(_lib.BLOCK_STRUCT_ORDER)
    sizes = (ctypes.c_int * n)()
    assert lib.mkda_block_struct_sizes(sizes, n) == n
    assert list(sizes) == [ctypes.sizeof(_lib.STRUCTS[s]) for s in _lib.BLOCK_STRUCT_ORDER]


def test_cpu_tensors_are_refused(lib):
    x, w, A = torch.randn(1, 5, 8), torch.randn(8, 4), -torch.rand(8, 16)
    bc = torch.randn(1, 5, 16)
    for call in (lambda: mk.causal_conv1d(x, w), lambda: mk.causal_conv1d(x, w, cu_seqlens=torch.tensor([0, 5])), lambda: mk.causal_conv1d_step(x[:, 0], x[:, :3], w),
                 lambda: mk.selective_scan(x, x, A, bc, bc), lambda: mk.selective_scan_step(x[:, 0], x[:, 0], A, bc[:, 0], bc[:, 0], torch.zeros(1, 8, 16)),
                 lambda: mk.rms_norm(x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(TypeError):
        mk.causal_conv1d(None, w)
    with pytest.raises(ValueError):
        mk.causal_conv1d(x, w, activation="gelu")


def test_tables_of_packed_sequences():
    table, dims = bounds_table(40, [0, 5, 5, 37], 16)
    assert table == [0, 5, 5, 37, 0, 1, 1, 2, 0, 1] and dims == (3, 0, 1, 3, 32)
    assert bounds_table(7, [0], 16) == ([0], (0, 0, 0, 0, 0))
    for bad in ([], [1, 7], [0, 5, 4], [0, 8]):
        with pytest.raises(ValueError):
            bounds_table(7, bad, 16)


def _filled(S, names, **numbers):
    for f in names:
        setattr(S, f, 0x30000)
    for f, v in numbers.items():
        setattr(S, f, v)
    return S


def _refused(lib, name, S, bad):
    from mogankda_b200 import _lib
    call = getattr(lib, name)
    assert call(None, None) == _lib.MKDA_ERR_ARG
    for path, value in bad:
        obj = S
        *outer, f = path.split(".")
        for o in outer:
            obj = getattr(obj, o)
        good = getattr(obj, f)
        setattr(obj, f, value)
        assert call(ctypes.byref(S), None) == _lib.MKDA_ERR_ARG, (name, path, value)
        setattr(obj, f, good)


def test_entry_points_refuse_without_launching(lib):
    """Fake addresses: every call has to come back from the checks."""
    from mogankda_b200 import _lib
    S = _lib.STRUCTS
    conv = [("W", 1), ("W", 5), ("D", 0), ("dtype", 3), ("dtype", -1), ("weight", 0)]
    seqs = [("S.N", 3), ("S.T", -1)]
    for name, struct, ptrs, more in (("mkda_conv_fwd", "MkdaConvFwd", ("x", "weight", "y"), [("x", 0), ("y", 0)]),
                                     ("mkda_conv_bwd", "MkdaConvBwd", ("x", "weight", "dy", "dx", "part"), [("dy", 0), ("dx", 0), ("part", 0), ("part_rows", 0), ("part_rows", 2)])):
        p = _filled(S[struct](), ptrs, D=8, W=4, dtype=1, x_stride=8)
        p.S.TT, p.S.N, p.S.T = 4, 2, 2
        if struct == "MkdaConvBwd":
            p.part_rows = 1
        _refused(lib, name, p, conv + seqs + more)
    p = _filled(S["MkdaConvStep"](), ("x", "weight", "state", "y"), D=8, W=4, dtype=1, N=2, x_stride=8)
    _refused(lib, "mkda_conv_step", p, conv + [("state", 0), ("N", 65536), ("N", -1)])
    scan = [("NST", 0), ("NST", 65), ("G", 0), ("G", 3), ("D", 0), ("dtype", 4), ("A", 0), ("A", 0x30004), ("x", 0), ("dt", 0), ("B", 0), ("C", 0)]
    numbers = dict(D=8, NST=16, G=2, dtype=1, x_stride=8, dt_stride=8, B_stride=32, C_stride=32)
    f = _filled(S["MkdaScanFwd"](), ("x", "dt", "B", "C", "A", "y", "ckpt"), **numbers)
    f.S.TT, f.S.N, f.S.T = 4, 2, 2
    _refused(lib, "mkda_scan_fwd", f, scan + seqs + [("y", 0), ("h0", 0x30008), ("ht", 0x30008), ("ckpt", 0x30008), ("S.cu", 0x30000), ("S.seg", 32), ("S.seg", -64), ("S.seg", 64)])
    b = _filled(S["MkdaScanBwd"](), ("dy", "dx", "ddt", "part_A", "part_B", "part_C"), slots=1, channel_blocks=lib.mkda_scan_bwd_channel_blocks(8, 2, 16))
    b.f = f
    _refused(lib, "mkda_scan_bwd", b, [("f." + n, v) for n, v in scan + seqs] + [("f.ckpt", 0), ("f.z", 0x30000), ("dy", 0), ("part_A", 0), ("part_B", 0), ("slots", 0),
                                      ("slots", 65536), ("channel_blocks", 1), ("dht", 0x30004), ("dh0", 0x30004), ("f.S.seg", 64)])
    p = _filled(S["MkdaScanStep"](), ("x", "dt", "B", "C", "A", "state", "y"), N=2, **numbers)
    _refused(lib, "mkda_scan_step", p, scan + [("state", 0), ("state", 0x30008), ("N", 65536)])
    p = _filled(S["MkdaNormFwd"](), ("x", "y"), rows=2, width=64, dtype=1, x_stride=64)
    _refused(lib, "mkda_norm_fwd", p, [("x", 0), ("y", 0), ("residual", 0x30000), ("out_e4m3", 1), ("width", 0), ("width", 32769), ("rows", -1), ("dtype", 9), ("group", 64), ("group", 128)])
    p = _filled(S["MkdaNormBwd"](), ("s", "dy", "dx"), rows=2, width=64, dtype=1, s_dtype=1, s_stride=64)
    _refused(lib, "mkda_norm_bwd", p, [("s", 0), ("dy", 0), ("dx", 0), ("width", 0), ("dtype", 9), ("s_dtype", -1), ("s_dtype", 2), ("part", 0x30000)])
    p = S["MkdaSumRows"]()
    j = p.job[0]
    j.out, j.rows, j.groups, j.pitch, j.cols, j.inner, j.valid = 0x30000, 2, 1, 8, 8, 8, 8
    bad = lib.mkda_sum_rows(ctypes.byref(p), None)
    setattr(j, "in", 0x30000)
    assert bad == _lib.MKDA_ERR_ARG
    for f, v in (("pitch", 4), ("inner", 0), ("out_dtype", 5), ("rows", -1), ("cols", 1 << 40)):
        good = getattr(j, f)
        setattr(j, f, v)
        if f == "cols":
            j.pitch = v
        assert lib.mkda_sum_rows(ctypes.byref(p), None) == _lib.MKDA_ERR_ARG, f
        setattr(j, f, good)
        j.pitch = 8


def test_scan_bwd_refuses_blocks_that_the_groups_do_not_have(lib):
    """Fake addresses: 8 channels in two groups are a block each."""
    from mogankda_b200 import _lib
    S = _lib.STRUCTS
    f = _filled(S["MkdaScanFwd"](), ("x", "dt", "B", "C", "A", "y", "ckpt"), D=8, NST=16, G=2, dtype=1, x_stride=8, dt_stride=8, B_stride=32, C_stride=32)
    f.S.TT, f.S.N, f.S.T = 4, 2, 2
    b = _filled(S["MkdaScanBwd"](), ("dy", "dx", "ddt", "part_A", "part_B", "part_C"), slots=1, channel_blocks=lib.mkda_scan_bwd_channel_blocks(8, 2, 16))
    b.f = f
    for first, blocks in ((1, 0), (-1, 1), (1, 1), (0, 2), (0, -1), (2 ** 31 - 1, 1)):
        b.first_block, b.blocks = first, blocks
        assert lib.mkda_scan_bwd(ctypes.byref(b), None) == _lib.MKDA_ERR_ARG and b"groups do not have" in lib.mkda_last_error()


def test_more_tokens_than_are_counted_in_32_bits_are_refused(lib):
    """The last run of tokens would end past 2^31 - 1.  Fake addresses."""
    from mogankda_b200 import _lib
    S, most = _lib.STRUCTS, 2 ** 31 - 1 - 65536
    calls = [("mkda_conv_fwd", _filled(S["MkdaConvFwd"](), ("x", "weight", "y"), D=8, W=4, dtype=1, x_stride=8)),
             ("mkda_scan_fwd", _filled(S["MkdaScanFwd"](), ("x", "dt", "B", "C", "A", "y"), D=8, NST=16, G=1, dtype=1, x_stride=8, dt_stride=8, B_stride=16, C_stride=16))]
    b = _filled(S["MkdaConvBwd"](), ("x", "weight", "dy", "dx", "part"), D=8, W=4, dtype=1, x_stride=8)
    b.part_rows = lib.mkda_conv_bwd_part_rows(most + 1, 8)
    calls.append(("mkda_conv_bwd", b))
    for name, p in calls:
        p.S.TT, p.S.N, p.S.T = most + 1, 1, most + 1
        assert getattr(lib, name)(ctypes.byref(p), None) == _lib.MKDA_ERR_ARG, name
