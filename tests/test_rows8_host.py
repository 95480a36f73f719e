"""8-bit rows and edge attention without a GPU: layouts, refusals before any launch, the C entry points' error codes, and the
row schedule."""
import ctypes
import math

import pytest
import torch


def _lib():
    from tango_b200 import _lib
    return _lib.lib


@pytest.mark.parametrize("cols,group,pitch,ld", [(1, 1, 4, 4), (3, 4, 4, 4), (8, 4, 4, 8), (9, 4, 4, 12), (5, 8, 8, 8), (12, 8, 8, 16),
                                                 (9, 9, 16, 16), (100, 128, 128, 112), (602, 128, 128, 608), (300, 100, 112, 336),
                                                 (250, 100, 112, 288), (1024, 1024, 1024, 1024), (0, 16, 16, 0)])
def test_layout(cols, group, pitch, ld):
    assert _lib().tango_rows8_pitch(group) == pitch and _lib().tango_rows8_ld(cols, group) == ld


class _Job(ctypes.Structure):
    _fields_ = [("x", ctypes.c_void_p), ("ldx", ctypes.c_int64), ("q", ctypes.c_void_p), ("scales", ctypes.c_void_p),
                ("scale_stride", ctypes.c_int64), ("interleaved", ctypes.c_int)]


class _Rows(ctypes.Structure):
    _fields_ = [("q", ctypes.c_void_p), ("scales", ctypes.c_void_p)]


class _Operands(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "kv", "o", "sq", "skv", "so")]


class _Plan(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_void_p), ("n_long", ctypes.c_int64), ("units", ctypes.c_void_p), ("n_units", ctypes.c_int64),
                ("heavy_first", ctypes.c_void_p), ("n_heavy", ctypes.c_int64)]


def _ref(x):
    return ctypes.cast(ctypes.byref(x), ctypes.c_void_p)


def test_pack_arguments_are_checked_before_any_launch():
    lib = _lib()
    ok = _Job(0x1000, 16, 0x2000, 0x3000, 1, 0)

    def pack(job=ok, n=1, rows=4, cols=16, group=16, kind=0, mode=1):
        return lib.tango_rows8_pack(_ref(job), n, rows, cols, group, kind, mode, 0, 0, None, None)

    assert pack(n=0) == -1 and pack(n=5) == -1 and pack(rows=-1) == -1 and pack(group=0) == -1 and pack(kind=3) == -1
    assert pack(mode=3) == -1 and pack(group=1025) == -5
    assert pack(job=_Job(0x1000, 8, 0x2000, 0x3000, 1, 0)) == -1           # leading dimension below the width
    assert pack(job=_Job(None, 16, 0x2000, 0x3000, 1, 0)) == -1
    assert pack(job=_Job(0x1002, 16, 0x2000, 0x3000, 1, 0)) == -2 and pack(job=_Job(0x1000, 16, 0x2002, 0x3000, 1, 0)) == -2
    assert pack(job=_Job(0x1000, 16, 0x2000, 0x3000, 0, 0)) == -1
    assert pack(rows=0) == 0 and pack(cols=0) == 0
    assert lib.tango_rows8_unpack(None, None, 4, 4, 4, 0, None, 4, None) == -1
    assert lib.tango_rows8_unpack(0x1000, 0x2000, 4, 4, 4, 0, 0x3000, 2, None) == -1
    assert lib.tango_act8_forward(3, _ref(ok), 4, 16, 16, 0, 0x4000, 16, 1, 0, 0, None, None) == -1
    half = _Job(0x1000, 16, None, 0x3000, 1, 0)                            # codes without scales or the reverse
    assert lib.tango_act8_forward(0, _ref(half), 4, 16, 16, 0, 0x4000, 16, 1, 0, 0, None, None) == -1
    assert lib.tango_act8_backward(-1, 0x1000, 0x2000, 4, 16, 16, 0, 0x3000, 16, 0x4000, 16, None) == -1
    assert lib.tango_act8_backward(0, 0x1000, 0x2000, 4, 16, 16, 0, 0x3000, 8, 0x4000, 16, None) == -1


def test_attention_arguments_are_checked_before_any_launch():
    lib = _lib()
    r = _Rows(0x1000, 0x2000)

    kept = []

    def x(q=0x1000, kv=0x1000, o=0x1000, skv=0x2000):
        kept.append(_Operands(q, kv, o, 0x2000, skv, 0x2000))
        return _ref(kept[-1])

    def forward(rows=4, heads=2, d=16, kind=0, x=x(o=None), out=0x3000, plan=None, ws=None, nbytes=0):
        return lib.tango_edge_attention(0x100, 0x200, rows, plan, heads, d, x, 1.0, out, kind, None, ws, nbytes, None)

    assert forward(rows=-1) == -1 and forward(heads=0) == -1 and forward(d=0) == -1 and forward(kind=7) == -1
    assert forward(d=513) == -5 and forward(heads=70000) == -5 and forward(rows=1 << 31) == -5
    assert forward(rows=0) == 0
    assert forward(x=x(q=None)) == -1 and forward(x=x(kv=None)) == -1 and forward(x=x(q=0x1008)) == -1 and forward(x=x(skv=None)) == -1 and forward(x=None) == -1
    assert forward(out=0x3004) == -2 and forward(x=x(skv=0x2004)) == -2 and forward(x=x(kv=0x1010)) == -2
    # long rows without a workspace that holds their units, and schedules that contradict themselves
    plan = _Plan(0x10, 2, 0x20, 3, 0x40, 1)
    assert forward(plan=_ref(plan)) == -1 and forward(plan=_ref(plan), ws=0x1000, nbytes=16) == -1
    assert forward(plan=_ref(_Plan(0x10, 0, 0x20, 3, 0x40, 1)), ws=0x1000, nbytes=1 << 20) == -1
    assert forward(plan=_ref(_Plan(0x10, 5, 0x20, 0, 0x40, 0))) == -1
    assert forward(plan=_ref(_Plan(0x10, 2, 0x20, 3, 0x40, 0))) == -1        # units of no row
    assert forward(plan=_ref(_Plan(0x10, 2, 0x20, 1, 0x40, 2)), ws=0x1000, nbytes=1 << 20) == -1
    assert forward(plan=_ref(_Plan(None, 2, None, 0, None, 0))) == -1 and forward(plan=_ref(_Plan(0x18, 2, None, 0, None, 0))) == -2
    def by_dst(x=x(), stats=0x4000, record=0x4000, qo=0x6000):
        return lib.tango_edge_attention_bwd_dst(0x100, 0x200, 4, None, 2, 16, x, 1.0, stats, 0x3000, 0, record, qo, None, 0, None)

    def by_src(kv=0x1000, skv=0x2000, qo=0x6000, record=0x4000):
        return lib.tango_edge_attention_bwd_src(0x100, 0x200, 4, None, 2, 16, kv, skv, qo, record, 0x3000, 0x3000, 0, None, 0, None)

    assert by_dst(x(o=None)) == -1 and by_dst(stats=None) == -1 and by_dst(stats=0x4004) == -2 and by_dst(qo=0x6010) == -2
    assert by_dst(record=None) == -1 and by_dst(qo=None) == -1
    assert by_src(kv=None) == -1 and by_src(qo=None) == -1 and by_src(record=None) == -1 and by_src(record=0x4008) == -2
    assert by_src(kv=0x1010) == -2 and by_src(skv=0x2004) == -2
    assert lib.tango_edge_attention_workspace_bytes(0, 3, 2, 16) == 3 * (4 + 32) * 4
    assert lib.tango_edge_attention_workspace_bytes(1, 3, 2, 41) == 3 * (4 + 2 * 96) * 4
    assert lib.tango_edge_attention_workspace_bytes(2, 3, 3, 8) == 3 * (2 * 24) * 4
    assert lib.tango_edge_attention_workspace_bytes(3, 3, 2, 16) == -1

    def rows(n=2, splits=1, d=16, ld=32, ws=None, nbytes=0, ids=0x500):
        return lib.tango_edge_attention_rows(0x100, 0x200, 4, ids, n, splits, 2, d, 0x1000, ld, 0, _ref(r), _ref(r), 1.0, 0x3000, ws, nbytes,
                                             1, 0, 0, None, None)

    assert rows(n=0) == 0 and rows(n=-1) == -1 and rows(splits=0) == -1 and rows(ld=31) == -1 and rows(ids=None) == -1
    assert rows(splits=4) == -1 and rows(splits=4, ws=0x1000, nbytes=64) == -1 and rows(d=600) == -5
    assert lib.tango_edge_attention_rows_splits(0, 10 ** 6) == 1 and lib.tango_edge_attention_rows_splits(5, 256) == 1
    assert lib.tango_edge_attention_rows_splits(10 ** 6, 10 ** 6) == 1
    assert 1 < lib.tango_edge_attention_rows_splits(1, 10 ** 6) <= 65535


def test_output_of_a_few_rows_starts_on_an_element():
    r = _Rows(0x1000, 0x2000)

    def rows(out, kind):
        return _lib().tango_edge_attention_rows(0x100, 0x200, 4, 0x500, 2, 1, 2, 16, 0x1000, 32, kind, _ref(r), _ref(r), 1.0, out, None, 0,
                                                1, 0, 0, None, None)

    assert rows(0x3002, 0) == -2 and rows(0x3001, 1) == -2 and rows(0x3003, 2) == -2


def _graph(n=20, e=60, seed=0):
    from tango_b200.graph import Graph
    gen = torch.Generator().manual_seed(seed)
    return Graph(torch.randint(0, n, (e,), generator=gen), torch.randint(0, n, (e,), generator=gen), n)


def test_refusals_before_any_launch():
    import tango_b200 as T
    x = torch.randn(4, 16)
    with pytest.raises(AssertionError, match="CUDA tensor"):
        T.pack8(x)
    with pytest.raises(AssertionError, match="CUDA tensor"):
        T.activation8(x)
    with pytest.raises(ValueError, match="relu"):
        T.activation8(x, "relu")
    with pytest.raises(ValueError, match="relu"):
        T.Activation8("relu")
    g = _graph()
    q = torch.randn(20, 2, 8)
    with pytest.raises(AssertionError, match="CUDA tensor"):
        T.edge_attention(g, q, q, q)
    with pytest.raises(AssertionError, match="heads, width"):
        T.edge_attention(g, q[0], q[0], q[0])
    with pytest.raises(AssertionError, match="width 1 to 512"):
        T.edge_attention(g, *[torch.randn(20, 1, 513)] * 3)
    with pytest.raises(TypeError, match="pack8"):
        T.edge_attention_rows(g, torch.tensor([1]), q[:1], q, q)
    codes, scales = torch.zeros(20, 16, dtype=torch.int8), torch.ones(20, 2)
    good = T.Packed8(codes, scales, (20, 2, 8), 8, torch.float32)
    for bad in (T.Packed8(codes, scales, (20, 16), 8, torch.float32), T.Packed8(codes, scales, (20, 2, 8), 16, torch.float32),
                T.Packed8(codes, scales, (19, 2, 8), 8, torch.float32)):
        with pytest.raises(ValueError, match="must be pack8"):
            T.edge_attention_rows(g, torch.tensor([1]), q[:1], good, bad)
    with pytest.raises(AssertionError, match="CUDA tensor"):
        T.edge_attention_rows(g, torch.tensor([1]), q[:1], good, good)


def test_packed_operands_of_another_type_are_refused_before_any_launch():
    """Bare pointers go to the kernel: scales of a half type would be read as fp32, twice as far as their buffer reaches."""
    import tango_b200 as T
    g = _graph()
    q = torch.randn(3, 2, 8)
    codes, scales = torch.zeros(20, 16, dtype=torch.int8), torch.ones(20, 2)
    good = T.Packed8(codes, scales, (20, 2, 8), 8, torch.float32)
    for c, s in ((codes, scales.bfloat16()), (codes, scales.half()), (codes, scales.double()), (codes.to(torch.uint8), scales),
                 (codes.float(), scales)):
        bad = T.Packed8(c, s, (20, 2, 8), 8, torch.float32)
        for k8, v8 in ((good, bad), (bad, good)):
            with pytest.raises(AssertionError, match="int8 codes and fp32 scales"):
                T.edge_attention_rows(g, torch.tensor([1, 2, 3]), q, k8, v8)


def test_activations_that_have_an_8_bit_form():
    import torch.nn as nn
    import torch.nn.functional as F
    from tango_b200.rows8 import Activation8, in_8_bits
    for a, kind in ((F.elu, "elu"), (F.gelu, "gelu"), (F.silu, "silu"), (nn.ELU(), "elu"), (nn.GELU(), "gelu"), (nn.SiLU(), "silu")):
        m = in_8_bits(a)
        assert isinstance(m, Activation8) and m.kind == kind
    for a in (F.relu, nn.ReLU(), nn.ELU(0.5), nn.GELU("tanh"), torch.tanh):
        with pytest.raises(ValueError, match="8-bit"):
            in_8_bits(a)
    from tango_b200.gnn import GAT
    with pytest.raises(ValueError, match="checkpoint"):
        GAT(None, 2, 8, 4, 3, [2, 1], checkpoint="int4")
    with pytest.raises(ValueError, match="8-bit"):
        GAT(None, 2, 8, 4, 3, [2, 1], activation=F.relu, checkpoint="int8")


def test_transformer_layers_of_earlier_files_run_the_chain():
    """A layer that was saved whole before the fused form existed has no attribute that says so."""
    import pickle
    from tango_b200.gnn import HGT
    layer = HGT(8, 16, 2)
    layer.__dict__.pop("_fused")
    old = pickle.loads(pickle.dumps(layer))
    assert "_fused" not in old.__dict__ and old._fused is False
    assert HGT(8, 16, 2, fused=True)._fused and pickle.loads(pickle.dumps(HGT(8, 16, 2, fused=True)))._fused


@pytest.mark.parametrize("scale", [1, 3000])
def test_units_cover_every_long_row_once(scale):
    """Also with enough edges for the limits to grow (lengths alone: the schedule reads nothing else)."""
    from tango_b200.graph import EdgeSchedule
    lengths = torch.tensor([0, 700, 5, 257, 256, 1, 3000, 0, 130, 49, 48]) * scale
    indptr = torch.zeros(lengths.numel() + 1, dtype=torch.int32)
    indptr[1:] = lengths.cumsum(0)
    s = EdgeSchedule(indptr)
    same = EdgeSchedule(indptr, int(indptr[-1]), torch.argsort(lengths, descending=True, stable=True).int())
    assert torch.equal(s.rows, same.rows) and torch.equal(s.units, same.units) and s.n_long == same.n_long
    assert s.longest == 3000 * scale
    rows = s.rows.long()
    length = rows[:, 2] - rows[:, 1]
    assert torch.equal(rows[:, 0].sort().values, torch.arange(11)) and (length.diff() <= 0).all()
    assert torch.equal(rows[:, 1], indptr.long()[rows[:, 0]]) and torch.equal(length, lengths[rows[:, 0]])
    assert s.n_heavy == int((lengths > s.threshold).sum()) <= s.n_long <= 11
    assert (length[:s.n_long] > 48).all()
    first = s.heavy_first.tolist()
    assert s.heavy_first.dtype == torch.int32 and first[0] == 0 and first[-1] == s.n_units and len(first) == s.n_heavy + 1
    for i in range(s.n_heavy):
        units = s.units[first[i]:first[i + 1]].tolist()
        assert [u[3] for u in units] == list(range(len(units))) and all(u[0] == int(rows[i, 0]) for u in units)
        assert units[0][1] == int(rows[i, 1]) and units[-1][2] == int(rows[i, 2])
        assert all(a[2] == b[1] and a[2] > a[1] for a, b in zip(units, units[1:]))
    for none in (torch.tensor([0, 3, 4], dtype=torch.int32), torch.tensor([0], dtype=torch.int32)):
        s = EdgeSchedule(none)
        assert s.heavy_first.tolist() == [0] and s.n_units == s.n_heavy == 0 and s.rows.shape == (none.numel() - 1, 4)


def test_quotients_without_division_are_exact():
    """The index arithmetic that finds row and group of an item: floor(i * m / 2^(32 + shift)) for every divisor met here and
    the largest indices, where a rounded-up multiplier would fail first."""
    for d in [2, 3, 4, 5, 7, 8, 9, 75, 76, 127, 128, 1000, 1023, 12345, 65535, 65537, (1 << 31) - 1]:
        shift = 0
        while (1 << (shift + 1)) < d:
            shift += 1
        m = ((1 << (32 + shift)) + d - 1) // d
        assert m < 1 << 32
        for i in {0, 1, d - 1, d, d + 1, (1 << 31) - 1, (1 << 31) - 2, ((1 << 31) - 1) // d * d, ((1 << 31) - 1) // d * d - 1}:
            if 0 <= i < 1 << 31:
                assert (i * m) >> (32 + shift) == i // d, (d, i)


def test_exact_rounding_in_32_bits():
    """The kernel's rule for values near a border, restated in fp32: product with an approximate reciprocal, and for the rest the
    exact remainder against half a step -- the quotient x / s rounded exactly, ties to even, for scales of all sizes."""
    import numpy as np
    rng = np.random.default_rng(3)
    f32 = np.float32
    for _ in range(300):
        m = f32(rng.uniform(1, 2) * 2.0 ** rng.integers(-110, 110))
        s = f32(m / f32(127))
        k = rng.integers(-127, 127, 64)
        x = ((k + 0.5) * float(s)).astype(f32)
        x = np.concatenate([x, np.nextafter(x, f32(np.inf)), np.nextafter(x, f32(-np.inf)), (rng.uniform(-1, 1, 64) * m).astype(f32)])
        x = x[np.abs(x) <= m]
        inv = f32(f32(1) / s)
        inv = np.nextafter(inv, f32(np.inf), dtype=f32)                    # one ulp off, as an approximate reciprocal may be
        t = x * inv
        q = np.rint(t).astype(f32)
        near = np.abs(t - q) > f32(0.4999)
        r = x.astype(np.float64) - q.astype(np.float64) * float(s)        # what the fused operation gives: exact in fp32
        assert (r[near] == r[near].astype(f32)).all()
        up = near & ((2 * np.abs(r) > s) | ((2 * np.abs(r) == s) & (q.astype(np.int64) % 2 != 0)))
        q = q + np.where(up, np.sign(r), 0)
        from fractions import Fraction
        for xi, qi in zip(x.tolist(), q.tolist()):
            assert round(Fraction(xi) / Fraction(float(s))) == qi, (xi, float(s))
    assert math.isclose(float(s) * 127, float(m), rel_tol=1e-6)


def test_exact_rounding_of_the_smallest_scales():
    """The same in the arithmetic of the kernel alone -- every operation rounded to fp32 -- for scales from the smallest normal
    number on, whose half may lie between two subnormal numbers: the remainder, doubled, against the scale and, for an odd code,
    against the number below it."""
    from fractions import Fraction
    import numpy as np
    f32 = np.float32
    rng = np.random.default_rng(4)

    def rounded(x, s, q):
        rest = (x.astype(np.float64) - q.astype(np.float64) * float(s)).astype(f32)     # one fused operation
        twice = np.abs(rest + rest)
        assert twice.dtype == f32
        limit = np.where(q.astype(np.int64) % 2 != 0, np.nextafter(s, f32(0)), s).astype(f32)
        return q + np.where(twice > limit, np.sign(rest), f32(0))

    for exponent in (-126, -126, -126, -125, -124, -120, 0, 100):
        for _ in range(40):
            s = f32(rng.uniform(1, 2) * 2.0 ** exponent)
            k = np.arange(-126, 126)
            x = ((k + 0.5) * float(s)).astype(f32)
            x = np.concatenate([x, np.nextafter(x, f32(np.inf)), np.nextafter(x, f32(-np.inf))])
            exact = [round(Fraction(float(a)) / Fraction(float(s))) for a in x]
            for side in (np.floor, np.ceil):             # whichever code the approximate quotient led to
                got = rounded(x, s, side(x.astype(np.float64) / float(s)).astype(f32))
                assert got.tolist() == exact, float(s)


def test_longest_row_is_found_once():
    """The row schedule of the incoming edges knows it; serving behind a training pass does not look for it again."""
    from tango_b200 import _native
    for first in (_native.edge_graph, _native.rows_graph):
        g = _graph()
        longest = int(torch.bincount(g.edges()[1].long()).max())
        handle = first(g, True) if first is _native.edge_graph else first(g)
        assert handle.knows_longest() and handle.longest() == longest
        assert handle.has_edge_schedule("csc") == handle.has_edge_schedule("csr") == (first is _native.edge_graph)
        assert _native.rows_graph(g) is handle


def test_rows_of_the_schedule_are_those_of_the_aggregations():
    """One list of the rows by decreasing length serves both kinds of kernels, and the units that are cut from it are the same."""
    from tango_b200 import _native
    from tango_b200.graph import EdgeSchedule, SpmmSchedule
    g = _graph(60, 20000)
    for fmt, indptr in (("csc", g.adj_csc[0]), ("csr", g.adj_csr[0])):
        plan = g._plans[fmt] = SpmmSchedule(indptr)
        kept, own = EdgeSchedule(indptr, g.num_edges(), rows=plan.row_info), EdgeSchedule(indptr)
        assert kept.rows is plan.row_info and torch.equal(kept.rows, own.rows) and torch.equal(kept.units, own.units)
        assert kept.n_units == own.n_units > 0 and torch.equal(kept.heavy_first, own.heavy_first)
        assert (kept.n_heavy, kept.n_long, kept.longest) == (own.n_heavy, own.n_long, own.longest)
    made = []
    init = EdgeSchedule.__init__
    try:
        EdgeSchedule.__init__ = lambda self, *a, **k: (init(self, *a, **k), made.append(self))[0]
        _native.edge_graph(g, True)
    finally:
        EdgeSchedule.__init__ = init
    assert [s.rows is g._plans[fmt].row_info for s, fmt in zip(made, ("csc", "csr"))] == [True, True]
