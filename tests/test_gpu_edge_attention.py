"""Edge attention on 8-bit rows, forward, backward and for a few rows, against the formulas in 64 bits on the same 8-bit values.

Tolerances, for fp32, with e = 2^-24.  A score is an exact integer times three roundings, its exponential in base 2 adds the
rounding of the difference to the maximum and 2 ulp of the hardware's exp2: relative error of a probability before
normalisation at most 8 e (|z|max + 1).  The sum of a row of n edges adds at most (n + 16) e, the normalisation 2 e, a
weighted sum (n + 16) e of the sum of its magnitudes.  All bounds below are c e times sums of magnitudes, with
c = 16 (|z|max + 1) + 4 n + 64, n the longest row that the value depends on.  Half types add their one rounding."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
# exp2 returns 0 below the normal numbers: a probability is off by up to 2^-126 (the largest of a row is 1 before it is
# normalised by a sum of at least 1), two of them meet in a gradient
FLUSHED = 2.0 ** -125
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -140, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def make_graph(kind, seed=0):
    import tango_b200 as T
    from tango_b200.graph import Graph
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def ints(hi, n):
        return torch.randint(0, hi, (n,), device="cuda", generator=gen)

    if kind == "one":                 # one node, one edge
        n, src, dst = 1, [0], [0]
    elif kind == "none":              # no edge at all
        n, src, dst = 5, [], []
    elif kind == "pair":              # one edge; the other rows are empty
        n, src, dst = 4, [2], [1]
    elif kind == "sparse":            # 0 to a dozen edges per node, some twice
        n = 700
        src, dst = ints(n, 2500), ints(n, 2500)
    elif kind == "classes":           # rows of every length around the kernels' classes, the last ones empty
        lengths = torch.tensor([0, 1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 47, 48, 49, 50, 63, 64, 65, 200, 511, 512, 513, 600,
                                1023, 1025, 2500], device="cuda")
        n = 60
        dst = torch.repeat_interleave(torch.arange(30, device="cuda"), lengths)
        src = ints(n, dst.numel())
    elif kind == "hubs":              # long rows and long columns: cut into units in both directions
        n = 300
        src = torch.cat([ints(n, 3000), torch.full((2000,), 7, device="cuda"), ints(n, 3000)])
        dst = torch.cat([torch.full((3000,), 11, device="cuda"), ints(n, 2000), ints(n, 3000)])
    src, dst = torch.as_tensor(src, device="cuda").long(), torch.as_tensor(dst, device="cuda").long()
    perm = torch.randperm(src.numel(), device="cuda", generator=gen)
    return T.graph_preprocess(Graph(src[perm], dst[perm], n), hub_block=0)


def values(t):
    """The 8-bit values of [N, H, D] in 64 bits."""
    import tango_b200 as T
    p = T.pack8(t, t.shape[2])
    return (T.unpack8(p, torch.float32)).double()      # a code times an fp32 scale, rounded to fp32: 2^-24, in the bounds


def reference(g, q, k, v, o, scale):
    """Outputs and sums of magnitudes, from 64-bit values; the gradients by autograd through the formula."""
    src, dst = (t.long() for t in g.edges())
    n, h, d = q.shape
    q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
    z = (q[dst] * k[src]).sum(-1) * scale
    top = torch.full((n, h), -math.inf, device=q.device, dtype=torch.float64).scatter_reduce(0, dst[:, None].expand(-1, h), z.detach(), "amax")
    p = torch.exp(z - top[dst])
    p = p / torch.zeros(n, h, device=q.device, dtype=torch.float64).index_add(0, dst, p)[dst]
    out = torch.zeros_like(q).index_add(0, dst, p.unsqueeze(-1) * v[src])
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), o)
    with torch.no_grad():
        zmax = float(z.abs().max()) if z.numel() else 0.0
        n_in = int(torch.bincount(dst, minlength=n).max())
        n_out = int(torch.bincount(src, minlength=n).max())
        c = 16 * (zmax + 1) + 4 * max(n_in, n_out) + 64
        adp = (o[dst].abs() * v[src].abs()).sum(-1)
        adelta = torch.zeros(n, h, device=q.device, dtype=torch.float64).index_add(0, dst, p * adp)
        full = (adp + adelta[dst]) * abs(scale)

        def magnitudes(p):
            ads = (p * full).unsqueeze(-1)
            p = p.unsqueeze(-1)
            return [torch.zeros_like(q).index_add(0, at, t) for at, t in ((dst, p * v[src].abs()), (dst, ads * k[src].abs()),
                                                                          (src, ads * q[dst].abs()), (src, p * o[dst].abs()))]

        bounds = [c * E * m + f for m, f in zip(magnitudes(p), magnitudes(torch.full_like(p, FLUSHED)))]
    return [out.detach(), dq, dk, dv], bounds


def check(got, want, bounds, dtype, names=("out", "dq", "dk", "dv")):
    for name, a, b, t in zip(names, got, want, bounds):
        assert a.dtype == dtype and a.shape == b.shape
        err = (a.double() - b).abs()
        bad = ~(err <= t + HALF[dtype] * b.abs() * 1.01 + TINY[dtype])
        assert not bad.any(), (name, float(err.max()), torch.nonzero(bad)[:3].tolist())


def run(g, q, k, v, o, scale=None):
    import tango_b200 as T
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    out = T.edge_attention(g, *leaves, scale)
    return [out.detach(), *torch.autograd.grad(out, leaves, o)]


def randn(seed, *shape, dtype=torch.float32, by=1.0):
    return (torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) * by).to(dtype)


def case(g, h, d, dtype=torch.float32, by=1.0, seed=1):
    n = g.num_nodes()
    return [randn(seed + i, n, h, d, dtype=dtype, by=by if i < 2 else 1.0) for i in range(4)]


SHAPES = [(1, 1), (1, 3), (2, 4), (3, 5), (8, 8), (5, 9), (1, 16), (4, 16), (3, 17), (6, 24), (4, 32), (3, 41), (1, 64), (16, 64), (2, 100),
          (1, 128), (2, 200), (1, 256), (3, 300), (1, 512), (33, 8), (40, 1)]


@pytest.mark.parametrize("kind", ["one", "none", "pair", "sparse", "classes", "hubs"])
@pytest.mark.parametrize("h,d", SHAPES)
def test_forward_and_gradients(cuda, kind, h, d):
    g = make_graph(kind)
    q, k, v, o = case(g, h, d)
    scale = 1 / math.sqrt(d)
    check(run(g, q, k, v, o), *reference(g, values(q), values(k), values(v), values(o), scale), torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("h,d", [(3, 5), (4, 32), (3, 41), (2, 100)])
def test_half_types(cuda, dtype, h, d):
    g = make_graph("hubs")
    q, k, v, o = case(g, h, d, dtype)
    check(run(g, q, k, v, o), *reference(g, values(q), values(k), values(v), values(o), 1 / math.sqrt(d)), dtype)


@pytest.mark.parametrize("scale,by", [(0.0, 1.0), (-0.5, 1.0), (3.0, 4.0), (1e-20, 1.0), (1.0, 1e-12)])
def test_scales(cuda, scale, by):
    """No scale, a negative one, scores of several hundred (one edge takes all), scores next to nothing."""
    g = make_graph("classes")
    q, k, v, o = case(g, 3, 24, by=by)
    check(run(g, q, k, v, o, scale), *reference(g, values(q), values(k), values(v), values(o), scale), torch.float32)


def test_gradients_against_differences(cuda):
    """Along a random direction of q, k and v: the loss <out, o> of the 64-bit formula at the 8-bit values."""
    g = make_graph("sparse")
    q, k, v, o = case(g, 2, 16)
    got = run(g, q, k, v, o)
    src, dst = (t.long() for t in g.edges())

    def loss(q, k, v):
        z = (q[dst] * k[src]).sum(-1) / 4
        p = torch.exp(z)
        p = p / torch.zeros(q.shape[:2], device="cuda", dtype=torch.float64).index_add(0, dst, p)[dst]
        return float((torch.zeros_like(q).index_add(0, dst, p.unsqueeze(-1) * v[src]) * values(o)).sum())

    at = [values(t) for t in (q, k, v)]
    for i in range(3):
        step = torch.randn(q.shape, device="cuda", dtype=torch.float64, generator=torch.Generator(device="cuda").manual_seed(i))
        h = 1e-5
        ends = [loss(*[t + s * h * step if j == i else t for j, t in enumerate(at)]) for s in (1, -1)]
        slope = (ends[0] - ends[1]) / (2 * h)
        grad = float((got[i + 1].double() * step).sum())
        size = float((got[i + 1].double() * step).abs().sum())
        # 64-bit differences: h^2 of the third derivative and 2^-52 of the loss over h; the kernel: the fp32 bounds above
        assert abs(slope - grad) <= 1e-5 * size + 1e-8


def test_8_bits_are_near_the_attention_of_the_inputs(cuda):
    """What the rounding of q, k, v and the gradient costs: each is within 1/254 of its group's largest magnitude, here about 3
    standard deviations, so a relative error of 3 / 254 / sqrt(3) = 0.7 % per operand; four of them, doubled for the softmax."""
    g = make_graph("sparse")
    q, k, v, o = case(g, 4, 32)
    got = run(g, q, k, v, o)
    want, _ = reference(g, *(t.double() for t in (q, k, v, o)), 1 / math.sqrt(32))
    for a, b in zip(got, want):
        assert float((a.double() - b).norm() / b.norm()) < 8 * 0.007


def test_repeats_bit_for_bit_and_rows_do_not_depend_on_their_neighbours(cuda):
    import tango_b200 as T
    from tango_b200.graph import Graph
    g = make_graph("hubs")
    q, k, v, o = case(g, 4, 16)
    a, b = run(g, q, k, v, o), run(g, q, k, v, o)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    # the same rows among others
    src, dst = g.edges()
    n = g.num_nodes()
    more = Graph(torch.cat([src, torch.randint(0, n, (900,), device="cuda").int()]),
                 torch.cat([dst, torch.randint(n, n + 90, (900,), device="cuda").int()]), n + 90)
    wide = [torch.cat([t, torch.randn(90, 4, 16, device="cuda")]) for t in (q, k, v)]
    with torch.no_grad():
        assert torch.equal(T.edge_attention(T.graph_preprocess(more, hub_block=0), *wide)[:n], a[0])


def test_rows_with_infinities_and_nan_stay_apart(cuda):
    g = make_graph("sparse")
    src, dst = (t.long() for t in g.edges())
    q, k, v, o = case(g, 2, 8)
    clean = run(g, q, k, v, o)
    bad = int(src[0])
    v2 = v.clone()
    v2[bad, 1, 3] = math.inf
    got = run(g, q, k, v2, o)
    hit = torch.zeros(g.num_nodes(), dtype=torch.bool, device="cuda")
    hit[dst[src == bad]] = True
    assert got[0][hit, 1].isnan().all() and torch.equal(got[0][:, 0], clean[0][:, 0]) and torch.equal(got[0][~hit], clean[0][~hit])
    q2 = q.clone()
    q2[int(dst[0]), 0, 0] = math.nan
    got = run(g, q2, k, v, o)
    rest = torch.ones_like(hit)
    rest[int(dst[0])] = False
    assert got[0][int(dst[0]), 0].isnan().all() and torch.equal(got[0][rest], clean[0][rest]) and torch.equal(got[1][rest], clean[1][rest])


@pytest.mark.parametrize("times", [1, 100, 700])
def test_scores_at_and_beyond_the_lowest_number(cuda, times):
    """Rows of a part of a warp, of a warp, and cut into units: a score close to the lowest number takes part like any other;
    one beyond it weighs nothing beside a finite one; a row of nothing else has no softmax, NaN in place of zeros."""
    import tango_b200 as T
    from tango_b200.graph import Graph
    pairs = [(1, 0), (1, 2), (3, 2), (4, 5), (4, 6), (3, 6), (4, 7), (1, 7)]
    src, dst = (torch.tensor(t, device="cuda").repeat(times) for t in zip(*pairs))
    g = T.graph_preprocess(Graph(src, dst, 9), hub_block=0)
    q = torch.ones(9, 1, 1, device="cuda")
    k, v = torch.zeros_like(q), torch.arange(9.0, device="cuda").view(9, 1, 1)
    k[1], k[4] = -2.2e38, -3e38              # times log2(e): -3.17e38 and minus infinity
    want = torch.tensor([1.0, 0, 3, 0, 0, math.nan, 3, 1, 0], device="cuda").view(9, 1, 1)
    out, dq, dk, dv = run(g, q, k, v, torch.ones_like(v), 1.0)
    bound = (2 * 4 * times + 32) * E * want.abs()       # equal weights: the sums of their row and one quotient
    assert torch.equal(out.isnan(), want.isnan()) and bool(((out - want).abs() <= bound)[~want.isnan()].all())
    assert dq[5].isnan().all() and not dq[[0, 1, 2, 3, 4, 6, 7, 8]].isnan().any()
    with torch.no_grad():
        assert torch.equal(T.edge_attention(g, q, k, v, 1.0).nan_to_num(-1), out.nan_to_num(-1))
    rows = T.edge_attention_rows(g, torch.arange(9, device="cuda"), q, T.pack8(k, 1), T.pack8(v, 1), 1.0)
    assert torch.equal(rows.isnan(), want.isnan()) and bool(((rows - want).abs() <= bound)[~want.isnan()].all())


def test_graph_that_was_not_preprocessed_and_strided_operands(cuda):
    import tango_b200 as T
    from tango_b200.graph import Graph
    g = make_graph("sparse")
    n = g.num_nodes()
    plain = Graph(*g.edges(), n)
    both = randn(5, n, 3, 2, 24)
    q, k, v = both[:, 0].transpose(1, 2), both[:, 1, :, 1:].transpose(1, 2), both[:, 2].transpose(1, 2)
    q, v = q[:, :23], v[:, :23]
    assert not q.is_contiguous() and q.shape == k.shape == (n, 23, 2)
    o = randn(6, 1, 23, 1).expand(n, 23, 2)
    want = run(g, q.contiguous(), k.contiguous(), v.contiguous(), o.contiguous())
    wide = torch.randn(n, 2 * 23 * 2, device="cuda")
    wide[:, 3:49] = q.reshape(n, 46)
    got = run(plain, wide[:, 3:49].view(n, 23, 2), k, v, o)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_only_some_gradients_and_saved_tensor_hooks(cuda):
    import tango_b200 as T
    g = make_graph("hubs")
    q, k, v, o = case(g, 2, 32)
    want = run(g, q, k, v, o)[1:]
    for needs in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(needs >> i & 1)) for i, t in enumerate((q, k, v))]
        T.edge_attention(g, *leaves).backward(o)
        for t, w in zip(leaves, want):
            assert (t.grad is None) == (not t.requires_grad) and (t.grad is None or torch.equal(t.grad, w))
    same = q.clone().requires_grad_()                     # one tensor in three places
    T.edge_attention(g, same, same, same).backward(o)
    parts = run(g, q, q, q, o)[1:]
    assert torch.allclose(same.grad, parts[0] + parts[1] + parts[2], rtol=1e-6, atol=1e-6)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    with torch.autograd.graph.save_on_cpu():
        out = T.edge_attention(g, *leaves)
    out.backward(o, retain_graph=True)
    out.backward(o)
    assert all(torch.equal(t.grad, 2 * w) for t, w in zip(leaves, want))
    with pytest.raises(RuntimeError, match="backward through the graph a second time"):
        out.backward(o)


def test_refusals(cuda):
    import tango_b200 as T
    g = make_graph("sparse")
    q, k, v, _ = case(g, 2, 8)
    for bad in ((q, k[1:], v), (q, k.half(), v), (q, k, v.cpu()), (q[:5], k[:5], v[:5]), (q.double(), k.double(), v.double()),
                (q.flatten(1), k.flatten(1), v.flatten(1))):
        with pytest.raises(AssertionError):
            T.edge_attention(g, *bad)
    for scale in (math.inf, math.nan, 1e300):
        with pytest.raises(AssertionError, match="finite"):
            T.edge_attention(g, q, k, v, scale)
    k8, v8 = T.pack8(k, 8), T.pack8(v, 8)
    ids = torch.tensor([1, 2], device="cuda")
    for rows, t in ((ids.float(), q[:2]), (ids[:1], q[:2]), (ids.cpu(), q[:2]), (ids.view(2, 1), q[:2])):
        with pytest.raises(AssertionError):
            T.edge_attention_rows(g, rows, t, k8, v8)
    with pytest.raises(AssertionError, match="no gradient"):
        T.edge_attention_rows(g, ids, q[:2].clone().requires_grad_(), k8, v8)
    with pytest.raises(ValueError, match="must be pack8"):
        T.edge_attention_rows(g, ids, q[:2], T.pack8(k, 16), v8)
    with pytest.raises(AssertionError, match="GPU"):
        T.edge_attention_rows(g, ids, q[:2], k8.to("cpu"), v8)


@pytest.mark.parametrize("h,d", [(2, 8), (3, 41), (1, 3)])
def test_keys_and_values_that_are_not_dense(cuda, h, d):
    """Packed rows of several layers kept in one array, and scales the other way round: the same bits as from dense ones."""
    import tango_b200 as T
    g = make_graph("sparse")
    n = g.num_nodes()
    q, k, v, _ = case(g, h, d)
    k8, v8 = T.pack8(k, d), T.pack8(v, d)
    ids = torch.tensor([1, 2, n - 1, 2], device="cuda")
    want = T.edge_attention_rows(g, ids, q[ids], k8, v8)
    codes = torch.stack([v8.codes, k8.codes, k8.codes + 1, v8.codes], 1)          # [N, layers, ld]
    scales = torch.stack([v8.scales, k8.scales, 2 * k8.scales, v8.scales], 1)

    def layer(i, scales=scales):
        return T.Packed8(codes[:, i], scales[:, i], (n, h, d), d, torch.float32)

    assert not layer(1).codes.is_contiguous()
    assert torch.equal(T.edge_attention_rows(g, ids, q[ids], layer(1), layer(3)), want)
    assert torch.equal(T.edge_attention_rows(g, ids, q[ids], layer(1), v8), want)
    turned = T.Packed8(k8.codes, k8.scales.t().contiguous().t(), (n, h, d), d, torch.float32)
    assert torch.equal(T.edge_attention_rows(g, ids, q[ids], turned, v8), want)
    for s in (k8.scales.t().contiguous(), k8.scales.flatten(), k8.scales[:1]):    # as many numbers, or fewer, in another shape
        if s.shape != k8.scales.shape:
            with pytest.raises(AssertionError, match="one group per head"):
                T.edge_attention_rows(g, ids, q[ids], T.Packed8(k8.codes, s, (n, h, d), d, torch.float32), v8)


@pytest.mark.parametrize("h,d,dtype", [(1, 3, torch.float32), (8, 8, torch.float16), (4, 32, torch.float32), (3, 41, torch.bfloat16),
                                       (2, 300, torch.float32), (33, 8, torch.float32)])
@pytest.mark.parametrize("kind", ["pair", "classes", "hubs"])
def test_few_rows(cuda, kind, h, d, dtype):
    import tango_b200 as T
    g = make_graph(kind)
    n = g.num_nodes()
    q, k, v, o = case(g, h, d, dtype)
    want, bounds = reference(g, values(q), values(k), values(v), values(o), 1 / math.sqrt(d))
    k8, v8 = T.pack8(k, d), T.pack8(v, d)
    gen = torch.Generator().manual_seed(3)
    for ids in (torch.arange(n), torch.tensor([n - 1]), torch.randint(0, n, (2 * n + 1,), generator=gen).int()):
        ids = ids.cuda()
        at = ids.long()
        got = T.edge_attention_rows(g, ids, q[at], k8, v8)
        check([got], [want[0][at]], [bounds[0][at]], dtype)
        assert torch.equal(got, T.edge_attention_rows(g, ids, q[at], k8, v8))


def test_few_rows_of_a_long_hub_and_unknown_ids(cuda):
    import tango_b200 as T
    from tango_b200.graph import Graph
    n, e = 5000, 150_000
    src = torch.randint(0, n, (e,), device="cuda")
    dst = torch.cat([torch.full((100_000,), 17, device="cuda"), torch.randint(0, n, (50_000,), device="cuda")])
    g = T.graph_preprocess(Graph(src, dst, n), hub_block=0)
    q, k, v, o = case(g, 2, 32)
    k8, v8 = T.pack8(k, 32), T.pack8(v, 32)
    want, bounds = reference(g, values(q), values(k), values(v), values(o), 1 / math.sqrt(32))
    ids = torch.tensor([17, 3, -1, 17, n, 4999, 1 << 40], device="cuda")
    known = torch.tensor([True, True, False, True, False, True, False], device="cuda")
    at = ids[known]
    queries = torch.randn(7, 2, 32, device="cuda")
    queries[known] = q[at]
    got = T.edge_attention_rows(g, ids, queries, k8, v8)
    assert got[~known].isnan().all()
    check([got[known]], [want[0][at]], [bounds[0][at]], torch.float32)
    one = T.edge_attention_rows(g, ids[:1], queries[:1], k8, v8)
    assert torch.equal(one[0], got[0]) and torch.equal(got[0], got[3])
    assert T.edge_attention_rows(g, ids[:0], queries[:0], k8, v8).shape == (0, 2, 32)
    # queries as columns of something wider
    wide = torch.randn(7, 100, device="cuda")
    wide[:, 30:94] = queries.flatten(1)
    assert torch.equal(T.edge_attention_rows(g, at, wide[known][:, 30:94].unflatten(1, (2, 32)), k8, v8), got[known])


def test_graph_without_nodes(cuda):
    import tango_b200 as T
    from tango_b200.graph import Graph
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    g = Graph(none, none, 0)
    x = torch.zeros(0, 2, 8, device="cuda")
    assert all(t.shape == (0, 2, 8) for t in run(g, x, x, x, x))
    k8, v8 = T.pack8(x, 8), T.pack8(x, 8)
    assert T.edge_attention_rows(g, none, x, k8, v8).shape == (0, 2, 8)
    assert T.edge_attention_rows(g, torch.tensor([0, -1], device="cuda"), torch.ones(2, 2, 8, device="cuda"), k8, v8).isnan().all()


def test_transformer_layer_asked_for_no_rows(cuda):
    from tango_b200.gnn import HGT
    g = make_graph("sparse")
    layer = HGT(12, 16, 2, fused=True).cuda()
    x = torch.randn(g.num_nodes(), 12, device="cuda")
    kept = layer.keys_values(x)
    ids = torch.zeros(0, dtype=torch.int64, device="cuda")
    got = layer.forward_rows(g, ids, x[ids], *kept)
    assert got.shape == (0, 16) and got.dtype == torch.float32


def test_streams_and_captured_graphs(cuda):
    """A run on a side stream, and two captured training passes replayed in turn with new inputs."""
    import tango_b200 as T
    g = make_graph("hubs")
    tensors = case(g, 4, 16)
    want = run(g, *tensors)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(g, *tensors)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))

    held = [[t.clone() for t in tensors] for _ in range(2)]
    captured = []
    with torch.cuda.stream(side):
        for h in held:
            run(g, *h)
    torch.cuda.current_stream().wait_stream(side)
    pool = torch.cuda.graph_pool_handle()
    for h in held:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs = run(g, *h)
            outs = [t.clone() for t in outs]
        captured.append((graph, outs))
    for seed in (10, 20):
        for i, (graph, outs) in enumerate(captured):
            new = case(g, 4, 16, seed=seed + i)
            for a, b in zip(held[i], new):
                a.copy_(b)
            graph.replay()
            for a, b in zip(outs, run(g, *new)):
                assert torch.equal(a, b)


def test_first_calls_inside_a_capture_are_refused(cuda):
    """With an error that says so, before any work: the capture and the process go on."""
    import tango_b200 as T
    g = make_graph("hubs")
    q, k, v, o = case(g, 4, 16)
    k8, v8, ids = T.pack8(k, 16), T.pack8(v, 16), torch.arange(5, device="cuda")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]

    def refused(f):
        x = torch.zeros(8, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            x.add_(1)
            with pytest.raises(RuntimeError, match="first call"):
                f()
            x.add_(1)
        graph.replay()
        assert x.eq(2).all()

    refused(lambda: T.edge_attention_rows(g, ids, q[:5], k8, v8))
    refused(lambda: T.edge_attention(g, q, k, v))
    want = T.edge_attention(g, q, k, v)
    refused(lambda: T.edge_attention(g, *leaves))           # the sources' schedule is still missing
    assert torch.equal(run(g, q, k, v, o)[0], want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(g, q, k, v, o)
        rows = T.edge_attention_rows(g, ids, q[:5], k8, v8)
    graph.replay()
    assert torch.equal(outs[0], want) and torch.equal(rows, T.edge_attention_rows(g, ids, q[:5], k8, v8))


def test_captured_backward_beside_a_living_graph_of_the_same_leaves(cuda):
    import tango_b200 as T
    g = make_graph("hubs")
    q, k, v, o = case(g, 2, 16)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    want = run(g, q, k, v, o)[1:]
    side = torch.cuda.Stream()          # (on the default stream PyTorch refuses to capture beside it, whatever the operator)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = T.edge_attention(g, *leaves)
        alive.backward(o, retain_graph=True)
        for t in leaves:
            t.grad.zero_()              # the captured pass adds to these
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        T.edge_attention(g, *leaves).backward(o)
    for n in (1, 2):
        graph.replay()
        assert all(torch.equal(t.grad, n * b) for t, b in zip(leaves, want))
    alive.backward(o)
    torch.cuda.synchronize()
    assert all(torch.equal(t.grad, 3 * b) or torch.allclose(t.grad, 3 * b, rtol=1e-6) for t, b in zip(leaves, want))


def test_first_calls_on_two_streams_and_from_two_threads(cuda):
    """The row schedules are made by whoever comes first; a call on another stream right behind it finds them whole."""
    import threading
    import tango_b200 as T
    want, graphs = None, [make_graph("hubs") for _ in range(3)]
    tensors = case(graphs[0], 4, 16)
    want = run(graphs[0], *tensors)
    g = graphs[1]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    res = [None, None]
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            res[i] = run(g, *tensors)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for r in res for a, b in zip(r, want))
    g, res = graphs[2], [None, None]

    def work(i):
        with torch.cuda.stream(streams[i]):
            res[i] = run(g, *tensors)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for r in res for a, b in zip(r, want))


def test_offsets_beyond_32_bits(cuda):
    """Codes, outputs and gradients of more than 2^32 bytes: rows at the far end of the tensors."""
    import tango_b200 as T
    from tango_b200.graph import Graph
    n, h, d = 4_300_000, 8, 64          # 2.2e9 elements a tensor, 4.4e9 bytes of interleaved codes
    if torch.cuda.mem_get_info()[0] < 100 << 30:
        pytest.skip("needs 100 GB")
    ends = torch.tensor([n - 1, n - 2, 5, n - 7, 3, n // 2], device="cuda")
    src, dst = ends.repeat(6), ends.repeat_interleave(6)
    g = Graph(src, dst, n)
    small = Graph(torch.arange(6, device="cuda").repeat(6), torch.arange(6, device="cuda").repeat_interleave(6), 6)
    parts = [randn(i, 6, h, d, dtype=torch.bfloat16) for i in range(4)]
    want = run(small, *parts)
    big = []
    for p in parts:
        t = torch.zeros(n, h, d, dtype=torch.bfloat16, device="cuda")
        t[ends] = p
        big.append(t)
    leaves = [t.requires_grad_() for t in big[:3]]
    out = T.edge_attention(g, *leaves)
    got = [out.detach()[ends]]
    grads = torch.autograd.grad(out, leaves, big[3])
    got += [t[ends] for t in grads]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del out, grads
    k8, v8 = T.pack8(big[1], d), T.pack8(big[2], d)
    with torch.no_grad():
        rows = T.edge_attention_rows(g, ends, parts[0], k8, v8)
    check([rows], [want[0].double()], [want[0].double().abs() * 2.0 ** -7 + 1e-3], torch.bfloat16)
    assert torch.equal(k8.unpack()[ends], T.pack8(parts[1], d).unpack())


@pytest.mark.parametrize("end", ["long", "middle", "short"])
def test_slots_at_the_end_of_32_bits(cuda, end):
    """Rows whose slots end at 2^31 - 1, the last of them of each of the kernels' classes: the same bits as of a graph whose slots
    begin at 0.  (The graph is symmetric, so that one array of 2^31 - 1 ids serves both directions.)"""
    import tango_b200 as T
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 20 GB")
    n = 90
    gen = torch.Generator(device="cuda").manual_seed(1)
    times = (torch.rand(n, n, device="cuda", generator=gen) < 0.05).int()          # rows of about nine edges,
    times[0], times[1, 2:] = 8, 1                                                  # one of some 700 and one of some 100
    times = torch.maximum(times, times.t())
    order = torch.arange(n, device="cuda").roll({"long": -1, "middle": -2, "short": 0}[end])     # the last of the new order: 0, 1, n - 1
    times = times[order][:, order]
    near = torch.repeat_interleave(torch.arange(n, device="cuda").repeat(n), times.flatten()).int()
    indptr = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int64), times.sum(1).cumsum(0)])
    e, most = near.numel(), 2 ** 31 - 1
    far = torch.zeros(most, dtype=torch.int32, device="cuda")
    far[most - e:] = near

    class Slots:
        def __init__(self, indptr, ids):
            self.adj_csc = self.adj_csr = (indptr.int(), ids, None)
            self.coo = near, near
            self._identity = {"csc": True, "csr": True}
            self._native = None

        def num_nodes(self):
            return n

        def num_edges(self):
            return e

    at_0, at_end = Slots(indptr, near), Slots(indptr + (most - e), far)
    assert int(at_end.adj_csc[0][-1]) == most
    for h, d in ((1, 3), (4, 32), (3, 41)):
        q, k, v, o = case(at_0, h, d)
        want = run(at_0, q, k, v, o)
        assert all(torch.equal(a, b) for a, b in zip(run(at_end, q, k, v, o), want))
        k8, v8 = T.pack8(k, d), T.pack8(v, d)
        for ids in (torch.arange(n, device="cuda"), torch.tensor([n - 1], device="cuda")):
            rows = T.edge_attention_rows(at_end, ids, q[ids], k8, v8)
            assert torch.equal(rows, T.edge_attention_rows(at_0, ids, q[ids], k8, v8))


def test_stochastic_rounding_draws_anew(cuda):
    import tango_b200 as T
    from tango_b200 import config, kernels
    g = make_graph("sparse")
    q, k, v, o = case(g, 2, 32)
    exact = run(g, q, k, v, o)
    config.set_rounding("stochastic", seed=3)
    try:
        kernels.set_call_counter(0)
        a = run(g, q, k, v, o)
        b = run(g, q, k, v, o)
        kernels.set_call_counter(0)
        c = run(g, q, k, v, o)
    finally:
        config.set_rounding("reference")
    for x, y, z, w in zip(a, b, c, exact):
        assert torch.equal(x, z) and not torch.equal(x, y)
        assert float((x - w).norm() / w.norm()) < 0.1


# ------------------------------------------------------------------------------------------------ bounds of every row's own
# As above, but with what a value itself depends on: c = 16 (|z|max of the row + 1) + 2 depth + 32, where depth is the most terms that
# meet one after another in a sum.  A row of up to 256 edges: that many.  A longer one on graphs of this size is cut into units of
# 128, which meet one by one; the slots of a warp (32 at most) before them.  Sources add their own depth to their destinations' c.
def depth_of(n):
    return torch.where(n <= 256, n, 128 + 32 + n // 128 + 1)


def own_bounds(g, q, k, v, o, scale, depth_of=depth_of):
    src, dst = (t.long() for t in g.edges())
    n, h, d = q.shape
    dev = q.device

    def total(at, t):
        return torch.zeros(n, *t.shape[1:], device=dev, dtype=torch.float64).index_add(0, at, t)

    z = (q[dst] * k[src]).sum(-1) * scale
    top = torch.full((n, h), -math.inf, device=dev, dtype=torch.float64).scatter_reduce(0, dst[:, None].expand(-1, h), z, "amax")
    zmax = torch.zeros(n, h, device=dev, dtype=torch.float64).scatter_reduce(0, dst[:, None].expand(-1, h), z.abs(), "amax")
    p = torch.exp(z - top[dst])
    p = p / total(dst, p)[dst]
    into, out_of = (depth_of(torch.bincount(t, minlength=n)).double()[:, None, None] for t in (dst, src))
    c = 16 * (zmax.unsqueeze(-1) + 1) + 2 * into + 32
    adp = (o[dst].abs() * v[src].abs()).sum(-1)

    def magnitudes(p):
        full = (p * (adp + total(dst, p * adp)[dst])).unsqueeze(-1) * abs(scale)
        p = p.unsqueeze(-1)
        return p * v[src].abs(), full * k[src].abs(), full * q[dst].abs(), p * o[dst].abs()

    out, dq, dk, dv = magnitudes(p)
    bounds = [c * E * total(dst, out), c * E * total(dst, dq)]
    bounds += [E * (total(src, c[dst] * t) + 2 * out_of * total(src, t)) for t in (dk, dv)]
    flushed = [total(at, t) for at, t in zip((dst, dst, src, src), magnitudes(torch.full_like(p, FLUSHED)))]
    return [a + b for a, b in zip(bounds, flushed)]


@pytest.mark.parametrize("kind", ["sparse", "classes", "hubs"])
@pytest.mark.parametrize("h,d", [(1, 3), (8, 8), (4, 32), (3, 41), (2, 100)])
def test_every_row_within_bounds_of_its_own(cuda, kind, h, d):
    g = make_graph(kind)
    q, k, v, o = case(g, h, d)
    at = [values(t) for t in (q, k, v, o)]
    want = reference(g, *at, 1 / math.sqrt(d))[0]
    check(run(g, q, k, v, o), want, own_bounds(g, *at, 1 / math.sqrt(d)), torch.float32)


def test_rows_without_a_schedule(cuda):
    """The kernels without a plan of the rows, every row by a warp, as C callers may have them."""
    from tango_b200 import _native
    for kind in ("pair", "classes", "hubs"):
        g = make_graph(kind)
        handle = _native.graph(g)
        assert not handle.has_edge_schedule("csc") and not handle.has_edge_schedule("csr")
        for h, d in ((1, 3), (4, 32), (3, 41)):
            q, k, v, o = case(g, h, d)
            at = [values(t) for t in (q, k, v, o)]
            want = reference(g, *at, 1 / math.sqrt(d))[0]
            leaves = [t.requires_grad_() for t in (q, k, v)]
            out = _native.ops.edge_attention(handle, *leaves, 1 / math.sqrt(d))
            got = [out.detach(), *torch.autograd.grad(out, leaves, o)]
            check(got, want, own_bounds(g, *at, 1 / math.sqrt(d), depth_of=lambda n: n), torch.float32)


def test_no_piece_of_a_long_row_is_lost(cuda):
    """A row of 100,000 edges asked for: cut into 64 pieces of 1563, a lane of the four warps takes at most a quarter of one, then 32
    slots, four warps and 64 pieces meet.  The bound is narrow enough to tell a lost piece: planted in the 64-bit form."""
    import tango_b200 as T
    from tango_b200._lib import lib
    from tango_b200.graph import Graph
    n, e, long = 5000, 140_000, 100_000
    gen = torch.Generator(device="cuda").manual_seed(7)
    src = torch.randint(0, n, (e,), device="cuda", generator=gen)
    dst = torch.cat([torch.full((long,), 17, device="cuda"), torch.randint(0, n, (e - long,), device="cuda", generator=gen)])
    g = T.graph_preprocess(Graph(src, dst, n), hub_block=0)
    q, k, v, o = case(g, 2, 32)
    at = [values(t) for t in (q, k, v, o)]
    scale = 1 / math.sqrt(32)
    want = reference(g, *at, scale)[0][0]
    indptr, ids = g.adj_csc[0], g.adj_csc[1].long()
    first, end = indptr[17:19].tolist()
    pieces = lib.tango_edge_attention_rows_splits(3, end - first)
    piece = -(-(end - first) // pieces)
    assert pieces == 64 and end - first > 99_999

    def depth(n):
        return torch.where(n <= 256, n, piece // 4 + 32 + 4 + pieces)

    bound = own_bounds(g, *at, scale, depth_of=depth)[0]
    rows = torch.tensor([17, 5, 4999], device="cuda")
    got = T.edge_attention_rows(g, rows, q[rows], T.pack8(k, 32), T.pack8(v, 32))
    check([got], [want[rows]], [bound[rows]], torch.float32)
    check([T.edge_attention(g, q, k, v)[17:18]], [want[17:18]], [bound[17:18]], torch.float32)
    key, value, query = at[1][ids[first:end]].cpu(), at[2][ids[first:end]].cpu(), at[0][17].cpu()
    p = torch.softmax((key * query).sum(-1) * scale, 0)
    for lost in (0, 31, pieces - 1):
        kept = torch.ones(end - first, 1)
        kept[lost * piece:(lost + 1) * piece] = 0
        wrong = (p * kept).unsqueeze(-1) * value
        wrong = wrong.sum(0) / (p * kept).sum(0).unsqueeze(-1)
        assert bool(((wrong - want[17].cpu()).abs() > bound[17].cpu()).any())


# ------------------------------------------------------------------------------------------------ models that call them
def test_transformer_layer_fused_against_the_chain_and_served(cuda):
    from tango_b200.gnn import HGT
    import tango_b200 as T
    from tango_b200.graph import rmat_graph
    g = T.graph_preprocess(rmat_graph(1500, 20000, 3, device="cuda"))
    torch.manual_seed(0)
    chain = HGT(48, 64, 4).cuda()
    fused = HGT(48, 64, 4, fused=True).cuda()
    fused.load_state_dict(chain.state_dict())
    x = torch.randn(1500, 48, device="cuda")
    o = torch.randn(1500, 64, device="cuda")
    res = []
    for m in (chain, fused):
        y = m(g, x)
        y.backward(o)
        # a bias of the keys shifts all scores of a row alike: its gradient is 0 but for rounding, nothing to compare
        res.append([y.detach()] + [p.grad for name, p in m.named_parameters() if name not in ("k_linear.bias", "attn_linear.bias")])
    # the chain rounds scores' operands, weights and values with one scale per tensor: 8 bits of noise on both sides
    for a, b in zip(*res):
        assert float(torch.nn.functional.cosine_similarity(a.flatten(), b.flatten(), 0)) > 0.98
    k8, v8 = fused.keys_values(x)
    rows = torch.tensor([5, 700, 5, 1499], device="cuda")
    every = fused.forward_rows(g, torch.arange(1500, device="cuda"), x, k8, v8)
    assert float((every - res[1][0]).norm() / res[1][0].norm()) < 1e-5       # all rows: the same int8 scales, another order of sums
    few = fused.forward_rows(g, rows, x[rows], k8, v8)
    assert float((few - res[1][0][rows]).norm() / res[1][0][rows].norm()) < 0.05
    assert not few.requires_grad


def test_attention_model_with_8_bit_activations(cuda):
    from tango_b200.gnn import GAT
    import tango_b200 as T
    from tango_b200.graph import rmat_graph
    import torch.nn.functional as F
    g = T.graph_preprocess(rmat_graph(1500, 20000, 3, device="cuda"))
    x, labels = torch.randn(1500, 48, device="cuda"), torch.randint(0, 5, (1500,), device="cuda")
    res = []
    for checkpoint in (None, "int8"):
        torch.manual_seed(1)
        m = GAT(g, 3, 48, 16, 5, [4, 4, 1], checkpoint=checkpoint).cuda()
        y = m(x)
        F.cross_entropy(y, labels).backward()
        res.append([y.detach()] + [p.grad for p in m.parameters()])
    # the same forward pass but for the last bits of exp; the gradients pass int8 quantizers, where those move single codes
    assert float((res[0][0] - res[1][0]).norm() / res[0][0].norm()) < 0.05
    for a, b in zip(*res):
        assert float(torch.nn.functional.cosine_similarity(a.flatten(), b.flatten(), 0)) > 0.98
