"""8-bit rows and the activations that keep them, against the formulas in 64 bits.

Tolerances.  Codes and scales are exact.  A value in fp32 is one product of a code and a scale, rounded once (2^-24 relative),
in bf16 and fp16 rounded once more (2^-8 and 2^-11).  Activations: CUDA's erff, expf and expm1f are within 2 ulp (4 * 2^-24
relative), the quotients within 2 ulp; with the two to four fp32 operations around them the outputs are within 16 * 2^-24 of
1 + |x| (GELU's 1 + erf cancels for negative x, so its error is relative to |x|, not to the result), a gradient within that of
|dy|.  Half types add their one rounding."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
ULPS = 16 * 2.0 ** -24
# half types: results below the normal numbers are rounded to multiples of the smallest one
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def reference(x, group):
    """(codes, scales, values) of a matrix, in 64 bits but for the fp32 scale."""
    rows, cols = x.shape
    groups = -(-cols // group)
    x = x.double()
    codes, values = torch.zeros_like(x), torch.zeros_like(x)
    scales = torch.zeros(rows, groups, dtype=torch.float32, device=x.device)
    for g in range(groups):
        at = slice(g * group, min(cols, (g + 1) * group))
        top = x[:, at].abs().amax(1)
        s = (top.float() / torch.full_like(top, 127.0).float())
        s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
        c = torch.where(s[:, None] > 0, (x[:, at] / s[:, None].double()).round(), torch.zeros_like(x[:, at]))
        codes[:, at], scales[:, g], values[:, at] = c, s, c * s[:, None].double()
    return codes, scales, values


def codes_of(p, rows, cols):
    """The codes of a packed matrix [rows, cols], and all its other bytes."""
    from tango_b200._lib import lib
    pitch, group = lib.tango_rows8_pitch(p.group), p.group
    place = torch.arange(cols, device=p.codes.device)
    place = place // group * pitch + place % group
    rest = torch.ones(p.codes.shape[1], dtype=torch.bool, device=p.codes.device)
    rest[place] = False
    return p.codes[:, place], p.codes[:, rest]


SHAPES = [(1, 1, 1), (1, 7, 4), (3, 5, 8), (2, 16, 16), (33, 31, 8), (257, 100, 128), (129, 602, 128), (65, 601, 64), (40, 300, 100),
          (19, 257, 256), (7, 3000, 1024), (5, 1500, 700), (70000, 8, 8), (1, 40000, 32), (1000, 41, 41), (9, 130, 33), (300, 64, 128), (77, 16, 1024),
          (50, 4, 128), (31, 9, 64), (40, 48, 1000), (64, 128, 128), (10, 512, 64), (999, 8, 4)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols,group", SHAPES)
def test_pack_and_unpack(cuda, rows, cols, group, dtype):
    import tango_b200 as T
    gen = torch.Generator(device="cuda").manual_seed(rows + cols)
    x = (torch.randn(rows, cols, device="cuda", generator=gen) * 10 ** torch.randn(rows, 1, device="cuda", generator=gen)).to(dtype)
    x[rows // 2, :group] = 0
    p = T.pack8(x, group)
    codes, scales, values = reference(x, group)
    got, rest = codes_of(p, rows, cols)
    assert torch.equal(got.double(), codes) and torch.equal(p.scales, scales) and not rest.any()
    y = p.unpack()
    assert y.shape == x.shape and y.dtype == dtype
    err = (y.double() - values).abs()
    bound = values.abs() * (2.0 ** -24 + (HALF_STEP[dtype] if dtype != torch.float32 else 0)) * 1.0001 + TINY[dtype]
    assert bool((err <= bound).all())
    assert torch.equal(T.unpack8(p, torch.float32).to(dtype), y)


def test_borders_between_codes(cuda):
    """Quotients on and next to a half: ties to even, and no neighbour rounded across."""
    import tango_b200 as T
    rng = np.random.default_rng(1)
    tops = (rng.uniform(1, 2, 400) * 2.0 ** rng.integers(-100, 100, 400)).astype(np.float32)
    rows = []
    for m in tops:
        s = float(np.float32(m / np.float32(127)))
        h = ((rng.integers(-126, 126, 41) + 0.5) * s).astype(np.float32)
        rows.append(np.concatenate([[m], h, np.nextafter(h, np.float32(np.inf)), np.nextafter(h, np.float32(-np.inf))]))
    rows.append(np.concatenate([[127.0], np.arange(-62, 61) + 0.5]))        # a scale of 1: exact ties
    x = torch.from_numpy(np.stack(rows).astype(np.float32)).cuda()
    p = T.pack8(x, 124)
    codes, scales, _ = reference(x, 124)
    # 64-bit quotients are exact enough to tell the sides of a half: x / s differs from it by 2^-24 of itself or is it
    got, _ = codes_of(p, *x.shape)
    assert torch.equal(got.double(), codes) and torch.equal(p.scales, scales)


def test_borders_between_codes_of_the_smallest_scales(cuda):
    """The same for scales of the lowest normal binades: half of such a scale may lie between two subnormal numbers."""
    import tango_b200 as T
    rng = np.random.default_rng(2)
    rows = []
    for exponent in (-126, -126, -126, -125, -124):
        for _ in range(200):
            s = float(np.float32(rng.uniform(1, 2) * 2.0 ** exponent))
            m = np.float32(127 * s)
            s = float(m / np.float32(127))
            h = ((rng.integers(-126, 126, 41) + 0.5) * s).astype(np.float32)
            rows.append(np.concatenate([[m], h, np.nextafter(h, np.float32(np.inf)), np.nextafter(h, np.float32(-np.inf))]))
    x = torch.from_numpy(np.stack(rows).astype(np.float32)).cuda()
    codes, scales, _ = reference(x, 124)
    assert bool((scales >= 2.0 ** -126).all())
    p = T.pack8(x, 124)
    got, _ = codes_of(p, *x.shape)
    assert torch.equal(p.scales, scales) and torch.equal(got.double(), codes)


def test_groups_without_numbers_and_without_size(cuda):
    import tango_b200 as T
    x = torch.randn(6, 64, device="cuda")
    x[0, 3], x[1, 40], x[2, 5], x[3] = math.nan, math.inf, -math.inf, 0
    x[4] = 1e-41                                   # scale below the normal numbers
    x[5, :32] = 3e38
    y = T.pack8(x, 32).unpack()
    bad = torch.zeros_like(x, dtype=torch.bool)
    bad[0, :32] = bad[1, 32:] = bad[2, :32] = True
    assert torch.equal(y.isnan(), bad)
    assert (y[3] == 0).all() and (y[4] == 0).all()
    _, _, want = reference(torch.where(bad, torch.zeros_like(x), x), 32)
    assert bool(((y.double() - want).abs()[~bad] <= want.abs()[~bad] * 2.0 ** -24).all())


def test_strides_empty_and_odd_tensors(cuda):
    import tango_b200 as T
    base = torch.randn(50, 77, device="cuda")
    for x in (base[:, 1:70], base.t(), base[::2, 3:], base[:, ::3], base[0], base[3:3], base[:, :0], base.view(25, 2, 77),
              base[:, :72].view(50, 9, 8).transpose(0, 1), torch.tensor(3.0, device="cuda"), base[:1, 1:33], base.expand(2, 50, 77)):
        p = T.pack8(x, 32)
        y = p.unpack()
        assert y.shape == x.shape and y.is_contiguous()
        if x.numel():
            m = x.reshape(x.shape[0] if x.dim() > 1 else 1, -1)
            _, _, want = reference(m, 32)
            assert bool(((y.reshape(m.shape).double() - want).abs() <= want.abs() * 2.0 ** -24).all())


def test_refusals(cuda):
    import tango_b200 as T
    x = torch.randn(4, 16, device="cuda")
    for group in (0, -3, 1025):
        with pytest.raises(AssertionError, match="groups of"):
            T.pack8(x, group)
    for bad in (x.double(), x.int(), x.cpu()):
        with pytest.raises(AssertionError, match="CUDA tensor"):
            T.pack8(bad)
        with pytest.raises(AssertionError, match="CUDA tensor"):
            T.activation8(bad)
    p = T.pack8(x, 16)
    with pytest.raises(AssertionError, match="do not belong"):
        T.unpack8(T.Packed8(p.codes, p.scales, (4, 40), 16, torch.float32))
    with pytest.raises(AssertionError, match="do not belong"):
        T.unpack8(T.Packed8(p.codes, p.scales[:, :0], (4, 16), 16, torch.float32))
    with pytest.raises(AssertionError, match="int8 codes"):
        T.unpack8(T.Packed8(p.codes.cpu(), p.scales.cpu(), (4, 16), 16, torch.float32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols,group", [(37, 41, 41), (50, 130, 64), (9, 601, 128), (21, 16, 16), (40, 3, 8), (11, 700, 700), (1, 67, 32),
                                             (64, 12, 4), (5, 1030, 1024)])
def test_where_a_row_begins_changes_nothing(cuda, rows, cols, group, dtype):
    # the same values behind every offset and at every pitch, in every rounding mode: the same bits as of a contiguous matrix
    import tango_b200 as T
    from tango_b200 import config, kernels
    x = torch.randn(rows, cols, device="cuda").to(dtype)
    dy = torch.randn(rows, cols, device="cuda").to(dtype)

    def all_of(x, dy):
        got = []
        for mode in ("reference", "trunc", "stochastic"):
            config.set_rounding(mode, seed=3)
            kernels.set_call_counter(0)
            p = T.pack8(x, group)
            leaf = x.detach().requires_grad_()
            y = T.activation8(leaf, "silu", group)
            g, = torch.autograd.grad(y, leaf, dy)
            got += [p.codes, p.scales, p.unpack(), y.detach(), g]
        return got
    try:
        want = all_of(x, dy)
        for before in range(4):
            for behind in range(4):
                wide = torch.full((rows, before + cols + behind), float("nan"), device="cuda", dtype=dtype)
                at = wide[:, before:before + cols]
                at.copy_(x)
                other = torch.full((rows, 1 + cols + behind), float("inf"), device="cuda", dtype=dtype)[:, 1:1 + cols]
                other.copy_(dy)
                for a, b in zip(all_of(at, other), want):
                    assert torch.equal(a, b)
    finally:
        config.set_rounding("reference")


@pytest.mark.parametrize("mode", ["trunc", "stochastic"])
def test_rounding_modes(cuda, mode):
    import tango_b200 as T
    from tango_b200 import config, kernels
    x = torch.randn(200, 90, device="cuda")
    _, scales, _ = reference(x, 32)
    quotient = x.double() / scales.repeat_interleave(32, 1)[:, :90].double()
    config.set_rounding(mode, seed=5)
    try:
        kernels.set_call_counter(0)
        p = T.pack8(x, 32)
        again = T.pack8(x, 32)
        kernels.set_call_counter(0)
        first = T.pack8(x, 32)
    finally:
        config.set_rounding("reference")
    got, rest = codes_of(p, 200, 90)
    got = got.double()
    assert torch.equal(p.scales, scales) and not rest.any() and torch.equal(first.codes, p.codes)
    if mode == "trunc":
        assert torch.equal(again.codes, p.codes)
        # the fp32 quotient may round up to a whole number that the exact one just misses
        assert bool(((got - quotient.trunc()).abs() <= ((quotient - quotient.round()).abs() < 1e-5).double()).all())
    else:
        assert not torch.equal(again.codes, p.codes)
        assert bool(((got - quotient).abs() < 1 + 1e-5).all())
        # the mean of 18,000 roundings, each uniform within a step (variance at most 1/4): 6 sigma
        assert abs(float((got - quotient).mean())) < 6 * 0.5 / math.sqrt(18000)


def f64(x, kind):
    if kind == "elu":
        return torch.where(x > 0, x, torch.expm1(x.clamp(max=0)))
    if kind == "gelu":
        return x * 0.5 * torch.special.erfc(-x / math.sqrt(2))
    return x * torch.sigmoid(x)


def slope64(t, kind):
    if kind == "elu":
        return torch.where(t > 0, torch.ones_like(t), t.clamp(max=0).exp())
    if kind == "gelu":
        return 0.5 * torch.special.erfc(-t / math.sqrt(2)) + t * torch.exp(-t * t / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(t)
    return s + t * s * torch.sigmoid(-t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind", ["elu", "gelu", "silu"])
@pytest.mark.parametrize("rows,cols,group", [(1, 1, 128), (300, 64, 128), (77, 601, 64), (33, 256, 256), (5, 1300, 600)])
def test_activation_and_its_gradient(cuda, rows, cols, group, kind, dtype):
    import tango_b200 as T
    gen = torch.Generator(device="cuda").manual_seed(cols)
    x = (torch.randn(rows, cols, device="cuda", generator=gen) * 3).to(dtype)
    dy = torch.randn(rows, cols, device="cuda", generator=gen).to(dtype)
    leaf = x.clone().requires_grad_()
    y = T.activation8(leaf, kind, group)
    with torch.no_grad():
        assert torch.equal(T.activation8(x, kind, group), y)
    y.backward(dy)
    assert y.dtype == dtype and leaf.grad.dtype == dtype
    want = f64(x.double(), kind)
    half = HALF_STEP[dtype] if dtype != torch.float32 else 0.0
    assert bool(((y.double() - want).abs() <= ULPS * (1 + x.double().abs()) + half * want.abs() * 1.01 + TINY[dtype]).all())
    t = reference(x, group)[2]
    want = dy.double() * slope64(t, kind)
    bound = (ULPS * (1 + t.abs()) * dy.double().abs() + half * want.abs() * 1.01 + TINY[dtype])
    assert bool(((leaf.grad.double() - want).abs() <= bound).all())
    # against differences of f at the copy: the error of a central difference of step h is h^2/6 |f'''| <= h^2 plus 2^-52 / h;
    # ELU has a kink in f'' at 0, where the difference is off by up to h / 2
    h = 1e-4
    slope = (f64(t + h, kind) - f64(t - h, kind)) / (2 * h)
    assert bool(((leaf.grad.double() - dy.double() * slope).abs() <= bound + dy.double().abs() * (h * 0.51 if kind == "elu" else 1e-7)).all())


def test_far_values_of_the_activations(cuda):
    import tango_b200 as T
    import torch.nn.functional as F
    x = torch.tensor([[-1e30, -200.0, -90.0, -30.0, 0.0, -0.0, 30.0, 90.0, 1e30]], device="cuda")
    for kind in ("elu", "gelu", "silu"):
        leaf = x.clone().requires_grad_()
        y = T.activation8(leaf, kind, 1)             # one number a group: the copy is x to 2^-24
        y.sum().backward()
        want = getattr(F, kind)(x.double())
        assert bool(((y.double() - want).abs() <= ULPS * x.abs().clamp(max=100).double() + want.abs() * ULPS).all()), kind
        assert bool(((leaf.grad.double() - slope64(x.double(), kind).nan_to_num(0)).abs() <= 1e-5).all()), kind
    bad = torch.tensor([[math.nan, 1.0], [2.0, 3.0]], device="cuda", requires_grad=True)
    T.activation8(bad, "elu", 2).sum().backward()
    assert bad.grad[0].isnan().all() and bad.grad[1].eq(1).all()


def test_activation_in_a_graph_of_operations(cuda):
    """Strided inputs and gradients, reuse of a graph, saved-tensor hooks, gradients of gradients refused."""
    import tango_b200 as T
    base = torch.randn(40, 3, 17, device="cuda")
    x = base.transpose(0, 2).detach().requires_grad_()
    y = T.activation8(x, "gelu", 16)
    g = torch.randn(3, device="cuda").view(1, 3, 1).expand(17, 3, 40)
    y.backward(g, retain_graph=True)
    once = x.grad.clone()
    y.backward(g)
    assert torch.equal(x.grad, 2 * once)
    with pytest.raises(RuntimeError, match="backward through the graph a second time"):
        y.backward(g)
    m = x.detach().reshape(17, 120)
    want = (g.reshape(17, 120).double() * slope64(reference(m, 16)[2], "gelu")).view(17, 3, 40)
    assert bool(((once.double() - want).abs() <= ULPS * (1 + x.detach().abs().max()) * g.abs().double()).all())
    with torch.autograd.graph.save_on_cpu():
        y = T.activation8(x, "gelu", 16)
    x.grad = None
    y.backward(g)
    assert torch.equal(x.grad, once)
    y = T.activation8(x, "silu")
    (dx,) = torch.autograd.grad((y * y).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()
    empty = torch.empty(0, 8, device="cuda", requires_grad=True)
    T.activation8(empty).sum().backward()
    assert empty.grad.shape == (0, 8)


def test_checkpoint_is_what_stays_in_memory(cuda):
    import tango_b200 as T
    x = torch.randn(4096, 1024, device="cuda").requires_grad_()
    torch.cuda.synchronize()
    h = x * 1.0
    requested = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]      # (allocated: by blocks, which may be larger)
    before = requested()
    y = T.activation8(h, "silu", 128)
    del h
    kept = requested() - before
    assert kept <= 4096 * 1024 * (1 + 4 / 128) + 8192          # y takes the place of h; the rest is the 8-bit copy
    y.sum().backward()


def test_packing_on_another_stream_and_in_a_captured_graph(cuda):
    import tango_b200 as T
    x = torch.randn(500, 200, device="cuda")
    want = T.pack8(x).unpack()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = T.pack8(x).unpack()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)

    leaf = torch.zeros_like(x).requires_grad_()
    dy = torch.zeros_like(x)

    def step():
        y = T.activation8(leaf, "elu")
        return (y.detach(), *torch.autograd.grad(y, leaf, dy))

    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in (1, 2):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        with torch.no_grad():
            leaf.copy_(torch.randn(x.shape, device="cuda", generator=gen))
            dy.copy_(torch.randn(x.shape, device="cuda", generator=gen))
        graph.replay()
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["groups", "pitch", "columns", "run"])
def test_indices_beyond_32_bits(cuda, kind):
    """More than 2^31 groups, rows further apart than 2^31 elements, more than 2^31 columns (the last a run of whole groups): the same
    bits as of parts that stay below."""
    import tango_b200 as T
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    gen = torch.Generator(device="cuda").manual_seed(5)

    def randn(n):
        x = torch.empty(n, device="cuda", dtype=torch.bfloat16)
        for part in x.split(1 << 28):
            part.normal_(generator=gen)
        return x

    if kind == "groups":
        x = randn(65537 * 32768).view(65537, 32768)
        p = T.pack8(x, 1)
        assert p.scales.numel() > 2 ** 31
        y = p.unpack()
        for at in (slice(0, 3), slice(32760, 32770), slice(65530, 65537)):
            part = T.pack8(x[at], 1)
            assert torch.equal(p.codes[at], part.codes) and torch.equal(p.scales[at], part.scales)
            assert torch.equal(y[at], part.unpack())
    elif kind == "pitch":
        far = 2 ** 31 + 1
        x, dy = (randn(far + 700) for _ in range(2))
        x, dy = x.as_strided((2, 601), (far, 1), 3), dy.as_strided((2, 601), (far, 1), 2)
        a, b = T.pack8(x, 64), T.pack8(x.contiguous(), 64)
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
        res = []
        for t, g in ((x, dy), (x.contiguous(), dy.contiguous())):
            leaf = t.detach().requires_grad_()
            y = T.activation8(leaf, "silu", 64)
            res.append((y.detach(), *torch.autograd.grad(y, leaf, g)))
        assert all(torch.equal(a, b) for a, b in zip(*res))
    else:
        whole = 2 ** 31
        x = randn(whole + (128 if kind == "run" else 67))
        rest = x[whole:]
        p = T.pack8(x)
        a, b = T.pack8(x[:whole].view(-1, 128)), T.pack8(rest)
        assert torch.equal(p.codes[0, :whole].view(-1, 128), a.codes) and torch.equal(p.codes[0, whole:], b.codes[0])
        assert torch.equal(p.scales[0, :-1], a.scales[:, 0]) and torch.equal(p.scales[0, -1:], b.scales[0])
        y = p.unpack()
        assert torch.equal(y[:whole].view(-1, 128), a.unpack()) and torch.equal(y[whole:], b.unpack())
        del p, a, b, y
        leaf = x.requires_grad_()
        y = T.activation8(leaf, "elu")
        tail = rest.detach().requires_grad_()
        z = T.activation8(tail, "elu")
        dy = torch.ones_like(y)
        dx, = torch.autograd.grad(y, leaf, dy)
        dz, = torch.autograd.grad(z, tail, dy[whole:])
        assert torch.equal(y[whole:], z) and torch.equal(dx[whole:], dz)
