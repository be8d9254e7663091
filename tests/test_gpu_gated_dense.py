"""The gated Dense layer on a B200 against its definition in 64 bits, element by element.

Bounds.  A product's error is that of its fp32 accumulation, at most ACC sum |x w| with ACC = 2^-17 for the tensor cores
(16-bit operands: exact products, sums of up to 2048 terms whose adds may truncate, 2^-23 each at the running size, which
stays below a sixteenth of sum |x w| per add on average) and for Float32 the 1e-5 of its product; an activation adds 2^-20 of
its value (exp and division of a few 2^-23), and every rounding half a step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ACC = {torch.float32: 2.0 ** -16, torch.float16: 2.0 ** -17, torch.bfloat16: 2.0 ** -17}
ACTS = ["silu", "gelu", "geluTanh", "sigmoid", "tanh", "relu", "identity"]


@pytest.fixture(scope="module")
def srt():
    import swiftrt_b200 as s
    assert torch.cuda.is_available()
    return s


def _act(name, z):
    """(value, slope, largest slope) in 64 bits"""
    s = torch.sigmoid(z)
    if name == "silu":
        return z * s, s * (1 + z * (1 - s)), 1.1
    if name == "sigmoid":
        return s, s * (1 - s), 0.25
    if name == "tanh":
        return torch.tanh(z), 1 - torch.tanh(z) ** 2, 1.0
    if name == "relu":
        return z.clamp_min(0), (z > 0).double(), 1.0
    if name == "gelu":
        p = 0.5 * torch.erfc(-z * 0.5 ** 0.5)
        return z * p, p + z * torch.exp(-z * z / 2) * 0.3989422804014327, 1.13
    if name == "geluTanh":
        a, c = 0.7978845608028654, 0.044715
        t = torch.tanh(a * (z + c * z ** 3))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * c * z * z), 1.13
    return z, torch.ones_like(z), 1.0


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _check(got, want, error, what):
    got, want = got.double().cpu(), want.cpu()
    dtype = what[1]
    limit = error.cpu() + _half(dtype) * (want.abs() + error.cpu()) + _tiny(dtype)
    off = (got - want).abs()
    assert bool((off <= limit).all()), f"{what[0]}: {int((~(off <= limit)).sum())} of {off.numel()} off, worst {float((off / limit).max()):.3g} times its bound"


def _make(M, K, H, dtype, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed + 3 * M + 5 * K + H)
    n = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(dtype).to(DEV)  # noqa: E731
    return n(M, K), n(K, H, scale=K ** -0.5), n(K, H, scale=K ** -0.5), n(H, scale=0.5) if bias else None, n(H, scale=0.5) if bias else None


def _products(x, w, b):
    z, size = x.double() @ w.double(), x.double().abs() @ w.double().abs()
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    return z, ACC[x.dtype] * size


def _check_forward(layer, x, act, y, kept=None, rounded=False):
    """`rounded`: the path that rounds both products before the activation."""
    dt = x.dtype
    g, eg = _products(x, layer.weight_gate, layer.bias_gate)
    u, eu = _products(x, layer.weight_up, layer.bias_up)
    if kept is not None:
        _check(kept[0], g, eg, ("gate", dt))
        _check(kept[1], u, eu, ("up", dt))
    if rounded:
        eg, eu = eg + _half(dt) * (g.abs() + eg) + _tiny(dt), eu + _half(dt) * (u.abs() + eu) + _tiny(dt)
    a, _, steep = _act(act, g)
    ea = steep * eg + 2.0 ** -20 * a.abs()
    _check(y, a * u, ea * (u.abs() + eu) + a.abs() * eu + 2.0 ** -23 * (a * u).abs(), ("y", dt))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,H", [(1, 64, 128), (1, 1024, 520), (3, 200, 264), (16, 128, 64), (17, 520, 136), (64, 256, 1000), (65, 72, 8), (130, 64, 130 * 8),
                                   (257, 192, 384), (300, 1000, 200), (5, 33, 40), (2, 64, 1), (31, 7, 13), (1, 1, 1), (600, 2048, 256)])
def test_forward_matches_the_definition(srt, dtype, M, K, H):
    dt = TYPES[dtype]
    act = ACTS[(M + K + H) % len(ACTS)]
    x, wg, wu, bg, bu = _make(M, K, H, dt, bias=(M + H) % 2 == 0)
    layer = srt.GatedDense(wg, wu, bg, bu, srt.ActivationType[act])
    rounded = dt == torch.float32 or K % 8 != 0 or H % 8 != 0
    _check_forward(layer, x, act, layer(x), rounded=rounded)
    y, kept = layer.forward_keep(x)
    _check_forward(layer, x, act, y, kept, rounded=rounded)
    assert srt.check_status() == 0


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [1, 20, 200])
def test_every_activation(srt, act, M):
    x, wg, wu, bg, bu = _make(M, 256, 256, torch.bfloat16)
    layer = srt.GatedDense(wg, wu, bg, bu, srt.ActivationType[act])
    y, kept = layer.forward_keep(x)
    _check_forward(layer, x, act, y, kept)
    _check_forward(layer, x, act, layer(x))


def _check_backward(layer, x, saved, act, dy, grads):
    dt = x.dtype
    g, u, d = saved[0].double(), saved[1].double(), dy.double()
    a, slope, _ = _act(act, g)
    rough = 2.0 ** -18             # slopes are sums of a few terms of size one, each to 2^-20 or better
    dg, du = d * u * slope, d * a
    eg = rough * (d * u).abs() * (1 + g.abs())
    eu = rough * du.abs()
    rg, ru = eg + _half(dt) * (dg.abs() + eg) + _tiny(dt), eu + _half(dt) * (du.abs() + eu) + _tiny(dt)
    wg, wu, xd = layer.weight_gate.double(), layer.weight_up.double(), x.double()
    acc = ACC[dt]
    p, q = dg @ wg.t(), du @ wu.t()
    size = (dg.abs() + rg) @ wg.abs().t() + (du.abs() + ru) @ wu.abs().t()
    error = rg @ wg.abs().t() + ru @ wu.abs().t() + acc * size
    extra = 0 if dt != torch.float32 and x.shape[1] % 8 == 0 and g.shape[1] % 8 == 0 else 1     # two products rounded before their sum
    _check(grads[0], p + q, error + extra * _half(dt) * (size + 2 * _tiny(dt)), ("x", dt))
    for got, z, r, name in ((grads[1], dg, rg, "weight gate"), (grads[2], du, ru, "weight up")):
        _check(got, xd.t() @ z, xd.abs().t() @ r + acc * (xd.abs().t() @ (z.abs() + r)), (name, dt))
    for got, z, e, name in ((grads[3], dg, eg, "bias gate"), (grads[4], du, eu, "bias up")):
        if got is not None:
            _check(got, z.sum(0), e.sum(0) + 2.0 ** -18 * z.abs().sum(0), (name, dt))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,H", [(1, 64, 128), (3, 200, 264), (33, 72, 8), (130, 64, 1040), (257, 320, 384), (300, 1000, 200), (5, 33, 40), (31, 7, 13), (1, 1, 1),
                                   (700, 256, 520)])
def test_backward_matches_the_definition(srt, dtype, M, K, H):
    dt = TYPES[dtype]
    act = ACTS[(M + K) % len(ACTS)]
    x, wg, wu, bg, bu = _make(M, K, H, dt, bias=H % 3 != 0)
    layer = srt.GatedDense(wg, wu, bg, bu, srt.ActivationType[act])
    _, saved = layer.forward_keep(x)
    dy = torch.randn(M, H, generator=torch.Generator().manual_seed(4)).to(dt).to(DEV)
    _check_backward(layer, x, saved, act, dy, layer.backward(x, saved, dy))
    assert srt.check_status() == 0


@pytest.mark.parametrize("act", ACTS)
def test_gradients_agree_with_differences_of_the_definition(srt, act):
    """Central differences of sum(v y) in 64 bits along a random direction of every input."""
    M, K, H = 20, 64, 72
    x, wg, wu, bg, bu = _make(M, K, H, torch.float32)
    layer = srt.GatedDense(wg, wu, bg, bu, srt.ActivationType[act])
    _, saved = layer.forward_keep(x)
    g = torch.Generator().manual_seed(6)
    v = torch.randn(M, H, generator=g, dtype=torch.float64).to(DEV)
    grads = layer.backward(x, saved, v.float())
    base = [t.double() for t in (x, wg, wu, bg, bu)]

    def value(x, wg, wu, bg, bu):
        return float((_act(act, x @ wg + bg)[0] * (x @ wu + bu) * v.float().double()).sum())

    for k, grad in enumerate(grads):
        direction = torch.randn(base[k].shape, generator=g, dtype=torch.float64).to(DEV)
        h = 1e-6 if act == "relu" else 1e-4          # relu: steps that cross a kink would be off by the kink
        up, down = list(base), list(base)
        up[k], down[k] = base[k] + h * direction, base[k] - h * direction
        slope, ours = (value(*up) - value(*down)) / (2 * h), float((grad.double() * direction).sum())
        size = float((grad.double() * direction).abs().sum())
        assert abs(slope - ours) <= 1e-4 * size, (k, slope, ours)


def test_transposed_weights_views_leading_dimensions_and_outputs(srt):
    """[outputSize x inputSize] weights, the two halves of one weight, padded rows, rank-3 inputs and no rows at all."""
    dt, M, K, H = torch.bfloat16, 70, 128, 192
    x, wg, wu, bg, bu = _make(M, K, H, dt)
    act = srt.ActivationType.silu
    want = srt.GatedDense(wg, wu, bg, bu, act)(x)
    both = torch.cat((wg, wu), 1)
    padded = torch.zeros(M, K + 8, dtype=dt, device=DEV)
    padded[:, :K] = x
    for m in (M, 1, 9):
        forms = {"transposed": (wg.t().contiguous().t(), wu.t().contiguous().t()), "halves": (both[:, :H], both[:, H:]),
                 "one of each": (wg.t().contiguous().t(), wu)}
        for name, (a, b) in forms.items():
            layer = srt.GatedDense(a, b, bg, bu, act)
            for t in (x[:m], padded[:m, :K], x[:m].t().contiguous().t()):
                y, kept = layer.forward_keep(t)
                _check_forward(layer, t, "silu", y, kept, rounded=True)
                _check_forward(layer, t, "silu", layer(t), rounded=True)
                dy = torch.randn(m, H, generator=torch.Generator().manual_seed(1)).to(dt).to(DEV)
                grads = layer.backward(t, kept, dy)
                if name != "one of each":
                    _check_backward(layer, t, kept, "silu", dy, grads)
    layer = srt.GatedDense(wg, wu, bg, bu, act)
    assert torch.equal(layer(x.view(7, 10, K)).view(M, H), want)
    assert layer(x[:0]).shape == (0, H)
    strided_bias = torch.stack((bg, bu), 1)
    assert torch.equal(srt.GatedDense(wg, wu, strided_bias[:, 0], strided_bias[:, 1], act)(x), want)


def test_rows_behind_and_columns_beside_are_left_alone(srt):
    """A result that is a view into a larger buffer: nothing outside it is written."""
    from swiftrt_b200 import _lib
    from swiftrt_b200.matmul import descriptor_args, enqueue
    for M, H in ((5, 72), (130, 136), (260, 264)):
        x, wg, wu, bg, bu = _make(M, 64, H, torch.bfloat16)
        wide = torch.full((M + 3, H + 16), 9.0, dtype=torch.bfloat16, device=DEV)
        enqueue(_lib.lib.srtMatmulGated, x.device, *descriptor_args(x, wg, wu, bg, bu), 8, *descriptor_args(None, None, wide[:M, 8:H + 8]))
        assert torch.equal(wide[:M, 8:H + 8], srt.GatedDense(wg, wu, bg, bu)(x))
        assert bool((wide[M:] == 9).all()) and bool((wide[:, :8] == 9).all()) and bool((wide[:, H + 8:] == 9).all())


def test_non_finite_rows_stay_in_their_row(srt):
    for M in (4, 100):
        x, wg, wu, bg, bu = _make(M, 128, 64, torch.bfloat16)
        layer = srt.GatedDense(wg, wu, bg, bu)
        want = layer(x)
        x[2, 5] = float("nan")
        x[3, 7] = float("inf")
        got = layer(x)
        assert bool(torch.isnan(got[2]).all()) and not bool(torch.isfinite(got[3]).all())
        rest = [r for r in range(M) if r not in (2, 3)]
        assert torch.equal(got[rest], want[rest])


def test_streams_graphs_and_repeats_give_the_same_bits(srt):
    for M in (2, 150):
        x, wg, wu, bg, bu = _make(M, 256, 264, torch.float16)
        layer = srt.GatedDense(wg, wu, bg, bu)
        dy = torch.randn(M, 264, device=DEV).half()

        def both():
            y, saved = layer.forward_keep(x)
            return (y, *saved, layer(x), *layer.backward(x, saved, dy))

        want = [t.clone() for t in both()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = both()
            side.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                captured = both()
        for t in captured:
            t.zero_()
        graph.replay()
        again = both()
        torch.cuda.synchronize()
        for a, b, c, d in zip(want, other, captured, again):
            assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)


def test_one_launch_where_the_header_says_so(srt):
    x, wg, wu, bg, bu = _make(100, 128, 136, torch.bfloat16)
    layer = srt.GatedDense(wg, wu, bg, bu)
    for call in (lambda: layer(x), lambda: layer.forward_keep(x), lambda: layer(x[:1])):
        before = srt.launch_count()
        call()
        assert srt.launch_count() == before + 1


def test_the_wait_limit_ends_the_fused_kernels_in_order(srt):
    """A limit of one nanosecond on every pipeline wait: the kernel ends, the status word says so, and the next call is right."""
    x, wg, wu, bg, bu = _make(600, 1024, 512, torch.bfloat16)
    layer = srt.GatedDense(wg, wu, bg, bu)
    want, saved = layer.forward_keep(x)
    dy = torch.randn(600, 512, device=DEV).to(torch.bfloat16)
    grads = layer.backward(x, saved, dy)
    try:
        srt.set_wait_limit(1)
        layer(x)
        assert srt.check_status() != 0
        layer.backward(x, saved, dy)
        assert srt.check_status() != 0
    finally:
        srt.set_wait_limit(0)
    assert torch.equal(layer(x), want) and srt.check_status() == 0
    for a, b in zip(grads, layer.backward(x, saved, dy)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,K,H", [(65, 96, 72), (520, 264, 300)])
def test_weight_gradients_wherever_the_pairs_lie(srt, dtype, M, K, H):
    """The second of dGate / dUp and of dWGate / dWUp before or behind the first one, apart or as column blocks of one
    matrix.  Small integers and the identity: every sum is exact, the result has one right value."""
    from swiftrt_b200._lib import lib
    from swiftrt_b200.matmul import descriptor_args, enqueue
    dt, g = TYPES[dtype], torch.Generator().manual_seed(M)
    ints = lambda *s: torch.randint(-1, 2, s, generator=g).to(dt).to(DEV)  # noqa: E731
    x, wg, wu, gate, up, dy = ints(M, K), ints(K, H), ints(K, H), ints(M, H), ints(M, H), ints(M, H)
    dg, du = dy.double() * up.double(), dy.double() * gate.double()
    want = [(x.double().t() @ d).to(dt) for d in (dg, du)]

    def pair(rows, cols, how):
        if how == "blocks":
            pitch = (cols + 7) // 8 * 8
            w = torch.full((rows, 2 * pitch), 7.0, dtype=dt, device=DEV)
            return w[:, :cols], w[:, pitch:pitch + cols], w
        w = torch.full((2, rows, cols), 7.0, dtype=dt, device=DEV)
        return (w[0], w[1], w) if how == "behind" else (w[1], w[0], w)

    for first in ("behind", "before", "blocks"):
        for second in ("behind", "before", "blocks"):
            dgate, dup, _ = pair(M, H, first)
            dwg, dwu, wide = pair(K, H, second)
            enqueue(lib.srtMatmulGatedBackward, x.device, *descriptor_args(dy, x, wg, wu, gate, up), int(srt.ActivationType.identity),
                    *descriptor_args(dgate, dup, None, None, dwg, dwu, None, None))
            srt.check_status(DEV)
            assert torch.equal(dgate.double(), dg) and torch.equal(dup.double(), du)
            assert torch.equal(dwg, want[0]) and torch.equal(dwu, want[1]), (first, second)
            if second == "blocks":
                pitch = wide.shape[1] // 2
                assert bool((wide[:, H:pitch] == 7).all()) and bool((wide[:, pitch + H:] == 7).all())


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("M,K,H", [(1, 136, 4096), (2, 1000, 8000), (40, 72, 3304), (300, 264, 4096), (1030, 520, 5000)])
def test_input_gradients_of_few_tiles_and_long_reductions(srt, dtype, M, K, H):
    """dX where its reduction is split, with the weights in either order, into a view, and captured (not split).  Small
    integers and the identity: the result has one right value."""
    from swiftrt_b200._lib import lib
    from swiftrt_b200.matmul import descriptor_args, enqueue
    dt, g = TYPES[dtype], torch.Generator().manual_seed(M)
    ints = lambda *s: torch.randint(-1, 2, s, generator=g).to(dt).to(DEV)  # noqa: E731
    x, gate, up, dy, both = ints(M, K), ints(M, H), ints(M, H), ints(M, H), ints(2, K, H)
    dg, du = dy.double() * up.double(), dy.double() * gate.double()
    for wg, wu in ((both[0], both[1]), (both[1], both[0])):
        want = (dg @ wg.double().t() + du @ wu.double().t()).to(dt)
        layer = srt.GatedDense(wg, wu, activation=srt.ActivationType.identity)
        assert torch.equal(layer.backward(x, (gate, up), dy)[0], want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = layer.backward(x, (gate, up), dy)[0]
        graph.replay()
        assert torch.equal(captured, want)
        wide = torch.full((M, K + 8), 7.0, dtype=dt, device=DEV)
        pair = torch.empty(2, M, H, dtype=dt, device=DEV)
        enqueue(lib.srtMatmulGatedBackward, x.device, *descriptor_args(dy, x, wg, wu, gate, up), int(srt.ActivationType.identity),
                *descriptor_args(pair[0], pair[1], wide[:, :K], None, None, None, None, None))
        assert torch.equal(wide[:, :K], want) and bool((wide[:, K:] == 7).all())
    srt.check_status(DEV)
