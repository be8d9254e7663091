"""Products with 4-bit weights on a B200 against their definition in 64 bits, element by element.

Bounds.  x and the integers q - z are exact in 16 bits and so are their products in fp32; what is lost is the adding up, at
most ACC sum |x (q - z) s| with ACC = 2^-18 (fp32 adds, truncating ones included, of at most 2^-23 of the running sum each, which
for these lengths stays below a thirty-second of the sum of sizes on average), an activation's 2^-20 and one rounding of the result."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ACC = 2.0 ** -18
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def srt():
    import swiftrt_b200 as s
    assert torch.cuda.is_available()
    return s


def _weight(srt, K, N, G, dtype, zeros, seed=0):
    g = torch.Generator().manual_seed(seed + K + 3 * N + G)
    groups = -(-K // G)
    packed = torch.randint(-2 ** 31, 2 ** 31, (-(-K // 8), N), generator=g).to(torch.int32).to(DEV)
    scales = ((0.5 + torch.rand(groups, N, generator=g)) * 0.4 * K ** -0.5).to(dtype).to(DEV)
    z = torch.randint(0, 16, (groups, N), generator=g).to(torch.uint8).to(DEV) if zeros else None
    return srt.Int4Weight(packed, scales, z, G, K)


def _value(w):
    """The weight in 64 bits."""
    K, N = w.shape
    rows = torch.arange(K, device=DEV)
    q = (w.packed.long()[rows // 8] >> (4 * (rows % 8))[:, None]) & 15
    z = 8 if w.zeros is None else (w.zeros.long() & 15)[rows // w.group]
    return (q - z).double() * w.scales.double()[rows // w.group]


def _act(name, z):
    s = torch.sigmoid(z)
    return {"identity": lambda: z, "relu": lambda: z.clamp_min(0), "silu": lambda: z * s, "sigmoid": lambda: s, "tanh": lambda: torch.tanh(z),
            "gelu": lambda: 0.5 * z * torch.erfc(-z * 0.5 ** 0.5),
            "geluTanh": lambda: 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z ** 3)))}[name]()


def _check(got, want, error):
    half = torch.finfo(got.dtype).eps / 2
    limit = error + half * (want.abs() + error) + torch.finfo(got.dtype).smallest_normal * half
    off = (got.double() - want).abs()
    assert bool((off <= limit).all()), f"{int((~(off <= limit)).sum())} of {off.numel()} off, worst {float((off / limit).max()):.3g} times its bound"


def _reference(x, w, bias):
    v = _value(w)
    z, e = x.double() @ v, ACC * (x.double().abs() @ v.abs())
    if bias is not None:
        z, e = z + bias.double(), e + 2.0 ** -23 * bias.double().abs()
    return z, e


def _check_single(srt, x, w, bias=None, act="identity"):
    got = srt.matmul_int4(x, w, bias, srt.ActivationType[act])
    z, e = _reference(x, w, bias)
    a = _act(act, z)
    _check(got, a, 1.2 * e + 2.0 ** -20 * a.abs())
    return got


SHAPES = [(1, 128, 32, 128), (1, 4096, 64, 128), (1, 1, 1, 32), (2, 7, 3, 32), (3, 33, 31, 32), (1, 100, 33, 64), (8, 256, 96, 64), (9, 520, 40, 32), (16, 1000, 36, 128),
          (17, 129, 35, 128), (31, 640, 100, 64), (33, 384, 64, 128), (70, 200, 72, 32), (4, 2048, 1001, 256), (1, 5000, 44, 128), (5, 1300, 128, 1408)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,K,N,G", SHAPES)
def test_products_match_the_definition(srt, dtype, zeros, M, K, N, G):
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(M)
    x = torch.randn(M, K, generator=g).to(dt).to(DEV)
    w = _weight(srt, K, N, G, dt, zeros)
    _check_single(srt, x, w)
    bias = torch.randn(N, generator=g).to(dt).to(DEV)
    _check_single(srt, x, w, bias, ("relu", "silu", "gelu", "geluTanh", "sigmoid", "tanh")[(M + K) % 6])
    # the gated form
    w1 = _weight(srt, K, N, G, dt, zeros, seed=5)
    b1 = torch.randn(N, generator=g).to(dt).to(DEV)
    for act in ("silu", "identity"):
        got = srt.GatedDense(w, w1, bias, b1, srt.ActivationType[act])(x)
        (g0, e0), (u0, e1) = _reference(x, w, bias), _reference(x, w1, b1)
        a, ea = _act(act, g0), 1.2 * e0 + 2.0 ** -20 * _act(act, g0).abs()
        _check(got, a * u0, ea * (u0.abs() + e1) + a.abs() * e1 + 2.0 ** -23 * (a * u0).abs())


def test_views_of_x_and_of_a_wider_weight(srt):
    """Column blocks of one packed weight at aligned and odd columns, x with any strides, leading dimensions, no rows."""
    K, N, G, dt = 300, 200, 64, torch.bfloat16
    w = _weight(srt, K, N, G, dt, True)
    g = torch.Generator().manual_seed(8)
    x = torch.randn(6, K, generator=g).to(dt).to(DEV)
    whole = _check_single(srt, x, w)
    for lo, hi in ((0, 64), (64, 200), (3, 50), (199, 200), (4, 9)):
        part = srt.Int4Weight(w.packed[:, lo:hi], w.scales[:, lo:hi], w.zeros[:, lo:hi], G, K)
        _check_single(srt, x, part)           # (how K is divided, and with it the order of the sums, depends on the columns)
    for view in (x.t().contiguous().t(), torch.cat((x, x), 1)[:, :K], torch.cat((x[:, :1], x), 1)[:, 1:], x.repeat_interleave(2, 1)[:, ::2],
                 x.repeat_interleave(2, 0)[::2]):
        assert torch.equal(srt.matmul_int4(view, w), whole)
    assert torch.equal(srt.matmul_int4(x[:1].expand(6, K), w), whole[:1].expand(6, N))
    assert torch.equal(srt.Dense(w, None, srt.ActivationType.identity)(x.view(2, 3, K)), whole.view(2, 3, N))
    assert srt.matmul_int4(x[:0], w).shape == (0, N)


def test_the_result_of_a_row_does_not_depend_on_its_neighbours(srt):
    w = _weight(srt, 640, 72, 128, torch.float16, False)
    x = torch.randn(8, 640, device=DEV).half()
    want = srt.matmul_int4(x, w)
    x[3, 100] = float("nan")
    x[5, 7] = float("inf")
    got = srt.matmul_int4(x, w)
    rest = [0, 1, 2, 4, 6, 7]
    assert torch.equal(got[rest], want[rest]) and bool(torch.isnan(got[3]).all()) and not bool(torch.isfinite(got[5]).any())


def _raw(w):
    """The C structure over the tensors as they are, without the copy that aligns their rows."""
    import ctypes

    from swiftrt_b200 import _lib
    from swiftrt_b200.tensor import data_type
    packed, scales, zeros, group, rows = w
    m = _lib.Int4Matrix(data_type(scales), group, rows, packed.shape[1], packed.data_ptr(), packed.stride(0), scales.data_ptr(), scales.stride(0),
                        zeros.data_ptr() if zeros is not None else None, zeros.stride(0) if zeros is not None else 0)
    return m, ctypes.addressof(m)


@pytest.mark.parametrize("M,K,N,G", [(1, 256, 33, 128), (3, 300, 70, 64), (9, 97, 31, 32), (20, 1000, 5, 128), (2, 2048, 130, 64)])
def test_rows_that_do_not_start_on_16_bytes(srt, M, K, N, G):
    """The C ABI takes packed weights at any column of a wider one; they run on the kernel without bulk loads."""
    from swiftrt_b200 import _lib
    from swiftrt_b200.matmul import descriptor_args, enqueue
    wide = [_weight(srt, K, N + 6, G, torch.float16, True, seed=s) for s in (0, 4)]
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(M)).half().to(DEV)
    for at in (0, 1, 3):
        parts = [(w.packed[:, at:at + N], w.scales[:, at:at + N], w.zeros[:, at:at + N], G, K) for w in wide]
        (m0, a0), (m1, a1) = (_raw(q) for q in parts)
        ref = [srt.Int4Weight(*q) for q in parts]
        out = torch.empty(M, N, dtype=torch.float16, device=DEV)
        enqueue(_lib.lib.srtMatmulInt4, x.device, *descriptor_args(x), a0, None, None, 5, *descriptor_args(out))
        z, e = _reference(x, ref[0], None)
        _check(out, z, e)
        enqueue(_lib.lib.srtMatmulGatedInt4, x.device, *descriptor_args(x), a0, a1, None, None, None, None, 5, *descriptor_args(out))
        u, f = _reference(x, ref[1], None)
        _check(out, z * u, e * (u.abs() + f) + z.abs() * f + 2.0 ** -23 * (z * u).abs())


def test_nothing_outside_the_result_is_written(srt):
    from swiftrt_b200 import _lib
    from swiftrt_b200.matmul import descriptor_args, enqueue
    for M, N in ((1, 33), (9, 64), (40, 100)):
        w = _weight(srt, 256, N, 128, torch.bfloat16, False)
        x = torch.randn(M, 256, device=DEV).to(torch.bfloat16)
        wide = torch.full((M + 2, N + 9), 5.0, dtype=torch.bfloat16, device=DEV)
        view = wide[:M, 4:N + 4]
        enqueue(_lib.lib.srtMatmulInt4, x.device, *descriptor_args(x), w.address, None, None, 5, *descriptor_args(view))
        assert torch.equal(view, srt.matmul_int4(x, w))
        assert bool((wide[M:] == 5).all()) and bool((wide[:, :4] == 5).all()) and bool((wide[:, N + 4:] == 5).all())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("K,N,G", [(128, 40, 128), (300, 33, 64), (31, 1, 32), (1, 5, 32), (700, 20, 256)])
def test_quantization_and_back_follow_their_formulas(srt, dtype, zeros, K, N, G):
    dt = TYPES[dtype]
    w = torch.randn(K, N, generator=torch.Generator().manual_seed(K)).to(dt)
    w[:, 0] = 0
    if N > 4:
        w[:, 1] = w[:, 1].abs()
        w[K // 2, 2], w[0, 3] = float("inf"), float("nan")
    q = srt.quantize_int4(w.to(DEV).t().contiguous().t() if K > 100 else w.to(DEV), G, zeros)
    groups = -(-K // G)
    for j in range(groups):
        part = w[j * G:(j + 1) * G].float()
        lo, hi = part.amin(0).clamp_max(0), part.amax(0).clamp_min(0)
        bad = ~torch.isfinite(part).all(0)
        scale = ((hi - lo) / 15 if zeros else torch.maximum(hi, -lo) / 7).to(dt)
        assert torch.equal(q.scales[j].cpu()[~bad], scale[~bad]) and bool(torch.isnan(q.scales[j].cpu()[bad]).all())
        s = scale.float()
        z = torch.where(s > 0, (torch.round(-lo / s)).clamp(0, 15), torch.full_like(s, 8.0)) if zeros else torch.full_like(s, 8.0)
        if zeros:
            assert torch.equal(q.zeros[j].cpu()[~bad].float(), z[~bad])
        want = torch.where(s > 0, (torch.round(part / s) + z).clamp(0, 15), z.expand_as(part))
        rows = torch.arange(j * G, min(K, (j + 1) * G))
        got = (q.packed.cpu().long()[rows // 8] >> (4 * (rows % 8))[:, None]) & 15
        assert torch.equal(got[:, ~bad].float(), want[:, ~bad])
    back = q.dequantize()
    good = torch.isfinite(q.scales.float()).all(0).cpu()
    assert torch.equal(back.cpu()[:, good], _value(q).cpu().to(dt)[:, good])
    # a weight is off by at most half a step of its scale, and the largest of a group by the rounding of the scale besides
    step = q.scales.float().cpu().repeat_interleave(G, 0)[:K]
    assert bool(((back.cpu().float() - w.float()).abs() <= step * (0.5 + 16 * torch.finfo(dt).eps) + 1e-7)[:, good].all())


def test_streams_graphs_and_repeats_give_the_same_bits(srt):
    for K, N in ((4096, 64), (512, 1000)):
        w, w1 = _weight(srt, K, N, 128, torch.bfloat16, True), _weight(srt, K, N, 128, torch.bfloat16, True, seed=2)
        x = torch.randn(3, K, device=DEV).to(torch.bfloat16)
        both = lambda: (srt.matmul_int4(x, w), srt.gated_matmul_int4(x, w, w1))  # noqa: E731
        before = srt.launch_count()
        want = [t.clone() for t in both()]
        assert srt.launch_count() == before + 2
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = both()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = both()
        for t in captured:
            t.zero_()
        graph.replay()
        again = both()
        torch.cuda.synchronize()
        for a, b, c, d in zip(want, other, captured, again):
            assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)


def test_a_weight_keeps_its_tensors(srt):
    """The library holds their addresses: elements may change in place, a tensor may not take another's place."""
    K, N = 128, 64
    w = _weight(srt, K, N, 64, torch.bfloat16, True)
    for name in ("packed", "scales", "zeros"):
        with pytest.raises(AttributeError):
            setattr(w, name, getattr(w, name).clone())
    x = torch.randn(2, K, device=DEV).to(torch.bfloat16)
    once = srt.matmul_int4(x, w)
    w.scales.mul_(2)
    assert torch.equal(srt.matmul_int4(x, w), once * 2)
