"""Few-row products at sizes where x takes most of a CTA's shared memory, against their definition in 64 bits on a sample of columns.

Bounds.  Products are exact in fp32, sums of n terms lose at most 2^-23 of the running sum per add (truncating ones included).  For
independent terms the running sum stays below 5 / sqrt(n) of the sum S of their sizes (five deviations; |x w| is 0.64 on average), 2/3 of that on
average over the adds.
  4-bit: within a group at most 16 truncating adds on the group's own sum, 2^-19 S at worst; then one add for every 128 (32 at least) rows, up
  to 768 of half a step (2^-24) of at most S / 20 on average: 2^-18.7 S.  Together below ACC = 2^-17.8.
  16-bit: K / 16 adds into one accumulator at most, 5.2 / sqrt(K) of S each: K sqrt(1 / K) 5.2 / 16 2^-23 S = 2^-17.3 S at K = 28672: ACC = 2^-17.
An activation adds 2^-20 of its value, slopes are below 1.1, and the result is rounded once."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
COLUMNS = 96


@pytest.fixture(scope="module")
def srt():
    import swiftrt_b200 as s
    assert torch.cuda.is_available()
    return s


def _randn(*shape, seed, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    out = torch.empty(shape, dtype=dtype, device=DEV)
    for part in out.split(4096):
        part.copy_(torch.randn(part.shape, generator=g, device=DEV) * scale)
    return out


def _columns(N, seed=1):
    g = torch.Generator().manual_seed(seed)
    picked = torch.cat((torch.randint(0, N, (COLUMNS,), generator=g), torch.tensor([0, N // 2, N - 1])))
    return picked.unique().to(DEV)


def _check(got, want, error):
    half = torch.finfo(got.dtype).eps / 2
    limit = error + half * (want.abs() + error) + torch.finfo(got.dtype).smallest_normal * half
    off = (got.double() - want).abs()
    assert bool((off <= limit).all()), f"{int((~(off <= limit)).sum())} of {off.numel()} off, worst {float((off / limit).max()):.3g} times its bound"


def _int4_weight(srt, K, N, G, dtype, zeros, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + K + 3 * N + G)
    groups = -(-K // G)
    packed = torch.randint(-2 ** 31, 2 ** 31, (-(-K // 8), N), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    scales = ((0.5 + torch.rand(groups, N, generator=g, device=DEV)) * (0.4 * K ** -0.5)).to(dtype)
    z = torch.randint(0, 16, (groups, N), generator=g, device=DEV, dtype=torch.int32).to(torch.uint8) if zeros else None
    return srt.Int4Weight(packed, scales, z, G, K)


def _int4_columns(w, columns):
    K, _ = w.shape
    rows = torch.arange(K, device=DEV)
    q = (w.packed[:, columns].long()[rows // 8] >> (4 * (rows % 8))[:, None]) & 15
    z = 8 if w.zeros is None else (w.zeros[:, columns].long() & 15)[rows // w.group]
    return (q - z).double() * w.scales[:, columns].double()[rows // w.group]


def _check_int4(srt, M, K, N, G, dtype, zeros):
    x = _randn(M, K, seed=M, dtype=dtype)
    w = _int4_weight(srt, K, N, G, dtype, zeros)
    columns = _columns(N)
    got = srt.matmul_int4(x, w)
    torch.cuda.synchronize()
    v = _int4_columns(w, columns)
    _check(got[:, columns], x.double() @ v, 2.0 ** -17.8 * (x.double().abs() @ v.abs()))
    assert srt.check_status() == 0


@pytest.mark.parametrize("M,K,N,G,dtype,zeros", [
    (32, 6144, 12288, 128, "bf16", False), (17, 12288, 14336, 128, "fp16", True), (17, 6144, 24576, 64, "bf16", True), (48, 6144, 8192, 32, "fp16", False),
    (32, 12288, 12288, 128, "bf16", True), (24, 8192, 16384, 128, "fp16", False), (33, 6400, 24576, 128, "bf16", False), (32, 24576, 4096, 32, "bf16", True),
    (17, 24576, 4104, 256, "fp16", True), (512, 6144, 6144, 128, "bf16", False)])
def test_4_bit_products_where_x_leaves_little_room(srt, M, K, N, G, dtype, zeros):
    _check_int4(srt, M, K, N, G, {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype], zeros)


@pytest.mark.parametrize("M,K,N,by_columns", [(12, 14336, 28672, False), (15, 24576, 8192, False), (16, 10240, 28672, False), (13, 28672, 8200, False),
                                              (16, 24576, 4096, True), (40, 10240, 12288, False), (8, 28672, 4096, False)])
def test_gated_products_where_x_leaves_little_room(srt, M, K, N, by_columns):
    x = _randn(M, K, seed=M)
    weights = [_randn(N, K, seed=s, scale=K ** -0.5).t() if by_columns else _randn(K, N, seed=s, scale=K ** -0.5) for s in (1, 2)]
    got = srt.GatedDense(*weights)(x)
    torch.cuda.synchronize()
    columns = _columns(N)
    (g, eg), (u, eu) = ((x.double() @ v, 2.0 ** -17 * (x.double().abs() @ v.abs())) for v in (w[:, columns].double() for w in weights))
    a = g * torch.sigmoid(g)
    ea = 1.1 * eg + 2.0 ** -20 * a.abs()
    _check(got[:, columns], a * u, ea * (u.abs() + eu) + a.abs() * eu + 2.0 ** -23 * (a * u).abs())
    assert srt.check_status() == 0


# x of these reductions fits beside no stage: the kernel that takes any view computes them
@pytest.mark.parametrize("M,K,N,G,dtype,zeros", [(8, 131072, 4096, 128, "bf16", False), (8, 110000, 32, 64, "fp16", True), (33, 120000, 100, 32, "bf16", True)])
def test_4_bit_products_without_room_for_x(srt, M, K, N, G, dtype, zeros):
    _check_int4(srt, M, K, N, G, {"bf16": torch.bfloat16, "fp16": torch.float16}[dtype], zeros)


@pytest.mark.parametrize("H", [60, 64])
def test_gated_products_without_room_for_x(srt, H):
    """Weights contiguous along K; results of 60 columns do not start on 16 bytes, which leaves the kernel without tiles."""
    M, K = 8, 131072
    x = _randn(M, K, seed=5)
    weights = [_randn(H, K, seed=s, scale=K ** -0.5).t() for s in (1, 2)]
    layer = srt.GatedDense(*weights)
    before = srt.launch_count()
    got = layer(x)
    torch.cuda.synchronize()
    assert srt.launch_count() == before + 1
    # (up to 131072 / 16 adds into one accumulator: 8192 5.2 / sqrt(131072) 2^-23 S)
    (g, eg), (u, eu) = ((x.double() @ w.double(), 2.0 ** -16 * (x.double().abs() @ w.double().abs())) for w in weights)
    a = g * torch.sigmoid(g)
    ea = 1.1 * eg + 2.0 ** -20 * a.abs()
    _check(got, a * u, ea * (u.abs() + eu) + a.abs() * eu + 2.0 ** -23 * (a * u).abs())
    assert srt.check_status() == 0


def test_gated_4_bit_product_without_room_for_x(srt):
    M, K, N = 8, 110000, 64
    x = _randn(M, K, seed=7)
    w = [_int4_weight(srt, K, N, 128, torch.bfloat16, True, seed=s) for s in (0, 1)]
    got = srt.gated_matmul_int4(x, *w)
    torch.cuda.synchronize()
    (g, eg), (u, eu) = ((x.double() @ v, 2.0 ** -17.8 * (x.double().abs() @ v.abs())) for v in (_int4_columns(i, torch.arange(N, device=DEV)) for i in w))
    a = g * torch.sigmoid(g)
    ea = 1.1 * eg + 2.0 ** -20 * a.abs()
    _check(got, a * u, ea * (u.abs() + eu) + a.abs() * eu + 2.0 ** -23 * (a * u).abs())
    assert srt.check_status() == 0


def test_more_rows_than_a_launch_has_room_for_are_refused(srt):
    w = _int4_weight(srt, 1, 4, 32, torch.bfloat16, False)
    x = torch.ones(1, 1, dtype=torch.bfloat16, device=DEV)
    most = 1048560
    assert torch.equal(srt.matmul_int4(x.expand(most, 1), w)[::4099], srt.matmul_int4(x, w).expand(256, 4))
    with pytest.raises(srt.MatmulError, match="too many rows"):
        srt.matmul_int4(x.expand(2200000, 1), w)
