"""Products into column blocks of a wider matrix: what lies behind a row of the block stays as it is, also where the block
starts on 16 bytes and ends between them.  The factors are small integers, so that every sum is exact in 32 bits and the
result has one right value."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("M,N,K", [(1, 70, 64), (40, 69, 128), (300, 70, 128), (515, 1001, 192), (2048, 1027, 256)])
def test_columns_behind_the_block_are_left_alone(dtype, M, N, K):
    import swiftrt_b200 as srt
    dt, g = TYPES[dtype], torch.Generator().manual_seed(M + N)
    a = torch.randint(-2, 3, (M, K), generator=g).to(dt).to(DEV)
    b = torch.randint(-2, 3, (K, N), generator=g).to(dt).to(DEV)
    pitch = (N + 15) // 8 * 8
    for wide in (torch.full((M, 2 * pitch), 7.0, dtype=dt, device=DEV), torch.full((M, pitch), 7.0, dtype=dt, device=DEV)):
        srt.matmul_into(wide[:, :N], a, False, b, False)
        srt.check_status(DEV)
        want = (a.double() @ b.double()).to(dt)
        assert torch.equal(wide[:, :N], want)
        assert bool((wide[:, N:] == 7).all()), "written behind the block"
