"""A state advanced in place by the CTAs of a cluster: each of them reads the state, one writes it."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,T,D", [(1, 65, 64), (1, 130, 40), (2, 500, 96), (3, 512, 33), (1, 2000, 256), (16, 100, 2048)])
@pytest.mark.parametrize("padded", [False, True])
def test_a_state_advances_in_place_as_it_does_into_a_new_tensor(dtype, B, T, D, padded):
    import swiftrt_b200 as srt
    g = torch.Generator().manual_seed(T + D)
    x, f = torch.randn(B, T, D, generator=g).to(dtype).to(DEV), (torch.randn(B, T, D, generator=g) + 3).to(dtype).to(DEV)
    lengths = torch.randint(0, T + 1, (B,), generator=g).to(torch.int32).to(DEV) if padded else None
    want = torch.randn(B, D, generator=g).to(DEV)
    states = [want.clone() for _ in range(3)]
    for step in range(40):
        hidden, new = srt.gated_recurrence(x, f, None, None, want, lengths)
        for s in states:
            got, same = srt.gated_recurrence(x, f, None, None, s, lengths, last=s)
            assert same is s and torch.equal(got, hidden)
        want = new
        x = x.roll(1, 1)
    for s in states:
        assert torch.equal(s, want)
    assert srt.check_status() == 0
