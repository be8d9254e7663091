"""The gated layer's backward pass with its tensors at changing places in memory, next to what is and is not mapped there."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("M,K,H,bias,odd", [(25, 304, 912, True, True), (25, 304, 912, False, False), (40, 96, 264, True, False), (2, 200, 3304, True, False)])
def test_gradients_do_not_depend_on_where_tensors_lie(M, K, H, bias, odd):
    import swiftrt_b200 as srt
    rng = random.Random(M + H)
    g = torch.Generator().manual_seed(H)
    h = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).half().to(DEV)  # noqa: E731
    src = [h(M, K), h(K, H + 8, scale=K ** -0.5), h(K, H + 3 if odd else H, scale=K ** -0.5), h(M, 2 * H), h(M, 2 * H), h(M, H + 32), h(H), h(H)]
    others, want = [], None
    for _ in range(150):
        for _ in range(rng.randint(0, 6)):
            others.append(torch.empty(rng.choice([300, 5000, 60000, 400000, 900000, 3000000]), dtype=torch.uint8, device=DEV))
        while len(others) > 60 or (others and rng.random() < 0.5):
            others.pop(rng.randrange(len(others)))
        x, wg, wu, gate, up, dy, bg, bu = (t.clone() for t in src)
        wu = wu[:, 1:1 + H] if odd else wu
        layer = srt.GatedDense(wg[:, 8:], wu, bg if bias else None, bu if bias else None)
        grads = [t for t in layer.backward(x, (gate[:, ::2], up[:, ::2]), dy[:, 16:16 + H]) if t is not None]
        want = want or [t.clone() for t in grads]
        assert all(torch.equal(a, b) for a, b in zip(grads, want))
    assert srt.check_status() == 0
