"""Layers of the recurrent block on inputs without elements: no rows in a batch, no steps, no batch items."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def srt():
    import swiftrt_b200 as s
    assert torch.cuda.is_available()
    return s


def _randn(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device=DEV).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lead", [(0,), (0, 3), (4, 0), (2, 0, 5)])
def test_gated_dense_without_rows(srt, dtype, lead):
    layer = srt.GatedDense(_randn(16, 24, dtype=dtype), _randn(16, 24, dtype=dtype))
    x = torch.empty(*lead, 16, device=DEV, dtype=dtype)
    assert layer(x).shape == (*lead, 24)
    y, (gate, up) = layer.forward_keep(x)
    assert y.shape == (*lead, 24) and gate.shape == up.shape == (0, 24)
    with pytest.raises(srt.MatmulError, match="without elements"):
        layer.backward(x, (gate, up), y)


@pytest.mark.parametrize("lead", [(0,), (0, 3), (4, 0)])
def test_4_bit_layers_without_rows(srt, lead):
    w, w1 = srt.quantize_int4(_randn(64, 24), 32), srt.quantize_int4(_randn(64, 24), 32)
    x = torch.empty(*lead, 64, device=DEV, dtype=torch.bfloat16)
    assert srt.matmul_int4(x, w).shape == (*lead, 24)
    assert srt.gated_matmul_int4(x, w, w1).shape == (*lead, 24)
    assert srt.Dense(w, None, srt.ActivationType.relu)(x).shape == (*lead, 24)
    assert srt.GatedDense(w, w1)(x).shape == (*lead, 24)


def test_gated_dense_of_no_terms_with_leading_dimensions(srt):
    b = _randn(24)
    layer = srt.GatedDense(_randn(0, 24), _randn(0, 24), None, b, srt.ActivationType.sigmoid)
    y = layer(torch.empty(2, 3, 0, device=DEV, dtype=torch.bfloat16))
    assert torch.equal(y, (0.5 * b).expand(2, 3, 24))


@pytest.mark.parametrize("blocks", [3, 4])
@pytest.mark.parametrize("B,T", [(0, 5), (3, 0), (0, 0)])
def test_recurrent_layer_without_items_or_steps(srt, blocks, B, T):
    cell = srt.LinearRecurrentCell(_randn(16, blocks * 8), _randn(blocks * 8), 8)
    x = torch.empty(B, T, 16, device=DEV, dtype=torch.bfloat16)
    state = torch.randn(B, 8, device=DEV)
    hidden, last = cell(x, state)
    assert hidden.shape == (B, T, 8) and torch.equal(last, state)
    hidden, last, saved = cell.forward_keep(x, state)
    assert hidden.shape == (B, T, 8) and torch.equal(last, state) and saved[1].shape == (B, 0 if T == 0 else 1, 8)
    assert cell.step(torch.empty(0, 16, device=DEV, dtype=torch.bfloat16), torch.empty(0, 8, device=DEV)).shape == (0, 8)
    with pytest.raises(srt.MatmulError):                    # no rows: there is no sum for the bias
        cell.backward(x, saved, hidden)
