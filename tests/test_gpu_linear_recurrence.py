"""The gated linear recurrence on a B200 against its definition in 64 bits, element by element."""
import pytest
import torch

import _recurrence_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def srt():
    import swiftrt_b200 as s
    assert torch.cuda.is_available()
    return s


def _make(B, T, D, dtype, gate_in, gate_out, seed=0):
    g = torch.Generator().manual_seed(seed + 31 * B + 7 * T + D)
    normal = lambda m, s: (torch.randn(B, T, D, generator=g) * s + m).clamp(-8, 8).to(dtype).to(DEV)  # noqa: E731
    return normal(0, 1), normal(2, 1.5), normal(0, 1) if gate_in else None, normal(0, 1) if gate_out else None


def _state(B, D, seed=1):
    return torch.randn(B, D, generator=torch.Generator().manual_seed(seed)).to(DEV)


def _check_forward(srt, tensors, initial, lengths, **kw):
    hidden, last, states = srt.gated_recurrence(*tensors, initial, lengths, keep=True, **kw)
    fw = ref.forward(*tensors, initial, lengths)
    for name, got in (("hidden", hidden), ("last", last), ("states", states)):
        ref.check(got, fw[name], fw[name + "_error"], name)
    plain = srt.gated_recurrence(*tensors, initial, lengths)
    assert torch.equal(plain[0], hidden) and torch.equal(plain[1], last), "keeping the states changes the result"
    return fw, hidden, last, states


def _check_backward(srt, tensors, fw, states, lengths, dy, dlast):
    update, forget, gate_in, gate_out = tensors
    grads = srt.gated_recurrence_backward(dy, *tensors, states, lengths, last_grad=dlast)
    want = ref.backward(dy, fw, update, gate_in, gate_out, dlast)
    for name, got in zip(("update", "forget", "input", "output", "initial"), grads):
        if name in want:
            ref.check(got, *want[name], "gradient of " + name)
        else:
            assert got is None
    return grads


SHAPES = [(1, 1, 1), (2, 3, 5), (3, 63, 64), (1, 64, 130), (2, 65, 66), (1, 129, 63), (2, 640, 192), (1, 1111, 257), (1, 2500, 64), (40, 9, 70)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("gates", [(False, False), (False, True), (True, False), (True, True)], ids=["f", "fo", "fi", "fio"])
@pytest.mark.parametrize("B,T,D", SHAPES)
def test_forward_and_backward_match_the_definition(srt, dtype, gates, B, T, D):
    dt = TYPES[dtype]
    tensors = _make(B, T, D, dt, *gates)
    initial = _state(B, D) if (B + T) % 2 else None
    lengths = None
    if B > 1 and T > 1:
        lengths = torch.tensor([(T, 0, T // 2, 1, 64, T - 1)[k % 6] for k in range(B)], dtype=torch.int32, device=DEV).clamp(max=T)
    fw, hidden, _, states = _check_forward(srt, tensors, initial, lengths)
    dy = (torch.randn(B, T, D, generator=torch.Generator().manual_seed(5))).to(dt).to(DEV)
    _check_backward(srt, tensors, fw, states, lengths, dy, _state(B, D, 9) if T % 2 else None)


def test_gradients_agree_with_differences_of_the_definition(srt):
    """d/dh of sum(w . hidden) + sum(v . last) along random directions, central differences in 64 bits: their own error
    is h^2 / 6 of a third derivative, below 1e-6 of the slope at h = 1e-4, and the Float32 gradients add 2^-20 per term."""
    B, T, D = 2, 70, 6
    tensors = _make(B, T, D, torch.float32, True, True)
    initial, lengths = _state(B, D), torch.tensor([T, 41], dtype=torch.int32, device=DEV)
    g = torch.Generator().manual_seed(3)
    w, v = torch.randn(B, T, D, generator=g), torch.randn(B, D, generator=g)
    states = srt.gated_recurrence(*tensors, initial, lengths, keep=True)[2]
    grads = srt.gated_recurrence_backward(w.to(DEV), *tensors, states, lengths, last_grad=v.to(DEV))

    def value(args):
        fw = ref.forward(*args, lengths)
        return float((fw["hidden"] * w).sum() + (fw["last"] * v).sum())

    base = [t.double().cpu() for t in (*tensors, initial)]
    for k, grad in enumerate(grads):
        direction = torch.randn(base[k].shape, generator=g, dtype=torch.float64)
        up, down = list(base), list(base)
        up[k], down[k] = base[k] + 1e-4 * direction, base[k] - 1e-4 * direction
        slope = (value(up) - value(down)) / 2e-4
        ours = float((grad.double().cpu() * direction).sum())
        size = float((grad.double().cpu() * direction).abs().sum())
        assert abs(slope - ours) <= 1e-5 * size, (k, slope, ours)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_column_blocks_other_strides_and_outputs_in_place_of_a_view(srt, dtype):
    """Gates as column blocks of one product, transposed and every-other-channel views, broadcast inputs."""
    dt, B, T, D = TYPES[dtype], 2, 150, 72
    g = torch.Generator().manual_seed(11)
    fused = torch.randn(B, T, 4 * D, generator=g).to(dt).to(DEV)
    blocks = [fused[..., k * D:(k + 1) * D] for k in range(4)]
    _check_forward(srt, (blocks[1], blocks[2], blocks[0], blocks[3]), _state(B, D), None)
    odd = torch.randn(B, T, 4 * D + 1, generator=g).to(dt).to(DEV)[..., 1:]           # rows at odd element offsets
    _check_forward(srt, (odd[..., :D], odd[..., D:2 * D], None, odd[..., 2 * D:3 * D]), None, None)
    steps_first = torch.randn(T, B, D, generator=g).to(dt).to(DEV).transpose(0, 1)
    channels_first = torch.randn(B, D, T, generator=g).to(dt).to(DEV).transpose(1, 2)
    every_other = torch.randn(B, T, 2 * D, generator=g).to(dt).to(DEV)[..., ::2]
    one_gate = torch.randn(1, 1, D, generator=g).to(dt).to(DEV).expand(B, T, D)
    state = torch.randn(D, B, generator=g).to(DEV).t()
    fw, _, _, states = _check_forward(srt, (steps_first, channels_first, one_gate, every_other), state, None)
    dy = torch.randn(T, B, D, generator=g).to(dt).to(DEV).transpose(0, 1)
    _check_backward(srt, (steps_first, channels_first, one_gate, every_other), fw, states, None, dy, _state(D, B).t())
    # gradients written into the column blocks of one tensor, its other columns untouched
    wide = torch.full((B, T, 4 * D + 8), 7.0, dtype=dt, device=DEV)
    outs = tuple(wide[..., k * D:(k + 1) * D] for k in (1, 2, 0, 3))
    srt.gated_recurrence_backward(dy, steps_first, channels_first, one_gate, every_other, states, out=outs)
    assert bool((wide[..., 4 * D:] == 7).all())
    want = ref.backward(dy, fw, steps_first, one_gate, every_other)
    for name, got in zip(("update", "forget", "input", "output"), outs):
        ref.check(got, *want[name], name)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("gate_in", [False, True], ids=["fo", "fio"])
@pytest.mark.parametrize("D", [66, 67, 68])
def test_column_blocks_that_start_but_do_not_end_on_16_bytes(srt, dtype, gate_in, D):
    """66 to 68 channels in blocks of 72: rows are aligned as for whole tiles, the last channel may have no partner, and
    what lies between the blocks stays as it is."""
    dt, B, T, pitch = TYPES[dtype], 3, 140, 72
    tensors = _make(B, T, D, dt, gate_in, True)

    def wide(fill):
        return torch.full((B, T, 5 * pitch), fill, dtype=dt, device=DEV)

    def blocks(w):
        return [w[..., k * pitch:k * pitch + D] for k in range(5)]

    source = wide(float("nan"))
    inputs = []
    for view, t in zip(blocks(source), tensors):
        inputs.append(None if t is None else view.copy_(t))
    lengths = torch.tensor([T, 70, 3], dtype=torch.int32, device=DEV)
    fw, _, _, states = _check_forward(srt, tuple(inputs), _state(B, D), lengths)
    dy = blocks(source)[4].copy_(torch.randn(B, T, D, generator=torch.Generator().manual_seed(4)).to(dt).to(DEV))
    result = wide(7.0)
    outs = [v if t is not None else None for v, t in zip(blocks(result), tensors)]
    srt.gated_recurrence_backward(dy, *inputs, states, lengths, out=tuple(outs))
    want = ref.backward(dy, fw, inputs[0], inputs[2], inputs[3])
    for k, (name, got) in enumerate(zip(("update", "forget", "input", "output"), outs)):
        if got is not None:
            ref.check(got, *want[name], name)
        assert bool((result[..., k * pitch + D:(k + 1) * pitch] == 7).all()), "written behind a block"


@pytest.mark.parametrize("T", [1, 70, 300])
def test_what_lies_behind_a_sequence_is_never_read(srt, T):
    """NaN and infinities behind the lengths, and lengths outside 0 .. T, which are taken as the nearest of them."""
    B, D = 4, 66
    tensors = _make(B, T, D, torch.bfloat16, True, True)
    n = [0, T, T // 2, 1]
    clean = srt.gated_recurrence(*tensors, _state(B, D), torch.tensor(n, dtype=torch.int32, device=DEV), keep=True)
    dy = torch.randn(B, T, D, device=DEV).to(torch.bfloat16)
    clean_grads = srt.gated_recurrence_backward(dy, *tensors, clean[2], torch.tensor(n, dtype=torch.int32, device=DEV))
    dirty, dirty_dy = [t.clone() for t in tensors], dy.clone()
    for k, bad in zip((*dirty, dirty_dy), (float("nan"), float("inf"), float("nan"), -float("inf"), float("nan"))):
        for b in range(B):
            k[b, n[b]:] = bad
    lengths = torch.tensor([-5, T + 9, n[2], n[3]], dtype=torch.int32, device=DEV)
    got = srt.gated_recurrence(*dirty, _state(B, D), lengths, keep=True)
    for a, b in zip(clean, got):
        assert torch.equal(a, b)
    for b in range(B):
        assert bool((got[0][b, n[b]:] == 0).all())
    for a, b in zip(clean_grads, srt.gated_recurrence_backward(dirty_dy, *dirty, clean[2], lengths)):
        assert torch.equal(a, b) and bool(torch.isfinite(b).all())


def test_saturated_gates_and_non_finite_values(srt):
    """Logits of any size: a closed gate contributes exactly nothing of a finite value; a NaN stays in its channel."""
    T, D = 80, 34
    update, forget, _, output = _make(1, T, D, torch.float32, False, True)
    forget[:, :, 0], forget[:, :, 1] = 200.0, -200.0
    forget[:, :, 2], forget[:, :, 3] = float("inf"), -float("inf")
    output[:, :, 4] = -float("inf")
    update[:, 20, 5] = float("nan")
    initial = _state(1, D)
    hidden, last = srt.gated_recurrence(update, forget, None, output, initial)
    assert torch.equal(last[0, 0], initial[0, 0]) and torch.equal(last[0, 2], initial[0, 2])
    assert torch.equal(last[0, 1], update[0, -1, 1]) and torch.equal(last[0, 3], update[0, -1, 3])
    assert bool((hidden[0, :, 4] == 0).all())
    assert bool(torch.isfinite(hidden[0, :20, 5]).all()) and bool(torch.isnan(hidden[0, 20:, 5]).all())
    others = [d for d in range(D) if d != 5]
    assert bool(torch.isfinite(hidden[..., others]).all())


def test_no_steps_no_items_and_one_step_forms(srt):
    D = 40
    state = _state(3, D)
    empty = torch.empty(3, 0, D, device=DEV)
    hidden, last, states = srt.gated_recurrence(empty, empty, None, None, state, keep=True)
    assert hidden.shape == (3, 0, D) and states.shape == (3, 0, D) and torch.equal(last, state)
    grads = srt.gated_recurrence_backward(empty, empty, empty, None, None, states, last_grad=state)
    assert torch.equal(grads[-1], state)
    assert bool((srt.gated_recurrence(empty, empty)[1] == 0).all())
    assert len(srt.gated_recurrence(empty, empty, keep=1)) == 3
    none = torch.empty(0, 4, D, device=DEV)
    assert srt.gated_recurrence(none, none)[0].shape == (0, 4, D)
    # rank 2 is one step; a state advances in place
    tensors = _make(3, 1, D, torch.float16, True, True)
    want = srt.gated_recurrence(*tensors, state)
    flat = [t[:, 0] for t in tensors]
    got = srt.gated_recurrence(*flat, state)
    assert torch.equal(got[0], want[0][:, 0]) and torch.equal(got[1], want[1])
    moving = state.clone()
    hidden, last = srt.gated_recurrence(*flat, moving, last=moving)
    assert last is moving and torch.equal(moving, want[1]) and torch.equal(hidden, want[0][:, 0])


def test_a_sequence_in_pieces_is_the_sequence(srt):
    """Prompt in two parts and single tokens behind it: the Float32 state carries everything across the calls."""
    B, T, D = 2, 200, 96
    tensors = _make(B, T, D, torch.bfloat16, False, True)
    fw = ref.forward(*tensors)
    state, parts = None, []
    for lo, hi in ((0, 130), (130, 197), (197, 198), (198, 199), (199, 200)):
        hidden, state = srt.gated_recurrence(*(t[:, lo:hi] if t is not None else None for t in tensors), state)
        parts.append(hidden)
    ref.check(torch.cat(parts, 1), fw["hidden"], fw["hidden_error"], "hidden")
    ref.check(state, fw["last"], fw["last_error"], "last")


def test_other_streams_graphs_and_repeated_calls_give_the_same_bits(srt):
    B, T, D = 2, 333, 200
    tensors = _make(B, T, D, torch.bfloat16, True, True)
    lengths = torch.tensor([T, 100], dtype=torch.int32, device=DEV)
    dy = torch.randn(B, T, D, device=DEV).to(torch.bfloat16)

    def both():
        out = srt.gated_recurrence(*tensors, None, lengths, keep=True)
        return (*out, *srt.gated_recurrence_backward(dy, *tensors, out[2], lengths))

    want = [t.clone() for t in both()]
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


def test_offsets_beyond_32_bits(srt):
    """Two batch items more than 2^32 elements apart in one buffer."""
    T, D = 70, 64
    far = (1 << 32) + 4096
    buffer = torch.zeros(far + T * D, dtype=torch.bfloat16, device=DEV)
    x = torch.as_strided(buffer, (2, T, D), (far, D, 1))
    x.copy_(torch.randn(2, T, D, device=DEV))
    _, forget, _, output = _make(2, T, D, torch.bfloat16, False, True)
    got = srt.gated_recurrence(x, forget, None, output)
    want = srt.gated_recurrence(x.contiguous(), forget, None, output)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_layer_trains_and_generates_like_its_definition(srt):
    """LinearRecurrentCell: the sequence form, its gradients against the composition of their parts, and token by token."""
    g = torch.Generator().manual_seed(2)
    B, T, nx, nh = 3, 75, 64, 40
    for blocks in (3, 4):
        w = (torch.randn(nx, blocks * nh, generator=g) * nx ** -0.5).to(DEV)
        bias = torch.randn(blocks * nh, generator=g).to(DEV)
        cell = srt.LinearRecurrentCell(w, bias, nh)
        x = torch.randn(B, T, nx, generator=g).to(DEV)
        state = torch.randn(B, nh, generator=g).to(DEV)
        hidden, last, saved = cell.forward_keep(x, state)
        z = x.double() @ w.double() + bias.double()
        z.requires_grad_(False)
        leaves = [t.double().cpu().requires_grad_() for t in (x, w, bias, state)]
        zz = leaves[0] @ leaves[1] + leaves[2]
        parts = zz.split(nh, -1)
        update, forget, gate, output = (parts[1], parts[2], parts[0], parts[3]) if blocks == 4 else (parts[0], parts[1], None, parts[2])
        c, hs = leaves[3], []
        for t in range(T):
            f = torch.sigmoid(forget[:, t])
            i = 1 - f if gate is None else torch.sigmoid(gate[:, t])
            c = f * c + i * update[:, t]
            hs.append(c * torch.sigmoid(output[:, t]))
        want = torch.stack(hs, 1)
        # the Float32 product is within 1e-5 (its tolerance); the recurrence does not amplify it: gates are at most one
        assert float((hidden.double().cpu() - want).norm() / want.norm()) <= 2e-5
        dy, dlast = torch.randn(B, T, nh, generator=g).to(DEV), torch.randn(B, nh, generator=g).to(DEV)
        torch.autograd.backward([want, c], [dy.double().cpu(), dlast.double().cpu()])
        for got, leaf in zip(cell.backward(x, saved, dy, dlast), leaves):
            assert float((got.double().cpu() - leaf.grad).norm() / leaf.grad.norm()) <= 4e-5
        moving = state.clone()
        for t in range(T):
            token = cell.step(x[:, t], moving)
            assert float((token.double().cpu() - want[:, t].detach()).norm() / want[:, t].detach().norm()) <= 2e-5
        assert float((moving - last).norm() / last.norm()) <= 2e-5
        assert torch.equal(cell(x, state)[0], hidden)


def test_python_refuses_what_the_header_refuses(srt):
    """Errors of the C ABI come as MatmulError with their code, bad arguments as ValueError, and nothing is launched."""
    x = torch.zeros(2, 3, 4, device=DEV)
    before = srt.launch_count()
    for bad in (torch.zeros(2, dtype=torch.int64, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV)[::2]):
        with pytest.raises(ValueError, match="lengths"):
            srt.gated_recurrence(x, x, lengths=bad)
    with pytest.raises(ValueError, match="different devices"):
        srt.gated_recurrence(x, x.cpu())
    with pytest.raises(ValueError, match="steps"):
        srt.gated_recurrence(x[0, 0], x[0, 0])
    with pytest.raises(srt.MatmulError, match="forget must be") as e:
        srt.gated_recurrence(x, x[:, :2])
    assert e.value.code == 1
    with pytest.raises(srt.MatmulError, match="not computed") as e:
        srt.gated_recurrence(x.double(), x.double())
    assert e.value.code == 801
    with pytest.raises(srt.MatmulError, match="Float32"):
        srt.gated_recurrence(x, x, initial=torch.zeros(2, 4, device=DEV, dtype=torch.float16))
    with pytest.raises(srt.MatmulError, match="states must be"):
        srt.gated_recurrence_backward(x, x, x, None, None, torch.zeros(2, 2, 4, device=DEV))
    assert srt.launch_count() == before


@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_wait_that_runs_out_is_reported_and_ends_in_order(srt, dtype):
    """A limit of one nanosecond on the waits for the tiles of a long sequence: the status word says so, the kernel ends, and
    the same calls with the default limit give what they gave before."""
    tensors = _make(2, 700, 256, TYPES[dtype], False, True)
    dy = torch.randn(2, 700, 256, device=DEV).to(TYPES[dtype])
    both = lambda: (r := srt.gated_recurrence(*tensors, keep=True), srt.gated_recurrence_backward(dy, *tensors, r[2]))  # noqa: E731
    want = both()
    assert srt.check_status() == 0
    try:
        srt.set_wait_limit(1)
        both()
        assert srt.check_status() != 0
    finally:
        srt.set_wait_limit(0)
    got = both()
    assert srt.check_status() == 0
    for a, b in zip(want[0] + want[1], got[0] + got[1]):
        assert a is b is None or torch.equal(a, b)
