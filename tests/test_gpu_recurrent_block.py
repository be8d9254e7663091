"""The language-model operators together: a residual block of a linear recurrence and a gated feed-forward layer, trained
on a padded batch, then quantized to 4 bits and run token by token."""
import os
import subprocess
import sys
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def srt():
    import swiftrt_b200 as s
    assert torch.cuda.is_available()
    return s


def _weights(nx, nh, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, scale: (torch.randn(*s, generator=g) * scale).to(dtype).to(DEV)  # noqa: E731
    return {"mix": n(nx, 3 * nx, scale=nx ** -0.5), "mix_bias": n(3 * nx, scale=0.5), "gate": n(nx, nh, scale=nx ** -0.5),
            "up": n(nx, nh, scale=nx ** -0.5), "down": n(nh, nx, scale=nh ** -0.5), "down_bias": n(nx, scale=0.1)}


def _reference(x, w, lengths):
    """x + recurrence(x) -> r;  r + down(gated(r)), in 64 bits with autograd."""
    B, T, nx = x.shape
    update, forget, output = (x @ w["mix"] + w["mix_bias"]).split(nx, -1)
    f, c, hs = torch.sigmoid(forget), torch.zeros(B, nx, dtype=x.dtype), []
    for t in range(T):
        on = (t < lengths)[:, None]
        c = torch.where(on, f[:, t] * c + (1 - f[:, t]) * update[:, t], c)
        hs.append(torch.where(on, c * torch.sigmoid(output[:, t]), torch.zeros_like(c)))
    r = x + torch.stack(hs, 1)
    return r + ((torch.nn.functional.silu(r @ w["gate"]) * (r @ w["up"])) @ w["down"] + w["down_bias"])


def _block(srt, w, nx):
    act = srt.ActivationType
    return (srt.LinearRecurrentCell(w["mix"], w["mix_bias"], nx), srt.GatedDense(w["gate"], w["up"], activation=act.silu),
            srt.Dense(w["down"], w["down_bias"], act.identity))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_training_step_of_a_block(srt, dtype):
    B, T, nx, nh = 3, 90, 64, 136
    w = _weights(nx, nh, dtype)
    mix, gated, down = _block(srt, w, nx)
    x = torch.randn(B, T, nx, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    lengths = torch.tensor([T, 0, 33], dtype=torch.int32, device=DEV)
    h, _, saved_mix = mix.forward_keep(x, lengths=lengths)
    r = x + h
    y1, saved_gate = gated.forward_keep(r)
    y2, kept = down.forward_keep(y1.view(-1, nh))
    y = r + y2.view_as(r)
    dy = torch.randn(B, T, nx, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    d1, d_down, d_down_bias = down.backward(y1.view(-1, nh), kept, dy.view(-1, nx))
    dr, d_gate, d_up, _, _ = gated.backward(r, saved_gate, d1.view(B, T, nh))
    dr = dr + dy
    dx, d_mix, d_mix_bias, _ = mix.backward(x, saved_mix, dr)
    dx = dx + dr
    leaves = {k: v.double().cpu().requires_grad_() for k, v in w.items()}
    x64 = x.double().cpu().requires_grad_()
    want = _reference(x64, leaves, lengths.cpu())
    want.backward(dy.double().cpu())
    # in relative 2-norm: Float32 products are within 1e-5 each, five of them in a row; every 16-bit tensor between two
    # operators is rounded by at most 2^-8, at most ten of them along a path
    limit = 5e-5 if dtype == torch.float32 else 10 * 2.0 ** -8
    for name, got, ref in (("y", y, want.detach()), ("x", dx, x64.grad), ("mix", d_mix, leaves["mix"].grad), ("mix bias", d_mix_bias, leaves["mix_bias"].grad),
                           ("gate", d_gate, leaves["gate"].grad), ("up", d_up, leaves["up"].grad), ("down", d_down, leaves["down"].grad),
                           ("down bias", d_down_bias, leaves["down_bias"].grad)):
        off = float((got.double().cpu() - ref).norm() / ref.norm())
        assert off <= limit, (name, off)


def test_generation_with_4_bit_weights_follows_the_sequence(srt):
    """A prompt through the 16-bit layers' dequantized weights, then the same block token by token through the 4-bit ones."""
    B, T, nx, nh = 2, 40, 128, 256
    act, dt = srt.ActivationType, torch.bfloat16
    w = _weights(nx, nh, dt, seed=3)
    q = {k: srt.quantize_int4(w[k], 64, zero_points=True) for k in ("mix", "gate", "up", "down")}
    exact = {**{k: v.dequantize() for k, v in q.items()}, "mix_bias": w["mix_bias"], "down_bias": w["down_bias"]}
    x = torch.randn(B, T, nx, generator=torch.Generator().manual_seed(4)).to(dt).to(DEV)
    want = _reference(x.double().cpu(), {k: v.double().cpu() for k, v in exact.items()}, torch.full((B,), T))
    mix, gated, down = _block(srt, exact, nx)
    h, state = mix(x[:, :20])
    r = x[:, :20] + h
    parts = [r + down(gated(r).view(-1, nh)).view_as(r)]
    mix4 = srt.Dense(q["mix"], w["mix_bias"], act.identity)
    gated4, down4 = srt.GatedDense(q["gate"], q["up"], activation=act.silu), srt.Dense(q["down"], w["down_bias"], act.identity)
    token, result = torch.empty(B, nx, dtype=dt, device=DEV), torch.empty(B, nx, dtype=dt, device=DEV)

    def step():
        update, forget, output = mix4(token).split(nx, -1)
        r = token + srt.gated_recurrence(update, forget, None, output, state, last=state)[0]
        result.copy_(r + down4(gated4(r)))

    before = state.clone()
    token.copy_(x[:, 20])
    step()
    state.copy_(before)
    graph = torch.cuda.CUDAGraph()                 # one token as a graph, replayed with a new token in place
    with torch.cuda.graph(graph):
        step()
    for t in range(20, T):
        token.copy_(x[:, t])
        graph.replay()
        parts.append(result.clone()[:, None])
    got = torch.cat(parts, 1).double().cpu()
    # rounding of at most 2^-8 at each of the five tensors between the operators, and 2^-9 for the dequantized weights
    off = float((got - want).norm() / want.norm())
    assert off <= 6 * 2.0 ** -8, off


FIRST_CALLS = """
import sys, torch
import swiftrt_b200 as srt
DEV = "cuda:0"
which = sys.argv[1]
r = lambda *s: torch.randn(*s, device=DEV).to(torch.bfloat16)
if which == "token":
    args = [r(2, 96) for _ in range(4)]
    call = lambda: srt.gated_recurrence(*args)
elif which == "sequence":
    args = [r(2, 200, 96) for _ in range(4)]
    call = lambda: srt.gated_recurrence(*args, keep=True)
elif which == "few":
    x, wg, wu = r(3, 128), r(128, 256), r(128, 256)
    call = lambda: (srt.GatedDense(wg, wu)(x),)
elif which == "tiles":
    x, wg, wu = r(300, 128), r(128, 256), r(128, 256)
    call = lambda: srt.GatedDense(wg, wu).forward_keep(x)[1]
elif which == "int4":
    x = r(3, 128)
    packed = torch.randint(-2 ** 31, 2 ** 31 - 1, (16, 96), device=DEV, dtype=torch.int64).to(torch.int32)
    w = srt.Int4Weight(packed, torch.rand(1, 96, device=DEV).to(torch.bfloat16), None, 128, 128)
    call = lambda: (srt.matmul_int4(x, w),)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = call()
for t in captured:
    t.zero_()
graph.replay()
torch.cuda.synchronize()
for a, b in zip(captured, call()):
    assert torch.equal(a, b)
srt.check_status(DEV)
print("right")
"""


@pytest.mark.parametrize("which", ["token", "sequence", "few", "tiles", "int4"])
def test_the_first_call_of_a_process_may_be_captured(which):
    """What a first call sets up (kernel attributes, the status word) is set up under a capture as well."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", FIRST_CALLS, which], capture_output=True, text=True, timeout=300,
                          env={**os.environ, "PYTHONPATH": root})
    assert done.returncode == 0 and "right" in done.stdout, done.stdout + done.stderr


def test_threads_and_graphs_at_once_give_the_same_bits(srt):
    """Four threads on their own streams, then two captured copies of the same calls replayed on two streams at once."""
    g = torch.Generator().manual_seed(6)
    r = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(torch.bfloat16).to(DEV)  # noqa: E731
    sequence, dy = [r(3, 300, 200) for _ in range(4)], r(3, 300, 200)
    layer = srt.GatedDense(r(256, 512, scale=0.06), r(256, 512, scale=0.06))
    rows, weight = [r(m, 256) for m in (1, 20, 100, 400)], srt.quantize_int4(r(256, 512))

    def work():
        kept = srt.gated_recurrence(*sequence, keep=True)
        out = [*kept, *srt.gated_recurrence_backward(dy, *sequence, kept[2])]
        for x in rows:
            y, saved = layer.forward_keep(x)
            out += [y, layer(x), srt.matmul_int4(x, weight), *(t for t in layer.backward(x, saved, y) if t is not None)]
        return out

    want = [t.clone() for t in work()]
    torch.cuda.synchronize()
    wrong = []

    def thread(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    got = work()
                    stream.synchronize()
                    wrong.extend((i, k) for k, (a, b) in enumerate(zip(want, got)) if not torch.equal(a, b))
                stream.synchronize()
        except Exception as e:  # noqa: BLE001  (shown by the assertion below)
            wrong.append((i, repr(e)))

    threads = [threading.Thread(target=thread, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:10]
    graphs, captured = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured.append(work())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    srt.check_status(DEV)
    for got in captured:
        assert [k for k, (a, b) in enumerate(zip(want, got)) if not torch.equal(a, b)] == []


@pytest.mark.parametrize("M,K,H", [(4096, 128, 256), (2500, 72, 120)])
def test_graphs_of_one_stream_share_no_workspace(srt, M, K, H):
    """Weight gradients of few tiles and a long reduction, which split it over a workspace of the stream when they are not
    captured: two captured copies over different inputs, replayed at once.  Small integers and the identity make every
    sum exact."""
    g = torch.Generator().manual_seed(8)
    ints = lambda *s: torch.randint(-1, 2, s, generator=g).to(torch.bfloat16).to(DEV)  # noqa: E731
    layer = srt.GatedDense(ints(K, H), ints(K, H), activation=srt.ActivationType.identity)
    inputs = [(ints(M, K), (ints(M, H), ints(M, H)), ints(M, H)) for _ in range(2)]
    want = [[t.clone() for t in layer.backward(*i)[:3]] for i in inputs]
    graphs, captured = [], []
    for i in inputs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured.append(layer.backward(*i)[:3])
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    srt.check_status(DEV)
    for x, (gate, up), dy in inputs[:1]:
        assert torch.equal(want[0][1], (x.double().t() @ (dy * up).double()).to(torch.bfloat16))
    for got, right in zip(captured, want):
        for a, b in zip(got, right):
            assert torch.equal(a, b)
