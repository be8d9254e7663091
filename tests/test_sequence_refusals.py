"""What the sequence operators refuse, through the C ABI with addresses that are never followed."""
import ctypes

import pytest

FAKE = 0x10000
F32, F64, F16, BF16 = 0, 1, 2, 14


def desc(dtype, shape, strides=None):
    from swiftrt_b200._lib import TensorDescriptor
    sz = ctypes.c_size_t
    if strides is None:
        strides, acc = [], 1
        for d in reversed(shape):
            strides.insert(0, acc)
            acc *= d
    n = 1
    for d in shape:
        n *= d
    sh, st = (sz * len(shape))(*shape), (sz * len(shape))(*strides)
    d = TensorDescriptor(dtype, len(shape), 1, n, n, sh, st, st)
    d._keep = (sh, st)
    return d


def pairs(*tensors):
    """(address, descriptor) arguments; None gives two nulls, a descriptor stands for a tensor at FAKE."""
    out = []
    for t in tensors:
        out += (None, None) if t is None else (FAKE, ctypes.addressof(t))
    return out


def forward(update, forget, input, output, initial, hidden, last, states):
    from swiftrt_b200 import _lib
    rc = _lib.lib.srtGatedRecurrence(*pairs(update, forget, input, output, initial), None, *pairs(hidden, last, states), None)
    return rc, _lib.last_error()


def seq(dtype=BF16, shape=(2, 70, 8), strides=None):
    return desc(dtype, shape, strides)


def state(shape=(2, 8), dtype=F32, strides=None):
    return desc(dtype, shape, strides)


@pytest.mark.parametrize("change,code,needle", [
    ({"update": seq(F64), "forget": seq(F64)}, 801, "not computed"),
    ({"forget": seq(F16)}, 1, "element type"),
    ({"forget": seq(shape=(2, 70, 9))}, 1, "forget must be"),
    ({"input": seq(shape=(2, 71, 8))}, 1, "input must be"),
    ({"output": seq(shape=(3, 70, 8))}, 1, "output must be"),
    ({"update": seq(shape=(2, 70, 8, 1))}, 1, "rank 3"),
    ({"hidden": seq(strides=(0, 8, 1))}, 1, "repeat"),
    ({"hidden": seq(strides=(560, 0, 1))}, 1, "repeat"),
    ({"hidden": None}, 1, "hidden"),
    ({"forget": None}, 1, "forget"),
    ({"initial": state(dtype=BF16)}, 1, "Float32"),
    ({"initial": state((2, 9))}, 1, "initial"),
    ({"last": state(strides=(8, 0))}, 1, "repeat"),
    ({"states": desc(F32, (2, 1, 8))}, 1, "states must be"),
    ({"states": desc(BF16, (2, 2, 8))}, 1, "states must be"),
])
def test_recurrence_refuses(change, code, needle):
    args = {"update": seq(), "forget": seq(), "input": None, "output": None, "initial": None, "hidden": seq(), "last": state(), "states": None}
    args.update(change)
    rc, text = forward(**args)
    assert rc == code and needle in text, (rc, text)


def test_recurrence_accepts_no_elements_without_a_device():
    none = desc(BF16, (0, 70, 8))
    assert forward(none, none, None, None, None, none, desc(F32, (0, 8)), None)[0] == 0


@pytest.mark.parametrize("change,code,needle", [
    ({"states": None}, 1, "states"),
    ({"states": desc(F32, (2, 3, 8))}, 1, "states must be"),
    ({"dUpdate": seq(F32)}, 1, "dUpdate"),
    ({"dForget": None}, 1, "dForget"),
    ({"dInput": None}, 1, "dInput"),
    ({"dOutput": seq(strides=(560, 8, 0))}, 1, "repeat"),
    ({"dInitial": state((2, 7))}, 1, "dInitial"),
    ({"outGrad": seq(shape=(2, 70, 7))}, 1, "outGrad"),
])
def test_recurrence_backward_refuses(change, code, needle):
    from swiftrt_b200 import _lib
    a = {"outGrad": seq(), "lastGrad": None, "update": seq(), "forget": seq(), "input": seq(), "output": seq(), "states": desc(F32, (2, 2, 8)),
         "dUpdate": seq(), "dForget": seq(), "dInput": seq(), "dOutput": seq(), "dInitial": state()}
    a.update(change)
    rc = _lib.lib.srtGatedRecurrenceBackward(
        *pairs(a["outGrad"], a["lastGrad"], a["update"], a["forget"], a["input"], a["output"], a["states"]), None,
        *pairs(a["dUpdate"], a["dForget"], a["dInput"], a["dOutput"], a["dInitial"]), None)
    assert rc == code and needle in _lib.last_error(), (rc, _lib.last_error())


def test_python_refuses_host_tensors_and_other_objects():
    import torch

    import swiftrt_b200 as srt
    x = torch.zeros(2, 3, 4)
    with pytest.raises(ValueError, match="device tensors"):
        srt.gated_recurrence(x, x)
    with pytest.raises(TypeError, match="update must be a tensor"):
        srt.gated_recurrence(None, x)
    with pytest.raises(TypeError, match="states must be a tensor"):
        srt.gated_recurrence_backward(x, x, x, None, None, None)
    with pytest.raises(ValueError, match="device tensors"):
        srt.GatedDense(torch.zeros(4, 6), torch.zeros(4, 6))(torch.zeros(2, 4))
    with pytest.raises(ValueError, match="fusedWeight"):
        srt.LinearRecurrentCell(torch.zeros(4, 10), None, 4)


# ------------------------------------------------------------------------------------------------ gated Dense
def mat(rows, cols, dtype=BF16, strides=None):
    return desc(dtype, (rows, cols), strides)


def vec(n, dtype=BF16, strides=None):
    return desc(dtype, (n,), strides)


def gated(change):
    from swiftrt_b200 import _lib
    a = {"x": mat(5, 16), "wg": mat(16, 24), "wu": mat(16, 24), "bg": vec(24), "bu": vec(24), "act": 8, "gate": None, "up": None, "out": mat(5, 24)}
    a.update(change)
    rc = _lib.lib.srtMatmulGated(*pairs(a["x"], a["wg"], a["wu"], a["bg"], a["bu"]), a["act"], *pairs(a["gate"], a["up"], a["out"]), None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("change,code,needle", [
    ({"x": None}, 1, "x"),
    ({"x": mat(5, 16, F64)}, 801, "not computed"),
    ({"wg": mat(17, 24)}, 1, "wGate must be"),
    ({"wu": mat(16, 25)}, 1, "wUp must be"),
    ({"wu": mat(16, 24, F16)}, 1, "element type"),
    ({"out": mat(5, 25)}, 1, "out must be"),
    ({"out": mat(5, 24, strides=(0, 1))}, 1, "repeat"),
    ({"out": desc(BF16, (1, 5, 24))}, 1, "rank 2"),
    ({"bg": vec(23)}, 1, "biasGate"),
    ({"bu": vec(24, F32)}, 1, "biasUp"),
    ({"act": 3}, 801, "coefficients"),
    ({"act": 99}, 1, "unknown activation"),
    ({"gate": mat(5, 24)}, 1, "both"),
    ({"gate": mat(5, 24), "up": mat(4, 24)}, 1, "up must be"),
])
def test_gated_refuses(change, code, needle):
    rc, text = gated(change)
    assert rc == code and needle in text, (rc, text)


def test_gated_without_rows_or_columns_launches_nothing():
    assert gated({"x": mat(0, 16), "out": mat(0, 24)})[0] == 0
    assert gated({"wg": mat(16, 0), "wu": mat(16, 0), "bg": None, "bu": None, "out": mat(5, 0)})[0] == 0


@pytest.mark.parametrize("change,code,needle", [
    ({"dy": mat(5, 23)}, 1, "outGrad must be"),
    ({"dg": None}, 1, "dGate"),
    ({"du": mat(5, 24, strides=(0, 1))}, 1, "repeat"),
    ({"dx": mat(5, 17)}, 1, "dX must be"),
    ({"dwu": mat(24, 16)}, 1, "dWUp must be"),
    ({"dbg": vec(24, strides=(0,))}, 1, "repeat"),
    ({"up": None}, 1, "up"),
    ({"act": 4}, 801, "coefficients"),
    ({"x": mat(0, 16), "dy": mat(0, 24), "gate": mat(0, 24), "up": mat(0, 24), "dg": mat(0, 24), "du": mat(0, 24), "dx": mat(0, 16)}, 1, "without elements"),
])
def test_gated_backward_refuses(change, code, needle):
    from swiftrt_b200 import _lib
    a = {"dy": mat(5, 24), "x": mat(5, 16), "wg": mat(16, 24), "wu": mat(16, 24), "gate": mat(5, 24), "up": mat(5, 24), "act": 8, "dg": mat(5, 24), "du": mat(5, 24),
         "dx": mat(5, 16), "dx2": None, "dwg": mat(16, 24), "dwu": mat(16, 24), "dbg": vec(24), "dbu": vec(24)}
    a.update(change)
    rc = _lib.lib.srtMatmulGatedBackward(*pairs(a["dy"], a["x"], a["wg"], a["wu"], a["gate"], a["up"]), a["act"],
                                         *pairs(a["dg"], a["du"], a["dx"], a["dx2"], a["dwg"], a["dwu"], a["dbg"], a["dbu"]), None)
    assert rc == code and needle in _lib.last_error(), (rc, _lib.last_error())


def test_silu_belongs_to_the_gated_and_4_bit_products():
    from swiftrt_b200 import _lib
    a, b, bias, out = mat(5, 16), mat(16, 24), vec(24), mat(5, 24)
    rc = _lib.lib.srtMatmulBiasActivation(FAKE, ctypes.byref(a), False, FAKE, ctypes.byref(b), False, FAKE, ctypes.byref(bias), 8, FAKE, ctypes.byref(out), None)
    assert rc == 801 and "silu" in _lib.last_error()


# ------------------------------------------------------------------------------------------------ 4-bit weights
def int4(rows=100, cols=24, group=64, type=BF16, packed=FAKE, ps=None, scales=FAKE, ss=None, zeros=None, zs=None):
    from swiftrt_b200 import _lib
    return _lib.Int4Matrix(type, group, rows, cols, packed, cols if ps is None else ps, scales, cols if ss is None else ss, zeros, cols if zs is None else zs)


@pytest.mark.parametrize("weight,change,code,needle", [
    ({"type": F32}, {}, 801, "Float16 or BFloat16"),
    ({"group": 0}, {}, 1, "groups are"),
    ({"group": 96}, {}, 1, "groups are"),
    ({"group": 16}, {}, 1, "groups are"),
    ({"packed": None}, {}, 1, "null"),
    ({"ps": 23}, {}, 1, "stride"),
    ({"zeros": FAKE, "zs": 3}, {}, 1, "stride"),
    ({"rows": 101}, {}, 1, "inner dimensions"),
    ({"cols": 25}, {}, 1, "out must be"),
    ({"type": F16}, {}, 1, "type of the weight"),
    ({}, {"x": desc(BF16, (1, 5, 100))}, 1, "rank 2"),
    ({}, {"bias": vec(23)}, 1, "bias"),
    ({}, {"bias": vec(24, F32)}, 1, "bias"),
    ({}, {"out": mat(5, 24, strides=(24, 0))}, 1, "repeat"),
    ({}, {"act": 4}, 801, "coefficients"),
    ({}, {"act": 77}, 1, "unknown activation"),
])
def test_int4_refuses(weight, change, code, needle):
    from swiftrt_b200 import _lib
    a = {"x": mat(5, 100), "bias": None, "act": 5, "out": mat(5, 24)}
    a.update(change)
    w = int4(**weight)
    rc = _lib.lib.srtMatmulInt4(*pairs(a["x"]), ctypes.addressof(w), *pairs(a["bias"]), a["act"], *pairs(a["out"]), None)
    assert rc == code and needle in _lib.last_error(), (rc, _lib.last_error())


def test_int4_gated_and_quantize_refuse():
    from swiftrt_b200 import _lib
    w, other = int4(), int4(group=32)
    call = lambda a, b: _lib.lib.srtMatmulGatedInt4(*pairs(mat(5, 100)), a, b, *pairs(None, None), 8, *pairs(mat(5, 24)), None)  # noqa: E731
    assert call(ctypes.addressof(w), None) == 1 and "wUp" in _lib.last_error()
    assert call(None, ctypes.addressof(w)) == 1 and "wGate" in _lib.last_error()
    assert call(ctypes.addressof(w), ctypes.addressof(other)) == 1 and "group size" in _lib.last_error()
    assert _lib.lib.srtQuantizeInt4(*pairs(mat(99, 24)), ctypes.addressof(w), None) == 1 and "w must be" in _lib.last_error()
    assert _lib.lib.srtQuantizeInt4(*pairs(mat(100, 24, F16)), ctypes.addressof(w), None) == 1
    assert _lib.lib.srtDequantizeInt4(ctypes.addressof(w), *pairs(mat(100, 25)), None) == 1 and "out must be" in _lib.last_error()
    # no rows of x: nothing to launch, whatever the machine
    assert _lib.lib.srtMatmulInt4(*pairs(mat(0, 100)), ctypes.addressof(w), None, None, 5, *pairs(mat(0, 24)), None) == 0


def test_int4_weight_checks_its_tensors():
    import torch

    import swiftrt_b200 as srt
    packed, scales = torch.zeros(13, 24, dtype=torch.int32), torch.zeros(2, 24, dtype=torch.float16)
    for args in ((packed.float(), scales, None, 64, 100), (packed[:12], scales, None, 64, 100), (packed, scales.float(), None, 64, 100),
                 (packed, scales, scales, 64, 100), (packed, scales[:1], None, 64, 100), (packed.t().contiguous().t(), scales, None, 64, 100)):
        with pytest.raises(ValueError):
            srt.Int4Weight(*args)
    with pytest.raises(ValueError, match="device tensors"):
        srt.Int4Weight(packed, scales, None, 64, 100)
