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


def test_python_refuses_host_tensors_and_bad_lengths():
    import torch

    import swiftrt_b200 as srt
    x = torch.zeros(2, 3, 4)
    with pytest.raises(ValueError, match="device tensors"):
        srt.gated_recurrence(x, x)
    from swiftrt_b200.linear_recurrent import _lengths
    for bad in (torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError, match="lengths"):
            _lengths(bad, 2)
    with pytest.raises(ValueError, match="fusedWeight"):
        srt.LinearRecurrentCell(torch.zeros(4, 10), None, 4)
