"""The descriptors of a call live as long as the call, whatever becomes of the cache that they come from."""
import ctypes
import importlib

import pytest
import torch


class _Stream:
    cuda_stream = 0


@pytest.mark.parametrize("tensors", [1, 11])
def test_descriptors_outlive_the_cache_while_a_call_runs(monkeypatch, tensors):
    matmul = importlib.import_module("swiftrt_b200.matmul")
    from swiftrt_b200._lib import TensorDescriptor
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda index: _Stream)
    given = [torch.zeros(3 + i, 2, 5) for i in range(tensors)]
    seen = []

    def churn(base):
        # what another thread's calls do to the cache: more geometries than it holds
        for n in range(2 * matmul._DESC_CACHE_MAX):
            matmul._descriptor(torch.empty(1).expand(base + n, 7))

    def callee(*args):
        churn(100000)
        for i in range(tensors):
            d = ctypes.cast(args[2 * i + 1], ctypes.POINTER(TensorDescriptor))[0]
            seen.append((d.rank, d.count, [d.shape[j] for j in range(3)] if d.rank == 3 else None))
        return 0

    proto = ctypes.CFUNCTYPE(ctypes.c_int, *[ctypes.c_void_p] * (2 * tensors + 3))
    args = matmul.descriptor_args(*given)
    churn(1000)
    matmul.enqueue(proto(callee), torch.device("cuda", 0), *args, *matmul.descriptor_args(None))
    assert seen == [(3, t.numel(), list(t.shape)) for t in given]


def test_one_call_may_have_more_geometries_than_the_cache_has_room_for(monkeypatch):
    matmul = importlib.import_module("swiftrt_b200.matmul")
    from swiftrt_b200._lib import TensorDescriptor
    monkeypatch.setattr(matmul, "_DESC_CACHE_MAX", 2)
    matmul._DESC_CACHE.clear()
    given = [torch.zeros(2, 3 + i) for i in range(8)]
    read = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p)(lambda at: ctypes.cast(at, ctypes.POINTER(TensorDescriptor))[0].shape[1])
    args = matmul.descriptor_args(*given)
    [torch.zeros(i + 1).tolist() for i in range(100)]
    assert [read(a) for a in args[1::2]] == [3 + i for i in range(8)]
