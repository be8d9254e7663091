"""What the 4-bit products read of a weight's tensors: rows one behind the other, each where the library is told that it starts."""
import pytest
import torch


def _read(t):
    """The tensor as the library reads it: its address, and max(stride, columns) elements from row to row."""
    from swiftrt_b200.int4 import _on_rows_of
    nbytes = {torch.int32: 16, torch.bfloat16: 8, torch.uint8: 4}[t.dtype]
    a = _on_rows_of(t, nbytes)
    step = max(a.stride(0), a.shape[1])
    inside = a.storage_offset() + (a.shape[0] - 1) * step + a.shape[1] <= a.untyped_storage().nbytes() // a.element_size()
    assert inside, "rows behind the end of the tensor's memory"
    return a.as_strided(a.shape, (step, 1))


@pytest.mark.parametrize("dtype", [torch.int32, torch.bfloat16, torch.uint8])
@pytest.mark.parametrize("rows,cols", [(1, 1), (5, 1), (1, 32), (6, 32), (6, 33), (3, 1001)])
def test_repeated_and_overlapping_rows_are_read_as_they_are(dtype, rows, cols):
    base = torch.arange(rows * cols + 64).remainder(200).to(dtype)
    views = [base[:rows * cols].view(rows, cols), base[:cols].expand(rows, cols), base[:1].expand(rows, cols).contiguous(),
             base.as_strided((rows, cols), (cols // 32 * 16, 1)), base.repeat(rows).view(rows, -1)[:, 3:3 + cols]]
    for v in views:
        assert torch.equal(_read(v), v)


@pytest.mark.gpu
def test_products_with_repeated_scales():
    import swiftrt_b200 as srt
    for cols in (64, 1):
        g = torch.Generator().manual_seed(cols)
        packed = torch.randint(-2 ** 31, 2 ** 31, (32, cols), generator=g).to(torch.int32).cuda()
        scales, zeros = (torch.rand(1, cols, generator=g) + 0.5).to(torch.bfloat16).cuda(), torch.randint(0, 16, (1, cols), generator=g).to(torch.uint8).cuda()
        x = torch.randn(3, 256, generator=g).to(torch.bfloat16).cuda()
        whole = srt.Int4Weight(packed, scales.repeat(8, 1), zeros.repeat(8, 1), 32, 256)
        for w in (srt.Int4Weight(packed, scales.expand(8, cols), zeros.expand(8, cols), 32, 256),
                  srt.Int4Weight(packed[:1].expand(32, cols), scales.expand(8, cols), zeros.expand(8, cols), 32, 256)):
            want = whole if w.packed.equal(packed) else srt.Int4Weight(packed[:1].repeat(32, 1), scales.repeat(8, 1), zeros.repeat(8, 1), 32, 256)
            assert torch.equal(srt.matmul_int4(x, w), srt.matmul_int4(x, want)) and torch.equal(w.dequantize(), want.dequantize())
