"""Where the operands of the row kernels lie, asked at the C ABI: many rows are copied in bulk, from memory of a GPU only."""
import pytest
import torch

from siglip_b200 import lib as L

DEV = "cuda"
BF16, F32, I8 = torch.bfloat16, torch.float32, torch.int8


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [300, 1152, 1153, 4304])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_rows_in_host_memory_are_refused(engine, cols, dtype):
    rows, lib, h, stream = 2000, engine._lib, engine._h, engine._stream(None)
    x = torch.randn((rows, cols), device=DEV).to(dtype)
    pinned, pageable = torch.zeros((rows, cols), dtype=dtype).pin_memory(), torch.zeros((rows, cols), dtype=dtype)
    out, scales, summed = torch.full((rows, cols), 85, dtype=I8, device=DEV), torch.full((rows,), -7.0, device=DEV), x.clone()
    kind = engine._dt(x)

    def rows_of(t):
        return lib.sl8_quantize_rows(h, t.data_ptr(), kind, rows, cols, cols, 1, out.data_ptr(), cols, scales.data_ptr(), stream)

    def norm_of(t, r):
        return lib.sl8_rmsnorm_quantize(h, t.data_ptr(), kind, rows, cols, cols, r.data_ptr(), cols, summed.data_ptr(), cols, None, 1e-6, 1, None, out.data_ptr(), cols,
                                        scales.data_ptr(), stream)

    for host in (pinned, pageable):
        for call in (lambda: rows_of(host), lambda: norm_of(host, x), lambda: norm_of(x, host)):
            assert call() == L.SL8_ERR_INVALID_VALUE and b"device memory" in lib.sl8_last_error_string(h)
    torch.cuda.synchronize()
    assert (out == 85).all() and (scales == -7).all() and torch.equal(summed, x)
    assert rows_of(x) == L.SL8_OK and norm_of(x, x) == L.SL8_OK
    engine.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [1152, 4305])
def test_many_rows_captured(engine, cols):
    """Asking where the operands lie is not in the way of a capture."""
    x = torch.randn((2000, cols), device=DEV).to(BF16)
    r = torch.randn((2000, cols), device=DEV).to(BF16)
    want = [t.clone() for t in (*engine.quantize_rows(x), *engine.rmsnorm_quantize_rows(x, residual=r))]
    other = torch.randn_like(x)
    held = other.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = (*engine.quantize_rows(held), *engine.rmsnorm_quantize_rows(held, residual=r))
    held.copy_(x)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    engine.device_status()
