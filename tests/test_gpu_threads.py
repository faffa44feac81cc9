"""Calls from several threads at once, straight at the C ABI (ctypes lets go of the interpreter lock while a call runs)."""
import ctypes as C
import threading

import pytest
import torch

from siglip_b200 import Engine
from siglip_b200 import lib as L

DEV = "cuda"
BF16, F32, I8, U8 = torch.bfloat16, torch.float32, torch.int8, torch.uint8


def from_threads(calls, turns):
    """Each call `turns` times from a thread of its own, all at once: the set of what each returned."""
    start, got = threading.Barrier(len(calls)), [set() for _ in calls]

    def work(i):
        start.wait()
        for _ in range(turns):
            got[i].add(calls[i]())

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("handles", [1, 2])
@pytest.mark.parametrize("rows,widths", [(1500, (4096, 8192, 12288)), (4, (10400, 11600, 12288))])
def test_row_kernels_of_different_widths(handles, rows, widths):
    """One kernel, as much shared memory as each width needs: no call takes from another what it has been granted."""
    engines = [Engine(0) for _ in range(handles)]
    g = torch.Generator(device=DEV).manual_seed(1)
    calls, checks, streams = [], [], [torch.cuda.Stream() for _ in range(2 * len(widths))]
    for i, stream in enumerate(streams):
        cols, e = widths[i % len(widths)], engines[i % handles]
        x, r = (torch.randn((rows, cols), generator=g, device=DEV).to(BF16) for _ in range(2))
        gamma = torch.rand((cols,), generator=g, device=DEV)
        want = engines[0].rmsnorm_quantize_rows(x, gamma, residual=r)
        q, s, h = torch.zeros_like(want[0]), torch.zeros_like(want[1]), torch.zeros_like(x)
        args = (e._h, x.data_ptr(), L.SL8_DT_BF16, rows, cols, cols, r.data_ptr(), cols, h.data_ptr(), cols, gamma.data_ptr(), 1e-6, L.SL8_CODE_INT8, None,
                q.data_ptr(), q.stride(0), s.data_ptr(), C.c_void_p(stream.cuda_stream))
        calls.append(lambda args=args, f=e._lib.sl8_rmsnorm_quantize: f(*args))
        checks.append(((q, s, h), want, x, r, gamma))
    torch.cuda.synchronize()
    assert from_threads(calls, 1500) == [{L.SL8_OK}] * len(calls)
    torch.cuda.synchronize()
    for e in engines:
        e.device_status()
        e.close()
    for got, want, *_ in checks:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_patch_unfolds_of_different_sizes():
    """The same of the patch unfold: patches of 64 x 64 and of 128 x 128 take 48 and 96 KiB in one kernel."""
    e = Engine(0)
    calls, checks, streams = [], [], [torch.cuda.Stream() for _ in range(4)]
    scale = torch.tensor([0.02], device=DEV)
    for i, stream in enumerate(streams):
        channels, patch = ((6, 64), (3, 128))[i % 2]
        pixels = torch.randn((8, channels, patch, patch), generator=torch.Generator(device=DEV).manual_seed(i), device=DEV).to(BF16)
        want = e.patchify_quantize(pixels, patch, scale)
        out = torch.zeros_like(want)
        args = (e._h, pixels.data_ptr(), L.SL8_DT_BF16, 8, channels, patch, patch, patch, scale.data_ptr(), out.data_ptr(), out.stride(0), C.c_void_p(stream.cuda_stream))
        calls.append(lambda args=args: e._lib.sl8_patchify_quantize_e4m3(*args))
        checks.append((out, want, pixels))
    torch.cuda.synchronize()
    assert from_threads(calls, 1500) == [{L.SL8_OK}] * len(calls)
    torch.cuda.synchronize()
    e.close()
    for out, want, _ in checks:
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_texts_of_calls_that_fail_at_once():
    """Refused calls of several threads on one handle: each text that is read is one that was written."""
    with Engine(0) as e:
        x, out, scales = torch.zeros((4, 64), dtype=BF16, device=DEV), torch.zeros((4, 64), dtype=I8, device=DEV), torch.zeros((4,), device=DEV)

        def refused(dtype, code_type, at):
            assert e._lib.sl8_quantize_rows(e._h, x.data_ptr() + at, dtype, 4, 64, 64, code_type, out.data_ptr(), 64, scales.data_ptr(), None) != L.SL8_OK
            return e._lib.sl8_last_error_string(e._h)

        calls = [lambda: refused(7, 1, 0), lambda: refused(1, 9, 0), lambda: refused(1, 1, 1)]
        texts = {call() for call in calls}
        assert len(texts) == 3 and all(texts)
        for got in from_threads(calls * 3, 20000):
            assert got <= texts
