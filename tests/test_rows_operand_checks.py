"""What the calls for operands with a scale per row refuse before any launch and what they let through, with and without the extension
module (tests/fake_abi.py); the formulas the GPU tests compare with, on the CPU."""
import json
import math

import numpy as np
import pytest
import torch

from tests import fake_abi
from tests.fake_abi import STREAM, cuda

U8, I8, F8, BF16, F32, F16 = torch.uint8, torch.int8, torch.float8_e4m3fn, torch.bfloat16, torch.float32, torch.float16
S = dict(stream=STREAM)


def x(rows=8, cols=32, dtype=BF16, **kw):
    return cuda(rows, cols, dtype=dtype, **kw)


def rows(e, **kw):
    kw = dict(out=cuda(8, 32, dtype=I8), scales=cuda(8, dtype=F32)) | kw
    return e.quantize_rows(kw.pop("x", x()), kw.pop("dtype", I8), **kw, **S)


def norm(e, **kw):
    kw = dict(out=cuda(8, 32, dtype=I8), scales=cuda(8, dtype=F32)) | kw
    return e.rmsnorm_quantize_rows(kw.pop("x", x()), kw.pop("gamma", None), 1e-6, kw.pop("dtype", I8), **kw, **S)


def static(e, **kw):
    kw = dict(out=cuda(8, 32)) | kw
    return e.rmsnorm_quantize(kw.pop("x", x()), kw.pop("gamma", None), 1e-6, kw.pop("scale", cuda(1, dtype=F32)), **kw, **S)


def linear(e, **kw):
    kw = dict(out=cuda(8, 64, dtype=BF16)) | kw
    return e.linear_scaled(kw.pop("A", cuda(8, 32, dtype=I8)), kw.pop("B", cuda(64, 32, dtype=I8)), kw.pop("sa", cuda(8, dtype=F32)),
                           kw.pop("sb", cuda(64, dtype=F32)), kw.pop("bias", None), **kw, **S)


host = torch.zeros
REFUSED = {
    "rows_few_rows": lambda e: rows(e, out=cuda(7, 32, dtype=I8)),
    "rows_few_columns": lambda e: rows(e, out=cuda(8, 24, dtype=I8, stride=(32, 1))),
    "rows_out_type": lambda e: rows(e, out=cuda(8, 32)),
    "rows_out_type_of_e4m3": lambda e: rows(e, dtype=F8),
    "rows_no_such_codes": lambda e: rows(e, dtype=BF16),
    "rows_x_type": lambda e: rows(e, x=x(dtype=F16)),
    "rows_x_strided": lambda e: rows(e, x=x(stride=(64, 2))),
    "rows_x_three_dimensions": lambda e: rows(e, x=cuda(2, 4, 32, dtype=BF16)),
    "rows_x_on_the_host": lambda e: rows(e, x=host(8, 32)),
    "rows_x_other_gpu": lambda e: rows(e, x=x(device=1)),
    "rows_scales_short": lambda e: rows(e, scales=cuda(7, dtype=F32)),
    "rows_scales_type": lambda e: rows(e, scales=cuda(8, dtype=BF16)),
    "rows_scales_strided": lambda e: rows(e, scales=cuda(8, dtype=F32, stride=(2,))),
    "rows_scales_on_the_host": lambda e: rows(e, scales=host(8)),
    "rows_out_on_the_host": lambda e: rows(e, out=host(8, 32, dtype=I8)),
    "norm_gamma_short": lambda e: norm(e, gamma=cuda(31, dtype=F32)),
    "norm_gamma_type": lambda e: norm(e, gamma=cuda(32, dtype=BF16)),
    "norm_residual_type": lambda e: norm(e, residual=x(dtype=F32)),
    "norm_residual_shape": lambda e: norm(e, residual=x(7)),
    "norm_residual_one_row": lambda e: norm(e, residual=x(1)),
    "norm_residual_strided": lambda e: norm(e, residual=x(stride=(64, 2))),
    "norm_residual_on_the_host": lambda e: norm(e, residual=host(8, 32, dtype=BF16)),
    "norm_summed_type": lambda e: norm(e, residual=x(), summed=x(dtype=F32)),
    "norm_summed_shape": lambda e: norm(e, residual=x(), summed=x(9)),
    "norm_summed_without_residual": lambda e: norm(e, summed=x()),
    "norm_scales_short": lambda e: norm(e, scales=cuda(7, dtype=F32)),
    "norm_out_type": lambda e: norm(e, out=cuda(8, 32, dtype=F8)),
    "static_out_int8": lambda e: static(e, out=cuda(8, 32, dtype=I8)),
    "static_scale_type": lambda e: static(e, scale=cuda(1, dtype=BF16)),
    "static_gamma_on_the_host": lambda e: static(e, gamma=host(32)),
    "linear_mixed": lambda e: linear(e, B=cuda(64, 32)),
    "linear_mixed_too": lambda e: linear(e, A=cuda(8, 32, dtype=F8)),
    "linear_bf16": lambda e: linear(e, A=cuda(8, 32, dtype=BF16), B=cuda(64, 32, dtype=BF16)),
    "linear_k": lambda e: linear(e, B=cuda(64, 48, dtype=I8)),
    "linear_a_strided": lambda e: linear(e, A=cuda(8, 32, dtype=I8, stride=(64, 2))),
    "linear_no_scale_a": lambda e: linear(e, sa=None),
    "linear_no_scale_b": lambda e: linear(e, sb=None),
    "linear_scale_a_of_the_tensor": lambda e: linear(e, sa=cuda(1, dtype=F32)),
    "linear_scale_b_short": lambda e: linear(e, sb=cuda(63, dtype=F32)),
    "linear_scale_a_type": lambda e: linear(e, sa=cuda(8, dtype=BF16)),
    "linear_scale_b_strided": lambda e: linear(e, sb=cuda(64, dtype=F32, stride=(0,))),
    "linear_scale_on_the_host": lambda e: linear(e, sa=host(8)),
    "linear_bias_short": lambda e: linear(e, bias=cuda(63, dtype=BF16)),
    "linear_bias_type": lambda e: linear(e, bias=cuda(64, dtype=F16)),
    "linear_bias_flag_contradicts": lambda e: linear(e, bias=cuda(64, dtype=BF16), flags=1),
    "linear_out_type": lambda e: linear(e, out=cuda(8, 64)),
    "linear_out_shape": lambda e: linear(e, out=cuda(9, 64, dtype=BF16)),
    "linear_other_gpu": lambda e: linear(e, sb=cuda(64, dtype=F32, device=1)),
}
TAKEN = {
    "rows": lambda e: rows(e),
    "rows_e4m3": lambda e: rows(e, dtype=F8, out=cuda(8, 32, dtype=F8)),
    "rows_raw": lambda e: rows(e, dtype=U8, out=cuda(8, 32)),
    "rows_raw_into_float8": lambda e: rows(e, dtype=U8, out=cuda(8, 32, dtype=F8)),
    "rows_f32": lambda e: rows(e, x=x(dtype=F32)),
    "rows_pitched": lambda e: rows(e, x=x(stride=(40, 1)), out=cuda(8, 32, dtype=I8, stride=(48, 1))),
    "rows_larger_buffers": lambda e: rows(e, out=cuda(10, 40, dtype=I8), scales=cuda(20, dtype=F32)),
    "rows_one_column": lambda e: rows(e, x=x(8, 1, stride=(16, 16)), out=cuda(8, 1, dtype=I8, stride=(16, 16))),
    "norm": lambda e: norm(e),
    "norm_gamma": lambda e: norm(e, gamma=cuda(32, dtype=F32)),
    "norm_residual_into_new": lambda e: norm(e, residual=x(), summed=x()),
    "norm_residual_pitched": lambda e: norm(e, residual=x(stride=(40, 1)), summed=x(stride=(64, 1))),
    "norm_e4m3": lambda e: norm(e, dtype=F8, out=cuda(8, 32, dtype=F8), residual=x(), summed=x()),
    "static": lambda e: static(e),
    "static_no_scale": lambda e: static(e, scale=None, gamma=cuda(32, dtype=F32), residual=x(), summed=x()),
    "linear": lambda e: linear(e),
    "linear_e4m3": lambda e: linear(e, A=cuda(8, 32, dtype=F8), B=cuda(64, 32)),
    "linear_gelu": lambda e: linear(e, bias=cuda(64, dtype=BF16), flags=16),
    "linear_f32_bias": lambda e: linear(e, bias=cuda(64, dtype=F32)),
    "linear_scales_of_more": lambda e: linear(e, sa=cuda(12, dtype=F32), sb=cuda(64, 2, dtype=F32)),
    "linear_one_row": lambda e: linear(e, A=cuda(1, 32, dtype=I8), sa=cuda(1, dtype=F32), out=cuda(1, 64, dtype=BF16)),
}
ALL = {f"refused_{k}": v for k, v in REFUSED.items()} | {f"taken_{k}": v for k, v in TAKEN.items()}


@pytest.fixture(scope="module")
def answers(tmp_path_factory):
    folder = tmp_path_factory.mktemp("fake")
    fake_abi.install(folder)
    r = fake_abi.run_child(folder, "tests.test_rows_operand_checks", "ALL")
    assert r.returncode == 0, r.stderr[-2000:]
    return json.loads(r.stdout.splitlines()[-1])


@pytest.mark.parametrize("name", sorted(REFUSED))
def test_refused(answers, name):
    for route, (error, message, calls) in answers[f"refused_{name}"].items():
        assert error in ("TypeError", "ValueError") and message and not calls, (route, error, message, calls)


@pytest.mark.parametrize("name", sorted(TAKEN))
def test_taken_alike_on_both_routes(answers, name):
    fast, slow = (answers[f"taken_{name}"][r] for r in ("extension", "python"))
    assert fast[0] is None and slow[0] is None, (fast, slow)
    assert len(fast[2]) == 1 and fast[2] == slow[2]


def test_null_handles():
    from siglip_b200 import build
    build.build()
    import siglip_b200.lib as L
    lib = L.load_library()
    assert lib.sl8_quantize_rows(None, None, 1, 1, 8, 8, 1, None, 8, None, None) == L.SL8_ERR_INVALID_VALUE
    assert lib.sl8_rmsnorm_quantize(None, None, 1, 1, 8, 8, None, 0, None, 0, None, 1e-6, 1, None, None, 8, None, None) == L.SL8_ERR_INVALID_VALUE
    assert lib.sl8_linear_scaled(None, None, 16, None, 16, 1, None, None, None, None, 16, 1, 16, 16, 0, None) == L.SL8_ERR_INVALID_VALUE


def test_the_predicted_codes_are_half_a_step_off_at_most(oracle):
    """The prediction that test_rows.py holds the kernels to, bit for bit, against the definition in 64 bits."""
    from tests.test_prep import nearest_e4m3
    from tests.test_rows import row_factors_of, row_scales_of
    rng = np.random.default_rng(0)
    y = (rng.standard_normal((200, 333)) * np.exp(rng.standard_normal((200, 1)) * 8)).astype(np.float32)
    y[3] = 0
    y[4] = 0
    y[4, 1] = 1e-39
    for top, half in ((127.0, lambda v, s: np.broadcast_to(s / 2, v.shape)), (448.0, lambda v, s: np.maximum(np.abs(v) / 16, s * 2.0 ** -10))):
        scale = row_scales_of(y, top)
        assert scale[3] == 1.0 and scale[4] == np.float32(2.0 ** -126)
        k = row_factors_of(y, top)[:, None]
        assert np.isfinite(k).all()
        if top == 127.0:
            v = np.rint(y.astype(np.float64) * k)
            assert np.abs(v).max() == 127
        else:
            v = oracle.e4m3_lut().astype(np.float64)[nearest_e4m3(oracle, (y * k).astype(np.float32))]
            assert np.abs(v).max() == 448
        s = scale.astype(np.float64)[:, None]
        assert (np.abs(v * s - y) <= half(y, s) + np.abs(y) * 2.0 ** -22).all()
        assert math.isclose(float(scale[0]), float(np.abs(y[0]).max()) / top, rel_tol=2.0 ** -23)
