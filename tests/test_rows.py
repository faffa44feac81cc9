"""Operands with a scale for each row: quantise_rows, RMS norm + residual + quantisation, the product that reads them.

Against plain formulas in 64 bits.  Where the fp32 steps are few enough to be written down (the quantisation of given rows) the
result is predicted bit for bit; elsewhere the bounds count the roundings (a half step each: bf16 2^-8, e4m3 2^-4, fp32 2^-24)."""
import math

import numpy as np
import pytest
import torch

from siglip_b200 import lib as L
from tests.test_prep import nearest_e4m3

DEV = "cuda"
BF16, F32, I8, F8, U8 = torch.bfloat16, torch.float32, torch.int8, torch.float8_e4m3fn, torch.uint8
TOP = {I8: 127.0, F8: 448.0, U8: 448.0}
TINY = 2.0 ** -126


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def activations(rows, cols, dtype, seed, std=1.0):
    g = gen(seed)
    x = torch.randn((rows, cols), generator=g, device=DEV) * torch.exp(0.5 * torch.randn((cols,), generator=g, device=DEV)) * std
    return x.to(dtype)


def row_scales_of(y32: np.ndarray, top: float) -> np.ndarray:
    """The scale of each row of fp32 values, in the kernels' fp32 steps."""
    amax = np.abs(y32).max(1).astype(np.float32)
    scale = np.maximum((amax / np.float32(top)).astype(np.float32), np.float32(TINY))
    return np.where(amax == 0, np.float32(1), scale).astype(np.float32)


def row_factors_of(y32: np.ndarray, top: float) -> np.ndarray:
    """What a row's values are multiplied by to become codes: top / max, or the reciprocal of a scale that was too small."""
    amax, scale = np.abs(y32).max(1).astype(np.float32), row_scales_of(y32, top)
    with np.errstate(divide="ignore", over="ignore"):
        return np.where((amax == 0) | (scale == np.float32(TINY)), np.float32(1) / scale, np.float32(top) / amax).astype(np.float32)


def rounding(values64: np.ndarray, scale64: np.ndarray, dtype) -> np.ndarray:
    """Half a step of a code around each value."""
    if dtype == I8:
        return np.broadcast_to(scale64 / 2, values64.shape)
    return np.maximum(np.abs(values64) * 2.0 ** -4, scale64 * 2.0 ** -10)


def decoded(codes: torch.Tensor, dtype) -> np.ndarray:
    return (codes if dtype == I8 else codes.view(F8)).double().cpu().numpy()


# ----------------------------------------------------------------------------- quantise_rows
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("codes", [I8, F8, U8])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 7), (5, 40), (2, 255), (7, 256), (9, 264), (4, 768), (33, 769), (6, 1152), (1000, 1280),
                                       (3, 1288), (8, 2048), (5, 2049), (2, 4096), (301, 4304), (1, 8192), (2, 9000), (3, 16384), (2, 16392),
                                       (1, 20001)])
def test_quantize_rows_bit_for_bit(engine, oracle, dtype, codes, rows, cols):
    x = activations(rows, cols, dtype, rows * 7 + cols)
    q, scales = engine.quantize_rows(x, codes)
    engine.device_status()
    assert q.dtype == codes and q.shape == (rows, cols) and scales.shape == (rows,) and scales.dtype == F32
    x32 = x.float().cpu().numpy()
    want_scale = row_scales_of(x32, TOP[codes])
    assert np.array_equal(scales.cpu().numpy(), want_scale)
    k = row_factors_of(x32, TOP[codes])[:, None]
    if codes == I8:
        want = np.rint(x32.astype(np.float64) * k.astype(np.float64))          # an fp32 product is exact in 64 bits
        assert np.abs(want).max() <= 127 and np.array_equal(q.cpu().numpy(), want.astype(np.int8))
    else:
        # (the search in the table may name either zero, rounding keeps the sign: shown for -1e-4 and 9e-4)
        scaled = (x32 * k).astype(np.float32)
        want = nearest_e4m3(oracle, scaled)
        want = np.where((want & 0x7F) == 0, np.where(np.signbit(scaled), 0x80, 0x00), want)
        assert np.array_equal(q.view(U8).cpu().numpy(), want)
    # and, whatever the steps: within half a step of x (the factor, the product and the scale are off by 2^-24 each)
    s64 = want_scale.astype(np.float64)[:, None]
    off = np.abs(decoded(q, codes) * s64 - x32)
    assert (off <= rounding(x32, s64, codes) + np.abs(x32) * 2.0 ** -22).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("offset,pitch,out_pitch", [(0, 648, 640), (8, 648, 656), (1, 641, 641), (3, 700, 643), (4, 644, 648)])
def test_quantize_rows_strides_and_neighbours(engine, dtype, offset, pitch, out_pitch):
    """Rows at any offset and pitch; what lies between the rows, before and behind them stays."""
    rows, cols = 37, 640
    buf = activations(1, offset + rows * pitch, dtype, 11).flatten()
    x = torch.as_strided(buf, (rows, cols), (pitch, 1), offset)
    codes = torch.full((offset + (rows + 2) * out_pitch,), 85, dtype=I8, device=DEV)
    out = torch.as_strided(codes, (rows, cols), (out_pitch, 1), out_pitch + offset)
    scales = torch.full((rows + 4,), -7.0, device=DEV)
    engine.quantize_rows(x, I8, out=out, scales=scales[2:2 + rows])
    plain, plain_scales = engine.quantize_rows(x.contiguous(), I8)
    assert torch.equal(out, plain) and torch.equal(scales[2:2 + rows], plain_scales)
    assert (scales[:2] == -7).all() and (scales[2 + rows:] == -7).all()
    written = torch.zeros_like(codes, dtype=torch.bool)
    torch.as_strided(written, (rows, cols), (out_pitch, 1), out_pitch + offset).fill_(True)
    assert (codes[~written] == 85).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cols", [40, 41, 1152, 4304, 16400])
def test_quantize_rows_zeros_infinities_nans(engine, dtype, cols):
    x = activations(8, cols, dtype, 5)
    x[1] = 0.0
    x[2, cols // 2] = math.inf
    x[3, cols - 1] = math.nan
    x[4] = -0.0
    x[5, 0] = -math.inf
    x[6] = 0.0
    x[6, 3] = 1e-38          # a scale that would leave the normal range
    for codes in (I8, F8):
        q, scales = engine.quantize_rows(x, codes)
        s = scales.cpu().numpy()
        assert s[1] == 1.0 and s[4] == 1.0 and np.isnan(s[[2, 3, 5]]).all() and s[6] == np.float32(TINY)
        v = decoded(q, codes)
        assert not v[1].any() and not v[4].any()
        step = 1 if codes == I8 else 0.0625
        assert abs(v[6, 3] * TINY - float(x[6, 3])) <= step * TINY and not np.delete(v[6], 3).any()
        good, good_scales = engine.quantize_rows(x[[0, 7]].contiguous(), codes)
        assert torch.equal(q[[0, 7]].view(U8), good.view(U8)) and torch.equal(scales[[0, 7]], good_scales)


# ----------------------------------------------------------------------------- RMS norm
def norm64(x, residual, gamma, eps):
    h = x.double() + (0 if residual is None else residual.double())
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    return y if gamma is None else y * gamma.double()


def norm_error(cols):
    """Relative error of an fp32 y: h, its square, h * gamma and the product with the reciprocal root 2^-24 each, the root itself 2 units;
    squares of one sign in a sum whose longest chain is a thread's (8 per group of elements) and some 40 additions across threads."""
    chain = 8 * math.ceil(cols / 4096) * 4 + 40
    return (2 + (chain + 2) / 2 + 4 + 2) * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("codes", [I8, F8, "static"])
@pytest.mark.parametrize("residual,gamma", [(True, True), (False, True), (True, False), (False, False)])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 13), (1, 1152), (65, 768), (1001, 1152), (5, 1157), (4, 2048), (3, 2056), (130, 4304), (2, 8192), (3, 16384),
                                       (2, 12288), (3, 12192), (7, 12160), (2, 10300), (2, 17000), (1, 33001)])
def test_rmsnorm_against_64_bits(engine, dtype, codes, residual, gamma, rows, cols):
    x = activations(rows, cols, dtype, cols + rows)
    r = activations(rows, cols, dtype, cols + rows + 1, std=3.0) if residual else None
    g = 1 + 0.2 * torch.randn((cols,), generator=gen(3), device=DEV) if gamma else None
    eps = 1e-5
    y = norm64(x, r, g, eps).cpu().numpy()
    rel = norm_error(cols)
    if codes == "static":
        scale = torch.tensor([6.0 / 448.0], device=DEV)
        got = engine.rmsnorm_quantize(x, g, eps, scale, residual=r)
        q, summed = got if residual else (got, None)
        assert q.dtype == U8
        s64, kind = np.full((rows, 1), float(scale)), F8
        y = np.clip(y, -448 * s64, 448 * s64)
    else:
        q, scales, *rest = engine.rmsnorm_quantize_rows(x, g, eps, codes, residual=r)
        summed = rest[0] if residual else None
        assert q.dtype == codes and len(rest) == int(residual)
        s64, kind = scales.double().cpu().numpy()[:, None], codes
        want = np.abs(y).max(1, keepdims=True) / TOP[codes]
        assert (np.abs(s64 - want) <= want * (rel + 2.0 ** -23)).all()
    engine.device_status()
    off = np.abs(decoded(q, kind) * s64 - y)
    assert (off <= rounding(np.abs(y) * (1 + 2 * rel), s64, kind) + np.abs(y) * 2 * (rel + 2.0 ** -22)).all()
    if residual:
        assert summed.dtype == dtype and torch.equal(summed, (x.float() + r.float()).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cols", [1152, 1153, 4304, 16400, 16401])
@pytest.mark.parametrize("into", ["x", "residual"])
def test_rmsnorm_sum_in_place(engine, dtype, cols, into):
    x, r = activations(19, cols, dtype, 1), activations(19, cols, dtype, 2)
    g = torch.rand((cols,), generator=gen(3), device=DEV)
    want = engine.rmsnorm_quantize_rows(x, g, residual=r)
    a, b = x.clone(), r.clone()
    got = engine.rmsnorm_quantize_rows(a, g, residual=b, summed=a if into == "x" else b)
    assert got[2] is (a if into == "x" else b)
    for u, v in zip(got, want):
        assert torch.equal(u, v)
    assert torch.equal(b if into == "x" else a, r if into == "x" else x)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [72, 75, 1152, 4096])
def test_rmsnorm_zeros_infinities_nans_and_overflow(engine, cols):
    x = activations(8, cols, F32, 9)
    x[1] = 0.0
    x[2, 1] = math.nan
    x[3, cols - 1] = -math.inf
    x[4, 5] = 1e30                     # its square is beyond fp32
    x[5] *= 1e-12                      # eps decides
    q, scales = engine.rmsnorm_quantize_rows(x, None, 1e-6)
    s = scales.cpu().numpy()
    assert s[1] == 1.0 and not q[1].any() and np.isnan(s[2:5]).all() and np.isfinite(s[[0, 5, 6, 7]]).all()
    y = norm64(x, None, None, 1e-6).cpu().numpy()
    for i in (0, 5, 6, 7):
        assert (np.abs(decoded(q, I8)[i] * float(s[i]) - y[i]) <= float(s[i]) * (0.5 + 127 * 4 * norm_error(cols))).all()
    flat = engine.rmsnorm_quantize(x, None, 1e-6, torch.tensor([0.05], device=DEV)).view(F8).float()
    assert torch.isnan(flat[2:5]).all() and torch.isfinite(flat[[0, 1, 5, 6, 7]]).all() and not flat[1].any()
    # eps = 0 and a row of zeros is 0 / 0
    _, scales = engine.rmsnorm_quantize_rows(x, None, 0.0)
    assert torch.isnan(scales[1]) and torch.isfinite(scales[0])


@pytest.mark.gpu
def test_rmsnorm_pitched_operands(engine):
    rows, cols = 50, 520
    def pitched(seed, pitch, off):
        return torch.as_strided(activations(1, off + rows * pitch, BF16, seed).flatten(), (rows, cols), (pitch, 1), off)
    g = torch.rand((cols + 1,), generator=gen(3), device=DEV)[1:]            # 4-byte aligned only
    for px, ox, pr, orr, ps, osum in ((528, 8, 1040, 0, 520, 16), (523, 1, 520, 3, 777, 5), (520, 0, 520, 0, 521, 0)):
        x, r = pitched(1, px, ox), pitched(2, pr, orr)
        whole = torch.full((osum + (rows + 1) * ps,), 9.0, dtype=BF16, device=DEV)
        summed = torch.as_strided(whole, (rows, cols), (ps, 1), osum)
        got = engine.rmsnorm_quantize_rows(x, g, residual=r, summed=summed)
        want = engine.rmsnorm_quantize_rows(x.contiguous(), g.clone(), residual=r.contiguous())
        # The codes come from the elements and the largest of them alone; the squares are added in another order element by element.
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
        assert ((got[1] - want[1]).abs() <= want[1] * 2 * norm_error(cols)).all()
        mask = torch.ones_like(whole, dtype=torch.bool)
        torch.as_strided(mask, (rows, cols), (ps, 1), osum).fill_(False)
        assert (whole[mask] == 9.0).all()


# ----------------------------------------------------------------------------- many rows: rings in shared memory, several rows per warp or block
# (rows, columns, elements ahead of the first row, pitch): whole vectors and not, each width that has a kernel of its own
MANY = [(6100, 8, 0, 8), (9001, 64, 0, 64), (20003, 72, 0, 1152), (7001, 128, 8, 144), (5999, 120, 0, 128), (1481, 40, 0, 40), (300001, 16, 0, 16),
        (5003, 1, 0, 1), (3001, 1, 5, 3), (4001, 4, 0, 4), (9003, 7, 1, 7), (8001, 63, 0, 63), (7777, 65, 0, 65), (6666, 100, 0, 100), (2222, 129, 1, 130), (3333, 200, 4, 201), (6001, 256, 8, 272), (6011, 504, 0, 512), (6003, 768, 0, 768), (6007, 1152, 16, 1160), (12345, 1280, 0, 1280), (1481, 1288, 8, 1296), (2999, 2048, 0, 2048),
        (1777, 4304, 0, 4304), (1483, 8192, 0, 8192), (1482, 12288, 0, 12288), (1490, 12296, 8, 12304), (1485, 16384, 0, 16384), (1481, 16392, 0, 16392),
        (1700, 9, 1, 9), (1600, 13, 0, 17), (1503, 255, 3, 255), (1502, 256, 1, 257), (2001, 333, 0, 333), (1600, 511, 5, 600), (1555, 767, 0, 768), (1500, 769, 7, 769),
        (3001, 1155, 0, 1155), (1490, 2047, 1, 2049), (1481, 2050, 0, 2050), (1482, 4305, 3, 4305), (1483, 12287, 0, 12287), (1484, 12290, 1, 12290), (1481, 16383, 0, 16383),
        (1481, 16385, 1, 16385)]


def surrounded(rows, cols, ahead, pitch, dtype, seed, std=1.0):
    """Rows inside a buffer that is NaN everywhere else."""
    x = activations(rows, cols, dtype, seed, std)
    buf = torch.full((ahead + (rows - 1) * pitch + cols + 5,), math.nan, dtype=dtype, device=DEV)
    view = torch.as_strided(buf, (rows, cols), (pitch, 1), ahead)
    view.copy_(x)
    return view, buf


def fenced_codes(rows, cols, pitch):
    codes = torch.full((16 + (rows + 1) * pitch,), 85, dtype=U8, device=DEV)
    written = torch.zeros_like(codes, dtype=torch.bool)
    torch.as_strided(written, (rows, cols), (pitch, 1), 16).fill_(True)
    return codes, torch.as_strided(codes, (rows, cols), (pitch, 1), 16), written


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols,ahead,pitch", MANY)
def test_quantize_many_rows_bit_for_bit(engine, dtype, rows, cols, ahead, pitch):
    x, _ = surrounded(rows, cols, ahead, pitch, dtype, rows + cols)
    x[rows // 2] = 0.0
    for codes in (I8, F8):
        flat, out, written = fenced_codes(rows, cols, (cols + 15) // 16 * 16 + 16)
        q, scales = engine.quantize_rows(x, codes, out=out.view(codes))
        engine.device_status()
        amax = x.float().abs().amax(1)
        top = torch.tensor(TOP[codes], device=DEV)
        assert torch.equal(scales, torch.where(amax == 0, torch.ones_like(amax), amax / top))
        k = torch.where(amax == 0, torch.ones_like(amax), top / amax)[:, None]
        for r in range(0, rows, 2048):          # (products of two fp32 numbers are exact in 64 bits)
            v = x[r:r + 2048].float()
            want = torch.round(v.double() * k[r:r + 2048].double()).to(I8) if codes == I8 else (v * k[r:r + 2048]).clamp(-448.0, 448.0).to(F8)
            assert torch.equal(q[r:r + 2048].view(U8), want.view(U8)), r
        assert (flat[~written] == 85).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols,ahead,pitch", MANY)
def test_rmsnorm_of_many_rows(engine, dtype, rows, cols, ahead, pitch):
    """Against 64 bits: with a residual of another pitch into a third buffer, and without; the sum in place."""
    x, whole = surrounded(rows, cols, ahead, pitch, dtype, rows + cols)
    r, _ = surrounded(rows, cols, ahead + 8, pitch + 8, dtype, rows + cols + 1, std=3.0)
    g = 1 + 0.2 * torch.randn((cols,), generator=gen(3), device=DEV)
    rel = norm_error(cols)
    for residual, codes in ((r, I8), (None, F8), (r, "static")):
        flat, out, written = fenced_codes(rows, cols, (cols + 15) // 16 * 16)
        if codes == "static":
            q, summed = engine.rmsnorm_quantize(x, g, 1e-5, torch.tensor([0.02], device=DEV), residual=residual, out=out)
            scales, kind = torch.full((rows,), 0.02, device=DEV), F8
        else:
            q, scales, *rest = engine.rmsnorm_quantize_rows(x, g, 1e-5, codes, residual=residual, out=out.view(codes))
            summed, kind = (rest + [None])[0], codes
        engine.device_status()
        for lo in range(0, rows, 2048):
            part = slice(lo, lo + 2048)
            y = norm64(x[part], None if residual is None else residual[part], g, 1e-5)
            s = scales[part].double()[:, None]
            if codes == "static":
                y = y.clamp(-448 * 0.02, 448 * 0.02)
            else:
                want = y.abs().amax(1, keepdim=True) / TOP[codes]
                want = torch.where(want == 0, 1.0, want)         # (a row of zeros: of one column, x = -residual)
                assert ((s - want).abs() <= want * (rel + 2.0 ** -23)).all()
            half = (s / 2).expand_as(y) if kind == I8 else torch.maximum(y.abs() * (1 + 2 * rel) * 2.0 ** -4, s * 2.0 ** -10)
            value = (q[part] if kind == I8 else q[part].view(F8)).double() * s
            assert ((value - y).abs() <= half + y.abs() * 2 * (rel + 2.0 ** -22)).all(), lo
        assert (flat[~written] == 85).all()
        if residual is not None:
            assert torch.equal(summed, (x.float() + residual.float()).to(dtype))
    want = engine.rmsnorm_quantize_rows(x, g, residual=r)
    before = whole.clone()
    got = engine.rmsnorm_quantize_rows(x, g, residual=r, summed=x)
    assert got[2] is x and all(torch.equal(a, b) for a, b in zip(got, want))
    inside = torch.zeros_like(whole, dtype=torch.bool)
    torch.as_strided(inside, (rows, cols), (pitch, 1), ahead).fill_(True)
    assert torch.equal(whole[~inside].isnan(), before[~inside].isnan())


# ----------------------------------------------------------------------------- the product
def operand(rows, cols, codes, seed, pitch=None):
    g = gen(seed)
    pitch = (cols + 15) // 16 * 16 if pitch is None else pitch
    buf = torch.randint(0, 256, (rows, pitch), generator=g, device=DEV, dtype=torch.int32)
    if codes == I8:
        q = (buf - 128).to(I8)
    else:                      # any finite code, most of them of ordinary size
        q = torch.randn((rows, pitch), generator=g, device=DEV).mul_(20).clamp_(-448, 448).to(F8)
        q = torch.where(buf % 64 == 0, (buf & 0xFE).clamp(max=0xFE).to(U8), q.view(U8))
        q[(q & 0x7F) == 0x7F] = 0x10
        q = q.view(F8) if codes == F8 else q
    scales = torch.exp(torch.randn((rows,), generator=g, device=DEV)) * 1e-2
    return q[:, :cols], scales


def gelu64(y):
    return 0.5 * y * (1 + np.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))


def check_linear(got, A, B, sa, sb, bias, gelu, codes):
    as64 = lambda t: (t if codes == I8 else t.view(F8)).double()  # noqa: E731
    a, b = as64(A), as64(B)
    acc = a @ b.T
    p = (acc * sa.double()[:A.shape[0], None] * sb.double()[:B.shape[0]]).cpu().numpy()
    size = (a.abs() @ b.abs().T * sa.double()[:A.shape[0], None] * sb.double()[:B.shape[0]]).cpu().numpy()
    y = p + (0 if bias is None else bias.double().cpu().numpy())
    # the sum: exact for int8; for e4m3 K additions in fp32, off by less than a whole step (2^-23) each; then three roundings
    err = np.abs(p) * 2.0 ** -22 + np.abs(y) * 2.0 ** -23
    if codes != I8:
        err = err + size * A.shape[1] * 2.0 ** -23
    if gelu:
        y = gelu64(y)
        err = 1.13 * err + np.abs(y) * 2.0 ** -14 + TINY       # slope; ex2.approx and rcp.approx with an argument below 140
    off = np.abs(got.double().cpu().numpy() - y)
    bad = off > np.abs(y) * 2.0 ** -8 + err * (1 + 2.0 ** -8)
    assert not bad.any(), (np.argwhere(bad)[:5], got.shape)


SHAPES = [(1, 16, 1), (1, 1152, 4304), (2, 48, 16), (3, 128, 31), (8, 144, 128), (15, 272, 129), (16, 4304, 1152), (17, 256, 300), (31, 1168, 588), (32, 64, 2048),
          (33, 400, 1155), (63, 128, 640), (64, 1152, 4304), (65, 1152, 300), (100, 16, 32), (127, 48, 33), (128, 112, 4304), (129, 240, 257), (300, 336, 1155),
          (65, 144, 6144), (128, 400, 12333), (97, 2048, 6200), (61, 272, 2048), (10, 2048, 8192), (50, 2064, 8000), (729, 1152, 588), (257, 4304, 100), (1000, 592, 999)]


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [I8, F8])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_linear_scaled(engine, codes, M, N, K):
    A, sa = operand(M, K, codes, M + K)
    B, sb = operand(N, K, codes, N + K + 1)
    bias = torch.randn((N,), generator=gen(4), device=DEV)
    for b, gelu in ((bias.to(BF16), False), (None, False), (bias, True)):
        D = engine.linear_scaled(A, B, sa, sb, b, flags=L.SL8_FLAG_GELU if gelu else 0)
        engine.device_status()
        check_linear(D, A, B, sa, sb, b, gelu, codes)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [3, 40, 64, 200])
def test_linear_scaled_writes_its_matrix_only(engine, M):
    N, K = 176, 300
    for codes in (I8, U8):
        A, sa = operand(M, K, codes, 1, pitch=400)
        B, sb = operand(N, K, codes, 2, pitch=320)
        D = torch.full((M + 3, N + 24), 5.0, dtype=BF16, device=DEV)
        engine.linear_scaled(A, B, sa, sb, out=D[1:1 + M, 8:8 + N])
        check_linear(D[1:1 + M, 8:8 + N], A, B, sa, sb, None, False, codes)
        D[1:1 + M, 8:8 + N] = 5.0
        assert (D == 5.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [I8, F8])
@pytest.mark.parametrize("variant", [1, 2, 3, 14, 15, 18, 19, 20, 21])
def test_linear_scaled_every_variant(engine, codes, variant):
    """Tails of N that a CTA pair has to round up for kind::i8, tails of K and M."""
    from siglip_b200 import Engine
    with Engine(0) as e:
        e.set_variant(variant)
        for M, N, K in ((5, 16, 64), (130, 272, 200), (300, 528, 4304), (777, 1168, 96), (257, 144, 1155)):
            A, sa = operand(M, K, codes, M)
            B, sb = operand(N, K, codes, N)
            bias = torch.randn((N,), generator=gen(4), device=DEV).to(BF16)
            D = e.linear_scaled(A, B, sa, sb, bias, flags=L.SL8_FLAG_GELU)
            e.device_status()
            check_linear(D, A, B, sa, sb, bias, True, codes)


@pytest.mark.gpu
@pytest.mark.parametrize("M", [2, 70])
def test_int8_sums_are_exact_to_the_last_product(engine, M):
    """The largest K with the largest products; then a sum of which one product is left."""
    K, N = 131071, 128
    A = torch.full((M, K + 1), -128, dtype=I8, device=DEV)[:, :K]
    B = torch.full((N, K + 1), -128, dtype=I8, device=DEV)[:, :K]
    one = torch.ones((max(M, N),), device=DEV)
    D = engine.linear_scaled(A, B, one, one)
    assert (D.float() == float(torch.tensor(128.0 * 128.0 * K).to(BF16))).all()
    B = B.clone()
    B[:, :K // 2] = 127
    B[:, K // 2:K // 2 * 2] = -127
    B[:, -1] = 1
    D = engine.linear_scaled(A, torch.nn.functional.pad(B, (0, 1))[:, :K], one, one)
    assert (D.float() == -128.0).all()
    with pytest.raises(L.SL8Error) as e:
        engine.linear_scaled(torch.zeros((M, 131072), dtype=I8, device=DEV), torch.zeros((N, 131072), dtype=I8, device=DEV), one, one)
    assert e.value.code == L.SL8_ERR_UNSUPPORTED


@pytest.mark.gpu
@pytest.mark.parametrize("M", [5, 300])
def test_a_row_that_is_no_number_stays_alone(engine, M):
    x = activations(M, 512, BF16, 3)
    clean = engine.quantize_rows(x)
    x[2, 100] = math.nan
    W, sw = operand(160, 512, I8, 7)
    q, s = engine.quantize_rows(x)
    D = engine.linear_scaled(q, W, s, sw)
    want = engine.linear_scaled(*((clean[0], W, clean[1], sw)))
    assert torch.isnan(D[2]).all()
    keep = [i for i in range(M) if i != 2]
    assert torch.equal(D[keep], want[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", [(400, 2000), (1152, 4304), (272, 100)])
def test_rows_do_not_depend_on_their_neighbours(engine, N, K):
    """int8: the same rows alone and among others are the same bit for bit, whichever kernel the number of rows calls for."""
    A, sa = operand(300, K, I8, 1)
    B, sb = operand(N, K, I8, 2)
    bias = torch.randn((N,), generator=gen(4), device=DEV)
    for flags in (0, L.SL8_FLAG_GELU):
        whole = engine.linear_scaled(A, B, sa, sb, bias, flags=flags)
        for lo, hi in ((0, 1), (5, 6), (10, 26), (20, 50), (63, 64), (100, 164), (10, 139)):
            assert torch.equal(engine.linear_scaled(A[lo:hi], B, sa[lo:hi].clone(), sb, bias, flags=flags), whole[lo:hi])


@pytest.mark.gpu
def test_the_same_call_twice(engine):
    """e4m3 sums are fp32: the order of their parts is fixed."""
    for M in (1, 16, 30, 64, 500):
        A, sa = operand(M, 4304, F8, 1)
        B, sb = operand(1152, 4304, F8, 2)
        first = engine.linear_scaled(A, B, sa, sb)
        for _ in range(5):
            assert torch.equal(engine.linear_scaled(A, B, sa, sb), first)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(engine):
    """Rows that lie more than 2^31 elements apart from first to last, read and written."""
    cols = 1152
    for rows, pitch in ((3, 1 << 30), (1500, 1 << 21), (1500, (1 << 21) + 1)):
        buf = torch.empty(((rows - 1) * pitch + cols,), dtype=BF16, device=DEV)
        x = torch.as_strided(buf, (rows, cols), (pitch, 1))
        x.copy_(activations(rows, cols, BF16, 1))
        assert all(torch.equal(a, b) for a, b in zip(engine.quantize_rows(x), engine.quantize_rows(x.contiguous())))
        want = engine.rmsnorm_quantize_rows(x.contiguous(), residual=x.contiguous())
        got = engine.rmsnorm_quantize_rows(x, residual=x, summed=x)
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
        del buf, x, got
    for M, pitch in ((16, 1 << 28), (130, 1 << 25)):
        A, sa = operand(M, 256, I8, 1)
        B, sb = operand(144, 256, I8, 2)
        buf = torch.empty(((M - 1) * pitch + 144,), dtype=BF16, device=DEV)
        D = torch.as_strided(buf, (M, 144), (pitch, 1))
        engine.linear_scaled(A, B, sa, sb, out=D)
        assert torch.equal(D, engine.linear_scaled(A, B, sa, sb))
        del buf, D
    engine.device_status()


# ----------------------------------------------------------------------------- together
def block(engine, s, x, stream=None):
    """What a block with int8 operands runs between its attentions, residual additions in the norms."""
    kw = dict(stream=stream)
    q, sq, h = engine.rmsnorm_quantize_rows(x, s["g1"], residual=s["r"], **kw)
    qkv = engine.linear_scaled(q, s["qkv"], sq, s["s_qkv"], s["b_qkv"], **kw)
    o, so = engine.quantize_rows(qkv[:, :s["d"]], **kw)
    a = engine.linear_scaled(o, s["proj"], so, s["s_proj"], **kw)
    q2, sq2, h2 = engine.rmsnorm_quantize_rows(a, s["g2"], residual=h, **kw)
    f = engine.linear_scaled(q2, s["fc1"], sq2, s["s_fc1"], s["b_fc1"], flags=L.SL8_FLAG_GELU, **kw)
    f8, sf = engine.quantize_rows(f, **kw)
    return engine.linear_scaled(f8, s["fc2"], sf, s["s_fc2"], **kw), h2


def block64(s, x):
    def rows(y):
        scale = y.abs().amax(1, keepdim=True) / 127
        return torch.round(y / scale) * scale
    w = lambda n: s[n].double() * s["s_" + n].double()[:, None]  # noqa: E731
    h = x.double() + s["r"].double()
    qkv = rows(norm64(h, None, s["g1"], 1e-6)) @ w("qkv").T + s["b_qkv"].double()
    a = rows(qkv[:, :s["d"]]) @ w("proj").T
    h2 = a + h
    f = rows(norm64(h2, None, s["g2"], 1e-6)) @ w("fc1").T + s["b_fc1"].double()
    f = 0.5 * f * (1 + torch.tanh(math.sqrt(2 / math.pi) * (f + 0.044715 * f ** 3)))
    return rows(f) @ w("fc2").T, h2


def block_state(engine, rows, d, ff):
    s = dict(d=d, r=activations(rows, d, BF16, 2))
    g = gen(1)
    for name, n, k in (("qkv", 3 * d, d), ("proj", d, d), ("fc1", ff, d), ("fc2", d, ff)):
        s[name], s["s_" + name] = engine.quantize_rows(torch.randn((n, k), generator=g, device=DEV) / math.sqrt(k))
    s["b_qkv"] = (0.1 * torch.randn((3 * d,), generator=g, device=DEV)).to(BF16)
    s["b_fc1"] = 0.1 * torch.randn((ff,), generator=g, device=DEV)
    s["g1"], s["g2"] = (1 + 0.1 * torch.randn((d,), generator=g, device=DEV) for _ in range(2))
    return s


@pytest.mark.gpu
@pytest.mark.parametrize("rows,d,ff", [(1, 768, 2048), (9, 1152, 4304), (197, 768, 2048), (729, 1152, 4304)])
def test_a_block_of_them(engine, rows, d, ff):
    s = block_state(engine, rows, d, ff)
    x = activations(rows, d, BF16, 6)
    got, stream = block(engine, s, x)
    engine.device_status()
    want, h2 = block64(s, x)
    # Each of four quantisations leaves uniform errors of up to half a step, a step being the largest of a row (about 4.5 of its
    # root mean square) over 127: 4.5 / 127 / sqrt(12) = 1 % of the rms each, bf16 between the calls 0.2 % each.
    rms = lambda t: float(t.double().square().mean().sqrt())  # noqa: E731
    assert rms(got.double() - want) <= 0.03 * rms(want)
    assert rms(stream.double() - h2) <= 0.01 * rms(h2)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 300])
def test_streams_and_graphs(engine, rows):
    """On a stream of its own, captured and replayed on new inputs, two graphs of one engine in turn, and beside eager calls."""
    s = block_state(engine, rows, 768, 1024)
    xs = [activations(rows, 768, BF16, 20 + i) for i in range(3)]
    want = [[t.clone() for t in block(engine, s, x)] for x in xs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = block(engine, s, xs[1])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    held = [x.clone() for x in xs[:2]]
    graphs, outs = [], []
    for x in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(block(engine, s, x))
        graphs.append(g)
    for turn in range(3):
        for i in (0, 1):
            held[i].copy_(xs[(turn + i) % 3])
            graphs[i].replay()
        eager = block(engine, s, xs[2])
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[(turn + i) % 3]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[2]))
    engine.device_status()


@pytest.mark.gpu
def test_two_streams_at_once(engine):
    """Overlapping calls on one handle have nothing between them."""
    s = block_state(engine, 33, 768, 1024)
    xs = [activations(33, 768, BF16, 40 + i) for i in range(2)]
    want = [[t.clone() for t in block(engine, s, x)] for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(block(engine, s, xs[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


@pytest.mark.gpu
def test_clusters_beside_pairs_on_another_stream():
    """The kernels for few rows share SMs with those of CTA pairs that leave them room: neither waits for its partners while it holds
    what the other's partners wait for (tensor memory)."""
    from siglip_b200 import Engine
    with Engine(0) as pairs, Engine(0) as few:
        pairs.set_variant(13)                     # the least shared memory of the pairs
        A, _ = operand(3000, 1152, F8, 1)
        W, _ = operand(1024, 1152, F8, 2)
        x, sx = operand(5, 1152, I8, 3)
        w, sw = operand(1152, 1152, I8, 4)
        one = torch.tensor([0.01], device=DEV)
        want_a, want_b = pairs.linear_bias(A, W, None, scale_a=one), few.linear_scaled(x, w, sx, sw)
        torch.cuda.synchronize()
        got_a, got_b = torch.empty_like(want_a), torch.empty_like(want_b)
        streams = [torch.cuda.Stream() for _ in range(3)]
        for _ in range(100):
            pairs.linear_bias(A, W, None, scale_a=one, out=got_a, stream=streams[0])
            for st in streams[1:]:
                for _ in range(4):
                    few.linear_scaled(x, w, sx, sw, out=got_b, stream=st)
        torch.cuda.synchronize()
        pairs.device_status()
        few.device_status()
        assert torch.equal(got_a, want_a) and torch.equal(got_b, want_b)


@pytest.mark.gpu
def test_static_norm_feeds_the_layers_that_were_there(engine):
    x, r = activations(197, 768, BF16, 1), activations(197, 768, BF16, 2)
    scale = torch.tensor([8.0 / 448.0], device=DEV)
    q, _ = engine.rmsnorm_quantize(x, None, 1e-6, scale, residual=r)
    W, _ = operand(256, 768, F8, 3)
    D = engine.linear_bias(q, W, None, scale_a=scale)
    y = norm64(x, r, None, 1e-6)
    want = (q.view(F8).double() * float(scale)) @ W.double().T
    assert (D.double() - want).abs().max() <= want.abs().max() * 2.0 ** -7
    assert float((q.view(F8).double() * float(scale) - y).norm() / y.norm()) < 0.04


@pytest.mark.gpu
def test_a_wait_that_runs_out(monkeypatch):
    """The kernels for few rows give up like the others: a copy that is never issued, a short budget, an error status, and the next
    call is right."""
    from siglip_b200 import Engine
    monkeypatch.setenv("SL8_TEST_DROP_B", "1")
    dropping = Engine(0)
    monkeypatch.delenv("SL8_TEST_DROP_B")
    A, sa = operand(4, 2048, I8, 1)
    B, sb = operand(256, 2048, I8, 2)
    dropping.set_wait_budget_us(3000)
    dropping.linear_scaled(A, B, sa, sb)
    with pytest.raises(L.SL8Error) as e:
        dropping.device_status()
    assert e.value.code == L.SL8_ERR_DEVICE_TIMEOUT
    dropping.close()
    with Engine(0) as e:
        check_linear(e.linear_scaled(A, B, sa, sb), A, B, sa, sb, None, False, I8)
        e.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("cols", [1152, 1153, 4304])
def test_a_row_that_never_comes(monkeypatch, cols):
    """The same of the kernels that bring rows into shared memory."""
    from siglip_b200 import Engine
    monkeypatch.setenv("SL8_TEST_DROP_B", "1")
    dropping = Engine(0)
    monkeypatch.delenv("SL8_TEST_DROP_B")
    x = activations(9000, cols, BF16, 1)
    dropping.set_wait_budget_us(3000)
    dropping.quantize_rows(x)
    with pytest.raises(L.SL8Error) as e:
        dropping.device_status()
    assert e.value.code == L.SL8_ERR_DEVICE_TIMEOUT and dropping.last_status_detail[0] == 7 and dropping.last_status_detail[2] == 1
    dropping.close()
    with Engine(0) as e:
        q, s = e.quantize_rows(x)
        e.device_status()
        assert torch.equal(q[:64], e.quantize_rows(x[:64])[0])


@pytest.mark.gpu
def test_pinned_memory_is_refused(engine):
    x, host = activations(8, 64, BF16, 1), torch.zeros((8, 64), dtype=BF16).pin_memory()
    for call in (lambda: engine.quantize_rows(host), lambda: engine.quantize_rows(x, out=torch.zeros((8, 64), dtype=I8).pin_memory()),
                 lambda: engine.quantize_rows(x, scales=torch.zeros(8).pin_memory()), lambda: engine.rmsnorm_quantize_rows(host),
                 lambda: engine.rmsnorm_quantize_rows(x, torch.zeros(64).pin_memory()), lambda: engine.rmsnorm_quantize_rows(x, residual=host),
                 lambda: engine.rmsnorm_quantize_rows(x, residual=x, summed=host.clone().pin_memory()), lambda: engine.rmsnorm_quantize(x, scale=torch.ones(1).pin_memory())):
        with pytest.raises(ValueError):
            call()


@pytest.mark.gpu
def test_the_library_refuses(engine):
    """Straight at the C ABI: what the Python checks would stop."""
    lib, h = engine._lib, engine._h
    x = activations(4, 64, BF16, 1)
    out, sc = torch.zeros((4, 64), dtype=I8, device=DEV), torch.zeros((4,), device=DEV)
    p = lambda t, off=0: t.data_ptr() + off  # noqa: E731
    stream = engine._stream(None)
    quant = lambda **k: lib.sl8_quantize_rows(*({"h": h, "x": p(x), "dt": 1, "r": 4, "c": 64, "ld": 64, "t": 1, "o": p(out), "lo": 64, "s": p(sc), "st": stream} | k).values())  # noqa: E731
    assert quant() == L.SL8_OK
    for bad in (dict(x=None), dict(o=None), dict(s=None), dict(dt=2), dict(t=2), dict(t=-1), dict(r=0), dict(c=0), dict(ld=63), dict(lo=63)):
        assert quant(**bad) == L.SL8_ERR_INVALID_VALUE, bad
    assert quant(h=None) == L.SL8_ERR_INVALID_VALUE
    assert quant(r=1, c=(1 << 30) + 8, ld=1 << 31, lo=1 << 31) == L.SL8_ERR_UNSUPPORTED
    for bad in (dict(x=p(x, 1)), dict(s=p(sc, 2))):
        assert quant(**bad) == L.SL8_ERR_ALIGNMENT, bad
    norm = lambda **k: lib.sl8_rmsnorm_quantize(*({"h": h, "x": p(x), "dt": 1, "r": 4, "c": 64, "ld": 64, "res": None, "lr": 0, "sum": None, "ls": 0, "g": None, "eps": 1e-6, "t": 1,  # noqa: E731
                                                   "scale": None, "o": p(out), "lo": 64, "s": p(sc), "st": stream} | k).values())
    y = x.clone()
    assert norm() == L.SL8_OK and norm(t=0, s=None) == L.SL8_OK and norm(res=p(x), lr=64, sum=p(y), ls=64) == L.SL8_OK
    for bad in (dict(s=None), dict(scale=p(sc)), dict(res=p(x), lr=64), dict(sum=p(y), ls=64), dict(res=p(x), lr=63, sum=p(y), ls=64), dict(eps=-1.0), dict(eps=math.nan),
                dict(res=p(x), lr=64, sum=p(y), ls=63)):
        assert norm(**bad) == L.SL8_ERR_INVALID_VALUE, bad
    assert norm(g=p(sc, 2)) == L.SL8_ERR_ALIGNMENT
    A, B, D = torch.zeros((4, 64), dtype=I8, device=DEV), torch.zeros((32, 64), dtype=I8, device=DEV), torch.zeros((4, 32), dtype=BF16, device=DEV)
    sb = torch.ones((32,), device=DEV)
    lin = lambda **k: lib.sl8_linear_scaled(*({"h": h, "A": p(A), "lda": 64, "B": p(B), "ldb": 64, "t": 1, "sa": p(sc), "sb": p(sb), "bias": None, "D": p(D), "ldd": 32, "M": 4, "N": 32,  # noqa: E731
                                               "K": 64, "f": 0, "st": stream} | k).values())
    assert lin() == L.SL8_OK
    for bad in (dict(A=None), dict(B=None), dict(D=None), dict(sa=None), dict(sb=None), dict(t=2), dict(M=0), dict(N=0), dict(K=0), dict(lda=48), dict(ldd=16), dict(f=4), dict(f=8), dict(f=32)):
        assert lin(**bad) == L.SL8_ERR_INVALID_VALUE, bad
    for bad in (dict(A=p(A, 8)), dict(lda=72), dict(ldb=72), dict(ldd=36), dict(D=p(D, 8)), dict(sa=p(sc, 2)), dict(sb=p(sb, 2)), dict(bias=p(sb, 4))):
        assert lin(**bad) == L.SL8_ERR_ALIGNMENT, bad
    assert lin(N=24) == L.SL8_ERR_UNSUPPORTED
    torch.cuda.synchronize()
