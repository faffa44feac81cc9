"""Codes of bf16 rows against the quotient in whole numbers: a bf16 number has eight bits, so that x * 127 / max and x * 448 / max often lie
exactly between two codes, and these go to the even one."""
from fractions import Fraction

import numpy as np
import pytest
import torch

from tests.test_rows import MANY, activations, fenced_codes, surrounded

DEV = "cuda"
BF16, I8, F8, U8 = torch.bfloat16, torch.int8, torch.float8_e4m3fn, torch.uint8


def parts(x):
    """Whole mantissas (128 .. 255, or 0) and exponents of bf16 numbers."""
    fraction, exponent = torch.frexp(x.double())
    return (fraction * 256).long(), exponent.long() - 8


def exact_values(x, codes):
    """What the codes of each row of x stand for in steps of its scale: the nearest, ties to even (zeros in a row of zeros)."""
    m, e = parts(x)
    top, top_e = parts(x.abs().amax(1, keepdim=True))
    down = (top_e - e).clamp(max=38)                 # (beyond, the quotient is far below half of any code)
    unit = 1 if codes == I8 else 512                 # e4m3: in its smallest steps, 2^-9
    num, den = m.abs() * (127 if codes == I8 else 448 * 512), top.clamp(min=1) << down
    if codes == F8:                                  # three bits behind the leading one
        log2 = sum((num >= den << j).long() for j in range(1, 18))
        den = den << (log2 - 3).clamp(min=0)
    q = num // den
    twice = 2 * (num - q * den)
    q = q + ((twice > den) | ((twice == den) & (q % 2 == 1))).long()
    if codes == F8:
        q = q << (log2 - 3).clamp(min=0)
    return m.sign() * q.double() / unit


def every_pair():
    """[128, 3840]: in row i every bf16 number of both signs from its largest one, 128 + i, down to a thirty-thousandth of it."""
    top = torch.arange(128, 256).double()[:, None]
    steps = (torch.arange(128, 256).double()[None] * torch.ldexp(torch.ones(15, dtype=torch.float64), -torch.arange(15))[:, None]).flatten()[None]
    x = torch.where(steps <= top, steps, top)
    return torch.cat((x, -x), 1).to(BF16)


def test_the_whole_numbers():
    """exact_values against fractions, on a few of the pairs; all of them against the fp32 steps that the kernels take."""
    x = every_pair()
    rng = np.random.default_rng(0)
    i8, f8 = exact_values(x, I8), exact_values(x, F8)
    grid = sorted({Fraction(m) * Fraction(2) ** e for m in range(16) for e in range(-9, 6)} - {Fraction(480)})
    for i, j in zip(rng.integers(0, 128, 400), rng.integers(0, x.shape[1], 400)):
        v, top = Fraction(float(x[i, j])), Fraction(float(x[i].abs().max()))
        assert round(v * 127 / top) == int(i8[i, j])                       # (Python rounds halves to even)
        want = abs(v) * 448 / top
        off = min(abs(g - want) for g in grid)
        near = [g for g in grid if abs(g - want) == off]
        got = abs(Fraction(float(f8[i, j])))
        assert got in near
        if len(near) == 2:
            code = int(torch.tensor([float(got)]).to(F8).view(torch.uint8))
            assert code % 2 == 0
    halves = (exact_values(x, I8) - x.double() * 127 / x.double().amax(1, keepdim=True)).abs() == 0.5
    assert halves.any(1).all()                       # (half of the largest is in every row)

    v, top = x.float().numpy(), x.float().numpy().max(1, keepdims=True)
    up = (np.float32(127) / top).astype(np.float32)
    up = np.where(up.astype(np.float64) * top < 127, np.nextafter(up, np.float32(np.inf)), up)          # the quotient rounded up
    assert np.array_equal(np.rint(v.astype(np.float64) * up), i8.numpy())
    k = (np.float32(448) / top).astype(np.float32)
    rest = ((448 - k.astype(np.float64) * top) / top).astype(np.float32)
    q = (v.astype(np.float64) * k + (v * rest).astype(np.float64)).astype(np.float32)
    assert torch.equal(torch.from_numpy(q).to(F8).double(), f8)


def check(engine, x):
    for codes in (I8, F8):
        q, scales = engine.quantize_rows(x, codes)
        engine.device_status()
        assert torch.equal(q.double(), exact_values(x, codes)), codes
        top = torch.tensor(127.0 if codes == I8 else 448.0, device=DEV)
        assert torch.equal(scales, x.float().abs().amax(1) / top)


@pytest.mark.gpu
@pytest.mark.parametrize("times", [1, 12, 47])
@pytest.mark.parametrize("columns", [3840, 768, 256, 128, 64])
def test_every_pair_of_numbers(engine, times, columns):
    """From a row per block to a ring or several rows per warp; the largest of each row in front of whatever part of it comes."""
    x = every_pair().to(DEV)
    for lo in range(0, x.shape[1], columns):
        part = x[:, lo:lo + columns].clone()
        part[:, 0] = x[:, 0:128].amax(1)
        check(engine, part.repeat(times, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(1, 7), (3, 40), (5, 1152), (7, 4304), (4, 4305), (2, 9000), (2, 16392), (1, 20001), (1601, 7), (2000, 63), (2000, 64), (1999, 100), (1777, 256), (1500, 333),
                                       (2001, 1152), (6007, 1152), (1490, 769), (1500, 4304), (1482, 4305), (1481, 12296), (1481, 16385)])
def test_rows_of_any_width(engine, rows, cols):
    g = torch.Generator(device=DEV).manual_seed(rows + cols)
    x = (torch.randn((rows, cols), generator=g, device=DEV) * torch.exp(3 * torch.randn((rows, 1), generator=g, device=DEV))).to(BF16)
    x[:, cols // 2] = x.abs().amax(1) / 2            # 63.5 steps of int8
    x[x == 0] = 1e-3
    check(engine, x)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(7, 256), (9, 264), (4, 768), (33, 769), (6, 1152), (1000, 1280), (8, 2048), (5, 2049), (301, 4304), (2, 16392)])
def test_few_rows(engine, rows, cols):
    x = activations(rows, cols, BF16, rows * 7 + cols)
    check(engine, x)
    q, scales = engine.quantize_rows(x, U8)
    assert q.dtype == U8 and torch.equal(q.view(F8).double(), exact_values(x, F8)) and torch.equal(scales, engine.quantize_rows(x, F8)[1])


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,ahead,pitch", MANY)
def test_many_rows(engine, rows, cols, ahead, pitch):
    """Rows with NaN all around them and a row of zeros among them; codes with others' bytes around them."""
    x, _ = surrounded(rows, cols, ahead, pitch, BF16, rows + cols)
    x[rows // 2] = 0.0
    for codes in (I8, F8):
        flat, out, written = fenced_codes(rows, cols, (cols + 15) // 16 * 16 + 16)
        q, scales = engine.quantize_rows(x, codes, out=out.view(codes))
        engine.device_status()
        amax = x.float().abs().amax(1)
        assert torch.equal(scales, torch.where(amax == 0, 1.0, amax / torch.tensor(127.0 if codes == I8 else 448.0, device=DEV)))
        for r in range(0, rows, 2048):
            part = x[r:r + 2048]
            assert torch.equal(q[r:r + 2048].double(), exact_values(part, codes)), r
            if codes == F8:          # zeros keep their sign
                assert torch.equal(q[r:r + 2048].view(U8) >= 128, torch.signbit(part)), r
        assert (flat[~written] == 85).all()
