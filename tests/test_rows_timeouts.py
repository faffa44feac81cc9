"""A row that never comes leaves the residual stream as it was, also where the sum goes in place: the call can be made again."""
import pytest
import torch

from siglip_b200 import Engine
from siglip_b200 import lib as L

DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("cols", [1152, 1288, 2050, 4304, 4305])
@pytest.mark.parametrize("into", ["x", "residual"])
def test_the_sum_of_a_row_that_never_comes(monkeypatch, dtype, cols, into):
    monkeypatch.setenv("SL8_TEST_DROP_B", "1")
    dropping = Engine(0)
    monkeypatch.delenv("SL8_TEST_DROP_B")
    g = torch.Generator(device=DEV).manual_seed(cols)
    x, r = (torch.randn((9000, cols), generator=g, device=DEV).to(dtype) for _ in range(2))
    summed = x if into == "x" else r
    before, both = summed.clone(), (x.float() + r.float()).to(dtype)
    dropping.set_wait_budget_us(3000)
    dropping.rmsnorm_quantize_rows(x, residual=r, summed=summed)
    with pytest.raises(L.SL8Error) as e:
        dropping.device_status()
    assert e.value.code == L.SL8_ERR_DEVICE_TIMEOUT and dropping.last_status_detail[0] == 7 and dropping.last_status_detail[2] == 1
    dropping.close()
    assert torch.equal(summed[1], before[1])
    # every other row has its sum, or is as it was
    done = (summed == both).all(1)
    assert (done | (summed == before).all(1)).all() and done.sum() > 4000
