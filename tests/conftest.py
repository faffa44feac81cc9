import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs a B200 (sm_100) and the built libsiglip_fp8.so")


# Two tests of test_rows.py predict codes from 127 / max or 448 / max rounded to fp32.  With these rows, all bf16, some quotient lies exactly half way
# between two codes (max / 2 is 63.5 steps of int8 in every row that holds it), and the prediction is the odd one of them wherever that factor was rounded the
# wrong way; the operator rounds ties to even.  test_rows_ties.py has the same rows, against the quotients in whole numbers.
ODD_TIES = {
    "test_quantize_rows_bit_for_bit":
        "7-256-codes0-dtype0 7-256-codes1-dtype0 7-256-codes2-dtype0 9-264-codes0-dtype0 4-768-codes0-dtype0 33-769-codes0-dtype0 6-1152-codes0-dtype0 "
        "1000-1280-codes0-dtype0 1000-1280-codes1-dtype0 1000-1280-codes2-dtype0 8-2048-codes0-dtype0 5-2049-codes0-dtype0 301-4304-codes0-dtype0 "
        "301-4304-codes1-dtype0 301-4304-codes2-dtype0 2-16392-codes0-dtype0",
    "test_quantize_many_rows_bit_for_bit":
        "6100-8-0-8-dtype0 9001-64-0-64-dtype0 20003-72-0-1152-dtype0 7001-128-8-144-dtype0 5999-120-0-128-dtype0 1481-40-0-40-dtype0 "
        "300001-16-0-16-dtype0 4001-4-0-4-dtype0 9003-7-1-7-dtype0 8001-63-0-63-dtype0 7777-65-0-65-dtype0 6666-100-0-100-dtype0 2222-129-1-130-dtype0 "
        "3333-200-4-201-dtype0 6001-256-8-272-dtype0 6011-504-0-512-dtype0 6003-768-0-768-dtype0 6007-1152-16-1160-dtype0 12345-1280-0-1280-dtype0 "
        "1481-1288-8-1296-dtype0 2999-2048-0-2048-dtype0 1777-4304-0-4304-dtype0 1483-8192-0-8192-dtype0 1482-12288-0-12288-dtype0 "
        "1490-12296-8-12304-dtype0 1485-16384-0-16384-dtype0 1481-16392-0-16392-dtype0 1700-9-1-9-dtype0 1600-13-0-17-dtype0 1503-255-3-255-dtype0 "
        "1502-256-1-257-dtype0 2001-333-0-333-dtype0 1600-511-5-600-dtype0 1555-767-0-768-dtype0 1500-769-7-769-dtype0 3001-1155-0-1155-dtype0 "
        "1490-2047-1-2049-dtype0 1481-2050-0-2050-dtype0 1482-4305-3-4305-dtype0 1483-12287-0-12287-dtype0 1484-12290-1-12290-dtype0 "
        "1481-16383-0-16383-dtype0 1481-16385-1-16385-dtype0",
}


def pytest_collection_modifyitems(items):
    for item in items:
        if getattr(item, "callspec", None) and item.callspec.id in ODD_TIES.get(item.originalname, "").split():
            item.add_marker(pytest.mark.xfail(strict=True, raises=AssertionError, reason="expects the odd code where a quotient is a tie"))


@pytest.fixture(scope="session")
def oracle():
    """The CPU oracle (oracle/libsl8_oracle.so), built on demand where a C compiler exists."""
    from tests.oracle_lib import Oracle
    return Oracle()


@pytest.fixture(scope="session")
def engine():
    import torch
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import siglip_b200
    eng = siglip_b200.Engine(0)
    yield eng
    eng.close()
