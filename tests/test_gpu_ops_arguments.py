"""Arguments that the C entries refuse before any launch."""
import pytest

from ptq_int8_lab_b200 import engine as E

pytestmark = pytest.mark.gpu

INVALID = 1   # PTQ8_ERR_INVALID


@pytest.fixture(scope="module")
def ops():
    from ptq_int8_lab_b200.ops import Int8Ops
    return Int8Ops(0)


def rows_call(ops, x=0, ldx=16, x_rows=0, rows=0, n_rows=0, codes=0, ldc=16, scale=0, width=16, x_type=0):
    from ptq_int8_lab_b200.ops import _ROWS
    args = _ROWS.pack(x, ldx, x_rows, rows, n_rows, codes, ldc, scale, width, x_type)
    rc = E.lib().ptq8_quantize_rows(ops._h, args, None)
    return rc, E.lib().ptq8_ops_last_error(ops._h).decode()


@pytest.mark.parametrize("width,rc", [(0x7FFFFFF0, 0), (0x7FFFFFF1, INVALID), (0x7FFFFFFF, INVALID), (0, INVALID), (-5, INVALID)])
def test_row_width(ops, width, rc):
    """Rows whose last vector would end past an int are refused.  (No rows: nothing is launched either way.)"""
    got, text = rows_call(ops, width=width, ldx=1 << 31, ldc=1 << 31)
    assert got == rc and (rc == 0 or "width" in text)
