"""Arguments that the C entries refuse before any launch."""
import pytest
import torch

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


def linear_call(ops, grouped=False, **change):
    from ptq_int8_lab_b200.ops import _LINEAR
    a = dict(x=0, ldx=64, x_scale=0, w=0, ldw=64, w_group_stride=64 * 32, w_scale=0, bias=0, y=0, ldy=32, offsets=0, rows=2,
             in_features=64, out_features=32, groups=1, w_bits=8, epilogue=0, y_type=0)
    assert not set(change) - set(a)
    a.update(change)
    call = E.lib().ptq8_linear_grouped if grouped else E.lib().ptq8_linear
    rc = call(ops._h, _LINEAR.pack(*a.values()), None)
    return rc, E.lib().ptq8_ops_last_error(ops._h).decode()


def test_misaligned_tensors(ops):
    """A pointer that is no multiple of its element's size: refused, one operand at a time."""
    buf = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    at = [buf.data_ptr() + i * 8192 for i in range(8)]
    good = dict(x=at[0], x_rows=2, n_rows=2, codes=at[1], scale=at[2], ldx=64, ldc=64, width=64)
    assert rows_call(ops, **good)[0] == 0 and rows_call(ops, **good, rows=at[3])[0] == 0
    for change in (dict(scale=at[2] + 2), dict(rows=at[3] + 1), dict(x=at[0] + 2), dict(x=at[0] + 1, x_type=2)):
        rc, text = rows_call(ops, **{**good, **change})
        assert rc == INVALID and "aligned" in text
    good = dict(x=at[0], x_scale=at[1], w=at[2], w_scale=at[3], bias=at[4], y=at[5])
    assert linear_call(ops, **good)[0] == 0 and linear_call(ops, True, **good, offsets=at[6])[0] == 0
    for change in (dict(x_scale=at[1] + 2), dict(w_scale=at[3] + 1), dict(bias=at[4] + 2), dict(y=at[5] + 2), dict(y=at[5] + 1, y_type=2)):
        for grouped in (False, True):
            rc, text = linear_call(ops, grouped, **{**good, "offsets": at[6], **change})
            assert rc == INVALID and "aligned" in text
    rc, text = linear_call(ops, True, **good, offsets=at[6] + 2)
    assert rc == INVALID and "aligned" in text
    assert linear_call(ops, False, **good, offsets=at[6] + 2)[0] == 0   # not looked at there
    torch.cuda.synchronize()


def test_outputs_never_require_gradients(ops):
    """Inputs may (weights kept as parameters, hidden states of a layer before): the outputs are those without, and say so."""
    x = torch.randn((6, 64), device="cuda", requires_grad=True)
    codes, scale = ops.quantize_rows(x)
    again = ops.quantize_rows(x.detach())
    assert not scale.requires_grad and torch.equal(codes, again[0]) and torch.equal(scale, again[1])
    w = torch.randint(-128, 128, (32, 64), device="cuda", dtype=torch.int8)
    ws = torch.nn.Parameter(torch.rand(32, device="cuda"))
    y = ops.linear(codes, scale, w, ws, bias=ws)
    assert not y.requires_grad and torch.equal(y, ops.linear(codes, scale, w, ws.detach(), bias=ws.detach()))
