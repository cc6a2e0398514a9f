"""Token operators without a GPU: what is exported, packed and refused."""
import ctypes

import pytest
import torch

from ptq_int8_lab_b200 import engine as E


def test_argument_structs():
    """The packed formats have the C structs' sizes (the library asserts the same numbers)."""
    from ptq_int8_lab_b200 import ops
    assert ops._ROWS.size == 72 and ops._LINEAR.size == 120


def test_null_handles():
    L = E.lib()
    assert L.ptq8_linear(None, None, None) == 1 and L.ptq8_linear_grouped(None, None, None) == 1
    assert L.ptq8_quantize_rows(None, None, None) == 1
    assert L.ptq8_ops_check_device_error(None, None) == 1 and L.ptq8_ops_set_wait_test(None, 0, 0) == 1
    assert L.ptq8_ops_last_error(None) == b"null handle"
    L.ptq8_ops_destroy(None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="needs a machine without a GPU")
def test_no_gpu_is_an_error():
    from ptq_int8_lab_b200.ops import Int8Ops
    with pytest.raises(E.Ptq8Error, match="ptq8_ops_create"):
        Int8Ops(0)
    err = ctypes.create_string_buffer(4)   # a short buffer gets a cut message
    assert not E.lib().ptq8_ops_create(0, err, len(err))
    assert len(err.value) == 3


def test_weights_are_quantized_like_the_engine_s():
    """lay_weights' codes and scales are quantize_weight's: checked on the host parts it is made of."""
    import numpy as np
    from ptq_int8_lab_b200.package import pack_w4, unpack_w4
    w = np.random.default_rng(0).normal(0, 1, (5, 33)).astype(np.float32)
    codes, scale = E.quantize_weight(w, 4)
    assert np.array_equal(unpack_w4(pack_w4(codes), 33), codes) and scale.shape == (5,)
