"""CPU checks of linear_cross_entropy, keep8 and linear(checkpoint=True): argument refusals (they come before
any device work) and the sizes of the work spaces."""
import pytest

import endia_b200 as nd
from endia_b200 import _lib
from endia_b200._array import Array, ArrayShape
from endia_b200.functional.keep_ops import keeps_sign, rows_and_cols


def meta(*shape, requires_grad=False, is_complex=False):
    """An array without storage: enough for every check that must come before a kernel is enqueued."""
    a = Array(ArrayShape(list(shape)))
    a.requires_grad_flag = requires_grad
    a.is_complex_flag = is_complex
    return a


def refused(status, fn, *args, **kw):
    with pytest.raises(_lib.EndiaError) as e:
        fn(*args, **kw)
    assert e.value.status == status, e.value


def test_cross_entropy_refusals():
    f = nd.linear_cross_entropy
    x, w, t = meta(4, 8), meta(8, 16), meta(4)
    refused(_lib.EINVAL, f, x, w, t, reduction="avg")
    refused(_lib.EINVAL, f, meta(4, 8, is_complex=True), w, t)
    refused(_lib.EINVAL, f, x, w, meta(4, requires_grad=True))
    refused(_lib.ESHAPE, f, x, meta(9, 16), t)
    refused(_lib.ESHAPE, f, x, w, meta(5))
    refused(_lib.ESHAPE, f, x, w, meta(4, 1))
    refused(_lib.ESHAPE, f, meta(8), w, meta(1))
    refused(_lib.ESHAPE, f, x, w, t, bias=meta(8))
    refused(_lib.ESHAPE, f, x, w, t, bias=meta(1, 16))
    refused(_lib.ESHAPE, f, meta(4, 0), meta(0, 16), t)
    refused(_lib.ESHAPE, f, x, meta(8, 0), t)
    refused(_lib.ELIMIT, f, meta(4, 1), meta(1, (1 << 24) + 1), t)


def test_checkpointed_layer_refusals():
    f = nd.nn.linear
    refused(_lib.EINVAL, f, meta(2, 3, 4), meta(4, 5), checkpoint=True)
    refused(_lib.EINVAL, f, meta(3, 4, is_complex=True), meta(4, 5), checkpoint=True)
    refused(_lib.EINVAL, f, meta(3, 4), meta(4, 5), meta(1, 5), checkpoint=True)
    refused(_lib.ESHAPE, f, meta(3, 4), meta(5, 4), checkpoint=True)
    refused(_lib.ESHAPE, f, meta(3, 4), meta(4, 5), meta(4), checkpoint=True)
    refused(_lib.ESHAPE, f, meta(3, 0), meta(0, 5), checkpoint=True)


def test_keep8_refusals():
    refused(_lib.EINVAL, nd.keep8, meta(4, 4, is_complex=True))
    refused(_lib.EINVAL, nd.keep8, meta(4, 4, requires_grad=True))       # a parameter
    view = meta(4, 4)
    view.is_view = True
    refused(_lib.EINVAL, nd.keep8, view)
    strided = Array(ArrayShape([4, 4], [1, 4]))
    refused(_lib.EINVAL, nd.keep8, strided)
    empty = meta(0, 4)
    assert nd.keep8(empty) is empty


def test_rows_and_cols_and_sign_rule():
    assert rows_and_cols(meta(6)) == (1, 6)
    assert rows_and_cols(meta(2, 3, 4)) == (6, 4)
    assert rows_and_cols(meta(3, 0)) == (0, 0)
    a = meta(2, 2)
    assert not keeps_sign(a)
    a.name = "relu"
    assert keeps_sign(a)
    b = meta(2, 2)
    b._lin_act = _lib.ACT_RELU
    assert keeps_sign(b)
    b._lin_act = _lib.ACT_TANH
    assert not keeps_sign(b)


def test_work_space_sizes():
    lib = _lib.lib
    # 8.25 bits per value, rows filled up to 32
    assert lib.endia_b200_keep8_bytes(0, 5) == 0
    assert lib.endia_b200_keep8_bytes(1, 1) == 256
    assert lib.endia_b200_keep8_bytes(1024, 4096) == 1024 * 4096 * 33 // 32
    assert lib.endia_b200_keep8_bytes(-1, 4) == 0
    assert lib.endia_b200_linear_ce_state_bytes(7) >= 4 * (1 + 7)
    # the work space does not grow with the vocabulary beyond a piece: 1/64 of the logits for the row
    # statistics is all that does
    M, K = 4096, 1024
    for back in (0, 1):
        small, large = (lib.endia_b200_linear_ce_scratch_bytes(M, K, v, back) for v in (1 << 15, 1 << 19))
        assert large - small <= 4 * M * ((1 << 19) - (1 << 15)) // 64 + (160 << 20), back
        assert large < (900 << 20) < 4 * M * (1 << 19)
    # up to 16 rows without a backward pass: no pairs
    assert lib.endia_b200_linear_ce_scratch_bytes(16, 4096, 1 << 17, 2) < (1 << 20)
    assert lib.endia_b200_linear_ce_scratch_bytes(17, 4096, 1 << 17, 2) > (1 << 20)
    # piece floor: many rows
    assert lib.endia_b200_linear_ce_scratch_bytes(1 << 20, 64, 1 << 17, 1) < 4 * (1 << 20) * (1 << 17) // 16


def test_no_cpu_fallback_of_the_entry_points():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    lib = _lib.lib
    assert lib.endia_b200_linear_ce_fwd(None, 1, None, 1, None, None, 1, 1, 1, 0, None, None, None, None) == _lib.ENODEV
    assert lib.endia_b200_linear_ce_bwd(None, 1, None, 1, None, None, 1, 1, 1, 0, None, None, None, None, None, None,
                                        None) == _lib.ENODEV
    assert lib.endia_b200_keep8(None, 1, 1, 1, 0, None, None) == _lib.ENODEV
    assert lib.endia_b200_keep8_read(None, 1, 1, None, None) == _lib.ENODEV
    assert lib.endia_b200_linear_keep_fwd(None, 1, None, 1, None, 0, 1, 1, 1, None, None, 0, None, None) == _lib.ENODEV
    assert lib.endia_b200_linear_keep_bwd(None, None, 1, None, None, 0, None, 1, 1, 1, None, None, None, None,
                                          None) == _lib.ENODEV
