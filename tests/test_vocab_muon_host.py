"""The argument checks of the vocabulary cross entropy and the Muon step that run before any device work (no GPU): sizes
that do not fit are refused by the binding, a null context by the library."""
import ctypes
from types import SimpleNamespace

import numpy as np
import pytest

from laya_amd import _native, ops


def _array(*shape, dtype=np.float32):
    return SimpleNamespace(ptr=16, shape=shape, size=int(np.prod(shape)), dtype=np.dtype(dtype))


def _parameter(*shape):
    return SimpleNamespace(ctx=SimpleNamespace(handle=None), shape=shape, data=_array(*shape), trainable=False)


def test_vocab_ce_refuses_arrays_that_do_not_fit():
    W, b = _parameter(50, 8), _parameter(50)
    x, t, r = _array(6, 8), _array(6, dtype=np.int32), _array(6)
    with pytest.raises(ValueError, match="for 7 rows"):
        ops.vocab_ce(W, b, x, t, 7, r, r)
    with pytest.raises(ValueError, match="for -1 rows"):
        ops.vocab_ce(W, b, x, t, -1, r, r)
    with pytest.raises(ValueError, match="int32"):
        ops.vocab_ce(W, b, x, _array(6), 6, r, r)
    with pytest.raises(ValueError, match="row weights"):
        ops.vocab_ce(W, b, x, t, 6, r, r, row_weights=_array(5))
    with pytest.raises(ValueError, match="bias"):
        ops.vocab_ce(W, _parameter(49), x, t, 6, r, r)
    with pytest.raises(ValueError, match="bf16"):
        ops.vocab_ce(W, b, x, t, 6, r, r, weight16=_array(50, 7, dtype=np.uint16))
    with pytest.raises(ValueError, match="lse"):
        ops.vocab_ce(W, b, x, t, 6, r, _array(5))
    with pytest.raises(ValueError, match="lse"):
        ops.vocab_ce_backward(W, b, x, t, 6, _array(5), None)
    with pytest.raises(ValueError, match="dx"):
        ops.vocab_ce_backward(W, b, x, t, 6, r, _array(6, 7))


def test_muon_refuses_arrays_that_do_not_fit():
    ctx = SimpleNamespace(handle=None)
    with pytest.raises(ValueError, match="2 offsets"):
        ops.MuonMatrices(ctx, [0, 8], [2], [4, 4])
    with pytest.raises(ValueError, match="negative"):
        ops.MuonMatrices(ctx, [-8], [2], [4])
    m = SimpleNamespace(ctx=ctx, handle=None, end=100)
    with pytest.raises(ValueError, match="up to 100"):
        ops.muon(m, _array(100), _array(99), _array(100), 0.1)
    with pytest.raises(ValueError, match="3 matrices"):
        ops.orthogonalize(ctx, _array(3, 4, 5), 3, 4, 5, _array(59))
    with pytest.raises(ValueError):
        ops.orthogonalize(ctx, _array(3, 4, 5), -1, 4, 5, _array(60))


def test_the_library_refuses_a_null_context():
    L, f = _native.lib(), ctypes.c_float(1.0)
    h = ctypes.c_void_p()
    assert L.laya_vocab_ce_fwd(None, 16, 1, 8, 16, None, 8, None, 16, None, f, 16, 16, None, None) == _native.ERR_ARGUMENT
    assert L.laya_vocab_ce_bwd(None, 16, 1, 8, 16, None, 8, None, 16, None, f, 16, None, None, None) == _native.ERR_ARGUMENT
    assert L.laya_orthogonalize(None, 16, 1, 4, 4, 5, 16) == _native.ERR_ARGUMENT
    assert L.laya_matrices_create(None, None, None, None, None, 0, ctypes.byref(h)) == _native.ERR_ARGUMENT
    assert L.laya_muon(None, None, 16, 32, 48, 0.1, 0.9, 1, 0.0, 5, None, 0) == _native.ERR_ARGUMENT
    assert b"null context" in L.laya_last_error()


def test_a_borrowed_array_is_not_freed():
    from laya_amd.device import DeviceArray
    owner = SimpleNamespace()
    a = DeviceArray.borrow(SimpleNamespace(handle=1), 4096, (3, 5), np.uint16, owner=owner)
    assert (a.size, a.nbytes, a.shape, a.dtype) == (15, 30, (3, 5), np.uint16) and a.owner is owner
    a.free()  # with a handle, memory of its own would go to the library
    assert a.ptr is None and a.owner is None
