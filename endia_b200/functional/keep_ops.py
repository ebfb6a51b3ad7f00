"""Activations held in 8 bits for the backward pass.

The reference keeps every op's float32 result until the graph is dropped (endia/_array/_array.mojo:
125-131). keep8(h) replaces the storage of an activation that the forward pass has finished with by
8.25 bits per value (endia_b200_keep8: signed integers with one power-of-two scale per 32 features); the
layers of nn.linear(..., checkpoint=True) read that form in their backward pass, any other reader gets
the values it stands for in float32."""
from .. import _lib
from .._array import Array, alloc, stream, flush_readers, await_pending


class Kept8(Array):
    """An array whose values are held in 8 bits. The first access of `buf` writes the values they stand
    for to float32 storage, which then stays."""
    _buf = None

    @property
    def buf(self):
        if self._buf is None and self._kept8 is not None:
            rows, cols = rows_and_cols(self)
            out = alloc(self.size())
            _lib.call("endia_b200_keep8_read", self._kept8.data_ptr(), rows, cols, out.data_ptr(), stream())
            self._buf = out
        return self._buf

    @buf.setter
    def buf(self, value):
        self._buf = value

    def held(self):
        return self._buf is None and self._kept8 is not None


def rows_and_cols(arr):
    cols = arr.shape()[-1]
    return (arr.size() // cols if cols else 0), cols


def keeps_sign(arr):
    """Whether `arr` is a ReLU's output: its 8-bit form then keeps every positive value positive, so that
    the derivative taken from it is exact."""
    return arr.name == "relu" or getattr(arr, "_lin_act", None) == _lib.ACT_RELU


def quantise(arr, ld=None):
    """The 8-bit form of a row-major array (torch buffer; see endia_b200_keep8)."""
    rows, cols = rows_and_cols(arr)
    kept = alloc((_lib.lib.endia_b200_keep8_bytes(rows, cols) + 3) // 4)
    _lib.call("endia_b200_keep8", arr.data_ptr(), cols if ld is None else ld, rows, cols, int(keeps_sign(arr)),
              kept.data_ptr(), stream())
    return kept


def keep8(arr):
    """Hold the values of `arr` in 8 bits from here on and release its float32 storage; returns `arr`.

    For activations between two layers, after the last forward use and before backward(): what the
    backward pass (or anything else) reads of `arr` afterwards are the values its 8-bit form stands for
    (at most half of 1/63.75 of the largest of 32 neighbours off). A layer with checkpoint=True that has
    taken `arr` as its input has made the form already. Refused: complex arrays, views and
    non-contiguous arrays (their storage belongs to another array), leaves that require a gradient
    (their values are parameters)."""
    if arr.is_complex():
        raise _lib.EndiaError(_lib.EINVAL, "keep8: real arrays only")
    if arr.is_view or arr.base_ is not None or not arr.is_contiguous():
        raise _lib.EndiaError(_lib.EINVAL, "keep8: a view shares its storage with another array and cannot be held in 8 bits")
    if arr.requires_grad() and not arr.args_:
        raise _lib.EndiaError(_lib.EINVAL, "keep8: a leaf that requires a gradient is not an activation")
    if isinstance(arr, Kept8) and arr.held() or arr.ndim() == 0 or arr.size() == 0:
        return arr
    flush_readers(arr)
    await_pending(arr)
    kept = getattr(arr, "_kept8", None)
    if kept is None or not arr.args_:      # (a leaf's storage may have been rewritten since)
        kept = quantise(arr)
    arr.buf = None
    if not isinstance(arr, Kept8):
        arr.__dict__.pop("buf", None)
        arr.__class__ = Kept8
    arr._buf = None
    arr._kept8 = kept
    arr._tf32_lo = arr._pair16 = None
    return arr
