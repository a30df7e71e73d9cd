"""The Python handles of device memory."""
import weakref

import pytest


def test_a_buffer_takes_attributes_of_its_users():
    """Programs hang notes of their own on the buffers they own (a name, the host copy it came from); weak references work too."""
    from rtensors_amd import hip as H
    b = H.HipBuf(None, 0, 3, H.F32)
    b.name = "bias"
    assert b.name == "bias" and (b.len, b.dtype) == (3, H.F32) and weakref.ref(b)() is b


def test_a_borrowed_view_is_a_plain_record():
    from rtensors_amd import hip as H
    v = H.HipView(None, 64, 3, H.F32)
    assert not isinstance(v, H.HipBuf) and (v.ptr, v.len, v.dtype) == (64, 3, H.F32)
    with pytest.raises(AttributeError):
        v.name = "bias"
