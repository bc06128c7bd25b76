"""vt_stream_create without a device."""
import ctypes

import pytest

from veritac_amd import _lib


def test_a_stream_needs_a_place_to_go():
    assert _lib.load_library().vt_stream_create(None) == _lib.VT_EINVAL
    assert "null" in _lib.last_error()


@pytest.mark.skipif(_lib.load_library().vt_device_count() > 0, reason="for hosts without a device")
def test_no_stream_without_a_device():
    out = ctypes.c_void_p()
    assert _lib.load_library().vt_stream_create(ctypes.byref(out)) == _lib.VT_ENODEV and not out.value
    with pytest.raises(_lib.HipGemmError):
        _lib.stream_create()
