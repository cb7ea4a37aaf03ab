"""Host side of the device's own status word, without a GPU."""
import ctypes as C

from streamk_b200 import _lib as L


def test_refusals(lib):
    assert lib.sk_device_status(None) == L.SK_ERR_ARG


def test_the_flag_is_its_own():
    others = (L.SK_FLAG_PDL, L.SK_FLAG_NO_TABLE, L.SK_FLAG_BF16, L.SK_FLAG_OFFSETS_64, L.SK_FLAG_OUT_F32, L.SK_FLAG_ZERO_REST,
              *L.SK_FLAG_Q4_GROUP.values(), 1 << 30)
    assert all(L.SK_FLAG_DEVICE_STATUS & f == 0 for f in others)
    assert L.SK_DEVICE_STATUS_BYTES >= C.sizeof(L.SkStatus)


def test_the_shortcut_is_told_of_captures():
    m = L.load_host()
    assert m.set_captured(63, True) is None and m.set_captured(63, False) is None and m.set_captured(63, False) is None
    for bad in ((), (0,), ("0", True), (0, True, 1)):
        try:
            m.set_captured(*bad)
        except TypeError:
            continue
        raise AssertionError(bad)
