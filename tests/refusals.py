"""What the tests of refused calls share: calls that are refused before
anything reaches a device, with a zeroed block in the handle's place."""
import ctypes as C

_HANDLE = C.create_string_buffer(4096)


def fake_handle():
    return C.addressof(_HANDLE)


def refused(status, code):
    from streamoe_amd import _abi

    assert _abi.STATUS[status] == "SMOE_ERR_" + code, (_abi.STATUS.get(status), code)
