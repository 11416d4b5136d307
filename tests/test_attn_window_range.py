"""attn_decode from Python passes a window on as it is, or refuses it: on the CPU,
with stand-ins for device tensors and a library that keeps what it was given."""
import pytest
import torch

from test_kv_buffers import Cache4, _cache, _tok
from test_serving_buffers import BAD, On, k  # noqa: F401 (a fixture)


@pytest.mark.parametrize("window", [0, 1, 1000, 2 ** 31, 2 ** 32 - 1, 2 ** 32, 2 ** 32 + 5, 2 ** 40, -1, -2 ** 32])
def test_window(k, monkeypatch, window):  # noqa: F811
    from streamoe_amd import _abi

    def decode(*args):  # the window as the C call would get it
        given.append(_abi.PROTOTYPES["smoe_attn_decode"][1][8](args[8]).value)
        return 0

    given = []
    monkeypatch.setattr(k.lib, "smoe_attn_decode", decode, raising=False)
    status = k.attn_decode(_cache(), *_tok(), Cache4(5, 8, 64), 0.1, window, On(5, 8, 64), 8, 5, On(1 << 16, dtype=torch.uint8))
    assert (status, given) == ((0, [window]) if 0 <= window < 2 ** 32 else (BAD, []))
