"""The number of parts of an adapter's hidden values, as the C entries take it (no GPU)."""
import pytest

OK = 4096  # (an aligned address that is never read: every call here is refused on the host)


def _forward(L, dtype, parts):
    return L.lib.ufpn_lateral_adapters_parts(dtype, OK, OK, OK, OK, OK, OK, None, 1.0, None, 2 * OK, OK, parts, 1, 64, 4,
                                             4, 8, 2, 0, 0, None)


def _backward(L, dtype, parts):
    return L.lib.ufpn_lateral_adapters_backward_parts(dtype, OK, OK, None, OK, OK, OK, OK, None, 1.0, OK, parts, OK, OK,
                                                      OK, 1, 64, 4, 4, 8, 2, OK, 1 << 40, None)


@pytest.mark.parametrize("call", [_forward, _backward])
@pytest.mark.parametrize("dtype,parts", [(1, 1), (1, 4), (1, 0), (1, -1), (2, 2), (2, 1), (2, 4)])
def test_refused_parts(call, dtype, parts):
    from unified_fpn import _lib
    assert call(_lib, dtype, parts) == _lib.ERR_INVALID_ARG
    assert b"parts" in _lib.lib.ufpn_last_error()
