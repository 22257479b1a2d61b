"""CPU: numbers that the C ABI's 32 bits do not hold are refused before the call."""
import pytest

from opensplat_amd import cabi


@pytest.mark.parametrize("v", [2 ** 31, 2 ** 32, 2 ** 32 + 1, -2 ** 31 - 1, 2 ** 63])
def test_int32_refuses(v):
    with pytest.raises(ValueError):
        cabi._int32("a size", 5, v)


def test_int32_passes():
    cabi._int32("a size", 0, 2 ** 31 - 1, -2 ** 31)
