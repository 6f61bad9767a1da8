"""A scale whose product with log2(e) is no finite fp32 number is refused, on the host (0 times it would be NaN)."""
import pytest

from tests.test_attention_abi import _fails, _packed, _paged


@pytest.mark.parametrize("name,make", [("attention_packed", _packed), ("attention_paged", _paged)])
@pytest.mark.parametrize("scale", [3.4e38, 2.4e38])
def test_scale_that_overflows(name, make, scale):
    assert "scale" in _fails(name, *make(scale=scale))
