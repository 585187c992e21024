"""Calls of the 8-bit operators that would give wrong answers are refused on the host."""
import numpy as np
import pytest

import pywelvet


@pytest.mark.parametrize("codes", [np.array([[1, 200]]), np.array([[-128, 0]], np.int8), np.array([[0.5, 1.0]]),
                                   np.array([[-300, 1]], np.int64), np.array([[np.nan, 1.0]])])
def test_codes_that_are_not_whole_numbers_of_a_byte(codes):
    with pytest.raises(pywelvet.WelvetError) as e:
        pywelvet.Int8Layer.from_codes(codes, np.ones(1))
    assert e.value.code == 1 and "[-127, 127]" in str(e.value)


def test_scales_of_another_count():
    for scales in (np.ones(2), np.ones((3, 1)), np.ones(4)):
        with pytest.raises(pywelvet.WelvetError) as e:
            pywelvet.Int8Layer.from_codes(np.zeros((3, 5), np.int8), scales)
        assert e.value.code == 1 and "scales" in str(e.value)
