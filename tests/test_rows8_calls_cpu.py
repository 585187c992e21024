"""Calls of the 8-bit operators that would give wrong answers are refused on the host."""
import numpy as np
import pytest

import pywelvet
from test_rows8_cpu import accepted, refused


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


def test_swiglu_in_the_place_of_an_input_that_rows_keep():
    """h in gate's or up's place: other threads look again at what is overwritten, so the
    scales of rows that are asked for would be anything.  By itself h may lie there."""
    rows = pywelvet.rows8(64, 64, 64)
    call = lambda place, **kw: pywelvet.rows8_swiglu(1, 3, 60, 128, 192, d_h=place, status=True, **kw)  # noqa: E731
    for place in (128, 192):
        for asked in ("gate", "up", "h"):
            refused(call(place, **{asked: rows}), "place")
        refused(call(place, h_stride=61), "stride")
        accepted(call(place))
    accepted(call(place, gate_stride=61, h_stride=60))  # up's place, up's stride


def test_backward_into_what_it_still_reads():
    """dx in dy's or dpre's place: blocks of few rows write dx beside others that read dy."""
    layer = type("Layer", (), {"h": None})()  # refused before a layer is looked into
    call = lambda **kw: pywelvet.rows8_backward(-1, 1, 3, 60, 60, 64, layer=layer, ws=1 << 20, ws_bytes=1 << 62,  # noqa: E731
                                                status=True, **kw)
    refused(call(d_dx=64), "place")
    refused(call(d_dx=128, d_dpre=128), "place")
    refused(call(d_dx=128, d_dpre=192), "layer")


def test_rules_are_not_changed_by_a_call():
    """Rules may be applied from two threads, or to two vocabularies in turn."""
    rules = pywelvet.LogitRules(masks=1, d_masks=64)
    before = bytes(rules.desc)
    for vocab in (100, 1000):
        rules.apply(1, 2, vocab, 64, None, status=True)  # refused: nothing is launched
        assert bytes(rules.desc) == before
