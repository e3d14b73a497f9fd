"""Windows and sinks as the attention calls take them, without a GPU: the quick way past the checks answers as they do."""
import numpy as np
import pytest

from bitween_amd.attention import _window


@pytest.mark.parametrize("window", [None, 1, 1024, 2 ** 62, 2 ** 62 + 1, 2 ** 100])
@pytest.mark.parametrize("sinks", [0, 4, 2 ** 62, 2 ** 63, 2 ** 100])
def test_numbers_that_are_taken(window, sinks):
    assert _window("x", window, sinks) == (min(window or 0, 2 ** 62), min(sinks, 2 ** 62))


class Count(int):
    pass


def test_whole_numbers_of_another_class_are_numbers():
    assert _window("x", Count(7), Count(2)) == (7, 2)


@pytest.mark.parametrize("window,sinks,error", [(0, 0, ValueError), (-1, 0, ValueError), (None, -1, ValueError), (5, -2 ** 70, ValueError), (True, 0, TypeError), (None, False, TypeError),
                                                (2.0, 0, TypeError), (4, None, TypeError), (np.int64(4), 0, TypeError), ("4", 0, TypeError), (None, 0.0, TypeError)])
def test_numbers_that_are_refused(window, sinks, error):
    with pytest.raises(error, match="(window|sinks) must be"):
        _window("x", window, sinks)
