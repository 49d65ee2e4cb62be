"""CPU tests of prompt_layer.pack: positions that int32 cannot hold are refused."""
from __future__ import annotations

import pytest

from lynnreal_omni_b200.prompt_layer import pack


def test_last_positions():
    most = 2 ** 31 - 1
    assert pack([3, 0, 1], "cpu", start=most - 2).positions.tolist() == [most - 2, most - 1, most, most - 2]
    for lengths, start in (([3, 1], most - 1), ([1], most + 1), ([4], 2 ** 40)):
        with pytest.raises(ValueError, match="position"):
            pack(lengths, "cpu", start=start)
