# SPDX-License-Identifier: Apache-2.0
import math

import pytest

from kotflash_b200 import rotary_frequencies


@pytest.mark.parametrize("trained_length", [math.nan, -1, 0])
def test_a_trained_length_is_a_positive_number(trained_length):
    with pytest.raises(ValueError, match="trained_length"):
        rotary_frequencies(8, scaling="yarn", factor=2.0, trained_length=trained_length)
