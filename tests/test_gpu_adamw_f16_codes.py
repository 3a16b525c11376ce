"""8-bit moments of float16 parameters, bit by bit as those of the other
types."""

import pytest

import test_gpu_adamw as base

pytestmark = pytest.mark.gpu


def test_8_bit_state_bit_by_bit(cuda):
    base.test_8_bit_state_bit_by_bit(cuda, "float16")
