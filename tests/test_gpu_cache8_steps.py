"""Steps of models whose attention layers keep their keys and values in 8 bits: the error word, steps that fail."""
from __future__ import annotations

import pytest
import torch

from cpi_b200.csrc import lib as K
from test_gpu_cache8_engine import engine

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("word", [1, 2, 3, 4, 5])
def test_the_error_word_says_which_kind_it_was(word):
    """A wait that ran out in a kernel on CTA pairs is not an index outside of the cache."""
    e = engine("dense", "int8")
    e.check_device_errors()
    K.device_error_flags(torch.device(DEV))[0] = word
    with pytest.raises(RuntimeError, match="outside of the cache" if word == K.INDEX_OUTSIDE else "gave up waiting"):
        e.check_device_errors()
    e.check_device_errors()
