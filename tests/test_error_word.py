"""The numbers that kernels write into the error word, read from the sources: an index outside of the cache has its own."""
from __future__ import annotations

import os
import re

from cpi_b200.csrc import lib as K

CSRC = os.path.dirname(K.__file__)


def test_waits_and_indices_have_different_numbers():
    indices, waits = set(), set()
    for name in sorted(os.listdir(CSRC)):
        if name.endswith((".cu", ".cuh")):
            for what in re.findall(r"atomicExch\((?:p\.)?error_flag, (\w+)\)", open(os.path.join(CSRC, name)).read()):
                (waits if what.isdigit() else indices).add((name, what))
    assert {n for n, _ in indices} == {"attention_decode_kv8.cu", "attention_prefill_kv8.cu", "kv8_stage.cu"}
    assert {w for _, w in indices} == {"kIndexOutside"} and len(waits) >= 8
    value = re.search(r"constexpr int kIndexOutside = (\d+);", open(os.path.join(CSRC, "common.cuh")).read()).group(1)
    assert int(value) == K.INDEX_OUTSIDE and {int(w) for _, w in waits} == {1, 2, 4, 5}
