"""bench.py's list of the decode kernels' sources, by which it tells whether the committed counter summary still holds."""

import os
import re

from test_bench_contract import ROOT, _bench

CSRC = os.path.join(ROOT, "nano-vllm-practice_amd", "csrc")


def included(name, seen):
    """``name`` and the files of csrc that it includes, directly or not."""
    if name not in seen and os.path.exists(os.path.join(CSRC, name)):
        seen.add(name)
        with open(os.path.join(CSRC, name)) as f:
            for other in re.findall(r'^#include "([\w.]+)"', f.read(), re.M):
                included(other, seen)
    return seen


def test_every_source_of_the_decode_kernels_is_listed():
    listed = [os.path.basename(x) for x in _bench().DECODE_SOURCES]
    assert sorted(listed) == sorted(included("paged_decode.hip", set()))
