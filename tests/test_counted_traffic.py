"""The counters that bench.py reports as traffic are of the engine's kernels as
they are: each summary is bound to the bytes of the source it was counted on."""
import glob
import os

import pytest

import bench

SUMMARIES = sorted(glob.glob(os.path.join(bench.ROOT, "profiles", "*_traffic.json")))


@pytest.mark.parametrize("path", SUMMARIES, ids=[os.path.basename(p) for p in SUMMARIES])
def test_counted_on_the_source_there_is(path):
    count, note = bench.counted_traffic(path)
    assert count, note
