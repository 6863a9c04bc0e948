"""The benchmark's recorded HBM bytes hold for the sources they name: those have to be all that the grouped GEMMs compile from."""

import os
import re
import sys

from conftest import ROOT

CSRC = os.path.join(ROOT, "architecture-zarelga-superposition_amd", "csrc")


def compiled_from(name, seen):
    if name not in seen and os.path.exists(os.path.join(CSRC, name)):
        seen.add(name)
        for inc in re.findall(r'^#include "([^"]+)"', open(os.path.join(CSRC, name)).read(), flags=re.M):
            compiled_from(inc, seen)
    return seen


def test_traffic_sources_are_complete():
    sys.path.insert(0, ROOT)
    import bench

    assert set(bench.TRAFFIC_C3_SOURCES) == compiled_from("gemm.hip", set())
    note = open(os.path.join(ROOT, bench.TRAFFIC_C3_PROFILE)).read()
    assert bench.TRAFFIC_C3_GEMM_SHA256[:12] in note and all(f"csrc/{s}" in note for s in bench.TRAFFIC_C3_SOURCES)
