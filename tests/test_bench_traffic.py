"""bench.py withholds `roofline.traffic` where the scoring kernels are not the ones whose counters were read: those of this tree are."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("section,sources", [("headline", ("score.hip", "score_geom.h", "score_lists.h")), ("exact", ("score_x3.hip", "score_x3.h"))])
def test_the_counters_are_those_of_the_kernels(section, sources):
    spec = importlib.util.spec_from_file_location("bench_of_the_tree", os.path.join(ROOT, "bench.py"))
    bench = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(bench)
    traffic, code, _ = bench.traffic_from_profile(section, 9830400, sources, False)
    assert traffic and traffic > 1e10, code
