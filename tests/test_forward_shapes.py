"""Shapes with routed feed-forward layers that the path walk cannot take are refused when they are made: a gated part was
left out without a word, and the sumcheck over the experts takes a power of two of them."""
import dataclasses

import pytest

from tests.test_path_workload import load_workloads_without_gpu


@pytest.mark.parametrize("change", [dict(glu=True), dict(experts=3), dict(experts=6), dict(experts_per_token=5),
                                    dict(experts_per_token=0), dict(experts=-4)])
def test_routed_shapes_that_are_refused(change):
    wl = load_workloads_without_gpu()
    with pytest.raises(ValueError, match="routed layers"):
        dataclasses.replace(wl.TINY_EXPERTS, **change)


def test_routed_shapes_that_are_taken():
    wl = load_workloads_without_gpu()
    for change in (dict(experts=1, experts_per_token=1), dict(experts=8, experts_per_token=8), dict(experts=0, glu=True)):
        assert dataclasses.replace(wl.TINY_EXPERTS, **change).name == "tiny-experts"
