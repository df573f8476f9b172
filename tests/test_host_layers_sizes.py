"""Rows in numbers that the layer operators do not count, on the CPU under sanitizers."""
import shutil

import pytest

from test_host_layers_results import run_host_check


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
def test_too_many_rows_are_refused_before_a_result_is_resized(tmp_path):
    assert "sizes of layers ok" in run_host_check(tmp_path, "host_layers_sizes_check")
