"""The units and workspace places of linear attention's chunked form, on the host."""
import shutil

import pytest

from test_host_mirror_cpu import _run_host_check


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")
def test_no_unit_leaves_the_workspace(tmp_path):
    assert "linear plan: ok" in _run_host_check(tmp_path, "linear_plan_check")


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")
def test_what_is_under_way_is_waited_for(tmp_path):
    assert "linear drain: ok" in _run_host_check(tmp_path, "linear_drain_check")
