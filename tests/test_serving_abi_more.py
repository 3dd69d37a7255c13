"""CPU tests of what the entry points of a decode step refuse, beside those of tests/test_serving_abi.py."""
import ctypes
import importlib

import pytest


@pytest.fixture(scope="module")
def adapters(package):
    return importlib.import_module("nemotron_inference_b200.adapters")


def test_results_that_begin_where_y_does_have_its_rows(adapters):
    lib, at = adapters._lib(), 1 << 21  # (addresses that are never followed)
    pool = ctypes.byref(adapters._Adapters(adapters=3, rank=16, inner=64, outer=128, a=at, b=at, scales=at))
    needed = lib.nmoe_adapters_workspace_bytes(pool, 10, 2)
    for y_stride, out_stride in ((128, 256), (256, 128), (136, 128)):
        assert lib.nmoe_adapters_add(pool, None, at, 64, at, y_stride, at, out_stride, 10, at, at, 2, at, needed, at) == 1
