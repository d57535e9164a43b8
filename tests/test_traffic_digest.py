"""The digest that counter figures of the products carry: of the products' sources and flags, and of nothing else.  No GPU needed."""
import os
import shutil

import pytest

import bench


@pytest.fixture
def csrc(tmp_path):
    there = os.path.join(bench.ROOT, "hopper_spmm_amd", "csrc")
    for name in os.listdir(there):
        if os.path.isfile(os.path.join(there, name)):
            shutil.copy(os.path.join(there, name), tmp_path)
    return tmp_path


def changed(csrc, name, text="\n// another line\n"):
    with open(csrc / name, "a") as f:
        f.write(text)
    return bench.kernel_sources_digest(str(csrc))


def test_the_cache_is_no_part_of_the_products(csrc):
    before = bench.kernel_sources_digest()
    assert bench.kernel_sources_digest(str(csrc)) == before
    for name in bench.CACHE_SOURCES:
        assert changed(csrc, name) == before
    assert changed(csrc, "Makefile", "SRCS += another.hip\n") == before


@pytest.mark.parametrize("name,text", [("spmm_mfma_kernel.hpp", "\n"), ("hspmm_run.hip", "\n"), ("hspmm_pack.cpp", "\n"), ("lane_ranges.hpp", "\n"), ("Makefile", "FLAGS += -O2\n")])
def test_the_products_sources_and_flags_are(csrc, name, text):
    assert changed(csrc, name, text) != bench.kernel_sources_digest()
