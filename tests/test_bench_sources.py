"""bench.py's counter figures go stale with the sources of the kernels that
were counted, and with no others."""

import os
import shutil
import sys

import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join("ascend-spmm_amd", "csrc")


@pytest.fixture()
def copied(tmp_path, monkeypatch):
    sys.path.insert(0, REPO)
    import bench

    shutil.copytree(os.path.join(REPO, CSRC), tmp_path / CSRC)
    before = bench.kernel_sources_hash()
    monkeypatch.setattr(bench, "REPO", str(tmp_path))
    assert bench.kernel_sources_hash() == before
    return bench, tmp_path / CSRC, before


@pytest.mark.parametrize("name", ["layer_norm.hip", "orthogonalize.hip", "mma_ring.h", "preprocess.hip", "another.hip"])
def test_other_operators_do_not_count(copied, name):
    bench, csrc, before = copied
    with open(csrc / name, "a") as f:
        f.write("// changed\n")
    assert bench.kernel_sources_hash() == before


@pytest.mark.parametrize("name", ["spmm_gather.hip", "spmm_block.hip", "permute_rows.hip", "spmm_capi.hip", "common.h", "lanevec.h",
                                  "wgsearch.h"])
def test_the_counted_kernels_do(copied, name):
    bench, csrc, before = copied
    with open(csrc / name, "a") as f:
        f.write("// changed\n")
    assert bench.kernel_sources_hash() != before
    assert bench.measured_traffic(2, "csr", 128)[1].startswith("stale")
