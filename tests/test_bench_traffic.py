"""The benchmark's traffic figures belong to the kernels that they were collected from: to their sources and compiler
flags, not to every file beside them."""
import json
import os
import re
import shutil

import pytest

import bench
from recommend_amd import build as rbuild

CSRC = os.path.join(bench.ROOT, "recommend_amd", "csrc")


@pytest.fixture
def copy(tmp_path, monkeypatch):
    shutil.copytree(CSRC, tmp_path / "recommend_amd" / "csrc")
    os.makedirs(tmp_path / "profiles")
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    return tmp_path


def test_every_source_of_the_kernels_is_listed():
    found, todo = set(), ["eval.hip", "eval_filter.hip", "spmm.hip"]
    while todo:
        name = todo.pop()
        found.add(name)
        with open(os.path.join(CSRC, name)) as f:
            todo += [h for h in re.findall(r'#include "([^/"]+)"', f.read()) if h not in found]
    assert found == set(bench.TRAFFIC_SOURCES)


def test_figures_outlive_changes_of_other_sources(copy, monkeypatch):
    doc = {"shape": "elec", "emb_dim": 64, "kernel_source_digest": bench.kernel_source_digest(),
           "groups": {"spmm_hop": {"traffic_bytes": 5}}}
    (copy / bench.TRAFFIC).write_text(json.dumps(doc))
    assert bench.pmc_traffic("spmm_hop", "elec", 64, 1) == (5, bench.TRAFFIC)
    for name in ("embedding.hip", "torch_ops.cpp", "elem.h"):
        with open(copy / "recommend_amd" / "csrc" / name, "a") as f:
            f.write("// changed\n")
    assert bench.pmc_traffic("spmm_hop", "elec", 64, 1)[0] == 5
    assert bench.pmc_traffic("spmm_hop", "baby", 64, 1)[0] is None and bench.pmc_traffic("spmm_hop", "elec", 64, 2)[0] is None
    monkeypatch.setattr(rbuild, "FLAGS", rbuild.FLAGS + ["-g"])
    assert "other kernel sources" in bench.pmc_traffic("spmm_hop", "elec", 64, 1)[1]
    monkeypatch.undo()
    monkeypatch.setattr(bench, "ROOT", str(copy))
    with open(copy / "recommend_amd" / "csrc" / "spmm.hip", "a") as f:
        f.write("// changed\n")
    assert "other kernel sources" in bench.pmc_traffic("spmm_hop", "elec", 64, 1)[1]
