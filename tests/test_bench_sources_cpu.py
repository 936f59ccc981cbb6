"""bench.py's sha of the measured path's kernel sources: what voids a committed counter summary, and what does not."""
import json
import os
import re
import shutil
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "ur-mvo_amd", "csrc")


@pytest.fixture(scope="module")
def bench():
    sys.path.insert(0, ROOT)
    import bench
    return bench


def test_the_sha_covers_the_path_and_its_flags_alone(bench, tmp_path):
    here = bench.kernel_source_sha()
    tree = str(tmp_path / "csrc")
    shutil.copytree(CSRC, tree, ignore=shutil.ignore_patterns("build*"))
    shutil.copy(os.path.join(CSRC, "build_info.hip"), tree)
    assert bench.kernel_source_sha(tree) == here
    make = open(os.path.join(CSRC, "Makefile")).read()
    operators = set(re.search(r"^OPERATORS := (.*)$", make, re.M).group(1).split())
    assert operators | {"probes.hip"} == {f for f in bench.OFF_THE_PATH if f.endswith(".hip")}
    for f in sorted(os.listdir(tree)):
        path = os.path.join(tree, f)
        text = open(path).read()
        # a header of the operators is included by them alone
        if f not in bench.OFF_THE_PATH:
            assert not re.search(r"#include \"(attention_op|operator_common)\.h\"", text), f
        if f == "Makefile":
            continue
        open(path, "a").write("// changed\n")
        assert (bench.kernel_source_sha(tree) == here) == (f in bench.OFF_THE_PATH), f
        open(path, "w").write(text)
    open(os.path.join(tree, "Makefile"), "w").write(make + "\n# a comment\n")
    assert bench.kernel_source_sha(tree) == here
    open(os.path.join(tree, "Makefile"), "w").write(make.replace("-O3", "-O2"))
    assert bench.kernel_source_sha(tree) != here


def test_a_summary_is_found_by_its_sources(bench, monkeypatch, tmp_path):
    os.mkdir(tmp_path / "profiles")
    monkeypatch.setattr(bench, "ROOT", str(tmp_path))
    monkeypatch.setattr(bench, "kernel_source_sha", lambda: "this")
    assert bench._summary("pmc_hbm")[0] is None
    for name, sha in (("a_pmc_hbm", "this"), ("b_pmc_hbm", "other"), ("c_pmc_hbm_exact", "this")):
        json.dump({"source_sha": sha, "name": name}, open(tmp_path / "profiles" / f"{name}.json", "w"))
    assert bench._summary("pmc_hbm")[0]["name"] == "a_pmc_hbm" and bench._summary("pmc_hbm")[1] == "a_pmc_hbm.json"
    assert bench._summary("pmc_hbm_exact")[0]["name"] == "c_pmc_hbm_exact"
    assert bench._summary("pmc_mfma")[0] is None
