"""The profiles' hash covers what the profiled kernels are compiled from, and nothing else."""

import re
import shutil
from pathlib import Path

import pytest

import bench_profiles
from nanotitan_amd.build import HIP_SOURCES

ROOT = Path(__file__).resolve().parent.parent
# Kernels beside the training layer's path, which no profile with a hash measures.
BESIDE = {"few_tokens.hip", "block_norm.hip", "block_norm_backward.hip", "checkpoint8.hip"}


@pytest.fixture
def tree(tmp_path):
    shutil.copytree(ROOT / "nanotitan_amd" / "csrc", tmp_path / "nanotitan_amd" / "csrc",
                    ignore=shutil.ignore_patterns("__pycache__"))
    shutil.copytree(ROOT / "include", tmp_path / "include")
    return tmp_path


def _changes(tree, path):
    before = bench_profiles.kernel_source_hash(tree)
    with open(tree / path, "a") as fh:
        fh.write("\n// another line\n")
    return bench_profiles.kernel_source_hash(tree) != before


def test_every_source_is_profiled_or_named():
    assert set(bench_profiles.PROFILED_SOURCES) | BESIDE == set(HIP_SOURCES)


@pytest.mark.parametrize("path,counts", [
    ("nanotitan_amd/csrc/grouped_gemm.hip", True), ("nanotitan_amd/csrc/common.hpp", True),
    ("nanotitan_amd/csrc/gemm_common.hpp", True), ("nanotitan_amd/csrc/gelu.hpp", True),
    ("nanotitan_amd/csrc/gen_gelu_table.py", True), ("include/nanotitan_moe.h", True),
    ("nanotitan_amd/csrc/few_tokens.hip", False), ("nanotitan_amd/csrc/block_norm.hpp", False),
    ("nanotitan_amd/csrc/torch_ext.cpp", False)])
def test_what_counts(tree, path, counts):
    assert _changes(tree, path) == counts


def test_a_new_header_counts(tree):
    csrc = tree / "nanotitan_amd" / "csrc"
    (csrc / "inner.hpp").write_text("#pragma once\n")
    (csrc / "outer.hpp").write_text('#pragma once\n  #  include "inner.hpp"\n')
    src = csrc / "router.hip"
    src.write_text('#include "outer.hpp"\n' + src.read_text())
    assert _changes(tree, "nanotitan_amd/csrc/inner.hpp")
    (csrc / "inner.hpp").unlink()
    with pytest.raises(FileNotFoundError, match="inner.hpp"):
        bench_profiles.kernel_source_hash(tree)


def test_every_quoted_include_is_covered():
    files = bench_profiles.profiled_files(ROOT)
    names = {p.name for p in files}
    for p in files:
        if p.suffix != ".py":
            for inc in re.findall(r'#\s*include\s+"([^"]+)"', p.read_text()):
                assert bench_profiles.GENERATED.get(inc, inc) in names, (p.name, inc)
