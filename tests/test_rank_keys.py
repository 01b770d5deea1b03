"""The keys by which log probabilities rank logits (CPU): tests/rank_keys.hip takes rows with NaN, infinities,
zeros of both signs and ties through the library's own key arithmetic."""

from __future__ import annotations

import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


@pytest.fixture(scope="module")
def broken(tmp_path_factory):
    binary = str(tmp_path_factory.mktemp("ranks") / "rank_keys")
    subprocess.run(["hipcc", "--offload-arch=gfx950", "-O1", "-std=c++17", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "-I" + os.path.join(ROOT, "residualquant_amd", "csrc"),
                    os.path.join(HERE, "rank_keys.hip"), "-o", binary], check=True)
    out = subprocess.run([binary], check=True, capture_output=True, text=True, timeout=300).stdout
    return {line.split()[0]: int(line.split()[1]) for line in out.splitlines()}


@pytest.mark.parametrize("name", ["range", "index", "passes"])
def test_rank_keys(broken, name):
    assert broken[name] == 0
