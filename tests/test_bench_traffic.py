"""The benchmark line's traffic figures: reported while the optimizer's sources
are those that they were measured on, whatever else the library holds."""

import re
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
sys.path.insert(0, str(ROOT))
import bench  # noqa: E402

CSRC = ROOT / "cresso_amd" / "csrc"


@pytest.mark.parametrize("workload", sorted(bench.TRAFFIC_FILES))
def test_profiles_are_of_the_current_sources(workload):
    nbytes, note = bench.measured_traffic(workload)
    assert nbytes and nbytes > 0, note


def test_the_optimizer_includes_no_operator_source():
    """What is left out of the digest does not reach a kernel of the optimizer's step."""
    files = {p.name: p.read_text() for pat in bench.SOURCE_GLOBS for p in ROOT.glob(pat)}
    assert bench.OPERATOR_SOURCES <= set(files)
    for name in set(files) - bench.OPERATOR_SOURCES:
        for included in re.findall(r'#include "([^"]+)"', files[name]):
            assert Path(included).name not in bench.OPERATOR_SOURCES, (name, included)


def test_a_changed_optimizer_source_makes_them_stale(tmp_path, monkeypatch):
    copy = tmp_path / "cresso_amd" / "csrc"
    copy.mkdir(parents=True)
    for p in CSRC.iterdir():
        if p.is_file():
            (copy / p.name).write_bytes(p.read_bytes())
    (tmp_path / "profiles").symlink_to(ROOT / "profiles")
    monkeypatch.setattr(bench, "ROOT", tmp_path)
    (copy / "distill.hip").write_text("// another operator\n")
    assert bench.measured_traffic("c2")[0]
    (copy / "spectral_route.hip").write_text("// another kernel\n")
    assert bench.measured_traffic("c2")[0] is None
