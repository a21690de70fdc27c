"""bench.py where the reference engine is neither built nor there as sources: its arm says so in one line and ends well, and the
framework's own arm leaves its figure out."""
import json
import sys

import pytest

import bench
import oracle


@pytest.fixture
def nowhere(monkeypatch, tmp_path):
    monkeypatch.setattr(oracle, "REF_SO", str(tmp_path / "libclref.so"))
    monkeypatch.delenv("CLUTOR_REF_DIR", raising=False)
    monkeypatch.delenv("RANK", raising=False)


@pytest.mark.parametrize("args", [[], ["--workload", "model"], ["--workload", "prompt"], ["--workload", "prefill64"], ["--gpus", "2"]])
def test_reference_arm_is_unavailable(nowhere, monkeypatch, capsys, args):
    monkeypatch.setattr(sys, "argv", ["bench.py", "--impl", "reference", "--steps", "1", "--warmup", "0", *args])
    bench.main()
    lines = capsys.readouterr().out.splitlines()
    assert len(lines) == 1
    line = json.loads(lines[0])
    assert set(line) == {"impl", "unavailable"} and line["impl"] == "reference"
    assert "CLUTOR_REF_DIR" in line["unavailable"] and "\n" not in line["unavailable"]


def test_reference_arm_other_ranks_are_silent(nowhere, monkeypatch, capsys):
    monkeypatch.setenv("RANK", "1")
    monkeypatch.setattr(sys, "argv", ["bench.py", "--impl", "reference", "--gpus", "2"])
    bench.main()
    assert capsys.readouterr().out == ""


def test_own_arms_baseline(nowhere):
    assert "CLUTOR_REF_DIR" in bench.cpu_baseline(lambda: pytest.fail("there is nothing to time"))["unavailable"]


def test_baseline_where_the_reference_is(monkeypatch, tmp_path):
    so = tmp_path / "libclref.so"
    so.write_bytes(b"")
    monkeypatch.setattr(oracle, "REF_SO", str(so))
    assert bench.cpu_baseline(lambda: {"value": 3.0}) == {"value": 3.0}
