"""Tests against the reference engine where there is none: skipped with the reason, while every other missing file still fails."""
import pytest

import oracle


def test_missing_reference_and_other_files(monkeypatch, tmp_path):
    monkeypatch.setattr(oracle, "_libs", {})
    monkeypatch.setattr(oracle, "REF_SO", str(tmp_path / "libclref.so"))
    monkeypatch.delenv("CLUTOR_REF_DIR", raising=False)
    with pytest.raises(oracle.ReferenceMissing, match="CLUTOR_REF_DIR"):
        oracle.ref_lib()
    monkeypatch.setenv("CLUTOR_REF_DIR", str(tmp_path))   # sources are given: what is missing is the build
    with pytest.raises(FileNotFoundError) as e:
        oracle.ref_lib()
    assert not isinstance(e.value, oracle.ReferenceMissing)
    monkeypatch.setattr(oracle, "ORACLE_SO", str(tmp_path / "liboracle.so"))
    with pytest.raises(FileNotFoundError) as e:
        oracle.oracle_lib()
    assert not isinstance(e.value, oracle.ReferenceMissing)


def test_such_tests_are_skipped():
    """The hook of conftest.py around a test's call."""
    from tests import conftest

    def through(error):
        hook = conftest.pytest_runtest_call(None)
        next(hook)
        hook.throw(error)

    with pytest.raises(pytest.skip.Exception, match="no reference"):
        through(oracle.ReferenceMissing("no reference"))
    with pytest.raises(FileNotFoundError, match="another"):
        through(FileNotFoundError("another"))
