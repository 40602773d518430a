"""The hook that skips comparisons with the reference's kernels where they are not built."""
import conftest
import pytest

from oracle import build as oracle_build
from oracle import ref_gpu


def outcome(monkeypatch, tmp_path, error, ask=(), built=False):
    """What the hook makes of a test that asks for libraries and then raises `error`."""
    monkeypatch.setattr(ref_gpu, "REF", tmp_path / "none")
    monkeypatch.setattr(oracle_build, "REFERENCE", tmp_path)
    if built:
        (tmp_path / "kernels").mkdir()
    hook = conftest.pytest_runtest_call(None)
    next(hook)
    for name in ask:
        assert not ref_gpu.available(name)
    with pytest.raises(BaseException) as caught:
        hook.throw(error)
    return caught.type


def test_only_a_missing_library_skips(monkeypatch, tmp_path):
    run = lambda *a, **k: outcome(monkeypatch, tmp_path, *a, **k)
    skipped, failed = pytest.skip.Exception, pytest.fail.Exception
    ref_gpu.MISSING.add("ref_gate.so")                      # an earlier test's
    assert run(ref_gpu.NotBuilt("ref_dense.so")) is skipped
    assert run(failed("oracle/_ref/ref_dense.so is missing: build it"), ask=["ref_dense.so"]) is skipped
    # failures of the comparison itself, whatever they say
    assert run(AssertionError("3 of 5 outputs differ from oracle/_ref/ref_dense.so"), ask=["ref_dense.so"]) is AssertionError
    assert run(failed("differs from the reference GPU oracle")) is failed
    assert run(failed("oracle/_ref/ref_gate.so is missing")) is failed
    assert run(failed("timings differ"), ask=["ref_dense.so"]) is failed
    assert run(FileNotFoundError("ref_dense.so"), ask=["ref_dense.so"]) is FileNotFoundError


def test_with_the_checkout_nothing_is_skipped(monkeypatch, tmp_path):
    assert outcome(monkeypatch, tmp_path, ref_gpu.NotBuilt("ref_dense.so"), built=True) is ref_gpu.NotBuilt
