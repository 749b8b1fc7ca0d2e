"""What can be said of a batch's results and their engine without a device."""
import pytest

from visualmesh_b200 import abi
from visualmesh_b200.engine import BatchResult, VisualMeshError


def test_waiting_without_an_engine_is_refused():
    assert abi.load().vm_wait_for(None, None) == abi.VM_ERR_INVALID_ARGUMENT
    assert abi.load().vm_last_error()


class FakeEngine:
    calls, closed = 3, False


@pytest.mark.parametrize("change", [dict(calls=4), dict(closed=True)])
def test_results_that_are_gone_cannot_be_had(change):
    """Their memory may have been freed: what is left to do is not to look."""
    engine = FakeEngine()
    raw = abi.vm_batch_result()
    raw.on_device = 1
    result = BatchResult(raw, engine)
    vars(engine).update(change)
    for read in (result.tensors, result.scores, lambda: result.advance(None, None), lambda: result.filtered(None)):
        with pytest.raises(VisualMeshError, match="gone"):
            read()


def test_scores_need_probabilities(monkeypatch):
    engine = FakeEngine()
    engine.gives_probabilities = False
    raw = abi.vm_batch_result()
    raw.on_device = 1
    result = BatchResult(raw, engine)
    monkeypatch.setattr(result, "_classifications", lambda: (None, None))
    with pytest.raises(VisualMeshError, match="probabilities"):
        result.scores()
