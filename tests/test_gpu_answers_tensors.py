"""What torch knows of the tensors that the operators on answers are given."""
import pytest
import torch

from visualmesh_b200.engine import VisualMeshError

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def answers():
    from visualmesh_b200 import answers
    return answers


def test_tensors_that_are_written_in_place_say_so(answers):
    state, x = torch.ones((6, 4), device="cuda"), torch.ones((6, 4), device="cuda")
    out = torch.zeros((6, 4), device="cuda")
    before = state._version, out._version, x._version
    answers.gated_step(state, x, x, out=out)
    assert state._version > before[0] and out._version > before[1] and x._version == before[2]
    # what autograd saved of them is refused, as after any other write in place
    for changed in (state, out):
        w = torch.ones((6, 4), device="cuda", requires_grad=True)
        loss = (w * changed).sum()
        answers.gated_step(state, x, x, out=out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    # a view's writes are its base's
    version = state._version
    answers.gated_step(state[:, :2], x[:, :2], x[:, :2])
    assert state._version > version
    with torch.inference_mode():
        state, x = torch.ones((6, 4), device="cuda"), torch.ones((6, 4), device="cuda")
        answers.gated_step(state, x, x)
    answers.gated_step(state, x, x)
    assert bool(torch.isfinite(state).all())
