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


def calls_of(answers, x):
    """Every operator, with x as each of its arguments that could carry a gradient."""
    plain = torch.ones((6, 4), device="cuda")
    row, states = torch.ones(6, device="cuda"), torch.ones((6, 1, 4), device="cuda")
    scored = answers.scores(plain)
    three, row_x = (x[:, None], plain[:, None]), x[:, 0].contiguous()
    labels = torch.zeros(6, dtype=torch.int64, device="cuda")
    return [lambda: answers.scores(x), lambda: answers.scores_backward(x, scored, d_entropy=row), lambda: answers.scores_backward(plain, scored, d_entropy=row_x),
            lambda: answers.scores_backward(plain, scored, labels, d_log_prob=row_x), lambda: answers.scores_backward(plain, scored, d_log_sum=row_x),
            lambda: answers.gated_scan(three[0], three[1]), lambda: answers.gated_scan(three[1], three[0]), lambda: answers.gated_scan(three[1], three[1], x.contiguous()),
            lambda: answers.gated_scan_backward(three[0], three[1], states), lambda: answers.gated_scan_backward(three[1], three[1], states, three[0]),
            lambda: answers.gated_scan_backward(three[1], three[1], states, None, x.contiguous()),
            lambda: answers.gated_step(plain.clone(), x, plain), lambda: answers.gated_step(plain.clone(), plain, x), lambda: answers.gated_step(x, plain, plain)]


def test_tangents_are_not_lost(answers):
    import torch.autograd.forward_ad as forward
    with forward.dual_level():
        x = forward.make_dual(torch.ones((6, 4), device="cuda"), torch.ones((6, 4), device="cuda"))
        for call in calls_of(answers, x):
            with pytest.raises(VisualMeshError, match="tangent"):
                call()
        answers.scores(forward.unpack_dual(x).primal)
    for call in calls_of(answers, torch.ones((6, 4), device="cuda")):
        call()


def test_views_without_values_of_their_own_are_refused(answers):
    negated = torch.complex(torch.ones((6, 4), device="cuda"), torch.ones((6, 4), device="cuda")).conj().imag
    assert negated.is_neg() and bool((negated == -1).all())
    with pytest.raises(VisualMeshError, match="resolve_neg"):
        answers.gated_step(torch.ones((6, 4), device="cuda"), torch.ones((6, 4), device="cuda"), negated)
    with pytest.raises(VisualMeshError, match="resolve_neg"):
        answers.scores(torch._efficientzerotensor((6, 4), device="cuda"))
    with pytest.raises(VisualMeshError, match="resolve_neg"):
        answers.gated_scan(torch.ones((6, 1, 4), device="cuda"), torch.ones((6, 1, 4), device="cuda"), torch._efficientzerotensor((6, 4), device="cuda"))
    answers.scores(negated.resolve_neg().contiguous())
