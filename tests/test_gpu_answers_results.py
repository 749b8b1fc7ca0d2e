"""Results that an engine left on the device, read by torch's streams while the engine goes on."""
import dataclasses

import pytest
import torch

import golden_io as G
from visualmesh_b200 import workloads as W
from visualmesh_b200.engine import Engine, FrameInput, Mesh, VisualMeshError

pytestmark = pytest.mark.gpu

LONG = 200_000_000  # cycles that a stream is kept busy for: a tenth of a second, many of the engine's calls


@pytest.fixture(scope="module")
def setup():
    case = G.Case("ring6_equisolid_rgba")
    mesh = Mesh.from_arrays(case.rays, case.nbrs, case.bsp)
    engine = Engine(case.network, device=0)
    fr = case.frames[0]

    def batch(seed, n=4):
        images = [W.random_bytes(seed + f, fr["image"].size).reshape(fr["image"].shape) for f in range(n)]
        return engine.prepare_batch([FrameInput(mesh, fr["Hoc"], case.lens, image, case.format) for image in images])

    yield engine, mesh, batch(1), batch(100)
    engine.close()


def reads(mesh, classes):
    gate = torch.randn(classes, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    return [lambda r: r.scores(top=classes)[1:],
            lambda r: (r.advance(torch.full((mesh.n_nodes, classes), 1.0 / classes, device="cuda"), gate),),
            lambda r: r.filtered(gate)[:2]]


@pytest.mark.parametrize("which", range(3))
def test_the_next_batch_waits_for_what_reads_the_last(setup, which):
    engine, mesh, first, second = setup
    read = reads(mesh, engine.n_classes)[which]
    wanted = []
    for prepared in (first, second):
        wanted.append([v.clone() for v in read(engine.run_prepared(prepared, results_on_device=True))])
        torch.cuda.synchronize()
    assert not torch.equal(wanted[0][0], wanted[1][0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for stream in streams:
        torch.cuda.synchronize()
        result = engine.run_prepared(first, results_on_device=True)
        with torch.cuda.stream(stream):
            read(result)  # what it allocates is there from now on
            torch.cuda._sleep(LONG)
            got = read(result)
        again = read(engine.run_prepared(second, results_on_device=True))
        torch.cuda.synchronize()
        for a, b in zip(got, wanted[0]):
            assert torch.equal(a, b)
        for a, b in zip(again, wanted[1]):
            assert torch.equal(a, b)


def test_the_engine_waits_for_reads_of_ones_own(setup):
    engine, mesh, first, second = setup
    result = engine.run_prepared(first, results_on_device=True)
    x = result.tensors()["classifications"]
    want = x.clone()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    copies = [torch.empty_like(x) for _ in streams]
    for stream, copy in zip(streams, copies):
        with torch.cuda.stream(stream):
            torch.cuda._sleep(LONG)
            copy.copy_(x)
        engine.wait_for(stream)
    engine.run_prepared(second, results_on_device=True)
    torch.cuda.synchronize()
    for copy in copies:
        assert torch.equal(copy, want)


def test_reads_of_results_are_captured(setup):
    """A graph of such a read is launched again for every batch whose results lie where those of the first did."""
    engine, mesh, first, second = setup
    result = engine.run_prepared(first, results_on_device=True)
    want = [v.clone() for v in result.scores()[1:]]
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = result.scores()[1:]
    stream = torch.cuda.Stream()
    for prepared in (first, second, first):
        engine.run_prepared(prepared, results_on_device=True)
        with torch.cuda.stream(stream):
            torch.cuda._sleep(LONG // 10)
            graph.replay()
        engine.wait_for(stream)
    engine.run_prepared(second, results_on_device=True)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_results_of_an_earlier_call_cannot_be_had(setup):
    engine, mesh, first, second = setup
    old = engine.run_prepared(first, results_on_device=True)
    new = engine.run_prepared(second, results_on_device=True)
    new.scores()
    with pytest.raises(VisualMeshError):
        old.scores()
    case = G.Case("ring6_equisolid_rgba")
    fr = case.frames[0]
    other = Engine(case.network, device=0)
    result = other.run_batch([FrameInput(mesh, fr["Hoc"], case.lens, fr["image"], case.format)], results_on_device=True)
    other.close()
    with pytest.raises(VisualMeshError):
        result.tensors()


@pytest.mark.parametrize("activation", [W.SELU, W.RELU, W.SOFTMAX, W.TANH])
def test_scores_of_answers_that_are_no_probabilities_are_refused(activation):
    from visualmesh_b200 import answers
    case = G.Case("ring6_equisolid_rgba")
    network = [list(group) for group in case.network]
    network[-1][-1] = dataclasses.replace(network[-1][-1], activation=activation)
    mesh, fr = Mesh.from_arrays(case.rays, case.nbrs, case.bsp), case.frames[0]
    engine = Engine(network, device=0)
    result = engine.run_batch([FrameInput(mesh, fr["Hoc"], case.lens, fr["image"], case.format)], results_on_device=True)
    if activation == W.SOFTMAX:
        assert bool(torch.isfinite(result.scores().entropy).all())
    else:
        with pytest.raises(VisualMeshError, match="probabilities"):
            result.scores()
        answers.scores(result.tensors()["classifications"])
    engine.close()
