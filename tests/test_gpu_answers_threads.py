"""Calls of several threads at once, and tensors on another device than the current one."""
import ctypes as C
import threading

import pytest
import torch

from visualmesh_b200 import abi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def answers():
    from visualmesh_b200 import answers
    return answers


def inputs(seed, device="cuda"):
    q = torch.Generator(device=device).manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, device=device, generator=q)
    return {"rows": normal(400, 77), "long": normal(3, 9001).bfloat16(), "labels": torch.randint(-1, 77, (400,), device=device, generator=q),
            "x": normal(2, 3000, 24), "gate": normal(2, 3000, 24) + 2, "table": normal(900, 8), "steps": normal(700, 8),
            "index": torch.randint(-1, 900, (700,), device=device, generator=q).int()}


def everything(answers, v):
    scored = answers.scores(v["rows"], v["labels"], 3)
    scan = answers.gated_scan(v["x"], v["gate"], keep=True)
    table = v["table"].clone()
    return [*scored, answers.scores_backward(v["rows"], scored, v["labels"], scored.log_prob, scored.entropy), *answers.scores(v["long"], top=5)[1:], *scan,
            *answers.gated_scan_backward(v["x"], v["gate"], scan.states, scan.y, scan.last), answers.gated_step(table, v["steps"], v["steps"], v["index"]), table]


def test_calls_of_several_threads_at_once(answers):
    """From a library whose kernels no thread has used yet, as far as other tests left any: function attributes are set by whoever comes first."""
    wanted = {seed: [t.clone() for t in everything(answers, inputs(seed))] for seed in range(6)}
    torch.cuda.synchronize()
    got, failed, start = {}, [], threading.Barrier(6)

    def run(seed):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                held = inputs(seed)
                start.wait()
                for _ in range(20):
                    got[seed] = everything(answers, held)
                torch.cuda.current_stream().synchronize()
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=run, args=(seed,)) for seed in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for seed in range(6):
        for a, b in zip(got[seed], wanted[seed]):
            assert torch.equal(a, b)


def test_messages_belong_to_the_thread_of_the_call():
    lib, seen = abi.load(), {}

    def refuse(name, **bad):
        for _ in range(200):
            assert lib.vm_scores(-1, bad.get("x", 4096), bad.get("type", 0), 3, 5, 5, 0, 4096, 0, None, 4096, 4096, None, None, None) == abi.VM_ERR_INVALID_ARGUMENT
            seen.setdefault(name, set()).add(lib.vm_last_error())

    threads = [threading.Thread(target=refuse, args=("type",), kwargs=dict(type=9)), threading.Thread(target=refuse, args=("null",), kwargs=dict(x=None))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(seen["type"]) == len(seen["null"]) == 1 and seen["type"] != seen["null"]


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="one device")
def test_tensors_of_another_device_than_the_current_one(answers):
    torch.cuda.set_device(0)
    want = everything(answers, inputs(1, "cuda:0"))
    held = {k: t.to("cuda:1") for k, t in inputs(1, "cuda:0").items()}
    got = everything(answers, held)
    assert torch.cuda.current_device() == 0
    for a, b in zip(got, want):
        assert a.device == torch.device("cuda:1") and torch.equal(a.cpu(), b.cpu())
    with pytest.raises(abi.VisualMeshError):
        answers.scores(held["rows"], held["labels"].to("cuda:0"))


def test_a_device_that_is_not_there_is_an_error_and_the_current_one_stays(answers):
    x, out = torch.zeros((3, 5), device="cuda"), torch.zeros(3, device="cuda")
    row = abi.vm_sequence(x.data_ptr(), 5, 5, 1)
    lib, none = abi.load(), torch.cuda.device_count() + 3
    assert lib.vm_scores(none, x.data_ptr(), abi.VM_F32, 3, 5, 5, 0, None, 0, None, out.data_ptr(), None, None, None, None) == abi.VM_ERR_CUDA
    assert lib.vm_gated_scan(none, abi.VM_F32, 3, 1, 5, C.byref(row), C.byref(row), None, None, None, None, None, None, 0, None) == abi.VM_ERR_CUDA
    assert torch.cuda.current_device() == 0
    assert bool(torch.isfinite(answers.scores(x).entropy).all())
