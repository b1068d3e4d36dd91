"""The experts' workspace of a model: what it keeps as steps grow."""

from __future__ import annotations

import pytest
import torch

from tests.test_layer_model_gpu import make_model

pytestmark = pytest.mark.gpu


def test_an_outgrown_workspace_that_no_capture_took_is_let_go():
    model = make_model()
    before = torch.cuda.memory_allocated()
    sizes = []
    for rows in (1, 64, 65, 300, 4000, 20):
        ws = model.expert_workspace(rows)
        sizes.append(ws.numel())
        del ws
        torch.cuda.synchronize()
        assert torch.cuda.memory_allocated() - before <= sizes[-1] + 512  # one, rounded up as it is allocated
    assert sizes[0] == sizes[1] < sizes[2] < sizes[3] < sizes[4] == sizes[5]


@torch.inference_mode()
def test_one_that_a_capture_took_stays_and_the_next_ones_do_not():
    model = make_model()
    x = torch.randn(40, 192, device="cuda", dtype=torch.float16)
    want = model._experts(0, x, None)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model._experts(0, x, None)
    first = model._expert_workspaces[0]
    for rows in (100, 1000, 5000):
        model.expert_workspace(rows)
        assert len(model._expert_workspaces) == 2 and model._expert_workspaces[0] is first
    graph.replay()
    assert torch.equal(out, want) and not first[:6200].any()


@torch.inference_mode()
def test_it_grows_behind_a_step_on_another_stream():
    """The old one's memory is not handed out on the stream that allocated it while that step runs."""
    model = make_model()
    x = torch.randn(64, 192, device="cuda", dtype=torch.float16)
    want = model._experts(0, x, None)  # allocates on this stream
    old, size = model._expert_workspaces[-1].data_ptr(), model._expert_workspaces[-1].numel()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # some 100 ms
        got = model._experts(0, x, None)
        model.expert_workspace(100)
    others = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(4)]
    assert old not in [t.data_ptr() for t in others] or side.query()  # unless it is done by now
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_a_step_of_no_tokens():
    model = make_model()
    x = torch.empty(0, 192, device="cuda", dtype=torch.float16)
    assert model._experts(0, x, None).shape == (0, 192)


@torch.inference_mode()
def test_a_size_that_is_refused_leaves_what_captures_hold():
    """More tokens than any call takes: refused each time, and the captured step's workspace is still there."""
    model = make_model()
    x = torch.randn(40, 192, device="cuda", dtype=torch.float16)
    want = model._experts(0, x, None)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model._experts(0, x, None)
    first = model._expert_workspaces[0]
    for grown in (False, True):
        if grown:
            model.expert_workspace(1000)
        for _ in range(2):
            with pytest.raises(ValueError):
                model.expert_workspace(2**24 + 1)
            assert model._expert_workspaces and model._expert_workspaces[0] is first
    graph.replay()
    assert torch.equal(out, want)
    assert torch.equal(model._experts(0, x, None), want)
