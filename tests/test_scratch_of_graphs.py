"""Scratch of recorded calls: it belongs to the graph, not to the buffers that eager calls share and outgrow."""
import contextlib

import pytest
import torch

import torchsso
from torchsso import _hip


@pytest.fixture
def scratch(monkeypatch):
    """A _Workspace on a pretended device: (workspace, set of the streams that are being captured, current stream)."""
    state = dict(captured=set(), current=[1], empty=torch.empty)

    class Stream(object):

        def __init__(self, handle):
            self.cuda_stream = handle

    @contextlib.contextmanager
    def use(stream):
        state['current'].append(stream.cuda_stream)
        yield
        state['current'].pop()
    monkeypatch.setattr(torch.cuda, 'is_initialized', lambda: True)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: state['current'][-1] in state['captured'])
    monkeypatch.setattr(torch.cuda, 'stream', use)
    monkeypatch.setattr(_hip, 'stream_ptr',
                        lambda device=None, stream=None: state['current'][-1] if stream is None else stream.cuda_stream)
    monkeypatch.setattr(torch, 'empty', lambda size, dtype, device: state['empty'](size, dtype=dtype))
    state.update(workspace=_hip._Workspace(), Stream=Stream, device=torch.device('cuda', 0))
    return state


def test_a_recorded_call_does_not_take_the_buffer_of_eager_ones(scratch):
    get, device = scratch['workspace'].get, scratch['device']
    eager, _ = get(device, 1000)
    scratch['captured'].add(1)
    recorded, size = get(device, 1000)
    assert size == recorded.numel() == 1000
    assert recorded.data_ptr() != eager.data_ptr()
    assert all(recorded is not b for b in scratch['workspace'].bufs.values())
    scratch['captured'].clear()
    assert get(device, 1000)[0] is eager


def test_nor_does_one_on_a_stream_that_the_recording_includes(scratch):
    get, device, side = scratch['workspace'].get, scratch['device'], scratch['Stream'](2)
    eager, _ = get(device, 1000, side)
    scratch['captured'].update((1, 2))
    recorded, _ = get(device, 1000, side)
    assert recorded.data_ptr() != eager.data_ptr()
    # a stream outside the recording is not touched by it
    scratch['captured'].remove(2)
    assert get(device, 1000, side)[0] is eager


@pytest.mark.gpu
def test_a_graph_outlives_the_scratch_that_it_was_recorded_with():
    g = torch.randn(200, 300, device='cuda')
    large = torch.randn(1500, 1500, device='cuda')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = torchsso.utils.orthogonalize(g)           # (the scratch of that stream)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = torchsso.utils.orthogonalize(g)
    with torch.cuda.stream(side):
        torchsso.utils.orthogonalize(large)              # (... which this outgrows)
    torch.cuda.synchronize()
    others = [torch.full((1 << 20,), 3., device='cuda') for _ in range(64)]
    with torch.cuda.stream(side):
        others += [torch.full((1 << 20,), 3., device='cuda') for _ in range(64)]
    torch.cuda.synchronize()
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        assert all(bool((t == 3.).all()) for t in others)
