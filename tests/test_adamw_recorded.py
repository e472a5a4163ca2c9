"""AdamW steps recorded into a graph where nothing is left for its kernel to do."""
import pytest
import torch

from evox_amd.utils import optimizers


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_recorded_step_of_empty_leaves(cuda, bits):
    """A tree of empty leaves counts its steps without reading the count on the host."""
    opt = optimizers.adamw(0.1, state_bits=bits)
    params = [torch.zeros(0, 3, device=cuda), torch.zeros(0, device=cuda, dtype=torch.bfloat16)]
    state = opt.init(params)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        new, after = opt.step(params, state, params)
    for k in range(3):
        state["count"].fill_(float(k))
        graph.replay()
        torch.cuda.synchronize()
        assert float(after["count"]) == k + 1 and set(after) == set(state)
        assert [p.shape for p in new] == [(0, 3), (0,)] and [p.dtype for p in new] == [torch.float32, torch.bfloat16]
