"""AdamW steps at the ends of its sizes: nothing left for the kernel to do, and more than a launch holds."""
import pytest
import torch

from evox_amd.ops import adamw as aw
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


@pytest.mark.gpu
def test_refuses_a_leaf_of_2_to_34_elements(cuda):
    """One number expanded, so that nothing of that size exists; the leaf is refused before the state is looked at."""
    leaf = torch.zeros(1, dtype=torch.bfloat16, device=cuda).expand(2 ** 34)
    state = aw.adamw_init([leaf[:1]], 8)
    with pytest.raises(ValueError, match="one launch"):
        aw.adamw_step([leaf[:1], leaf], [leaf[:1], leaf], state, learning_rate=0.1)
    with pytest.raises(ValueError, match="state"):
        aw.adamw_step([leaf[:2 ** 34 - 1024]], [leaf[:2 ** 34 - 1024]], state, learning_rate=0.1)
