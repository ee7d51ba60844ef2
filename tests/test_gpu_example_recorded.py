"""The video example's forward pass with dropout as a recorded graph: every replay draws the masks of an eager pass with that state."""
import pytest
import torch

from test_gpu_blocks_use import example

pytestmark = pytest.mark.gpu


def test_recorded_pass_draws_new_masks(device, aclnn):
    E = example()
    torch.manual_seed(0)
    model = E.Model(device)
    frames = torch.rand(2, E.FRAMES, 3, E.SIZE, E.SIZE, device=device)
    with torch.no_grad():
        model(frames, p=0.3)  # once outside the recording, so that libraries are set up
        state = model.state.clone()
        assert state.tolist() == [1234, 2 * E.BLOCKS]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            scores = model(frames, p=0.3)
        seen = []
        for _ in range(4):
            graph.replay()
            torch.cuda.synchronize()
            seen.append(scores.clone())
        assert model.state.tolist() == [1234, 5 * 2 * E.BLOCKS]
        assert all(not torch.equal(a, b) for a, b in zip(seen, seen[1:]))
        model.state.copy_(state)
        for got in seen:
            want = model(frames, p=0.3)
            assert got.isfinite().all() and torch.equal(got, want)
