"""Captured calls with block patterns, beside calls with other patterns."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _calls():
    from burn_dragon_amd import RotaryEmbedding
    from burn_dragon_amd.kernel.block_sparse import BlockPattern1d, BlockPattern2d
    from burn_dragon_amd.kernel.linear_attention import build_freqs, fused_state_aligned
    from burn_dragon_amd.kernel.relu_lowrank import fused_forward

    g = torch.Generator()
    g.manual_seed(1)
    r = lambda *shape: torch.randn(shape, generator=g).to(DEV)
    x, w = r(2, 1, 3, 32), r(1, 2, 32, 640)
    q, v, freqs = r(1, 2, 64, 32), r(1, 1, 64, 16), build_freqs(32, 65536.0, RotaryEmbedding.ROPE, DEV)
    latent = lambda size, blocks: fused_forward(x, w, None, 0.0, BlockPattern1d.from_blocks(size, blocks))
    time = lambda size, pairs: fused_state_aligned(q, v, freqs, None, BlockPattern2d.from_pairs(size, pairs), RotaryEmbedding.ROPE)
    return [(lambda: latent(64, [1, 4]), [lambda: latent(64, [0, 2, 9]), lambda: latent(1, [3])]),
            (lambda: time(16, [(1, 0), (3, 1)]), [lambda: time(16, [(2, 2)]), lambda: time(2, [(9, 1)])])]


def test_a_captured_call_keeps_its_pattern():
    for call, others in _calls():
        want = call().clone()
        torch.cuda.synchronize()
        assert want.abs().max() > 0
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        for other in others * 2:
            out.zero_()
            assert not torch.equal(other(), want)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
