"""fp8.PackedFp8 on the device: what reads a weight's codes right after they were packed again."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def test_a_graph_replayed_on_another_stream_reads_the_weight_packed_before():
    from flash_diffusion_amd import ops
    from flash_diffusion_amd.fp8 import PackedFp8
    w, x, p = _rand(4096, 2048).cuda(), _rand(300, 2048, seed=1, dtype=BF16).cuda(), PackedFp8()
    ops.gemm_fp8(x, p(w))
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        y = ops.gemm_fp8(x, p(w))
    for seed in (2, 3, 4, 5):
        new = _rand(4096, 2048, seed=seed).cuda()
        want = ops.gemm_fp8(x, ops.pack_weight_fp8(new))
        w.copy_(new)
        p(w)
        with torch.cuda.stream(other):       # (nothing tells this stream to wait for the one that packed)
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_transposed_data_of_a_square_weight():
    from flash_diffusion_amd.fp8 import PackedFp8
    w, p = torch.nn.Parameter(_rand(256, 256).cuda(), requires_grad=False), PackedFp8()
    before = p(w).values().clone()
    w.data = w.data.t()
    assert torch.equal(p(w).values(), before.t())                 # (square blocks: the transpose has the same codes)
