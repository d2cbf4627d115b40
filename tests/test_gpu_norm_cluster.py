"""GPU: the norm of few rows with one scale, whose CTAs exchange their maxima through distributed
shared memory: the same scale and codes from many launches, alone and beside other work."""
import pytest
import torch

from test_gpu_decoder_ops import close, gen, norm_exact

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("M,N", [(1, 64), (1, 4096), (3, 512), (7, 4096), (8, 16384), (9, 24), (16, 2048)])
def test_every_launch_has_the_scale_of_all_rows(M, N):
    """Most CTAs of the cluster have no row where M is small, and reach the exchange ahead of those that do."""
    from qik.rms_norm import fused_add_rms_norm_e4m3
    g = gen(M * N)
    w = torch.randn(N, generator=g, device=DEV).bfloat16()
    xs = [(torch.randn(M, N, generator=g, device=DEV) * 2.0 ** (i % 5 - 2)).bfloat16() for i in range(8)]
    rs = [torch.randn(M, N, generator=g, device=DEV).bfloat16() for _ in range(8)]
    want = []
    for x, r in zip(xs, rs):
        q, s, _ = fused_add_rms_norm_e4m3(x, r, w, 1e-6)
        y = norm_exact(x, r, w, 1e-6)[1]
        close(s, (y.abs().amax() / 448).reshape(1), 0)
        want.append((q, s))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = [[fused_add_rms_norm_e4m3(x, r, w, 1e-6)[:2] for x, r in zip(xs, rs)] for _ in range(20)]
    other, big = torch.cuda.Stream(), torch.randn(4096, 4096, device=DEV).bfloat16()
    other.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        with torch.cuda.stream(other):  # the clusters start in what another kernel leaves free
            big @ big
        graph.replay()
        for rep in got:
            for (q, s), (q0, s0) in zip(rep, want):
                assert torch.equal(s, s0) and torch.equal(q.view(torch.uint8), q0.view(torch.uint8))
    torch.cuda.synchronize()
