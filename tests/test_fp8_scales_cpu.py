"""CPU: the FP8 linears take one scale for the whole input; a scale for each row is refused before
anything is launched."""
import pytest
import torch


def e4m3(*shape):
    return torch.zeros(*shape).to(torch.float8_e4m3fn)


@pytest.mark.parametrize("scale", [torch.ones(4), torch.ones(4, 1), torch.ones(0), torch.ones(1, dtype=torch.bfloat16),
                                   torch.ones(1, device="meta")])
def test_only_one_scale_is_taken(scale):
    from qik.fp8 import FP8Linear, fp8_gemm
    one = torch.ones(1)
    lin = FP8Linear(256, 768)
    for call in (lambda: fp8_gemm(e4m3(4, 256), scale, e4m3(16, 256), one), lambda: fp8_gemm(e4m3(4, 256), one, e4m3(16, 256), scale),
                 lambda: lin.forward_e4m3(e4m3(4, 256), scale), lambda: lin.forward_swiglu_e4m3(e4m3(4, 256), scale),
                 lambda: lin.forward_qkv_rms_rope_e4m3(e4m3(1, 4, 256), scale, 2, torch.ones(128), torch.ones(128), None, 1e-6)):
        with pytest.raises(ValueError, match="one fp32 scale"):
            call()


def test_the_row_parallel_linear_too():
    from qik.tp_comm import PeerRowReduce
    r = object.__new__(PeerRowReduce)
    r.M, r.N = 4, 16
    with pytest.raises(ValueError, match="one fp32 scale"):
        r(e4m3(4, 256), torch.ones(4), e4m3(16, 256), torch.ones(1))


@pytest.mark.gpu
def test_row_scales_of_the_norm_are_refused():
    from qik.fp8 import FP8Linear, fp8_ffn_gelu
    from qik.rms_norm import fused_add_rms_norm_e4m3
    x = torch.randn(8, 256, device="cuda").bfloat16()
    q, s, _ = fused_add_rms_norm_e4m3(x, x, x[0].clone(), 1e-6, scales="row")
    up, down = FP8Linear(256, 512).cuda(), FP8Linear(512, 256).cuda()
    for call in (lambda: up.forward_e4m3(q, s), lambda: fp8_ffn_gelu(q, up, down, x_scale=s)):
        with pytest.raises(ValueError, match="one fp32 scale"):
            call()
    assert up.forward_e4m3(q[:1], s[:1]).shape == (1, 512)
