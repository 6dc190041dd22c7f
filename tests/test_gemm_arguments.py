"""Bias and residual of the bf16 GEMM: its epilogue reads them 16 bytes at a time
on the operands' device, so anything else is refused before the launch."""
import pytest
import torch

from aether_b200.ops import functional as F

M, N, K = 70, 48, 64


def case(g):
    a, b = torch.randn(M, K, generator=g).bfloat16().cuda(), torch.randn(N, K, generator=g).bfloat16().cuda()
    return a, b, torch.randn(N + 8, generator=g).bfloat16().cuda(), torch.randn(M, N + 16, generator=g).bfloat16().cuda()


@pytest.mark.gpu
def test_gpu_refusals():
    a, b, bias, res = case(torch.Generator().manual_seed(1))
    for kw in (dict(bias=bias[:N].cpu()), dict(bias=bias[1 : N + 1]), dict(bias=bias[4 : N + 4]), dict(bias=bias[:N].float()),
               dict(bias=bias), dict(residual=res[:, :N].cpu()), dict(residual=res[:, 1 : N + 1]), dict(residual=res[:, 4 : N + 4]),
               dict(residual=res[:, :N].half()), dict(residual=res[: M - 1, :N]), dict(residual=res[0, :N]),
               dict(residual=res[:, : N + 4].contiguous()[:, :N])):
        with pytest.raises(RuntimeError):
            F.gemm(a, b, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("off", [0, 8])
def test_gpu_slices_on_16_byte_boundaries(off):
    """One rounding of the result to bf16, and fp32 sums of 64 products."""
    a, b, bias, res = case(torch.Generator().manual_seed(2))
    y = F.gemm(a, b, bias=bias[off : off + N], residual=res[:, off : off + N]).double()
    want = a.double() @ b.double().t() + bias[off : off + N].double() + res[:, off : off + N].double()
    size = a.double().abs() @ b.double().abs().t() + bias[off : off + N].double().abs() + res[:, off : off + N].double().abs()
    assert ((y - want).abs() <= 2.0 ** -8 * want.abs() + 66 * 2.0 ** -23 * size).all()
