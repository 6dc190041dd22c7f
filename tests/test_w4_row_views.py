"""Token rows that share memory: one row repeated (stride 0) and windows that
overlap, for each way a product of at most 64 rows goes.

Bound: K products summed in fp32, one rounding to bf16 (2^-9)."""
import pytest
import torch

from aether_b200.ops import functional as F

CPU_GPU = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("M", [1, 5, 16, 17, 33, 64])
@pytest.mark.parametrize("stride", [0, 8, 3])
def test_rows_that_overlap(dev, M, stride):
    g = torch.Generator().manual_seed(M + stride)
    N, K, group = 130, 256, 64
    codes, scales = torch.randint(0, 16, (N, K), generator=g), (torch.randn(N, K // group, generator=g) * 0.01).half()
    w64 = (codes.double() - 8) * scales.double().repeat_interleave(group, 1)
    x = torch.randn(K + stride * M, generator=g).bfloat16().to(dev).as_strided((M, K), (stride, 1))
    got = F.linear_w4(x, F.pack_w4(codes, scales).to(dev)).cpu().double()
    x64 = x.cpu().double()
    want = x64 @ w64.t()
    tol = K * 2.0 ** -23 * (x64.abs() @ w64.abs().t()) + 2.0 ** -8 * want.abs() + 1e-6
    assert ((got - want).abs() <= tol).all()
