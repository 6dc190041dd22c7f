"""Products with 4-bit weights and group scales against the formula in 64 bits.

Bound, from the arithmetic: K products are summed in fp32 (an error of at most
K * 2^-23 * sum |w| |x|, in any order and with the tensor cores' truncation),
and the result is rounded once to bf16 (2^-9)."""
import pytest
import torch

from aether_b200.ops import functional as F
from aether_b200.ops import reference as ref

CPU_GPU = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def make(g, N, K, group):
    codes = torch.randint(0, 16, (N, K), generator=g)
    scales = (torch.randn(N, K // group, generator=g) * 0.01).half()
    return F.pack_w4(codes, scales), (codes.double() - 8) * scales.double().repeat_interleave(group, 1)


def check(dev, M, N, K, group, bias=False, residual=False, swiglu=False, seed=0, wide=0):
    g = torch.Generator().manual_seed(seed)
    w, w64 = make(g, N, K, group)
    x = torch.randn(M, K + wide, generator=g).bfloat16()
    b = torch.randn(N, generator=g).bfloat16() if bias else None
    n_out = N // 2 if swiglu else N
    r = torch.randn(M, n_out + wide, generator=g).bfloat16()[:, :n_out] if residual else None
    x64 = x[:, :K].double()
    y = x64 @ w64.t()
    e = K * 2.0 ** -23 * (x64.abs() @ w64.abs().t())
    if bias:
        y = y + b.double()
        e = e + 2.0 ** -23 * y.abs()
    if swiglu:
        a, u = y.chunk(2, 1)
        ea, eu = e.chunk(2, 1)
        act = a * torch.sigmoid(a)
        e = 1.1 * ea * (u.abs() + eu) + act.abs() * eu  # |silu'| <= 1.1
        y = act * u
    if residual:
        y = y + r.double()
    tol = e + 2.0 ** -8 * y.abs() + 1e-6
    out = torch.full((M, n_out + wide), 5.0, dtype=torch.bfloat16, device=dev)
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    got = F.linear_w4(x.to(dev)[:, :K], w.to(dev), bias=to(b), residual=to(r), swiglu=swiglu, out=out[:, :n_out])
    assert (out[:, n_out:] == 5.0).all()
    err = (got.cpu().double() - y).abs()
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("N,K", [(1, 128), (17, 384), (40, 1152), (256, 2048)])
@pytest.mark.parametrize("M", [1, 3, 8, 9, 64])
def test_linear(dev, M, N, K, group):
    check(dev, M, N, K, group)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("K,group", [(32, 32), (96, 32), (64, 64), (192, 64), (1056, 32), (18944, 64)])
def test_linear_columns_that_end_inside_a_tile(dev, K, group):
    check(dev, 5, 35, K, group, bias=True)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("M", [16, 17, 32, 33, 48, 64])
@pytest.mark.parametrize("N,K,group", [(35, 32, 32), (130, 96, 32), (300, 192, 64), (515, 1920, 128), (1000, 1056, 32)])
def test_linear_batches(dev, M, N, K, group):
    check(dev, M, N, K, group, bias=True, residual=True, wide=5)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("M,F_", [(17, 200), (40, 64), (64, 1000), (64, 33)])
def test_linear_batches_swiglu(dev, M, F_):
    check(dev, M, 2 * F_, 512, 64, bias=True, swiglu=True)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
def test_gpu_linear_more_row_tiles_than_sms(group):
    """A CTA walks over several row tiles, its pipelines running on."""
    check("cuda", 64, 128 * 330 + 7, 384, group)
    check("cuda", 20, 128 * 330 + 7, 384, group, bias=True)


@pytest.mark.gpu
@pytest.mark.parametrize("K,group", [(96, 32), (128, 128), (640, 64), (1152, 128)])
def test_gpu_linear_rings_across_row_tiles(K, group):
    """Columns that a warp's turns, the scales' stages and a row tile's end cut
    in other places for each row tile."""
    check("cuda", 50, 128 * 200 + 9, K, group)
    check("cuda", 18, 2 * (64 * 170 + 8), K, group, swiglu=True)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("M,N,K,bias,residual,swiglu", [(1, 200, 256, True, True, False), (4, 2 * 133, 512, False, False, True),
                                                        (16, 2 * 64, 384, True, False, True), (33, 130, 640, True, True, False),
                                                        (2, 6, 128, True, True, True)])
@pytest.mark.parametrize("wide", [0, 3])
def test_linear_epilogues_and_strides(dev, M, N, K, bias, residual, swiglu, wide):
    check(dev, M, N, K, 128, bias, residual, swiglu, wide=wide)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("M,N,swiglu", [(0, 64, False), (65, 48, False), (130, 35, False), (70, 96, True), (70, 2 * 33, True)])
def test_linear_many_rows(dev, M, N, swiglu):
    """More than a decode batch: the weights are expanded (bf16: one more
    rounding of each weight, 2^-9), or the rows are taken in parts."""
    g = torch.Generator().manual_seed(1)
    w, w64 = make(g, N, 256, 64)
    x = torch.randn(M, 256, generator=g).bfloat16()
    n_out = N // 2 if swiglu else N
    r = torch.randn(M, n_out, generator=g).bfloat16()
    y, e = x.double() @ w64.t(), 2.0 ** -8 * (x.double().abs() @ w64.abs().t())
    if swiglu:
        a, u = y.chunk(2, 1)
        ea, eu = e.chunk(2, 1)
        e = 1.1 * ea * (u.abs() + eu) + (a * torch.sigmoid(a)).abs() * eu + 2.0 ** -7 * (a * torch.sigmoid(a) * u).abs()
        y = a * torch.sigmoid(a) * u
    y = y + r.double()
    got = F.linear_w4(x.to(dev), w.to(dev), residual=r.to(dev), swiglu=swiglu).cpu().double()
    assert ((got - y).abs() <= e + 2.0 ** -8 * y.abs() + 1e-6).all()


@pytest.mark.parametrize("dev", CPU_GPU)
def test_every_code_and_column(dev):
    """One-hot rows read single weights back exactly."""
    K, N = 256, 32
    codes = (torch.arange(N)[:, None] * 7 + torch.arange(K)[None] * 3) % 16
    w = F.pack_w4(codes, torch.full((N, K // 32), 0.5)).to(dev)
    for k0 in range(0, K, 64):
        x = torch.zeros(64, K, dtype=torch.bfloat16)
        x[torch.arange(64), k0 + torch.arange(64)] = 1.0
        got = F.linear_w4(x.to(dev), w).cpu().float()
        assert torch.equal(got, (codes[:, k0 : k0 + 64].t().float() - 8) * 0.5)
    assert torch.equal(w.bf16().cpu().float(), (codes.float() - 8) * 0.5)


@pytest.mark.parametrize("dev", CPU_GPU)
def test_padding_holds_nothing(dev):
    """Rows and columns past N and K may hold anything finite."""
    g = torch.Generator().manual_seed(3)
    w, w64 = make(g, 19, 160, 32)
    c = torch.full((32, 256), 15)
    c[:19, :160] = (w64 / w64.abs().clamp(min=1e-30)).long() * 0 + torch.randint(0, 16, (19, 160), generator=g)
    s = torch.full((32, 8), 100.0)
    s[:19, :5] = torch.rand(19, 5, generator=g)
    full = F.pack_w4(c, s)
    part = F.W4Weight(full.q, full.s, 19, 160, 32).to(dev)
    x = torch.randn(2, 160, generator=g).bfloat16()
    want = x.double() @ ((c[:19, :160].double() - 8) * s[:19, :5].half().double().repeat_interleave(32, 1)).t()
    got = F.linear_w4(x.to(dev), part).cpu().double()
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 1e-3).all()
    assert part.bf16().shape == (19, 160)


@pytest.mark.parametrize("dev", CPU_GPU)
def test_non_finite_rows_stay_in_their_row(dev):
    g = torch.Generator().manual_seed(4)
    w, _ = make(g, 48, 256, 128)
    x = torch.randn(9, 256, generator=g).bfloat16()
    x[3, 17] = float("nan")
    x[8, 255] = float("inf")
    y = F.linear_w4(x.to(dev), w.to(dev)).cpu().float()
    ok = torch.ones(9, dtype=torch.bool)
    ok[[3, 8]] = False
    assert y[3].isnan().all() and not y[8].isfinite().any() and y[ok].isfinite().all()


def test_quantize():
    g = torch.Generator().manual_seed(5)
    w = torch.randn(40, 256, generator=g) * 0.02
    w[3, :128] = 0
    q = F.quantize_w4(w, 64)
    v = ref.w4_values(q.q, q.s, 40, 256, 64)
    step = (w.view(40, 4, 64).abs().amax(-1) / 7).repeat_interleave(64, 1)
    # half a step, and 2^-11 of up to seven steps for the fp16 scale; subnormal scales aside
    assert ((v - w).abs() <= 0.51 * step + 1e-7).all() and (v[3, :128] == 0).all()
    assert q.bytes() == 48 * 256 // 2 + 48 * 4 * 2 and q.shape == (40, 256)


@pytest.mark.gpu
def test_gpu_linear_repeats_bit_for_bit():
    g = torch.Generator().manual_seed(6)
    for M, N, K in ((1, 500, 3584), (16, 3584, 1536), (64, 96, 8960)):
        w = make(g, N, K, 128)[0].to("cuda")
        x = torch.randn(M, K, generator=g).bfloat16().cuda()
        first = F.linear_w4(x, w)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs = [F.linear_w4(x, w) for _ in range(4)]
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(o, first) for o in outs)


def test_refusals():
    c = torch.randint(0, 16, (8, 96))
    for s in (torch.ones(8, 2), torch.ones(8, 6), torch.ones(7, 3)):
        with pytest.raises(ValueError):
            F.pack_w4(c, s)
    for K, group in ((100, 32), (128, 16), (96, 64)):
        with pytest.raises(ValueError):
            F.quantize_w4(torch.zeros(4, K), group)
    w = F.pack_w4(c, torch.ones(8, 3))
    with pytest.raises(ValueError):
        F.linear_w4(torch.zeros(2, 95).bfloat16(), w)


@pytest.mark.gpu
def test_gpu_refusals():
    w = F.pack_w4(torch.randint(0, 16, (8, 96)), torch.ones(8, 3)).to("cuda")
    x = torch.zeros(2, 96, dtype=torch.bfloat16, device="cuda")
    F.linear_w4(x, w)
    W = F.W4Weight
    y = torch.zeros(2, 8, dtype=torch.bfloat16, device="cuda")
    bad = [lambda: F.linear_w4(x.float(), w), lambda: F.linear_w4(x[:, :64], w), lambda: F.linear_w4(x.cpu().t().cuda().t()[:, ::2], w),
           lambda: F.linear_w4(x, w, bias=y[0, :7]), lambda: F.linear_w4(x, w, bias=y[0].float()), lambda: F.linear_w4(x, w, residual=y[:1]),
           lambda: F.linear_w4(x, w, residual=y.float()), lambda: F.linear_w4(x, w, out=y.float()), lambda: F.linear_w4(x, w, out=y[:, :7]),
           lambda: F.linear_w4(x, W(w.q, w.s, 8, 96, 16)), lambda: F.linear_w4(x, W(w.q, w.s, 8, 128, 32)),
           lambda: F.linear_w4(x, W(w.q, w.s.float(), 8, 96, 32)), lambda: F.linear_w4(x, W(w.q.long(), w.s, 8, 96, 32)),
           lambda: F.linear_w4(x, W(w.q, w.s, 24, 96, 32)), lambda: F.linear_w4(x, W(w.q.cpu(), w.s, 8, 96, 32)),
           lambda: F.linear_w4(x, W(w.q, w.s, 7, 96, 32), swiglu=True), lambda: F.dequant_w4(w, out=y)]
    for f in bad:
        with pytest.raises(RuntimeError):
            f()
