"""Products with 4-bit weights of more rows than a decode batch take the same
arguments as smaller ones: any row stride and base, and the same refusals.

Bound: each weight is rounded once more to bf16 (2^-9), and so are gate, up and
SwiGLU's product; sums are fp32."""
import pytest
import torch

from aether_b200.ops import functional as F

CPU_GPU = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def slice_of(t, shift, wide):
    """t's values as rows of a wider tensor, `shift` elements in."""
    full = torch.full((t.shape[0], t.shape[1] + wide), 5.0, dtype=t.dtype, device=t.device)
    full[:, shift : shift + t.shape[1]] = t
    return full, full[:, shift : shift + t.shape[1]]


def check(dev, M, N, swiglu, wide, shift, same_rows=False):
    g = torch.Generator().manual_seed(1)
    K, group, n_out = 256, 64, N // 2 if swiglu else N
    codes, scales = torch.randint(0, 16, (N, K), generator=g), (torch.randn(N, K // group, generator=g) * 0.01).half()
    w64 = (codes.double() - 8) * scales.double().repeat_interleave(group, 1)
    x = torch.randn(1 if same_rows else M, K, generator=g).bfloat16().expand(M, K)
    b, r = torch.randn(N, generator=g).bfloat16(), torch.randn(M, n_out, generator=g).bfloat16()
    y, e = x.double() @ w64.t() + b.double(), 2.0 ** -8 * (x.double().abs() @ w64.abs().t() + b.double().abs())
    if swiglu:
        a, u = y.chunk(2, 1)
        ea, eu = e.chunk(2, 1)
        act = a * torch.sigmoid(a)
        y, e = act * u, 1.1 * ea * (u.abs() + eu) + act.abs() * eu + 2.0 ** -7 * (act * u).abs()
    y = y + r.double()
    dx = x.to(dev) if not same_rows else x[:1].to(dev).expand(M, K)
    if wide:
        dx = slice_of(dx, shift, wide)[1]
    db = torch.cat([b[:1], b]).to(dev)[1:] if shift else b.to(dev)  # two bytes off
    full, out = slice_of(torch.zeros(M, n_out, dtype=torch.bfloat16, device=dev), shift, wide)
    got = F.linear_w4(dx, F.pack_w4(codes, scales).to(dev), bias=db, residual=slice_of(r.to(dev), shift, wide)[1], swiglu=swiglu, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert (full[:, :shift] == 5.0).all() and (full[:, shift + n_out :] == 5.0).all()
    err = (got.cpu().double() - y).abs()
    assert (err <= e + 2.0 ** -8 * y.abs() + 1e-6).all(), float((err / (e + 2.0 ** -8 * y.abs())).max())


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("N,swiglu", [(48, False), (96, True), (35, False), (2 * 33, True)])
@pytest.mark.parametrize("wide,shift", [(0, 0), (5, 0), (3, 2), (8, 0), (8, 4), (8, 8), (9, 1)])
def test_strides_and_bases(dev, N, swiglu, wide, shift):
    check(dev, 65, N, swiglu, wide, shift)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("N,swiglu", [(48, False), (96, True), (35, False)])
def test_one_row_repeated(dev, N, swiglu):
    check(dev, 130, N, swiglu, 0, 0, same_rows=True)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [48, 35])
def test_gpu_refusals(N):
    M, K = 70, 96
    w = F.pack_w4(torch.randint(0, 16, (N, K)), torch.ones(N, 3)).to("cuda")
    x, b, r = (torch.zeros(s, dtype=torch.bfloat16, device="cuda") for s in ((M, K), (N,), (M, N)))
    F.linear_w4(x, w, bias=b, residual=r, out=r)
    bad = [dict(x=x.float()), dict(x=x[:, :64]), dict(x=x.t().contiguous().t()), dict(x=x[:, None]),
           dict(bias=b.cpu()), dict(bias=b.float()), dict(bias=b[1:]), dict(bias=torch.cat([b, b])[::2]), dict(residual=r.cpu()),
           dict(residual=r.float()), dict(residual=r[1:]), dict(residual=r[:1]), dict(residual=torch.cat([r, r])),
           dict(residual=r.t().contiguous().t()), dict(out=r.float()), dict(out=r[:, 1:]), dict(out=r.cpu()),
           dict(w=F.W4Weight(w.q, w.s, N, K, 16)), dict(w=F.W4Weight(w.q, w.s.cpu(), N, K, 32)), dict(w=F.W4Weight(w.q, w.s, N + 16, K, 32)),
           dict(w=w, swiglu=True, residual=r)]
    for kw in bad:
        with pytest.raises(RuntimeError):
            F.linear_w4(**dict(dict(x=x, w=w), **kw))


@pytest.mark.parametrize("M", [2, 70])
def test_cpu_refusals(M):
    N, K = 35, 96
    w = F.pack_w4(torch.randint(0, 16, (N, K)), torch.ones(N, 3))
    x, b, r = (torch.zeros(s, dtype=torch.bfloat16) for s in ((M, K), (N,), (M, N)))
    F.linear_w4(x, w, bias=b, residual=r, out=r)
    for kw in (dict(bias=b[:1]), dict(residual=r[:1]), dict(residual=r[:, :1]), dict(out=torch.cat([r, r])), dict(out=r[0]),
               dict(swiglu=True)):
        with pytest.raises(ValueError):
            F.linear_w4(x, w, **kw)
