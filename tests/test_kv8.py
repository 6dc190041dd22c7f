"""8-bit paged KV cache: append (rotation, quantisation, block scales), gather and
single-token attention, against statements in 64 bits.

Bounds, from the arithmetic: a stored value is within half a step of its fp32
value (one more half step for each time its block's scale grew); attention
rounds each weight once to fp16 (2^-11) and the output once to bf16 (2^-9), and
its fp32 logits and sums are far below that, so an output is within
2^-8 * sum_j p_j |v_j| of the exact one."""
import pytest
import torch

from aether_b200 import _ext
from aether_b200.ops import functional as F
from aether_b200.ops import reference as ref

CPU_GPU = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def make_cache(g, pages, Hkv, P, D):
    codes = (torch.randn(pages, Hkv, P, D, generator=g) * 35).round().clamp(-127, 127).add(128).to(torch.uint8)
    return codes, torch.exp(torch.randn(pages, Hkv, P // 16, generator=g) * 0.3) * 0.03


def make_table(g, rows, cols, first=1):
    return (torch.randperm(rows * cols, generator=g) + first).view(rows, cols).to(torch.int32)


def angles(n, D):
    return ref.rope_tables(n, D, 1e4)


def values64(codes, scale, pages, n):
    out = torch.empty(n, codes.shape[1], codes.shape[3], dtype=torch.float64)
    P = codes.shape[2]
    for t in range(n):
        p, r = int(pages[t // P]), t % P
        out[t] = (codes[p, :, r].double() - 128) * scale[p, :, r // 16].double()[:, None]
    return out


# ------------------------------------------------------------------ append
def run_append(dev, D, P, Hq, Hkv, spans, in_place, seed=0):
    """spans: (pos, n) of each sequence -> everything before and after."""
    g = torch.Generator().manual_seed(seed)
    B, T = len(spans), sum(n for _, n in spans)
    cols = max(-(-(p + n + 16) // P) for p, n in spans)
    kc, ks = make_cache(g, B * cols + 1, Hkv, P, D)
    vc, vs = make_cache(g, B * cols + 1, Hkv, P, D)
    table = make_table(g, B, cols)
    slot = torch.randperm(B, generator=g).to(torch.int32)
    row = (Hq + 2 * Hkv) * D
    qkv = torch.randn(T, row + 16, generator=g).bfloat16()[:, :row]
    qkv[:, Hq * D :] *= torch.exp(torch.randn(T, 1, generator=g))  # tokens of uneven size: scales grow
    cos, sin = angles(cols * P, D)
    pos = torch.tensor([p for p, _ in spans], dtype=torch.int32)
    start = torch.tensor([sum(n for _, n in spans[:i]) for i in range(B + 1)], dtype=torch.int32)
    before = [t.clone() for t in (kc, ks, vc, vs)]
    to = [t.to(dev) for t in (pos, slot, cos, sin, kc, ks, vc, vs, table)]
    x = torch.zeros(T, row + 16, dtype=torch.bfloat16, device=dev)[:, :row]
    x.copy_(qkv)
    out = None if in_place else torch.full((T, (Hq + Hkv) * D), 7.0, dtype=torch.bfloat16, device=dev)
    rs = None if all(n == 1 for _, n in spans) else start.to(dev)
    got = F.rope_kv8_append(x, *to, Hq, row_start=rs, out=out)
    return dict(qkv=qkv, pos=pos, slot=slot, start=start, cos=cos, sin=sin, table=table, before=before,
                after=[t.cpu() for t in to[4:8]], out=got.cpu(), x=x.cpu())


SPANS = {
    "one": [(0, 1)],
    "mid": [(5, 1), (16, 1), (31, 1), (63, 1), (64, 1)],
    "ragged": [(0, 40), (3, 0), (13, 1), (13, 3), (13, 4), (47, 90), (128, 16), (0, 1)],
}


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("spans", SPANS)
@pytest.mark.parametrize("D,P,Hq,Hkv,in_place", [(128, 64, 7, 1, True), (64, 16, 4, 2, False), (128, 16, 3, 3, False)])
def test_append(dev, spans, D, P, Hq, Hkv, in_place):
    spans = SPANS[spans]
    r = run_append(dev, D, P, Hq, Hkv, spans, in_place)
    touched = [set(), set()]
    for b, (p0, n) in enumerate(spans):
        if n == 0:
            continue
        x = r["qkv"][r["start"][b] : r["start"][b + 1]].double().view(n, -1, D)
        c, s = (t[p0 : p0 + n].double()[:, None] for t in (r["cos"], r["sin"]))
        a, bb = x[..., : D // 2], x[..., D // 2 :]
        y = torch.cat([a * c - bb * s, bb * c + a * s], -1)
        rows = r["out"][r["start"][b] : r["start"][b + 1], : (Hq + Hkv) * D].double()
        want = y[:, : Hq + Hkv].reshape(n, -1)
        assert ((rows - want).abs() <= 2.0 ** -8 * want.abs() + 1e-6).all()
        pages = r["table"][int(r["slot"][b])]
        for i, new in ((0, y[:, Hq : Hq + Hkv]), (1, x[:, Hq + Hkv :])):
            c0, s0, c1, s1 = r["before"][2 * i], r["before"][2 * i + 1], r["after"][2 * i], r["after"][2 * i + 1]
            old, now = (values64(c, s, pages, p0 + n) for c, s in ((c0, s0), (c1, s1)))
            assert torch.equal(now[: p0 // 16 * 16], old[: p0 // 16 * 16])
            for t in range(p0 // 16 * 16, p0 + n):
                page, blk = int(pages[t // P]), t % P // 16
                touched[i].add((page, blk))
                step = s1[page, :, blk].double()[:, None]
                base = t // 16 * 16
                part = new[max(0, base - p0) : base + 16 - p0]
                top = part.abs().amax((0, 2))[:, None] / 127
                if base < p0:  # older positions keep the scale from shrinking
                    top = torch.maximum(top, s0[page, :, blk].double()[:, None])
                assert ((step - top).abs() <= 1e-6 * top).all()
                exact = new[t - p0] if t >= p0 else old[t]
                assert ((now[t] - exact).abs() <= 0.5001 * step + 1e-12).all()
    for i in range(2):  # nothing else was written
        same = torch.ones(r["before"][2 * i + 1].shape[0], P // 16, dtype=torch.bool)
        for page, blk in touched[i]:
            same[page, blk] = False
        assert torch.equal(r["before"][2 * i + 1].transpose(1, 2)[same], r["after"][2 * i + 1].transpose(1, 2)[same])
        c0, c1 = (c.unflatten(2, (P // 16, 16)).transpose(1, 2)[same] for c in (r["before"][2 * i], r["after"][2 * i]))
        assert torch.equal(c0, c1)
    if in_place:  # v stays as it was
        assert torch.equal(r["x"][:, (Hq + Hkv) * D :], r["qkv"][:, (Hq + Hkv) * D :])


@pytest.mark.gpu
@pytest.mark.parametrize("spans", SPANS)
def test_append_cuda_equals_cpu_bit_for_bit(spans):
    a, b = (run_append(dev, 128, 32, 6, 2, SPANS[spans], False, seed=3) for dev in ("cpu", "cuda"))
    for x, y in zip(a["after"] + [a["out"]], b["after"] + [b["out"]]):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dev", CPU_GPU)
def test_append_token_by_token_keeps_the_block(dev):
    """Sixteen appends of one token, each larger than the last: at most one half
    step of the final scale for each growth."""
    g = torch.Generator().manual_seed(1)
    D, P = 128, 16
    kc, ks = (t.to(dev) for t in make_cache(g, 2, 1, P, D))
    vc, vs = kc.clone(), ks.clone()
    cos, sin = (t.to(dev) for t in angles(16, D))
    table = torch.tensor([[1]], dtype=torch.int32, device=dev)
    slot = torch.zeros(1, dtype=torch.int32, device=dev)
    x = torch.randn(16, 3 * D, generator=g).bfloat16() * (1.2 ** torch.arange(16)[:, None]).bfloat16()
    for t in range(16):
        F.rope_kv8_append(x[t : t + 1].to(dev), torch.tensor([t], dtype=torch.int32, device=dev), slot, cos, sin, kc,
                          ks, vc, vs, table, 1)
    got = values64(vc.cpu(), vs.cpu(), [1], 16)[:, 0]
    want = x[:, 2 * D :].double()
    step = float(vs[1, 0, 0])
    assert abs(step - float(want.abs().max()) / 127) <= 1e-6 * step
    # 1.2^-i of the final step for a rounding made i growths earlier: sum 1 / (1 - 1/1.2) = 6 halves, plus uneven maxima
    assert float((got - want).abs().max()) <= 0.5 * step * 8
    assert float((got - want).pow(2).mean().sqrt()) <= step  # and much less on average


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_append_zeros_and_non_finite(dev, bad):
    D, P = 64, 16
    g = torch.Generator().manual_seed(2)
    kc, ks = (t.to(dev) for t in make_cache(g, 4, 1, P, D))
    vc, vs = kc.clone(), ks.clone()
    cos, sin = (t.to(dev) for t in angles(16, D))
    table = torch.tensor([[1], [2], [3]], dtype=torch.int32, device=dev)
    qkv = torch.zeros(3, 3 * D, dtype=torch.bfloat16)
    qkv[1] = 1.0
    qkv[1, 2 * D + 5] = bad
    qkv[2] = 2.0 ** -120  # far below the smallest scale: rounds to zero
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    F.rope_kv8_append(qkv.to(dev), i32(0, 0, 0), i32(0, 1, 2), cos, sin, kc, ks, vc, vs, table, 1)
    v = values64(vc.cpu(), vs.cpu(), [1, 2, 3], 48)
    assert (v[0] == 0).all() and v[16].isnan().all() and (v[32] == 0).all()
    k = values64(kc.cpu(), ks.cpu(), [1, 2, 3], 48)
    assert (k[0] == 0).all() and k[16].isfinite().all()
    # the next token of that block reads as NaN too, a new block does not
    F.rope_kv8_append(torch.ones(1, 3 * D, dtype=torch.bfloat16, device=dev), i32(1), i32(1), cos, sin, kc, ks, vc, vs,
                      table, 1)
    assert values64(vc.cpu(), vs.cpu(), [2], 2).isnan().all()
    F.rope_kv8_append(torch.ones(1, 3 * D, dtype=torch.bfloat16, device=dev), i32(0), i32(1), cos, sin, kc, ks, vc, vs,
                      table, 1)
    assert (values64(vc.cpu(), vs.cpu(), [2], 1) - 1).abs().max() <= 0.5001 / 127


@pytest.mark.parametrize("dev", CPU_GPU)
def test_append_skips_negative_slots(dev):
    D = 64
    g = torch.Generator().manual_seed(2)
    kc, ks = (t.to(dev) for t in make_cache(g, 3, 1, 16, D))
    before = kc.clone(), ks.clone()
    cos, sin = (t.to(dev) for t in angles(16, D))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    x = torch.randn(2, 3 * D, generator=g).bfloat16().to(dev)
    table = torch.tensor([[1], [2]], dtype=torch.int32, device=dev)
    out = torch.zeros(2, 2 * D, dtype=torch.bfloat16, device=dev)
    F.rope_kv8_append(x, i32(0, 0), i32(-1, 1), cos, sin, kc, ks, kc.clone(), ks.clone(), table, 1, out=out)
    assert torch.equal(kc[:2], before[0][:2]) and not torch.equal(kc[2], before[0][2])
    assert (out[0] == 0).all() and (out[1] != 0).any()


# ------------------------------------------------------------------ gather
@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("D,P,first,n", [(128, 64, 0, 130), (64, 16, 7, 1), (128, 32, [3, 0, 40], 50), (64, 16, 0, 0)])
def test_gather(dev, D, P, first, n):
    g = torch.Generator().manual_seed(4)
    cols = -(-130 // P)
    codes, scale = make_cache(g, 3 * cols + 1, 2, P, D)
    table = make_table(g, 3, cols)
    slot = torch.tensor([2, 0, 1], dtype=torch.int32)
    f = torch.tensor(first, dtype=torch.int32).to(dev) if isinstance(first, list) else first
    got = F.gather_kv8(codes.to(dev), scale.to(dev), table.to(dev), slot.to(dev), f, n).cpu()
    assert got.shape == (3, n, 2, D)
    for b in range(3):
        f0 = first[b] if isinstance(first, list) else first
        want = values64(codes, scale, table[int(slot[b])], f0 + n)[f0:]
        assert torch.equal(got[b], want.float().bfloat16())


# ------------------------------------------------------------------ attention
def exact_attention(q, caches, table, slot, lens, Hq, scale, window, softcap):
    kc, ks, vc, vs = caches
    B, D, G = q.shape[0], kc.shape[3], Hq // kc.shape[1]
    out = torch.zeros(B, Hq * D, dtype=torch.float64)
    size = torch.zeros_like(out)
    for b in range(B):
        n = int(lens[b])
        if n == 0 or int(slot[b]) < 0:
            continue
        lo = max(0, n - window) if window else 0
        k, v = (values64(c, s, table[int(slot[b])], n)[lo:].repeat_interleave(G, 1) for c, s in ((kc, ks), (vc, vs)))
        x = torch.einsum("hd,lhd->hl", q[b, : Hq * D].double().view(Hq, D), k) * scale
        x = softcap * torch.tanh(x / softcap) if softcap else x
        p = torch.softmax(x, -1)
        out[b] = torch.einsum("hl,lhd->hd", p, v).reshape(-1)
        size[b] = torch.einsum("hl,lhd->hd", p, v.abs()).reshape(-1)
    return out, size


def check_attention(dev, Hq, Hkv, D, P, lens, window=0, softcap=0.0, qscale=2.0, seed=5, slot=None, poison=True):
    g = torch.Generator().manual_seed(seed)
    B, cols = len(lens), max(1, -(-max(lens) // P)) + 1
    caches = [t for _ in range(2) for t in make_cache(g, B * cols + 1, Hkv, P, D)]
    table = make_table(g, B, cols)
    slot = torch.randperm(B, generator=g).to(torch.int32) if slot is None else torch.tensor(slot, dtype=torch.int32)
    lens = torch.tensor(lens, dtype=torch.int32)
    scale = D ** -0.5
    q = (torch.randn(B, Hq * D + 8, generator=g) * qscale).bfloat16()  # a slice of wider rows
    want, size = exact_attention(q, caches, table, slot, lens, Hq, scale, window, softcap)
    if poison:  # scales of blocks that no key of a sequence lives in, the page of the unused table column among them
        used = torch.zeros(B * cols + 1, P // 16, dtype=torch.bool)
        for b in range(B):
            for t in range(0, int(lens[b]) if slot[b] >= 0 else 0, 16):
                used[int(table[int(slot[b]), t // P]), t % P // 16] = True
        for i in (1, 3):
            caches[i].transpose(1, 2)[~used] = float("nan")
    dq = q.to(dev)[:, : Hq * D]
    out = torch.full((B, Hq * D + 8), 3.0, dtype=torch.bfloat16, device=dev)
    args = [t.to(dev) for t in (*caches, table, slot, lens)]
    F.kv8_decode_attention(dq, *args, Hq, scale, out=out[:, : Hq * D], window=window, softcap=softcap)
    assert (out[:, Hq * D :] == 3.0).all()
    got = out[:, : Hq * D].cpu().double()
    assert torch.isfinite(got).all()
    err = (got - want).abs()
    assert (err <= 2.0 ** -8 * size + 1e-7).all(), float((err / (size + 1e-9)).max())
    return args, dq, scale


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("Hq,Hkv,D,P", [(7, 1, 128, 64), (8, 8, 64, 16), (12, 2, 128, 16), (12, 1, 64, 32),
                                        (32, 4, 128, 128), (17, 1, 128, 16)])
def test_attention_lengths(dev, Hq, Hkv, D, P):
    check_attention(dev, Hq, Hkv, D, P, [1, 0, 15, 16, 17, 63, 64, 65, 130, 333])


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("window,softcap", [(1, 0.0), (5, 0.0), (16, 30.0), (100, 0.0), (1000, 2.0), (0, 30.0)])
def test_attention_window_and_softcap(dev, window, softcap):
    check_attention(dev, 8, 2, 128, 32, [1, 16, 99, 100, 101, 257], window=window, softcap=softcap)


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("qscale", [0.0, 1e-30, 50.0, 1e4])
def test_attention_flat_and_peaked(dev, qscale):
    """All keys alike, and one key that takes everything."""
    check_attention(dev, 4, 2, 128, 16, [3, 200, 47], qscale=qscale)


@pytest.mark.parametrize("dev", CPU_GPU)
def test_attention_skips_negative_slots(dev):
    check_attention(dev, 4, 2, 64, 16, [30, 31, 32], slot=[2, -1, 0])


@pytest.mark.parametrize("dev", CPU_GPU)
@pytest.mark.parametrize("which", [1, 3])
def test_attention_reads_nan_blocks_as_nan(dev, which):
    args, q, scale = check_attention(dev, 4, 2, 64, 16, [40, 40], poison=False)
    page = int(args[4][int(args[5][0]), 1])
    args[which][page, 1, 0] = float("nan")
    out = F.kv8_decode_attention(q, *args, 4, scale).float().view(2, 4, 64)
    assert out[0, 2:].isnan().all() and out[0, :2].isfinite().all() and out[1].isfinite().all()


@pytest.mark.parametrize("dev", CPU_GPU)
def test_attention_tiny_values_behind_large_ones(dev):
    """The weight sits on a block whose v is 10^6 times smaller than the others'."""
    g = torch.Generator().manual_seed(9)
    kc, ks = make_cache(g, 5, 1, 16, 64)
    vc, vs = make_cache(g, 5, 1, 16, 64)
    table = torch.tensor([[1, 2, 3, 4]], dtype=torch.int32)
    vs[3] *= 1e-6
    kc[:] = 128
    kc[3, 0, 4] = 228
    q = torch.full((1, 64), 8.0).bfloat16()
    lens, slot = torch.tensor([64], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    want, size = exact_attention(q, (kc, ks, vc, vs), table, slot, lens, 1, 1.0, 0, 0.0)
    args = [t.to(dev) for t in (kc, ks, vc, vs, table, slot, lens)]
    got = F.kv8_decode_attention(q.to(dev), *args, 1, 1.0).cpu().double()
    assert (want.abs().max() < 1e-4) and ((got - want).abs() <= 2.0 ** -8 * size).all()


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,lens", [(28, 4, [5000]), (28, 4, [1, 4000, 17, 2500, 0, 900]), (8, 8, [70001]),
                                         (12, 2, [129] * 61)])
def test_gpu_attention_long_and_ragged(Hq, Hkv, lens):
    check_attention("cuda", Hq, Hkv, 128, 64, lens, poison=len(lens) > 1 and max(lens) < 10000)


@pytest.mark.gpu
def test_gpu_attention_repeats_bit_for_bit_and_on_other_streams():
    args, q, scale = check_attention("cuda", 28, 4, 128, 64, [3000, 100, 2048, 1])
    ws = F.kv8_workspace("cuda")
    first = F.kv8_decode_attention(q, *args, 28, scale, workspace=ws)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        outs = [F.kv8_decode_attention(q, *args, 28, scale, workspace=ws) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(s)
    outs.append(F.kv8_decode_attention(q, *args, 28, scale))
    for o in outs:
        assert torch.equal(o, first)


@pytest.mark.gpu
def test_gpu_offsets_past_32_bits():
    """Pools of 2.7e9 bytes: appended, gathered and attended at their far end."""
    pages, Hkv, P, D = 41000, 4, 128, 128
    kc = torch.zeros(pages, Hkv, P, D, dtype=torch.uint8, device="cuda")
    ks = torch.zeros(pages, Hkv, P // 16, device="cuda")
    vc, vs = torch.zeros_like(kc), torch.zeros_like(ks)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    g = torch.Generator().manual_seed(8)
    T, Hq = 200, 4
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).bfloat16()
    cos, sin = angles(256, D)
    F.rope_kv8_append(qkv.cuda(), i32(0), i32(0), cos.cuda(), sin.cuda(), kc, ks, vc, vs, table, Hq, row_start=i32(0, T))
    v = F.gather_kv8(vc, vs, table, i32(0), 0, T)[0].cpu()
    want = qkv[:, (Hq + Hkv) * D :].view(T, Hkv, D)
    assert float((v.float() - want.float()).abs().max()) <= 0.51 * float(want.float().abs().max()) / 127 + 2.0 ** -7
    q = torch.zeros(1, Hq * D, dtype=torch.bfloat16, device="cuda")
    o = F.kv8_decode_attention(q, kc, ks, vc, vs, table, i32(0), i32(T), Hq, 1.0).cpu().double().view(Hkv, D)
    assert ((o - v.double().mean(0)).abs() <= 2.0 ** -8 * v.double().abs().mean(0) + 2.0 ** -9 * v.double().abs().mean(0)).all()


# ------------------------------------------------------------------ refusals
@pytest.mark.gpu
def test_gpu_out_of_range_is_reported():
    _ext.check_status()
    g = torch.Generator().manual_seed(2)
    kc, ks = (t.cuda() for t in make_cache(g, 3, 1, 16, 64))
    vc, vs = kc.clone(), ks.clone()
    before = kc.clone()
    cos, sin = (t.cuda() for t in angles(64, 64))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    x = torch.randn(1, 3 * 64, generator=g).bfloat16().cuda()
    q = x[:, :64]
    for table, slot, pos in (([[1]], 0, 16), ([[1]], 1, 0), ([[9]], 0, 0), ([[-1]], 0, 0), ([[1, 2, 1, 2, 1]], 0, 64)):
        t = torch.tensor(table, dtype=torch.int32, device="cuda")
        F.rope_kv8_append(x.clone(), i32(pos), i32(slot), cos, sin, kc, ks, vc, vs, t, 1)
        assert _ext.check_status() == 5
    assert torch.equal(kc, before)
    t = torch.tensor([[1, 7]], dtype=torch.int32, device="cuda")
    assert (F.gather_kv8(kc, ks, t, i32(0), 16, 16) == 0).all() and _ext.check_status() == 5
    for slot, n in ((0, 20), (1, 5)):
        F.kv8_decode_attention(q, kc, ks, vc, vs, t, i32(slot), i32(n), 1, 1.0)
        assert _ext.check_status() == 5
    F.kv8_decode_attention(q, kc, ks, vc, vs, t, i32(0), i32(16), 1, 1.0)
    assert _ext.check_status() == 0


@pytest.mark.gpu
def test_gpu_refusals():
    g = torch.Generator().manual_seed(2)
    kc, ks = (t.cuda() for t in make_cache(g, 3, 2, 16, 64))
    t = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    i = torch.zeros(1, dtype=torch.int32, device="cuda")
    cos, sin = (a.cuda() for a in angles(16, 64))
    x = torch.zeros(1, 8 * 64, dtype=torch.bfloat16, device="cuda")

    def append(x=x, kc=kc, ks=ks, t=t, i=i, cos=cos, Hq=4, **kw):
        F.rope_kv8_append(x, i, i, cos, sin, kc, ks, kc, ks, t, Hq, **kw)

    def attend(q=x, kc=kc, ks=ks, t=t, i=i, Hq=8, **kw):
        return F.kv8_decode_attention(q, kc, ks, kc, ks, t, i, i, Hq, 1.0, **kw)

    append(), attend()
    bad = [lambda: append(x=x.float()), lambda: append(x=x[:, :100]), lambda: append(i=i.long()), lambda: append(Hq=5),
           lambda: append(kc=kc.char()), lambda: append(kc=kc[:, :, :8].contiguous()), lambda: append(kc=kc.transpose(1, 2)),
           lambda: append(kc=kc[..., :48].contiguous()), lambda: append(ks=ks.half()), lambda: append(ks=ks[:2]),
           lambda: append(t=t.long()), lambda: append(t=t.cpu()), lambda: append(cos=cos[:, :16]),
           lambda: append(x=x.expand(2, -1)), lambda: append(row_start=i), lambda: append(out=x[:, :64]),
           lambda: append(x=torch.zeros(1, 8 * 64 + 1, dtype=torch.bfloat16, device="cuda")[:, 1:]),
           lambda: attend(q=x.half()), lambda: attend(Hq=7), lambda: attend(q=x[:, :64]), lambda: attend(i=i[:0]),
           lambda: attend(window=-1), lambda: attend(softcap=-1.0), lambda: attend(kc=kc.int()),
           lambda: attend(out=x.float()), lambda: F.gather_kv8(kc, ks, t, i, -1, 1), lambda: F.gather_kv8(kc, ks, t, i.long(), 0, 1),
           lambda: F.gather_kv8(kc, ks, t, i, 0, 1, out=torch.zeros(1, 1, 2, 64, device="cuda"))]
    for f in bad:
        with pytest.raises((RuntimeError, ValueError)):
            f()


def test_cpu_refusals():
    kc, ks = make_cache(torch.Generator().manual_seed(2), 3, 2, 16, 64)
    t, i = torch.tensor([[1]], dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    cos, sin = angles(16, 64)
    with pytest.raises(ValueError):
        F.rope_kv8_append(torch.zeros(1, 8 * 64), i, i, cos, sin, kc, ks, kc, ks, t, 4)
    with pytest.raises(ValueError):
        F.rope_kv8_append(torch.zeros(2, 8 * 64).bfloat16(), i, i, cos, sin, kc, ks, kc, ks, t, 4)
    with pytest.raises(ValueError):
        F.kv8_decode_attention(torch.zeros(1, 8 * 64), kc, ks, kc, ks, t, i, i, 8, 1.0)
