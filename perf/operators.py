"""Cases of the quantised decode operators: appending to an 8-bit paged KV cache, attention of single tokens over
it, gathering a cached prefix back to bf16, and products with 4-bit weights.

Formats (all plain tensors, so both forms read the same bytes):
  * KV pools: uint8 [pages, Hkv, page, D], code + 128 with codes in -127..127; scales fp32 [pages, Hkv, page / 16], one
    for each 16 tokens of a page and KV head; a value is code * scale. The page table is int32 [rows, max_pages].
  * 4-bit weights [N, K]: int32 q [ceil(N/16), ceil(K/128), 2, 32, 4], fp16 scales [ceil(N/16), ceil(K/128) * 128 /
    group, 8, 2]; w = (nibble - 8) * scale. Tile (n, k) holds rows 16 n.. and columns 128 k..; [h, l, j] of it is row
    8 h + l // 4, and element e of its eight is column 16 (2 j + e // 4) + 4 (l % 4) + e % 4, kept in bits
    (0, 16, 4, 20, 8, 24, 12, 28)[e]. scales[n, g, r, h] belongs to row 8 h + r of tile n.
"""
import math

import torch

own = False

BLOCK = 16
SHIFTS = (0, 16, 4, 20, 8, 24, 12, 28)
WORKSPACE = 16 << 20


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one chat turn on a small model (12 query heads, 2 KV heads), a few dozen tokens in: latency counts
        _attn("attn 1x97", 1, 12, 2, 128, 64, 97),
        # a serving batch of uneven sequences on the 7B shape
        _attn("attn 16x2304 ragged", 16, 28, 4, 128, 64, 2304, ragged=True),
        # a full batch of long sequences: the cache is hundreds of MB a layer
        _attn("attn 64x4096", 64, 28, 4, 128, 64, 4096),
        # one very long document, grouped-query with eight KV heads
        _attn("attn 1x100001", 1, 32, 8, 128, 128, 100001),
        # the decode step's append, one token for each of a batch of sequences, most in mid-block
        _append("append 64 tokens", 64, 28, 4, 128, 64, 1, 2100, ragged=True),
        # prefill of uneven prompts into fresh and part-filled blocks
        _append("append 8x2048 ragged", 8, 28, 4, 128, 64, 2048, 300, ragged=True),
        # a shared prefix brought back for a chunk's prefill: one conversation, and a batch of them
        _gather("gather 1x1000", 1, 2, 128, 64, 1000),
        _gather("gather 8x4096", 8, 4, 128, 64, 4096),
        # QKV of a small model for one token; then the 7B shape: gate/up with SwiGLU for one token, the down projection
        # for sixteen and the output projection for a full batch
        _w4("w4 1x2048x1536", 1, 2048, 1536, 128, bias=True),
        _w4("w4 1x37888x3584 swiglu", 1, 37888, 3584, 128, swiglu=True),
        _w4("w4 16x3584x18944", 16, 3584, 18944, 64, residual=True),
        _w4("w4 64x3584x3584", 64, 3584, 3584, 32, residual=True),
    ]


def _attn(name, seqs, hq, hkv, dim, page, length, ragged=False, window=0, softcap=0.0):
    return dict(name=name, op="attn", seqs=seqs, hq=hq, hkv=hkv, dim=dim, page=page, length=length, ragged=ragged,
                window=window, softcap=softcap)


def _append(name, seqs, hq, hkv, dim, page, new, past, ragged=False):
    return dict(name=name, op="append", seqs=seqs, hq=hq, hkv=hkv, dim=dim, page=page, new=new, past=past, ragged=ragged)


def _gather(name, seqs, hkv, dim, page, length):
    return dict(name=name, op="gather", seqs=seqs, hkv=hkv, dim=dim, page=page, length=length)


def _w4(name, rows, n, k, group, bias=False, residual=False, swiglu=False):
    return dict(name=name, op="w4", rows=rows, n=n, k=k, group=group, bias=bias, residual=residual, swiglu=swiglu)


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("attn", "attn", "append", "gather", "w4", "w4"))
    dim = rng.choice((64, 128, 128))
    page = rng.choice((16, 32, 64, 128))
    hkv = rng.choice((1, 2, 4, 8))
    hq = hkv * rng.choice((1, 2, 4, 5, 6, 7, 8, 12))
    if op == "attn":
        seqs = _log(rng, 1, 64)
        length = _log(rng, 1, min(131072, 64 * 4 * 4096 * 128 // (seqs * hkv * dim)))
        window = rng.choice((0, 0, 0, _log(rng, 1, 2 * length)))
        c = _attn("", seqs, hq, hkv, dim, page, length, rng.random() < 0.6, window, rng.choice((0.0, 0.0, 0.0, 30.0)))
    elif op == "append":
        seqs = _log(rng, 1, 64)
        top = 200000000 // (seqs * dim * (4 * hq + 12 * hkv + 4))
        new = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, min(16384, top)))
        c = _append("", seqs, hq, hkv, dim, page, new, _log(rng, 1, 4000) - 1, rng.random() < 0.6)
    elif op == "gather":
        seqs = _log(rng, 1, 16)
        c = _gather("", seqs, hkv, dim, page, _log(rng, 1, min(131072, 32768 * 4 * 128 // (seqs * hkv * dim))))
    else:
        group = rng.choice((32, 64, 128))
        k = group * _log(rng, 1, 20480 // group)
        swiglu = rng.random() < 0.3
        rows = _log(rng, 1, 64)
        n = _log(rng, 1, min(40000, 37888 * 3584 // k, 5000000000 // (rows * k)))
        n = 2 * ((n + 1) // 2) if swiglu else n
        c = _w4("", rows, n, k, group, rng.random() < 0.4, rng.random() < 0.3 and not swiglu, swiglu)
    c.pop("name")
    return c


def _spread(n, top, ragged, low):
    """`n` whole numbers in low..top, the first of them top: all equal, or spread without a pattern."""
    if not ragged:
        return [top] * n
    return [top if i == 0 else low + int((top - low) * ((i * 0.6180339887 + 0.29) % 1.0)) for i in range(n)]


def work(case):
    op = case["op"]
    if op == "w4":
        m, n, k = case["rows"], case["n"], case["k"]
        n_out = n // 2 if case["swiglu"] else n
        b = n * k / 2 + 2 * n * (k // case["group"]) + 2 * m * k + 2 * m * n_out
        b += 2 * n if case["bias"] else 0
        b += 2 * m * n_out if case["residual"] else 0
        return {"bytes": b, "flops": 2 * m * n * k}
    hkv, d = case["hkv"], case["dim"]
    token = 2 * hkv * d * (1 + 4 / (BLOCK * d))  # 8-bit K and V of one token and its share of the scales
    if op == "gather":
        t = case["seqs"] * case["length"]
        return {"bytes": t * (token + 4 * hkv * d), "flops": 2 * t * hkv * d}
    if op == "attn":
        lens = _spread(case["seqs"], case["length"], case["ragged"], 1)
        keys = sum(min(x, case["window"]) if case["window"] else x for x in lens)
        return {"bytes": keys * token + 4 * case["seqs"] * case["hq"] * d, "flops": 4 * keys * case["hq"] * d}
    past, new, first, count = _append_plan(case)
    t, hq = sum(new), case["hq"]
    rows = 2 * t * (hq + 2 * hkv) * d + 4 * t * d + 2 * t * (hq + hkv) * d  # qkv and angles in, rotated q and k out
    back = 2 * case["seqs"] * count * 2 * hkv * d  # the blocks as they stand for afterwards
    return {"bytes": rows + t * token + back, "flops": 3 * t * (hq + hkv) * d + 2 * t * hkv * d}


def _append_plan(case):
    """Tokens before, new tokens, first position shown and how many positions are shown, for each sequence."""
    past = _spread(case["seqs"], case["past"], case["ragged"], 0)
    new = _spread(case["seqs"], case["new"], case["ragged"] and case["new"] > 1, 0)
    first = [p // BLOCK * BLOCK for p in past]
    count = max(p + n - f for p, n, f in zip(past, new, first))
    return past, new, first, -(-count // BLOCK) * BLOCK


# ------------------------------------------------------------------ inputs
def _cache(g, pages, hkv, page, dim):
    """One pool and its scales: normal values of uneven size, as projections give."""
    codes = (torch.randn(pages, hkv, page, dim, generator=g, device="cuda", dtype=torch.bfloat16) * 34).round_()
    codes = codes.clamp_(-127, 127).add_(128).to(torch.uint8)
    scale = torch.exp(torch.randn(pages, hkv, page // BLOCK, generator=g, device="cuda") * 0.3) * 0.03
    return codes, scale


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "w4":
        m, n, k, group = case["rows"], case["n"], case["k"], case["group"]
        nt, kt = -(-n // 16), -(-k // 128)
        # nibbles of a normal distribution: the sum of two smaller uniform ones
        lo = torch.randint(-(1 << 31), 1 << 31, (nt, kt, 2, 32, 4), generator=g, device="cuda").int() & 0x77777777
        hi = torch.randint(-(1 << 31), 1 << 31, (nt, kt, 2, 32, 4), generator=g, device="cuda").int() & 0x77777777
        s["q"] = lo + hi
        s["s"] = (torch.exp(torch.randn(nt, kt * 128 // group, 8, 2, generator=g, device="cuda") * 0.3) * 0.006).half()
        s["x"] = torch.randn(m, k, generator=g, device="cuda").bfloat16()
        s["b"] = torch.randn(n, generator=g, device="cuda").bfloat16() if case["bias"] else None
        n_out = n // 2 if case["swiglu"] else n
        s["r"] = torch.randn(m, n_out, generator=g, device="cuda").bfloat16() if case["residual"] else None
        return s
    seqs, hkv, dim, page = case["seqs"], case["hkv"], case["dim"], case["page"]
    if case["op"] == "append":
        past, new, first, count = _append_plan(case)
        top = max(f + count for f in first)
    else:
        lens = _spread(seqs, case["length"], case.get("ragged", False), 1)
        top = case["length"]
    per = -(-top // page)
    pages = seqs * per + 1
    s["kc"], s["ks"] = _cache(g, pages, hkv, page, dim)
    s["vc"], s["vs"] = _cache(g, pages, hkv, page, dim)
    s["table"] = (torch.randperm(pages - 1, generator=g, device="cuda").int() + 1).view(seqs, per).contiguous()
    s["slot"] = torch.randperm(seqs, generator=g, device="cuda").int()
    if case["op"] == "attn":
        s["seqlen"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["q"] = (torch.randn(seqs, case["hq"] * dim, generator=g, device="cuda") * 2).bfloat16()
        s["out"] = torch.empty(seqs, case["hq"] * dim, dtype=torch.bfloat16, device="cuda")
        s["workspace"] = torch.zeros(WORKSPACE, dtype=torch.uint8, device="cuda")
    elif case["op"] == "append":
        hq = case["hq"]
        t = sum(new)
        s["qkv"] = torch.randn(t, (hq + 2 * hkv) * dim, generator=g, device="cuda").bfloat16()
        s["out"] = torch.empty(t, (hq + hkv) * dim, dtype=torch.bfloat16, device="cuda")
        s["pos"] = torch.tensor(past, dtype=torch.int32, device="cuda")
        s["row_start"] = torch.tensor([sum(new[:i]) for i in range(seqs + 1)], dtype=torch.int32, device="cuda")
        s["first"] = torch.tensor(first, dtype=torch.int32, device="cuda")
        s["count"] = count
        angle = torch.arange(top, device="cuda", dtype=torch.float64)[:, None] * 1e6 ** (
            -torch.arange(dim // 2, device="cuda", dtype=torch.float64) * 2 / dim)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _own(s)
    return {"attn": _plain_attn, "append": _plain_append, "gather": _plain_gather, "w4": _plain_w4}[s["op"]](s)


def _own(s):
    from aether_b200.ops import functional as F

    if s["op"] == "attn":
        return F.kv8_decode_attention(s["q"], s["kc"], s["ks"], s["vc"], s["vs"], s["table"], s["slot"], s["seqlen"],
                                      s["hq"], s["dim"] ** -0.5, out=s["out"], workspace=s["workspace"],
                                      window=s["window"], softcap=s["softcap"])
    if s["op"] == "append":
        F.rope_kv8_append(s["qkv"], s["pos"], s["slot"], s["cos"], s["sin"], s["kc"], s["ks"], s["vc"], s["vs"],
                          s["table"], s["hq"], row_start=s["row_start"], out=s["out"])
        return {"qk": s["out"], "k": F.gather_kv8(s["kc"], s["ks"], s["table"], s["slot"], s["first"], s["count"]),
                "v": F.gather_kv8(s["vc"], s["vs"], s["table"], s["slot"], s["first"], s["count"])}
    if s["op"] == "gather":
        return {"k": F.gather_kv8(s["kc"], s["ks"], s["table"], s["slot"], 0, s["length"]),
                "v": F.gather_kv8(s["vc"], s["vs"], s["table"], s["slot"], 0, s["length"])}
    w = F.W4Weight(s["q"], s["s"], s["n"], s["k"], s["group"])
    return F.linear_w4(s["x"], w, bias=s["b"], residual=s["r"], swiglu=s["swiglu"])


def _values(codes, scale, table, slot, length):
    """fp32 [B, Hkv, length, D]: what the first `length` positions of each row's pages stand for."""
    pages = table[slot.long()].long()
    c = codes[pages].float() - 128
    b, n, h, p, d = c.shape
    v = c.view(b, n, h, p // BLOCK, BLOCK, d) * scale[pages][..., None, None]
    return v.view(b, n, h, p, d).permute(0, 2, 1, 3, 4).reshape(b, h, n * p, d)[:, :, :length]


def _plain_attn(s):
    b, hq, hkv, d = s["seqs"], s["hq"], s["hkv"], s["dim"]
    k = _values(s["kc"], s["ks"], s["table"], s["slot"], s["length"])
    q = s["q"].float().view(b, hkv, hq // hkv, d)
    x = (q @ k.transpose(2, 3)) * d ** -0.5
    del k
    if s["softcap"]:
        x = torch.tanh(x / s["softcap"]) * s["softcap"]
    j = torch.arange(s["length"], device="cuda")
    off = j >= s["seqlen"][:, None]
    if s["window"]:
        off = off | (j < s["seqlen"][:, None] - s["window"])
    x = x.masked_fill(off[:, None, None], float("-inf"))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    o = x @ _values(s["vc"], s["vs"], s["table"], s["slot"], s["length"])
    return o.reshape(b, hq * d).bfloat16()


def _shown(codes, scale, s):
    """bf16 [B, count, Hkv, D]: what positions first.. first + count stand for."""
    pos = s["first"].long()[:, None] + torch.arange(s["count"], device="cuda")
    page = s["table"][s["slot"].long()].long().gather(1, pos // s["page"])
    row = pos % s["page"]
    return ((codes[page, :, row].float() - 128) * scale[page, :, row // BLOCK][..., None]).bfloat16()


def _plain_store(y, codes, scale, page, row, old, unit, where, n_units):
    """Stores y [T, Hkv, D] at (page, row): a scale for each 16 positions, which takes in the older codes there."""
    t, h, d = y.shape
    top = torch.zeros(n_units, h, device="cuda").index_reduce_(0, unit, y.abs().amax(-1), "amax")
    new = top.clamp(min=2.0 ** -100) / 127
    upage, ublock = where
    before = scale[upage, :, ublock]
    new = torch.where(old[:, None] > 0, torch.maximum(before, new), new)
    r = torch.arange(BLOCK, device="cuda")
    rows = ublock[:, None] * BLOCK + r
    held = codes[upage[:, None], :, rows].float() - 128  # [units, 16, Hkv, D]
    held = torch.where((r < old[:, None])[:, :, None, None], (held * (before / new)[:, None, :, None]).round(), held)
    codes[upage[:, None], :, rows] = (held + 128).to(torch.uint8)
    codes[page, :, row] = ((y * (1 / new)[unit][..., None]).round().clamp(-127, 127) + 128).to(torch.uint8)
    scale[upage, :, ublock] = new


def _plain_append(s):
    hq, hkv, d, p = s["hq"], s["hkv"], s["dim"], s["page"]
    t = s["qkv"].shape[0]
    start = s["row_start"].long()
    tok = torch.arange(t, device="cuda")
    seq = (tok[:, None] >= start[None, 1:]).sum(1)
    pos = s["pos"].long()[seq] + tok - start[seq]
    x = s["qkv"].float().view(t, hq + 2 * hkv, d)
    c, sn = s["cos"][pos][:, None], s["sin"][pos][:, None]
    a, b = x[:, : hq + hkv, : d // 2], x[:, : hq + hkv, d // 2 :]
    qk = torch.cat([a * c - b * sn, b * c + a * sn], -1)
    page = s["table"][s["slot"].long()[seq], pos // p].long()
    row = pos % p
    per = s["count"] // BLOCK
    first = s["first"].long()
    unit = seq * per + (pos - first[seq]) // BLOCK
    at = first[:, None] + torch.arange(per, device="cuda") * BLOCK  # [B, per]: each block's first position
    old = (s["pos"].long()[:, None] - at).clamp(0, BLOCK)
    used = (at < (s["pos"].long() + start[1:] - start[:-1])[:, None]) & (start[1:] > start[:-1])[:, None]
    upage = s["table"][s["slot"].long()].long().gather(1, at // p)
    keep = used.reshape(-1).nonzero()[:, 0]
    number = torch.zeros(used.numel(), dtype=torch.long, device="cuda")
    number[keep] = torch.arange(keep.numel(), device="cuda")
    where = (upage.reshape(-1)[keep], (at % p // BLOCK).reshape(-1)[keep])
    old = old.reshape(-1)[keep]
    _plain_store(qk[:, hq:], s["kc"], s["ks"], page, row, old, number[unit], where, keep.numel())
    _plain_store(x[:, hq + hkv :], s["vc"], s["vs"], page, row, old, number[unit], where, keep.numel())
    return {"qk": qk.reshape(t, -1).bfloat16(), "k": _shown(s["kc"], s["ks"], s), "v": _shown(s["vc"], s["vs"], s)}


def _plain_gather(s):
    return {n: _values(s[n + "c"], s[n + "s"], s["table"], s["slot"], s["length"]).transpose(1, 2).bfloat16().contiguous()
            for n in ("k", "v")}


def _plain_w4(s):
    nt, kt = s["q"].shape[:2]
    w = (s["q"][..., None] >> torch.tensor(SHIFTS, device="cuda", dtype=torch.int32)) & 15
    w = w.view(nt, kt, 2, 8, 4, 4, 2, 4).permute(0, 2, 3, 1, 5, 6, 4, 7).reshape(nt * 16, -1, s["group"]).float() - 8
    w = (w * s["s"].float().permute(0, 3, 2, 1).reshape(nt * 16, -1, 1)).view(nt * 16, kt * 128)
    y = s["x"].float() @ w[: s["n"], : s["k"]].t()
    if s["b"] is not None:
        y = y + s["b"].float()
    if s["swiglu"]:
        a, u = y.chunk(2, -1)
        y = a / (1 + torch.exp(-a)) * u
    if s["r"] is not None:
        y = y + s["r"].float()
    return y.bfloat16()


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "append": _exact_append, "gather": _exact_gather, "w4": _exact_w4}[case["op"]](s)


def _row64(codes, scale, pages, length):
    """float64 [length, Hkv, D] of one sequence."""
    c = torch.cat(list(codes[pages.long()]), 1)[:, :length].double() - 128
    z = torch.cat(list(scale[pages.long()]), 1).double().repeat_interleave(BLOCK, 1)[:, :length]
    return (c * z[..., None]).transpose(0, 1)


def _exact_attn(s):
    out = []
    for b in range(s["seqs"]):
        n = int(s["seqlen"][b])
        pages = s["table"][int(s["slot"][b])]
        k, v = (_row64(s[x + "c"], s[x + "s"], pages, n) for x in "kv")
        lo = max(0, n - s["window"]) if s["window"] else 0
        q = s["q"][b].double().view(s["hkv"], -1, s["dim"])
        x = torch.einsum("hgd,lhd->hgl", q, k[lo:]) / math.sqrt(s["dim"])
        x = s["softcap"] * torch.tanh(x / s["softcap"]) if s["softcap"] else x
        out.append(torch.einsum("hgl,lhd->hgd", torch.softmax(x, -1), v[lo:]).reshape(-1))
    return torch.stack(out)


def _exact_gather(s):
    return {x: torch.stack([_row64(s[x + "c"], s[x + "s"], s["table"][int(i)], s["length"]) for i in s["slot"]]) for x in "kv"}


def _exact_append(s):
    hq, hkv, d = s["hq"], s["hkv"], s["dim"]
    start, rows, shown = s["row_start"].tolist(), [], {"k": [], "v": []}
    for b in range(s["seqs"]):
        past, n, first = int(s["pos"][b]), start[b + 1] - start[b], int(s["first"][b])
        x = s["qkv"][start[b] : start[b + 1]].double().view(n, hq + 2 * hkv, d)
        c, sn = (s[t][past : past + n].double()[:, None].repeat(1, 1, 2) for t in ("cos", "sin"))
        turned = torch.cat([-x[..., d // 2 :], x[..., : d // 2]], -1)
        y = (x * c + turned * sn)[:, : hq + hkv]
        rows.append(y.reshape(n, -1))
        for name, new in (("k", y[:, hq:]), ("v", x[:, hq + hkv :])):
            at = s["table"][int(s["slot"][b])].long()
            code = torch.cat(list(s[name + "c"][at]), 1).double().transpose(0, 1)[first : first + s["count"]] - 128
            scale = torch.cat(list(s[name + "s"][at]), 1).double().transpose(0, 1)[first // BLOCK :][: s["count"] // BLOCK]
            for i in range(0, past + n - first if n else 0, BLOCK):
                lo, hi = max(past, first + i), min(past + n, first + i + BLOCK)
                part, old = new[lo - past : hi - past], lo - first - i
                top = part.abs().amax((0, 2)).clamp(min=2.0 ** -100) / 127
                top = torch.maximum(top, scale[i // BLOCK]) if old else top
                code[i : i + old] = (code[i : i + old] * (scale[i // BLOCK] / top)[:, None]).round()
                code[i + old : hi - first] = (part / top[:, None]).round()
                scale[i // BLOCK] = top
            shown[name].append(code * scale.repeat_interleave(BLOCK, 0)[..., None])
    return {"qk": torch.cat(rows), "k": torch.stack(shown["k"]), "v": torch.stack(shown["v"])}


def _exact_w4(s):
    n, k, group = s["n"], s["k"], s["group"]
    nt, kt = s["q"].shape[:2]
    w = torch.empty(nt, 16, kt * 128, dtype=torch.int8, device="cuda")
    lane = torch.arange(32, device="cuda")
    for h in range(2):
        for j in range(4):
            for e in range(8):
                at = torch.arange(kt, device="cuda")[:, None] * 128 + 16 * (2 * j + e // 4) + 4 * (lane % 4) + e % 4
                w[:, 8 * h + lane // 4, at] = (((s["q"][:, :, h, :, j] >> SHIFTS[e]) & 15) - 8).to(torch.int8)
    scale = torch.cat([s["s"][..., 0], s["s"][..., 1]], 2).transpose(1, 2).reshape(nt * 16, -1).double()
    w, x, y = w.view(nt * 16, -1), s["x"].double(), []
    for i in range(0, n, 4096):
        part = w[i : min(n, i + 4096), :k].double()
        part = (part.view(part.shape[0], -1, group) * scale[i : i + part.shape[0], : k // group, None]).view(-1, k)
        y.append(x @ part.t())
    y = torch.cat(y, 1)
    if s["b"] is not None:
        y = y + s["b"].double()
    if s["swiglu"]:
        y = y[:, : n // 2] * torch.sigmoid(y[:, : n // 2]) * y[:, n // 2 :]
    return y + s["r"].double() if s["r"] is not None else y
