"""Slots, pages and positions out of range of an 8-bit paged cache: the CPU forms
raise where the kernels report, and neither touches another sequence's pages."""
import pytest
import torch

from aether_b200.ops import functional as F

D, P = 64, 16


def cache(fill=130):
    return torch.full((3, 1, P, D), fill, dtype=torch.uint8), torch.ones(3, 1, 1)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


TABLE = i32(1, 2)[:, None]


@pytest.mark.parametrize("table,slot,pos,n", [(TABLE, 2, 0, 1), (TABLE, 0, -3, 1), (TABLE, 0, 16, 1), (TABLE, 0, 10, 7),
                                              (i32(-1)[None], 0, 0, 1), (i32(3)[None], 0, 0, 1), (i32(1, 9)[None], 0, 0, 17),
                                              (i32(1, 2, 1)[None], 0, 32, 1)])
def test_append(table, slot, pos, n):
    kc, ks = cache()
    x = torch.ones(n, 3 * D).bfloat16()
    with pytest.raises(IndexError):
        F.rope_kv8_append(x, i32(pos), i32(slot), torch.ones(32, D // 2), torch.zeros(32, D // 2), kc, ks, kc, ks, table, 1,
                          row_start=i32(0, n))
    assert (kc == 130).all() and (ks == 1).all()


@pytest.mark.parametrize("start", [(0, 2), (-1, 0)])
def test_append_rows_outside_qkv(start):
    kc, ks = cache()
    with pytest.raises(IndexError):
        F.rope_kv8_append(torch.ones(1, 3 * D).bfloat16(), i32(0), i32(0), torch.ones(32, D // 2), torch.zeros(32, D // 2), kc, ks,
                          kc, ks, TABLE, 1, row_start=i32(*start))
    assert (kc == 130).all()


@pytest.mark.parametrize("table,slot,first,n", [(TABLE, -1, 0, 2), (TABLE, 2, 0, 2), (i32(-1)[None], 0, 0, 2), (i32(1, 3)[None], 0, 15, 2)])
def test_gather(table, slot, first, n):
    kc, ks = cache()
    with pytest.raises(IndexError):
        F.gather_kv8(kc, ks, table, i32(slot), first, n)


@pytest.mark.parametrize("first", [-3, i32(-3)])
def test_gather_before_the_sequence(first):
    kc, ks = cache()
    with pytest.raises(ValueError):
        F.gather_kv8(kc, ks, TABLE, i32(0), first, 2)


def test_gather_past_the_table_reads_zero():
    kc, ks = cache()
    v = F.gather_kv8(kc, ks, TABLE, i32(1), 14, 5)[0, :, 0, 0]
    assert v.tolist() == [2, 2, 0, 0, 0]


def test_entries_that_no_position_needs_are_not_looked_at():
    kc, ks = cache()
    t = i32(1, -1, 99)[None]
    assert (F.gather_kv8(kc, ks, t, i32(0), 3, 13) == 2).all()
    assert (F.kv8_decode_attention(torch.ones(1, D).bfloat16(), kc, ks, kc, ks, t, i32(0), i32(16), 1, 1.0) == 2).all()
    F.rope_kv8_append(torch.ones(16, 3 * D).bfloat16(), i32(0), i32(0), torch.ones(16, D // 2), torch.zeros(16, D // 2), kc, ks, kc, ks,
                      t, 1, row_start=i32(0, 16))
    assert (kc[0] == 130).all() and (kc[2] == 130).all()


@pytest.mark.parametrize("table,slot,n", [(TABLE, 2, 4), (TABLE, 0, 17), (i32(-1)[None], 0, 4), (i32(1, 3)[None], 0, 17)])
def test_attention(table, slot, n):
    kc, ks = cache()
    with pytest.raises(IndexError):
        F.kv8_decode_attention(torch.ones(1, D).bfloat16(), kc, ks, kc, ks, table, i32(slot), i32(n), 1, 1.0)


@pytest.mark.parametrize("dev", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("kw", [dict(window=-1), dict(softcap=-1.0), dict(softcap=float("inf")), dict(softcap=float("nan"))])
def test_attention_refuses(dev, kw):
    kc, ks = (t.to(dev) for t in cache())
    with pytest.raises((ValueError, RuntimeError)):
        F.kv8_decode_attention(torch.ones(1, D).bfloat16().to(dev), kc, ks, kc, ks, TABLE.to(dev), i32(0).to(dev), i32(4).to(dev), 1, 1.0,
                               **kw)
