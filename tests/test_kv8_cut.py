"""Attention over page tables of more than 1024 keys, whose sequences are cut into
ranges and joined by a second kernel: head_dim 64, several groups of eight query
heads, windows and softcaps, few and many parts. (Bound as in test_kv8.)"""
import pytest
import torch
from test_kv8 import check_attention

from aether_b200 import _ext
from aether_b200.ops import functional as F

RAGGED = [3000, 1, 0, 1200, 2047, 2049]


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[5000], RAGGED, [1100 + 37 * i for i in range(20)], [1025] * 40], ids=["one", "ragged", "20", "40"])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 64), (12, 1, 64), (17, 1, 128), (20, 2, 64)])
def test_gpu_heads(Hq, Hkv, D, lens):
    check_attention("cuda", Hq, Hkv, D, 64, lens)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window,softcap", [(1009, 0.0), (1500, 0.0), (2000, 30.0), (0, 30.0), (0, 2.0), (100000, 0.0)])
@pytest.mark.parametrize("lens", [[5000], RAGGED + [1499, 1500, 1501, 1009, 1010, 1024]], ids=["one", "ragged"])
def test_gpu_window_and_softcap(D, window, softcap, lens):
    check_attention("cuda", 12, 1, D, 32, lens, window=window, softcap=softcap)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_gpu_narrow_window_over_a_wide_table(D):
    """Few keys each: a CTA for each sequence, far into the table."""
    check_attention("cuda", 12, 1, D, 32, RAGGED + [5000], window=130, softcap=20.0)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,window,softcap", [(4, 4, 0, 30.0), (12, 1, 0, 5.0), (12, 1, 77, 30.0)])
def test_gpu_short_tables_of_head_dim_64(Hq, Hkv, window, softcap):
    check_attention("cuda", Hq, Hkv, 64, 16, [1, 16, 99, 0, 700, 257], window=window, softcap=softcap)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_gpu_a_sequence_alone_and_in_a_batch(D):
    """Whatever else is in the batch, where a sequence is cut is the most that changes: both within the bound of each
    other, and the same call repeats bit for bit."""
    args, q, scale = check_attention("cuda", 12, 1, D, 32, RAGGED, poison=False)
    all_ = F.kv8_decode_attention(q, *args, 12, scale)
    assert torch.equal(all_, F.kv8_decode_attention(q, *args, 12, scale))
    caches, table, slot, lens = args[:4], args[4], args[5], args[6]
    for b in (0, 3, 5):
        one = F.kv8_decode_attention(q[b : b + 1], *caches, table, slot[b : b + 1], lens[b : b + 1], 12, scale)
        v = F.gather_kv8(caches[2], caches[3], table, slot[b : b + 1], 0, int(lens[b]))
        assert (one[0].float() - all_[b].float()).abs().max() <= 2.0 ** -7 * v.abs().max().float()
    assert _ext.check_status() == 0
