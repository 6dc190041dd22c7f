"""A tensor-parallel model takes its own rank's shard and nothing else: the ranks'
products are summed, so whole weights would count once for each rank."""
import sys

import pytest

from aether_b200 import bench_serve
from aether_b200.models.qwen import QwenConfig, QwenModel, QwenWeights

TINY = dict(vocab=300, d_model=256, n_layers=1, n_heads=4, n_kv_heads=2, d_ff=512, max_seq=64)


class Rank:
    def __init__(self, rank, world):
        self.rank, self.world = rank, world


def build(weights, tp):
    return QwenModel(QwenConfig(**TINY), device="cpu", max_batch=1, weights=weights, tp=tp)


@pytest.mark.parametrize("w4", [False, True])
def test_whole_weights_are_refused(w4):
    w = QwenWeights(QwenConfig(**TINY), "cpu")
    if w4:
        w.quantize_w4(64)
    with pytest.raises(ValueError, match="shard"):
        build(w, Rank(0, 2))
    build(w, None)
    build(w, Rank(0, 1))


def test_another_ranks_shard_is_refused():
    full = QwenWeights(QwenConfig(**TINY), "cpu")
    w = QwenWeights.shard(full, 1, 2, "cpu")
    build(w, Rank(1, 2))
    for tp in (Rank(0, 2), Rank(1, 4), Rank(0, 1)):
        with pytest.raises(ValueError, match="shard"):
            build(w, tp)


@pytest.mark.parametrize("argv,world", [(["--w4", "128", "--tp", "2"], None), (["--w4", "128", "--emulate-tp", "8"], None),
                                        (["--w4", "64"], "2")])
def test_bench_serve_measures_4_bit_weights_on_one_gpu(monkeypatch, capsys, argv, world):
    def never(*a, **kw):
        raise AssertionError("went on")

    monkeypatch.setattr(bench_serve, "run", never)
    monkeypatch.setattr(bench_serve._ext, "C", never)
    monkeypatch.setattr(sys, "argv", ["bench_serve", *argv])
    if world:
        monkeypatch.setenv("WORLD_SIZE", world)
    with pytest.raises(SystemExit):
        bench_serve.main()
    assert "--w4" in capsys.readouterr().err
