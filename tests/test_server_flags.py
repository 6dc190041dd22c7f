"""Flags of the HTTP server that a model cannot honour end the program before
anything is built."""
import sys

import pytest

from aether_b200.models import deepseek, moe, qwen
from aether_b200.parallel import dist
from aether_b200.serving import server


@pytest.mark.parametrize("argv", [["--model", m, *f] for m in ("qwen2-moe", "mixtral", "deepseek-v2-lite")
                                  for f in (["--kv-bits", "8"], ["--w4", "64"])]
                         + [["--model", "tiny", "--w4", "128", "--tp", "2"], ["--model", "7b", "--kv-bits", "4"]])
def test_refused(monkeypatch, argv):
    def never(*a, **kw):
        raise AssertionError("went on")

    for mod, name in ((qwen, "QwenModel"), (qwen, "QwenWeights"), (moe, "MoEQwenModel"), (deepseek, "DeepSeekModel"), (dist, "init")):
        monkeypatch.setattr(mod, name, never)
    monkeypatch.setattr(sys, "argv", ["server", "--device", "cpu", *argv])
    with pytest.raises(SystemExit):
        server.main()


@pytest.mark.parametrize("argv,kw", [(["--kv-bits", "8", "--max-seq", "100", "--max-concurrent", "3"], dict(kv_bits=8, kv_pages=7)),
                                     ([], dict(kv_bits=16, kv_pages=0))])
def test_dense_models_take_them(monkeypatch, argv, kw):
    class Built(Exception):
        pass

    def model(cfg, **got):
        raise Built(got)

    monkeypatch.setattr(qwen, "QwenModel", model)
    monkeypatch.setattr(sys, "argv", ["server", "--device", "cpu", "--model", "tiny", *argv])
    with pytest.raises(Built) as e:
        server.main()
    assert {k: e.value.args[0][k] for k in kw} == kw
