"""The launch count of a timed region: every call is counted while counting is on,
however its function was come by, with the kernels that it launches."""
import pytest
import torch

from aether_b200 import _ext
from aether_b200.ops import functional as F


class Fake:
    version = 3

    def __init__(self):
        self.calls = 0

    def __getattr__(self, name):
        def f(*a, **kw):
            self.calls += 1
            return name

        return f

    def kv8_decode_kernels(self, q, kc, table, window):
        return 2


def test_functions_looked_up_before_counting(monkeypatch):
    proxy = _ext._CountingModule(Fake())
    monkeypatch.setattr(_ext, "_PROXY", proxy)
    early = proxy.swiglu_fwd
    assert early(1) == "swiglu_fwd" and proxy.version == 3
    _ext.count_launches(True)
    late = proxy.rmsnorm_bwd
    early(1), late(1), proxy.swiglu_fwd(2, x=1), proxy.read_and_clear_status()
    proxy.kv8_decode_attention(*range(12), window=0, cap=0.0)
    assert _ext.count_launches(False) == 1 + 2 + 1 + 0 + 2
    early(1), late(1), proxy.grad_norm()
    assert proxy.launches == 6 and proxy._mod.calls == 9
    _ext.count_launches(True)
    assert proxy.launches == 0
    early(1)
    assert _ext.count_launches(False) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("cols,window,want", [(16, 0, 1), (17, 0, 2), (64, 0, 2), (64, 1008, 1), (64, 1009, 2), (17, 5, 1)])
def test_gpu_attention_counts_its_join(cols, window, want):
    """Up to 1024 keys a CTA takes a sequence whole; more are cut and joined by a second kernel."""
    P, D = 64, 64
    kc = torch.full((cols, 1, P, D), 128, dtype=torch.uint8, device="cuda")
    ks = torch.ones(cols, 1, P // 16, device="cuda")
    table = torch.arange(cols, dtype=torch.int32, device="cuda")[None]
    i32 = lambda v: torch.tensor([v], dtype=torch.int32, device="cuda")  # noqa: E731
    q, slot, lens = torch.zeros(1, D, dtype=torch.bfloat16, device="cuda"), i32(0), i32(cols * P)
    ws, out = F.kv8_workspace("cuda"), torch.empty(1, D, dtype=torch.bfloat16, device="cuda")
    run = lambda q=q, slot=slot, lens=lens, out=out: F.kv8_decode_attention(  # noqa: E731
        q, kc, ks, kc, ks, table, slot, lens, 1, 1.0, out=out, workspace=ws, window=window)
    run()
    _ext.count_launches(True)
    run()
    assert _ext.count_launches(False) == want
    _ext.count_launches(True)
    run(q[:0], slot[:0], lens[:0], out[:0])
    assert _ext.count_launches(False) == 0
