"""Tensor-parallel serving over a paged KV cache on gloo ranks (CPU): the other
ranks' page tables follow rank 0's bookkeeping, and logits are those of one
rank.

Bound: the ranks' partial sums are added in fp32 and rounded to bf16 (2^-9)
where one rank rounds the whole sum, twice a layer; two layers and what follows
them leave well under 2 % of the logits' size, and a wrong page leaves 100 %."""
import os

import pytest
import torch
from test_tp_serve import _free_port, _GlooTP

TINY = dict(vocab=512, d_model=128, n_layers=2, n_heads=2, n_kv_heads=2, d_ff=256, max_seq=96, init_std=0.06)
STEPS = 12


def make_model(kv_bits, tp=None):
    from aether_b200.models.qwen import QwenConfig, QwenModel

    return QwenModel(QwenConfig(**TINY), device="cpu", seed=4, max_batch=2, kv_pages=13, page_size=16, kv_bits=kv_bits, tp=tp)


def waves():
    """Three waves over the same rows: two prompts of more than one page, two
    that begin with the first one's cached pages, two in swapped rows."""
    g = torch.Generator().manual_seed(1)
    first = torch.randint(0, 512, (2, 40), generator=g)
    again = first[:1].repeat(2, 1)
    again[:, 35:] = torch.randint(0, 512, (2, 5), generator=g)
    return [(first, [0, 1]), (again, [0, 1]), (first.flip(0), [1, 0])], torch.randint(0, 512, (STEPS, 2), generator=g)


def serve(model, cache):
    """Teacher-forced logits of every wave, by the calls that the engine makes."""
    out, hits = [], 0
    prompts, forced = waves()
    for p, slots in prompts:
        S = p.shape[1]
        for r in slots:
            cache.release(r)
        for i, r in enumerate(slots):
            n = cache.match_prefix(r, p[i].tolist())
            cache.ensure(r, S + STEPS)
            hits += n
            _, logits = model.prefill(p[i : i + 1, n:], slots=torch.tensor([r], dtype=torch.int32), start_pos=n, return_logits=True)
            cache.register_prompt(r, p[i].tolist())
            out.append(logits.clone())
        for t in range(STEPS):
            model.decode_step(forced[t], torch.full((2,), S + t, dtype=torch.int32), torch.tensor(slots, dtype=torch.int32),
                              use_graph=False, want_logits=True)
            out.append(model.buf["logits"][:2].clone())
    assert hits >= 2 * 32  # pages were shared
    return torch.cat(out)


def _worker(rank, world, port, q, kv_bits):
    os.environ.update(RANK=str(rank), WORLD_SIZE=str(world), MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    import torch.distributed as dist

    from aether_b200.serving.tp_serve import BroadcastModel, follow

    dist.init_process_group("gloo", rank=rank, world_size=world)
    ctrl = dist.new_group(backend="gloo")
    model = make_model(kv_bits, _GlooTP(rank, world))
    if rank == 0:
        bm = BroadcastModel(model, ctrl)
        logits = serve(bm, bm.cache)
        bm.stop()
        q.put(("logits", logits.numpy()))
    else:
        follow(model, ctrl)
    q.put((f"table{rank}", model.page_table.numpy()))
    dist.destroy_process_group()


@pytest.mark.parametrize("kv_bits", [8, 16])
def test_tp_paged_logits_match_one_rank(kv_bits):
    import multiprocessing as mp

    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    ps = [ctx.Process(target=_worker, args=(r, 2, port, q, kv_bits)) for r in range(2)]
    for p in ps:
        p.start()
    got = dict(q.get(timeout=300) for _ in range(3))
    for p in ps:
        p.join(timeout=60)
        assert p.exitcode == 0
    assert (got["table0"] == got["table1"]).all() and (got["table0"][:2, :3] > 0).all()
    one = make_model(kv_bits)
    want = serve(one, one.cache)
    rel = (torch.from_numpy(got["logits"]) - want).norm(dim=-1) / want.norm(dim=-1)
    assert float(rel.max()) < 0.02, rel


def test_changes_of_another_cache():
    from aether_b200.serving.kv import Paged8KVCache

    a, b = (Paged8KVCache(1, 1, 64, 9, 16, 3, 64, "cpu") for _ in range(2))
    a.ensure(0, 40)
    a.ensure(2, 1)
    first = a.take_changes()
    assert [r for r, _ in first] == [0, 2] and a.take_changes() == []
    b.apply_changes(first)
    assert torch.equal(a.table, b.table)
    a.ensure(0, 41)  # no new page
    assert a.take_changes() == []
    a.release(0)
    a.ensure(1, 64)
    b.apply_changes(a.take_changes())
    assert torch.equal(a.table, b.table) and b.pages == a.pages
    for bad in ([(3, [1])], [(0, [9])], [(0, [0])], [(0, [1] * 5)], [(-1, [])]):
        with pytest.raises(ValueError):
            b.apply_changes(bad)
