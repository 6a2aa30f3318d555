"""A windowed decoder split over 2 gloo ranks (context parallel, Ulysses, tensor parallel) against the unsplit one."""

import os
import socket
from dataclasses import replace

import pytest
import torch
import torch.multiprocessing as mp


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _worker(rank, world, port, q, kind):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(rank), WORLD_SIZE=str(world),
                      LOCAL_RANK=str(rank))
    import torch.distributed as dist
    torch.set_num_threads(1)
    from psrl_b200.models import PRESETS, build_model, packed_positions
    a = replace(PRESETS["tiny"], sliding_window=7, attention_sinks=2, window_from_layer=1)
    lens = [13, 29, 6]
    T = sum(lens)
    g = torch.Generator().manual_seed(11)
    ids = torch.randint(0, a.vocab_size, (T,), generator=g)
    labels = torch.randint(0, a.vocab_size, (T,), generator=g)
    wts = torch.randn(T, generator=g)
    pos, cu, mx = packed_positions(lens, "cpu")
    if kind == "tp":
        from psrl_b200.config import load_config
        from psrl_b200.parallel.dist import init_distributed
        from psrl_b200.trainer.actor import PolicyWorker
        init_distributed("cpu", timeout_s=300)
        cfg = load_config(preset="cpu_tiny_grpo")
        full = PolicyWorker(cfg, a, "cpu", seed=3).model
        split = PolicyWorker(cfg, a, "cpu", seed=3, tp_group=dist.group.WORLD).model
        x, y = (m.hidden_states(ids, pos, cu, mx).detach() for m in (full, split))
        q.put({"out": float((x - y).abs().max() / x.abs().max()), "grad": 0.0})
        dist.destroy_process_group()
        return
    dist.init_process_group("gloo", rank=rank, world_size=world)
    model = build_model(a, "cpu", torch.float32, seed=5)
    lp_full, _ = model.logprobs(ids, pos, cu, mx, labels)
    (lp_full * wts).sum().backward()
    ref = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad(set_to_none=True)
    if kind == "ulysses":
        from psrl_b200.parallel.ulysses import UlyssesShard as Shard
    else:
        from psrl_b200.parallel.cp import CPShard as Shard
    sh = Shard(cu, dist.group.WORLD)
    lp, _ = model.logprobs(sh.local(ids), sh.positions(), sh.plan, sh.plan.max_q, sh.local(labels))
    (lp * sh.local(wts, 0.0)).sum().backward()
    worst = 0.0
    for n, p in model.named_parameters():
        s = p.grad.clone()
        dist.all_reduce(s)
        worst = max(worst, float((s - ref[n]).abs().max() / (ref[n].abs().max() + 1e-12)))
    q.put({"out": float((sh.full(lp.detach()) - lp_full.detach()).abs().max()), "grad": worst})
    dist.destroy_process_group()


@pytest.mark.parametrize("kind", ["cp", "ulysses", "tp"])
def test_windowed_model_split_over_ranks(kind):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, 2, port, q, kind)) for r in range(2)]
    for p in procs:
        p.start()
    res = [q.get(timeout=300) for _ in procs]
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    # fp32 sums in another order: 2^-24 times a few hundred terms
    for r in res:
        assert r["out"] < 1e-4 and r["grad"] < 1e-4, r
