"""AdamW under data parallelism (two gloo ranks on the 64-bit backend): the gradients are clipped by the norm of their mean over the
ranks, and the replicas stay the same bits."""
import os
import socket
import tempfile

import pytest
import torch
import torch.multiprocessing as mp

WORLD, S = 2, 12


def _worker(rank, port, outdir, bits):
    import torch.distributed as dist
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    dist.init_process_group("gloo", rank=rank, world_size=WORLD)
    torch.set_num_threads(2)
    from downscaling.engine.networks import DiscriminatorNet, GeneratorNet
    from downscaling.engine.trainer import AdamW, DistSync, GanEngine, PhiloxSource
    from oracle.torch_backend import TorchOps
    ops = TorchOps()
    gen, disc = GeneratorNet(ops, S, 3, 2, 2, 1, feature_channels=32, seed=5), DiscriminatorNet(ops, S, S, 3, 2, 1, feature_channels=8, seed=6)
    eng = GanEngine(gen, disc, PhiloxSource(ops, seed=99, rank=rank), 0.1, n_critic=1, sync=DistSync())
    go, do = AdamW(1e-3, global_clipnorm=0.1, state_bits=bits), AdamW(1e-3, global_clipnorm=0.1, state_bits=bits)
    g = torch.Generator().manual_seed(100 + rank)
    for _ in range(2):
        eng.train_step(*(torch.randn(1, 1, S, S, c, generator=g, dtype=torch.float64) for c in (3, 2)), go, do)
    for net in (gen, disc):
        eng._flush(net)
    torch.save({"w": [net.params.flat.clone() for net in (gen, disc)], "norm": [float(o.grad_norm) for o in (go, do)],
                "mean": [float(net.params.grads.norm()) / WORLD for net in (gen, disc)], "steps": [go.iterations, do.iterations]}, os.path.join(outdir, f"rank{rank}.pt"))
    dist.destroy_process_group()


@pytest.mark.timeout(300)
@pytest.mark.parametrize("bits", [32, 8])
def test_two_ranks_clip_the_mean_gradient(bits):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    with tempfile.TemporaryDirectory() as out:
        mp.spawn(_worker, args=(port, out, bits), nprocs=WORLD, join=True)
        a, b = (torch.load(os.path.join(out, f"rank{i}.pt")) for i in range(WORLD))
    assert a["steps"] == b["steps"] == [2, 2] and a["norm"] == b["norm"]
    assert all(torch.equal(x, y) for x, y in zip(a["w"], b["w"]))
    assert abs(a["norm"][0] - a["mean"][0]) < 1e-12 * a["mean"][0]      # the generator's last gradients are still there
