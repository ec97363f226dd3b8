"""HipOps.concurrent_streams measures the streams, not the host: a host that is slow to enqueue finds the same streams."""
import os
import time

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("host_us", [0, 100])
def test_streams_are_found_on_a_slow_host(host_us, monkeypatch):
    if os.environ.get("GPU_MAX_HW_QUEUES", "4") in ("1", "2", "3"):
        pytest.skip("fewer than four hardware queues by configuration")
    from downscaling.engine.hipops import HipOps
    ops, sleep = HipOps("cuda:0"), torch.cuda._sleep

    def slow(cycles):
        until = time.perf_counter() + host_us * 1e-6
        while time.perf_counter() < until:
            pass
        sleep(cycles)
    monkeypatch.setattr(torch.cuda, "_sleep", slow)
    streams = ops.concurrent_streams(3)
    print(ops._cstreams_probe, flush=True)
    assert ops._cstreams_probe["concurrent_found"] == 3
    assert len({s.cuda_stream for s in streams} | {torch.cuda.current_stream().cuda_stream}) == 4
