"""AdamW at the list sizes that take the other two step kernels: chunks of 1024 streamed past the cache (96 MiB and more in fewer than 16 M
elements) and chunks of 4096 that are not (thousands of short tensors), and a train step whose decay is larger than its tolerance.
Tolerances: those of test_adamw_gpu.py."""
import pytest
import torch

from tests.test_adamw_gpu import BF16, F16, F32, make, step_close

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,sizes,types", [
    (32, [8000001, 77], (F32, F32, None)),
    (32, [7000003, 1 << 20, 5], (F32, F32, BF16)),
    (8, [12000001, 77], (F32, F32, None)),
    (8, [12000001, 1 << 20, 5], (F32, BF16, F16)),
], ids=str)
def test_streamed_short_chunks(bits, sizes, types, hip_ops):
    p, g, copy = types
    b, buffers = make(hip_ops, sizes, p, g, copy, bits, seed=31, shift=1)
    held = sum(sizes) * ((12 if bits == 32 else 6) + (4 if g is F32 else 2) + (2 if copy else 0))
    assert held >= 96 << 20 and sum(-(-n // 4096) for n in sizes) < 4096
    step_close(b, 3)
    norm = torch.zeros(1, device="cuda")
    step_close(b, 4, grad_scale=0.5, max_norm=0.5, norm=norm)
    for buf, s, n in buffers:
        assert (buf[:s] == 7).all() and (buf[s + n:] == 7).all()


@pytest.mark.parametrize("types", [(F32, F32, None), (F32, BF16, BF16), (F16, F16, None)], ids=lambda t: "-".join(str(x).replace("torch.", "") for x in t))
@pytest.mark.parametrize("bits", [32, 8])
def test_thousands_of_short_tensors(bits, types, hip_ops):
    p, g, copy = types
    sizes = [1 + (i * 37) % 300 for i in range(4199)] + [4096, 5000]
    b, buffers = make(hip_ops, sizes, p, g, copy, bits, seed=32)
    step_close(b, 3)
    norm = torch.zeros(1, device="cuda")
    step_close(b, 4, grad_scale=0.5, max_norm=0.5, norm=norm)
    for buf, s, n in buffers:
        assert (buf[:s] == 7).all() and (buf[s + n:] == 7).all()
    assert sum(-(-n // 4096) for n in sizes) >= 4096


def test_table_is_refused_while_capturing(hip_ops):
    """A batch cannot be made inside a capture, and the optimizer does not count steps inside one: both say so themselves, and the capture
    goes on."""
    from downscaling.engine.trainer import AdamW
    p, g, out = torch.zeros(10, device="cuda"), torch.ones(10, device="cuda"), torch.zeros(10, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out.add_(g)
        with pytest.raises(RuntimeError, match="while a graph is captured"):
            hip_ops.make_adamw([(p, g, 1.0)])
        with pytest.raises(RuntimeError, match="counts its steps on the host"):
            AdamW().apply_gradients(None)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
    assert (out == 3).all() and (p == 0).all()


def test_step_refusals_name_their_reason(hip_ops):
    from downscaling.engine.native import NativeError
    b, _ = make(hip_ops, [100])
    for bad, why in ((dict(t=0), "count from 1"), (dict(t=1, lr=-1.0), "not negative"), (dict(t=1, beta1=1.0), "beta1 and beta2"), (dict(t=1, eps=float("inf")), "finite")):
        with pytest.raises(NativeError, match=why):
            b.step(**{"lr": 1e-3, **bad})


def test_train_step_decays_what_it_should():
    """One train step of both networks with lr * weight_decay = 5e-3, fifty times the tolerance, against the same step on the 64-bit backend:
    the kernels are decayed, and nothing else is."""
    from downscaling.engine.hipops import HipOps
    from tests.test_adamw_decay_cpu import train_step_weights
    from tests.helpers import rel_err
    got, want = train_step_weights(HipOps("cuda:0")), train_step_weights()
    for a, b in zip(got, want):
        assert max(rel_err(a[k], b[k]) for k in b) < 1e-4
