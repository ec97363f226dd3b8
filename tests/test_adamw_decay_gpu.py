"""The weight decay of an AdamW step where it is smaller than half a step of fp32 below one (csrc/adamw.hip)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("lr,decay", [(2e-6, 0.01), (4e-6, 0.01), (1e-5, 0.01)])
def test_small_decay_accumulates(lr, decay, bits, hip_ops):
    """2000 steps of 65536 weights between 1 and 2 with gradients of either sign: the mean of the weights drifts by what the 64-bit run says,
    lr decay sum of the weights — 6e-5 to 3e-4 here.

    Tolerance.  A step rounds a weight below 2 to 2^-24 at most, in either direction, as the updates move the weights over many steps of
    their grid: 2000 independent roundings of 2^-24 / sqrt(3) give 1.6e-6 per weight, and over 65536 weights a mean of 6e-9.  The updates differ
    from the 64-bit ones by 20 u of themselves (8-bit moments: by a few percent, of either sign with m): at most 2000 * 20 u * 0.5 lr = 1e-8
    for one weight with 32 bits; 2000 steps of 0.05 * 0.5 lr with a tenth of them left after their signs cancel, over sqrt(65536): below 1e-8.
    The product lr decay carries 2 u.  All together stay below 1e-7; a decay that is wrong by one part in a hundred is off by 5e-7 and more."""
    n, steps, pool = 65536, 2000, 61
    gen = torch.Generator(device="cuda").manual_seed(17)
    p = 1.25 + 0.5 * torch.rand(n, generator=gen, device="cuda")
    start, w = p.double(), p.double()
    grads = torch.randn(pool, n, generator=gen, device="cuda")
    g = torch.empty(n, device="cuda")
    b1, b2, eps = 0.9, 0.99, 1e-8
    m, v = torch.zeros_like(w), torch.zeros_like(w)
    b = hip_ops.make_adamw([(p, g, 1.0)], state_bits=bits)
    for t in range(1, steps + 1):
        g.copy_(grads[t % pool])
        b.step(t, lr, b1, b2, eps, decay)
        gg = grads[t % pool].double()
        m.mul_(b1).add_(gg, alpha=1 - b1)
        v.mul_(b2).addcmul_(gg, gg, value=1 - b2)
        w.mul_(1 - lr * decay).sub_(m / (torch.sqrt(v / (1 - b2 ** t)) + eps), alpha=lr / (1 - b1 ** t))
    off, drift = float((p.double() - w).mean()), float((w - start).mean())
    expected = lr * decay * steps * float(start.mean())
    print(lr, decay, bits, "drift", drift, "off", off, "of", expected, flush=True)
    assert abs(off) < 5e-7 and abs(off) < 0.02 * expected


@pytest.mark.parametrize("decay,lr", [(1.0, 0.01), (0.0, 0.01), (1.0, 0.5)])
def test_infinite_weights(decay, lr, hip_ops):
    """An infinite weight stays what the formula makes of it, inf (1 - lr weight_decay d) minus a number; a NaN stays one."""
    inf = math.inf
    p = torch.tensor([inf, -inf, math.nan, 3.0e38, -3.0e38, 1.0], device="cuda")
    g = torch.tensor([1.0, -1.0, 1.0, 0.5, 0.5, 0.0], device="cuda")
    b = hip_ops.make_adamw([(p, g, decay)])
    b.step(1, lr, 0.9, 0.99, 1e-3, 0.1)
    keep = 1 - lr * 0.1 * decay
    got = p.tolist()
    assert got[0] == inf and got[1] == -inf and math.isnan(got[2])
    for x, start in zip(got[3:], (3.0e38, -3.0e38, 1.0)):
        assert abs(x - start * keep) <= 2 * U * abs(start)
