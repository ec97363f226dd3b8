"""8-bit second moments at the low end of fp32 (csrc/adamw.hip): one that is above zero never reads as zero, so that an update without an
epsilon divides by none."""
import pytest
import torch

pytestmark = pytest.mark.gpu
FLOOR = 2.0 ** -94      # the smallest scale of a block that holds any second moment: code 1 of it is still a normal number


@pytest.mark.parametrize("name,grads", [
    ("one size", [2.0 ** -57] * 256),                                              # block maximum near 2^-121
    ("far apart", [2.0 ** 20] + [2.0 ** -60] * 255),                                 # quotient to the block's maximum below 2^-149
    ("subnormal", [2.0 ** -69, 2.0 ** -68] * 128),                                   # the moments themselves below 2^-126
    ("a wide range", [2.0 ** -k for k in range(30, 62)] * 8),
    ("ordinary", [1e-3, 1e-4, 1e-5, 3e-8] * 64),
], ids=lambda x: x if isinstance(x, str) else "")
def test_second_moment_never_reads_as_zero(name, grads, hip_ops):
    g = torch.tensor(grads, device="cuda")
    g[7] = 0.0
    p = torch.ones(256, device="cuda")
    b = hip_ops.make_adamw([(p, g, 0.0)], state_bits=8)
    h = dict(lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-30)
    b.step(1, **h)
    m, v = torch.empty(256, device="cuda"), torch.empty(256, device="cuda")
    b.moments(m, v)
    # the second moment as fp32 holds it: zero where the square is below half of fp32's smallest number
    want = torch.tensor(1 - 0.99, dtype=torch.float64).float().cuda() * (g * g)
    some = want > 0
    assert some.sum() == 255 and (v[some] > 0).all() and v[7] == 0 and (v[some] >= torch.finfo(torch.float32).tiny).all()
    # the value that is read is the one of the nearest code, 1 at least
    top = max(float(want.max()), FLOOR)
    code = 255 * (want.double() / top) ** 0.25
    read = 255 * (v.double() / top) ** 0.25
    off = (read - code.clamp(min=1.0)).abs()
    assert (off[some] <= 0.5 + 2e-4).all(), float(off[some].max())
    # moments that are left without a gradient move their weights by a number
    g.zero_()
    for t in (2, 3, 4):
        b.step(t, **{**h, "eps": 0.0})
    b.moments(m, v)
    held = torch.ones(256, dtype=torch.bool, device="cuda")
    held[7] = False                     # (0 / 0 without an epsilon, as the formula says)
    assert p[held].isfinite().all() and (v[held] > 0).all()


def test_blocks_without_moments_stay_zero(hip_ops):
    p, g = torch.ones(600, device="cuda"), torch.zeros(600, device="cuda")
    g[:256] = 2.0 ** -60
    b = hip_ops.make_adamw([(p, g, 0.0)], state_bits=8)
    b.step(1, 1e-3)
    assert (b.v[256:] == 0).all() and (b.v_scale[1:] == 0).all() and float(b.v_scale[0]) == FLOOR and (b.v[:256] >= 1).all()


@pytest.mark.parametrize("k", [-120, -110, -96, -94, -90])
def test_matches_the_oracle(k, hip_ops):
    """The same step on the 64-bit backend: codes differ by one at most, where a value lies on a border between two."""
    from oracle.torch_backend import TorchOps
    gen = torch.Generator().manual_seed(5)
    g = torch.randn(512, generator=gen) * 2.0 ** (k / 2)
    p = torch.ones(512)
    o = TorchOps().make_adamw([(p.double(), g.double(), 0.0)], state_bits=8)
    b = hip_ops.make_adamw([(p.cuda(), g.cuda(), 0.0)], state_bits=8)
    o.step(1, 1e-3, 0.9, 0.5)
    b.step(1, 1e-3, 0.9, 0.5)
    assert (b.v.cpu().int() - o.v.int()).abs().max() <= 1 and (b.m.cpu().int() - o.m.int()).abs().max() <= 1
    assert ((b.v_scale.cpu().double() - o.v_scale).abs() <= 1e-5 * o.v_scale).all() and (o.v_scale >= FLOOR).all()
