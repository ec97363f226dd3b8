"""The clipped step's decision on a norm that is not finite is the one that the norm it hands out shows (csrc/adamw.hip)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [300, 20000], ids=["norm in the step's launch", "norm before it"])
@pytest.mark.parametrize("bits", [32, 8])
def test_norm_beyond_fp32(bits, n, hip_ops):
    """Gradients of 2^126: each of them is a number, their norm is above fp32's largest.  The caller reads infinity, so nothing has changed;
    scaled back into range the same gradients make a step."""
    p, g = torch.ones(n, device="cuda"), torch.full((n,), 2.0 ** 126, device="cuda")
    b = hip_ops.make_adamw([(p, g, 0.0)], state_bits=bits)
    norm = torch.zeros(1, device="cuda")
    b.step(1, 0.5, max_norm=1.0, norm=norm)
    assert norm.isinf().all() and (p == 1).all() and all((s == 0).all() for s in b.state)
    b.step(1, 0.5, max_norm=1.0)                          # the same without handing it out
    assert (p == 1).all() and all((s == 0).all() for s in b.state)
    b.step(1, 0.5, grad_scale=2.0 ** -20, max_norm=1.0, norm=norm)
    assert abs(float(norm) - 2.0 ** 106 * n ** 0.5) <= 2.0 ** -22 * float(norm)
    assert ((p - 0.5).abs() <= 1e-5).all()                  # the first step moves by lr g / (|g| + eps), with |g| = n^-0.5 after clipping


def test_the_oracle_decides_alike():
    from oracle.torch_backend import TorchOps
    p, g = torch.ones(300, dtype=torch.float64), torch.full((300,), 2.0 ** 126, dtype=torch.float64)
    norm = torch.zeros(1)
    b = TorchOps().make_adamw([(p, g, 0.0)])
    b.step(1, 0.5, max_norm=1.0, norm=norm)
    assert norm.isinf().all() and (p == 1).all()
