"""What a comparison of weights after an AdamW train step can see: on the 64-bit backend a step without decay, and one that decays every
variable, differ from the right one by far more than the tolerance of the comparison (1e-4)."""
import torch

from tests.helpers import randomize, rel_err, weights64


def train_step_weights(ops=None, weight_decay=5.0, decays=None):
    """({name: weights} of the generator, of the discriminator) after one train step of small networks, lr = 1e-3."""
    from downscaling.engine.networks import DiscriminatorNet, GeneratorNet
    from downscaling.engine.trainer import AdamW, GanEngine, PhiloxSource
    from oracle.torch_backend import TorchOps
    cv = (lambda t: t) if ops is None else (lambda t: t.float().to(ops.device))
    ops = ops or TorchOps()
    S, T = 32, 1
    g = torch.Generator().manual_seed(0)
    low, high = (torch.randn(2, T, S, S, c, generator=g, dtype=torch.float64) for c in (3, 2))
    gen, disc = GeneratorNet(ops, S, 3, 4, 2, T, feature_channels=32, seed=5), DiscriminatorNet(ops, S, S, 3, 2, T, feature_channels=8, seed=6)
    randomize(gen, 21), randomize(disc, 22)
    # (epsilon as the networks' own optimizers: the update stays a smooth function of the gradient where that is near zero)
    go, do = (AdamW(1e-3, 0.5, 0.9, 0.1, weight_decay=weight_decay, global_clipnorm=clip, decays=decays) for clip in (0.5, None))
    GanEngine(gen, disc, PhiloxSource(ops, seed=99), noise_std=0.1, n_critic=1).train_step(cv(low), cv(high), go, do)
    return weights64(gen), weights64(disc)


def test_a_wrong_decay_is_seen():
    right = train_step_weights()
    for wrong in (train_step_weights(weight_decay=0.0), train_step_weights(decays=lambda name: True), train_step_weights(weight_decay=4.5)):
        for a, b in zip(wrong, right):
            assert max(rel_err(a[k], b[k]) for k in b) > 3e-4
