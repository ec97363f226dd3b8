"""AdamW without a GPU: what the list, the step and the optimizer refuse, the oracle's arithmetic against hand-computed values and
torch's, the 8-bit format, and a train step of the engine on the oracle backend."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from downscaling.engine import native
from oracle.torch_backend import TorchOps


@pytest.fixture(scope="module")
def ops():
    """The HIP backend's argument checks on CPU tensors: nothing that passes them is called here."""
    from downscaling.engine.hipops import HipOps
    o = object.__new__(HipOps)
    o.device, o.lib = torch.device("cpu"), native.load()
    return o


def entry(n=10, p=torch.float32, g=torch.float32, copy=None):
    return (torch.zeros(n, dtype=p), torch.zeros(n, dtype=g), 1.0) + ((torch.zeros(n, dtype=copy),) if copy else ())


@pytest.mark.parametrize("bad", [
    (torch.zeros(10, dtype=torch.float64), torch.zeros(10), 1.0), (torch.zeros(10), torch.zeros(11), 1.0), (torch.zeros(20)[::2], torch.zeros(10), 1.0),
    (torch.zeros(10), torch.zeros(20)[::2], 1.0), (torch.zeros(10), torch.zeros(10, dtype=torch.int32), 1.0), (torch.zeros(10), torch.zeros(10), 1.0, torch.zeros(10)),
    (torch.zeros(10), torch.zeros(10), 1.0, torch.zeros(9, dtype=torch.bfloat16)), (torch.zeros(10), torch.zeros(10)), (torch.zeros(10), None, 1.0),
    (torch.zeros(10), torch.zeros(10), torch.ones(1)), (torch.zeros(10), torch.zeros(10), 1.0, None, None), (torch.zeros(10, device="meta"), torch.zeros(10), 1.0),
])
def test_list_refuses(ops, bad):
    with pytest.raises(ValueError):
        ops.make_adamw([entry(), bad])


def test_list_refuses_overlap_and_values(ops):
    p, g, d = entry()
    for second in ((p, torch.zeros(10), d), (torch.zeros(10), p, d), (p[5:], torch.zeros(5), d)):
        with pytest.raises(native.NativeError, match="overlap"):
            ops.make_adamw([(p, g, d), second])
    with pytest.raises(native.NativeError, match="overlap"):
        ops.make_adamw([(p, p, d)])
    m = torch.zeros(256)
    with pytest.raises(native.NativeError, match="overlap"):
        ops.make_adamw([(p, g, d)], state=(m, m))
    for decay in (-1.0, float("nan"), float("inf")):
        with pytest.raises(native.NativeError, match="decay"):
            ops.make_adamw([(p, g, decay)])
    with pytest.raises(ValueError, match="32 or 8"):
        ops.make_adamw([(p, g, d)], state_bits=16)
    for state in ((m,), (m, torch.zeros(255)), (m, torch.zeros(256, dtype=torch.float64))):
        with pytest.raises(ValueError, match="state"):
            ops.make_adamw([(p, g, d)], state=state)
    with pytest.raises(ValueError, match="state"):
        ops.make_adamw([(p, g, d)], state_bits=8, state=(m, m.clone()))


def test_c_entries_refuse():
    lib, h, base = native.load(), C.c_void_p(), 1 << 20      # (addresses are never read)
    ok = dict(p=base, g=2 * base, m=3 * base, v=4 * base, m_scale=5 * base, v_scale=6 * base, copy=0, n=1000, p_type=0, g_type=0, copy_type=0, decay=1.0)

    def create(bits=32, n=1, **change):
        arr = (native.AdamWTensor * 1)(native.AdamWTensor(*{**ok, **change}.values()))
        return lib.wdg_adamw_create(C.byref(h), arr, n, bits)
    for change in (dict(n=-1), dict(p=0), dict(g=0), dict(m=0), dict(v=0), dict(p_type=3), dict(g_type=-1), dict(copy=7 * base, copy_type=0), dict(p=base + 2),
                   dict(g=2 * base + 1), dict(m=3 * base + 2), dict(copy=7 * base + 1, copy_type=1), dict(g=base + 3996)):
        assert create(**change) == -1, change
    assert create(bits=8, m_scale=0) == -1 and create(bits=16) == -1
    # 8-bit codes span whole blocks: 1000 elements hold 1024 bytes
    assert create(bits=8, v=3 * base + 1000) == -1
    assert lib.wdg_adamw_create(None, None, 0, 32) == -1 and lib.wdg_adamw_create(C.byref(h), None, 1, 32) == -1
    args = native.AdamWArgs(1e-3, .9, .999, 1e-8, .01, 1.0, 0.0, 1, 0, 0)
    assert lib.wdg_adamw_step(None, C.byref(args), 0, 0, 0) == -1
    for bits in (32, 8):
        assert create(bits=bits) == 0 and lib.wdg_adamw_table_bytes(h) > 0
        assert lib.wdg_adamw_step(h, C.byref(args), 0, 0, 0) == -1 and b"bind" in lib.wdg_last_error()      # no table yet
        assert lib.wdg_adamw_bind(h, None, 0, None) == -1
        assert lib.wdg_adamw_destroy(h) == 0
    # an empty list needs no table: its step checks its numbers and launches nothing
    assert lib.wdg_adamw_create(C.byref(h), None, 0, 32) == 0 and lib.wdg_adamw_table_bytes(h) == 0
    assert lib.wdg_adamw_step(h, C.byref(args), 0, 0, 0) == 0
    for field, value in (("lr", -1.0), ("lr", math.nan), ("beta1", 1.0), ("beta1", -0.1), ("beta2", 1.0), ("beta2", math.nan), ("eps", -1e-9), ("eps", math.inf),
                         ("weight_decay", -1.0), ("grad_scale", math.nan), ("grad_scale", -1.0), ("max_norm", math.nan), ("max_norm", math.inf), ("step", 0)):
        a = native.AdamWArgs(1e-3, .9, .999, 1e-8, .01, 1.0, 0.0, 1, 0, 0)
        setattr(a, field, value)
        assert lib.wdg_adamw_step(h, C.byref(a), 0, 0, 0) == -1, field
    a = native.AdamWArgs(1e-3, .9, .999, 1e-8, .01, 1.0, 1.0, 1, 0, 0)
    assert lib.wdg_adamw_step(h, C.byref(a), 0, 0, 0) == -2
    assert lib.wdg_adamw_grad_norm(h, 1.0, 0, 0, 0, 0) == -1 and lib.wdg_adamw_grad_norm(h, math.nan, base, base, 4096, 0) == -1
    assert lib.wdg_adamw_grad_norm(h, 1.0, base, base, 8, 0) == -2
    assert lib.wdg_adamw_destroy(h) == 0 and lib.wdg_adamw_destroy(None) == 0
    assert lib.wdg_adamw_moments(0, 0, 0, 0, 0, base, base, 0, 0) == 0 and lib.wdg_adamw_moments(0, 0, 0, 0, 4, 0, 0, 0, 0) == 0
    assert lib.wdg_adamw_moments(0, base, base, base, 4, base, 0, 0, 0) == -1 and lib.wdg_adamw_moments(base, base, base, base, 4, base, 0, 3, 0) == -1
    assert lib.wdg_adamw_moments(base, base, base, base, -1, base, 0, 0, 0) == -1


def test_oracle_known_answers():
    """One element: g = 0.5, first step: m_hat = g, v_hat = g^2, so p moves by lr g / (|g| + eps) after its decay; clipping halves g."""
    o = TorchOps()
    p, g = torch.tensor([2.0], dtype=torch.float64), torch.tensor([0.5], dtype=torch.float64)
    b = o.make_adamw([(p, g, 1.0)])
    b.step(1, 0.1, 0.9, 0.99, 0.1, 0.2)
    assert abs(float(p) - (2.0 * (1 - 0.02) - 0.1 * 0.5 / 0.6)) < 1e-12
    q, n = torch.tensor([2.0], dtype=torch.float64), torch.zeros(1)
    o.make_adamw([(q, g, 0.0)]).step(1, 0.1, 0.9, 0.99, 0.1, 0.2, max_norm=0.25, norm=n)
    assert abs(float(q) - (2.0 - 0.1 * 0.25 / 0.35)) < 1e-12 and float(n) == 0.5


def test_oracle_against_torch():
    gen = torch.Generator().manual_seed(1)
    ws = [torch.randn(s, generator=gen, dtype=torch.float64) for s in (7, 300)]
    gs = [torch.zeros_like(w) for w in ws]
    par = [torch.nn.Parameter(w.clone()) for w in ws]
    opt = torch.optim.AdamW(par, lr=1e-2, betas=(0.8, 0.95), eps=1e-6, weight_decay=0.1)
    b = TorchOps().make_adamw([(w, g, 1.0) for w, g in zip(ws, gs)])
    for t in range(1, 6):
        for g, q in zip(gs, par):
            g.copy_(torch.randn(g.shape, generator=gen, dtype=torch.float64))
            q.grad = g.clone()
        torch.nn.utils.clip_grad_norm_(par, 3.0)
        opt.step()
        b.step(t, 1e-2, 0.8, 0.95, 1e-6, 0.1, max_norm=3.0)
    # (torch's clipping divides by norm + 1e-6)
    assert all(float((w - q.detach()).abs().max()) < 1e-6 for w, q in zip(ws, par))


def test_eight_bit_format():
    """Every code survives decoding and encoding; the value an element decodes to is the nearest on the companded scale; a second
    moment above zero never reads as zero; zero blocks stay zero, blocks that are not finite turn NaN."""
    o = TorchOps()
    b = o.make_adamw([(torch.zeros(512, dtype=torch.float64), torch.zeros(512, dtype=torch.float64), 0.0)], state_bits=8)
    b.m[:255] = torch.arange(-127, 128, dtype=torch.int16).to(torch.int8)
    b.m[255] = 5
    b.v[:256] = torch.arange(256, dtype=torch.int16).to(torch.uint8)
    b.m_scale.fill_(0.03)
    b.v_scale.fill_(2e-5)
    m, v = b.values()
    for x, code, second in ((m, b.m, False), (v, b.v, True)):
        q, top = b.encode(x, second)
        assert torch.equal(q, code) and (top[1] == 0) and abs(float(top[0]) / (2e-5 if second else 0.03) - 1) < 1e-12
    tiny = torch.zeros(256, dtype=torch.float64)
    tiny[0], tiny[1] = 1.0, 1e-30
    assert b.encode(tiny, True)[0].tolist()[:3] == [255, 1, 0] and b.encode(tiny, False)[0].tolist()[:3] == [127, 0, 0]
    tiny[2] = float("inf")
    assert b.encode(tiny, True)[1].isnan().all() and b.encode(tiny, False)[0].abs().max() <= 127


def test_optimizer_refuses_and_defaults():
    from downscaling.engine.trainer import AdamW
    from downscaling.gan import train
    assert train.AdamW is AdamW
    for bad in (dict(beta_1=1.0), dict(beta_2=-0.1), dict(epsilon=-1.0), dict(weight_decay=-1.0), dict(state_bits=16), dict(global_clipnorm=0.0)):
        with pytest.raises(ValueError):
            AdamW(**bad)
    o = AdamW(learning_rate=3e-4)
    assert o.lr == 3e-4 and o.decays("layer_with_weights-0/layer/w") and o.decays("a/cell/recurrent_kernel") and o.decays("a/kernel")
    assert not any(o.decays(n) for n in ("a/bias", "a/gamma", "a/beta", "layer/layer/bias"))


@pytest.mark.parametrize("bits", [32, 8])
def test_engine_train_step_on_the_oracle(bits):
    """GanEngine.train_step drives AdamW as it drives AdamTF: weights move, biases are not decayed, the norm is kept."""
    from downscaling.engine.networks import DiscriminatorNet, GeneratorNet
    from downscaling.engine.trainer import AdamW, GanEngine, PhiloxSource
    ops = TorchOps()
    gen, disc = GeneratorNet(ops, 32, 3, 4, 2, 1, feature_channels=16, seed=5), DiscriminatorNet(ops, 32, 32, 3, 2, 1, feature_channels=8, seed=6)
    g = torch.Generator().manual_seed(0)
    low, high = (torch.randn(2, 1, 32, 32, c, generator=g, dtype=torch.float64) for c in (3, 2))
    before = {n: w.copy() for n, w in gen.params.get_weights().items()}
    go, do = AdamW(1e-3, global_clipnorm=0.5, state_bits=bits), AdamW(1e-3, weight_decay=0.0, state_bits=bits)
    GanEngine(gen, disc, PhiloxSource(ops, seed=9), noise_std=0.1, n_critic=1).train_step(low, high, go, do)
    assert go.iterations == do.iterations == 1 and float(go.grad_norm) > 0 and do.grad_norm is None
    after = gen.params.get_weights()
    moved = [n for n in before if np.abs(after[n] - before[n]).max() > 0]
    assert any(n.endswith("/w") for n in moved) and any(n.endswith("bias") for n in moved)
    with pytest.raises(ValueError, match="another network"):
        go.apply_gradients(disc.params)
