"""What layernorm_fwd / layernorm_bwd refuse, and the oracle's gradients against differences.  No GPU: refused calls never launch."""
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


def args(P=6, C=10, dtype=torch.float32):
    return dict(x=torch.zeros(P, C, dtype=dtype), gamma=torch.ones(C), beta=torch.zeros(C), eps=1e-3, z=torch.zeros(P, C, dtype=dtype),
                mean_rstd=torch.zeros(P, 2))


@pytest.mark.parametrize("change", [
    dict(x=torch.zeros(6, 10, dtype=torch.float64)), dict(x=torch.zeros(60)), dict(z=torch.zeros(6, 9)), dict(z=torch.zeros(6, 10, dtype=torch.bfloat16)),
    dict(z=torch.zeros(1, 10).expand(6, 10)), dict(x=torch.zeros(10, 6).t()), dict(gamma=torch.ones(9)), dict(gamma=torch.ones(20)[::2]),
    dict(gamma=torch.ones(10, dtype=torch.float16)), dict(beta=torch.zeros(10, dtype=torch.float64)), dict(mean_rstd=torch.zeros(6, 3)),
    dict(mean_rstd=torch.zeros(6, 2, dtype=torch.float64)), dict(mean_rstd=torch.zeros(5, 2)), dict(x=torch.zeros(6, 0), z=torch.zeros(6, 0)),
    dict(x=torch.zeros(6, 10, device="meta")),
])
def test_forward_refuses(ops, change):
    with pytest.raises(ValueError):
        ops.layernorm_fwd(**{**args(), **change})


def test_forward_refuses_overlap(ops):
    buf = torch.zeros(6, 24)
    with pytest.raises(ValueError, match="overlaps"):
        ops.layernorm_fwd(**{**args(), "x": buf[:, :10], "z": buf[:, 5:15]})
    with pytest.raises(ValueError, match="overlaps"):
        ops.layernorm_fwd(**{**args(), "x": buf[:, :10], "z": buf.view(-1)[1:61].view(6, 10)})
    h = torch.zeros(6, 10, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="one type"):
        ops.layernorm_fwd(**{**args(), "x": h, "z": torch.zeros_like(h), "gamma": torch.ones(10, dtype=torch.bfloat16)})
    rows = lambda t: ops._ln_rows("x", t, t)      # noqa: E731
    for a, b in ((buf[:, :10], buf[:, 10:20]), (buf[:, 14:24], buf[:, :10]), (buf[:, :10], buf[:, 14:]), (buf[:3], buf[3:]), (buf, buf)):      # two halves of a concatenation
        ops._ln_apart("z", rows(a), {"x": rows(b)}, a.shape[1], 4)
    for a, b in ((buf[:, :10], buf[:, 9:19]), (buf[:, 9:19], buf[:, :10]), (buf[:3, 1:], buf[2:5, 1:])):
        with pytest.raises(ValueError, match="overlaps"):
            ops._ln_apart("z", rows(a), {"x": rows(b)}, a.shape[1], 4)


@pytest.mark.parametrize("change", [
    dict(dz=torch.zeros(6, 9)), dict(dz=torch.zeros(6, 10, dtype=torch.float16)), dict(mean_rstd=None), dict(mean_rstd=torch.zeros(12)),
    dict(dx=torch.zeros(1, 10).expand(6, 10)), dict(dgamma=torch.zeros(10, dtype=torch.bfloat16)), dict(dgamma=torch.zeros(11)),
    dict(dbeta=torch.zeros(20)[::2]), dict(gamma=torch.ones(10, 1)),
])
def test_backward_refuses(ops, change):
    a = dict(dz=torch.zeros(6, 10), x=torch.zeros(6, 10), mean_rstd=torch.zeros(6, 2), gamma=torch.ones(10), dx=torch.zeros(6, 10),
             dgamma=torch.zeros(10), dbeta=torch.zeros(10))
    with pytest.raises(ValueError):
        ops.layernorm_bwd(**{**a, **change})


def test_backward_refuses_overlap(ops):
    buf, vec = torch.zeros(6, 24), torch.zeros(16)
    a = dict(dz=torch.zeros(6, 10), x=buf[:, :10], mean_rstd=torch.zeros(6, 2), gamma=torch.ones(10), dx=buf[:, 4:14])
    with pytest.raises(ValueError, match="overlaps"):
        ops.layernorm_bwd(**a)
    with pytest.raises(ValueError, match="overlaps"):
        ops.layernorm_bwd(**{**a, "dx": torch.zeros(6, 10), "dgamma": vec[:10], "dbeta": vec[6:]})


def test_c_entries_refuse():
    lib = native.load()
    p = 1 << 20      # (never read: every call is refused)
    ok = dict(x=p, ldx=8, gamma=0, beta=0, eps=1e-3, z=2 * p, ldz=8, mr=0, P=4, C=8, type=0, ptype=0, stream=0)
    for change in (dict(type=3), dict(type=-1), dict(ptype=1), dict(type=1, ptype=2), dict(P=-1), dict(C=0), dict(C=(1 << 24) + 1), dict(x=0), dict(z=0),
                   dict(ldz=7), dict(ldx=-1), dict(x=p + 2), dict(type=1, z=2 * p + 1), dict(gamma=p + 1), dict(mr=p + 2), dict(eps=-1.0), dict(eps=float("nan"))):
        assert lib.wdg_layernorm_fwd(*{**ok, **change}.values()) == -1, change
        assert lib.wdg_last_error()
    assert lib.wdg_layernorm_fwd(*{**ok, "P": 0, "x": 0, "z": 0}.values()) == 0
    b = dict(dz=p, lddz=8, x=p, ldx=8, mr=p, gamma=0, dx=2 * p, lddx=8, dg=p, db=p, acc=0, P=4, C=8, type=0, ptype=0, ws=p, wsb=1 << 16, stream=0)
    for change in (dict(type=5), dict(ptype=2), dict(P=-2), dict(C=0), dict(dz=0), dict(mr=0), dict(dx=0), dict(lddx=5), dict(dg=p + 2), dict(ws=p + 1), dict(dz=p + 1), dict(gamma=p + 2)):
        assert lib.wdg_layernorm_bwd(*{**b, **change}.values()) == -1, change
    for change in (dict(ws=0), dict(wsb=4)):
        assert lib.wdg_layernorm_bwd(*{**b, **change}.values()) == -2, change
    assert lib.wdg_layernorm_bwd_ws_bytes(0, 8, 0) == 0 and lib.wdg_layernorm_bwd_ws_bytes(5, 0, 0) == 0
    assert lib.wdg_layernorm_bwd_ws_bytes(1, 8, 1) >= 2 * 8 * 4


@pytest.mark.parametrize("P,C", [(1, 5), (4, 3), (7, 32)])
def test_oracle_gradients_against_differences(P, C):
    """The oracle's dx, dgamma and dbeta against central differences of its forward pass, in 64 bits."""
    o, gen = TorchOps(), torch.Generator().manual_seed(P * C)
    r = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)      # noqa: E731
    x, gamma, beta, dz = r(P, C), 1 + 0.3 * r(C), r(C), r(P, C)

    def loss(x, gamma, beta):
        z = torch.empty(P, C, dtype=torch.float64)
        o.layernorm_fwd(x, gamma, beta, 1e-3, z)
        return float((z * dz).sum())
    mr, dx, dg, db = (torch.empty(*s, dtype=torch.float64) for s in ((P, 2), (P, C), (C,), (C,)))
    o.layernorm_fwd(x, gamma, beta, 1e-3, torch.empty(P, C, dtype=torch.float64), mr)
    o.layernorm_bwd(dz, x, mr, gamma, dx, dg, db, accumulate=False)
    h = 1e-5
    for which, grad in enumerate((dx, dg, db)):
        way = r(*grad.shape)
        a = [x, gamma, beta]
        up, down = list(a), list(a)
        up[which], down[which] = a[which] + h * way, a[which] - h * way
        slope = (loss(*up) - loss(*down)) / (2 * h)
        assert abs(slope - float((grad * way).sum())) < 1e-6 * (1 + abs(slope))
