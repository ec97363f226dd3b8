"""AdamW (csrc/adamw.hip) against the 64-bit formulas, one step at a time from the states that the kernel itself holds.

Tolerances, derived: u = 2^-24 is half a step of fp32.  g' = g gs carries 2 u; m = beta1 m + (1 - beta1) g' adds a rounding for each
constant, product and the sum: 6 u of the terms' magnitudes (8-bit states: 4 u more for the decoded value).  v likewise 10 u of itself (all
its terms are positive; 8-bit: 8 u more).  The update lr / bc1 m / (sqrt(v) rbc2 + eps) adds half of v's relative error, and 8 u for the
constants, root, sum, quotient and product.  p keeps 4 u of itself for the decay and half a step of its own type.
An 8-bit code c = 127 sqrt(|m| / M) (or 255 (v / V)^(1/4)) may miss the nearest integer by what the error of m moves it, and 6 u of
itself for the roots (one unit in the last place each, halved again by the roots that follow) and the product."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HYPER = dict(lr=2e-3, beta1=0.9, beta2=0.99, eps=1e-6, weight_decay=0.1)
SIZES = {"one": [1], "nine small ones": [300] * 9, "around a block": [3, 255, 256, 257, 513], "around a chunk": [4095, 4096, 4097, 12288, 1], "with empty ones": [0, 5, 0, 700, 0], "ragged": [70001, 33, 2, 9000]}


def make(ops, sizes, p=F32, g=F32, copy=None, bits=32, seed=0, shift=0, spread=True, zero=False):
    """(batch, buffers): every tensor `shift` elements into a buffer of its own, with 7s around it."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    buffers, entries = [], []
    for i, n in enumerate(sizes):
        size = math.exp(-3 + (i % 4)) if spread else 1.0
        made = []
        for kind, scale in ((p, 0.5), (g, size), (copy, 0.0)):
            if kind is None:
                continue
            buf = torch.full((n + shift + 8,), 7.0, dtype=kind, device="cuda")
            v = buf[shift:shift + n]
            v.copy_(torch.randn(n, generator=gen, device="cuda") * scale * (torch.exp(torch.randn(n, generator=gen, device="cuda")) if spread and kind is g else 1))
            buffers.append((buf, shift, n))
            made.append(v)
        entries.append((made[0], made[1], float(i % 3 != 1)) + tuple(made[2:]))
    b = ops.make_adamw(entries, state_bits=bits)
    if not zero:                                     # moments as earlier steps leave them
        r = lambda: torch.randn(b.total, generator=gen, device="cuda")      # noqa: E731
        if bits == 32:
            b.m.copy_(0.1 * r())
            b.v.copy_(r().square() * torch.exp(r()) * 0.01)
        else:
            b.m.copy_(torch.randint(-127, 128, (b.total,), generator=gen, device="cuda"))
            b.v.copy_(torch.randint(0, 256, (b.total,), generator=gen, device="cuda"))
            b.m_scale.copy_(torch.rand(b.total // 256, generator=gen, device="cuda") * 0.2)
            b.v_scale.copy_(torch.rand(b.total // 256, generator=gen, device="cuda") * 0.02)
            for o, n in zip(b.offsets, sizes):       # behind a tensor's end a block holds zeros
                end = o + -(-n // 256) * 256
                b.m[o + n:end] = 0
                b.v[o + n:end] = 0
    return b, buffers


def values(b):
    if b.state_bits == 32:
        return b.m.double(), b.v.double()
    q, c = b.m.double(), b.v.double()
    return q * q.abs() / 127.0 ** 2 * b.m_scale.double().repeat_interleave(256), (c / 255.0) ** 4 * b.v_scale.double().repeat_interleave(256)


def check_codes(code, x, tol, levels, power, n):
    """8-bit codes of a tensor's values x (64-bit, `tol` off at most), whole blocks; returns nothing, asserts."""
    full = torch.zeros(-(-n // 256) * 256, dtype=torch.float64, device=x.device)
    full[:n], t = x.abs(), torch.zeros_like(full)
    t[:n] = tol
    top = full.view(-1, 256).amax(1, keepdim=True).expand(-1, 256).reshape(-1)
    safe = torch.where(top > 0, top, torch.ones_like(top))
    c = levels * (full / safe) ** (1 / power)
    up = levels * ((full + t) / safe) ** (1 / power) - c + levels * (t / safe) / power
    down = c - levels * ((full - t).clamp(min=0) / safe) ** (1 / power) + levels * (t / safe) / power
    got = code.double().abs()
    least = torch.where((full > 0) & (levels == 255), torch.ones_like(c), torch.zeros_like(c))
    slack = 6 * U * c + 1e-12
    assert (got <= torch.maximum(c + 0.5 + up + slack, least)).all() and (got >= torch.minimum(c - 0.5 - down - slack, got.new_tensor(float(levels)))).all()
    assert (got >= least).all() and (got[n:] == 0).all()
    return top.view(-1, 256)[:, 0], (t.view(-1, 256).amax(1))


def step_close(b, t, grad_scale=1.0, max_norm=None, norm=None, h=HYPER, call=None):
    """One step of batch b, compared with the formulas on what b held before it."""
    old = [(p.double(), g.double()) for p, g, _, _ in b.entries]
    m0, v0 = values(b)
    extra = 0 if b.state_bits == 32 else 1
    scales = None if not extra else (b.m_scale.clone(), b.v_scale.clone())
    assert scales is None or all(s.isfinite().all() for s in scales)
    (call or (lambda: b.step(t, **h, grad_scale=grad_scale, max_norm=max_norm, norm=norm)))()
    gs = grad_scale
    if max_norm is not None:
        total = grad_scale * math.sqrt(sum(float((g * g).sum()) for _, g in old))
        gs = grad_scale * max_norm / max(total, max_norm)
        if norm is not None:
            assert abs(float(norm) - total) <= 4 * U * total
    bc1, bc2 = 1 - h["beta1"] ** t, 1 - h["beta2"] ** t
    for (p, g, decay, copy), (p0, g0), o in zip(b.entries, old, b.offsets):
        n = p.numel()
        if n == 0:
            continue
        gg = g0 * gs
        m = h["beta1"] * m0[o:o + n] + (1 - h["beta1"]) * gg
        v = h["beta2"] * v0[o:o + n] + (1 - h["beta2"]) * gg * gg
        tm = (6 + 4 * extra) * U * (h["beta1"] * m0[o:o + n].abs() + (1 - h["beta1"]) * gg.abs()) + 1e-37
        rv = (10 + 8 * extra) * U
        den = torch.sqrt(v / bc2) + h["eps"]
        upd = h["lr"] / bc1 * m / den
        new = p0 * (1 - h["lr"] * h["weight_decay"] * decay) - upd
        tol = 4 * U * p0.abs() + h["lr"] / bc1 * tm / den + upd.abs() * (rv + 12 * U)
        for out, where in ((p, "p"), (copy, "copy")):
            if out is not None:
                half = torch.finfo(out.dtype).eps / 2 * (new.abs() + tol) + (2.0 ** -25 if out.dtype == F16 else 1e-37)
                off = (out.double() - new).abs()
                assert (off <= tol + half).all(), (where, n, float((off / (tol + half)).max()))
        if b.state_bits == 32:
            assert ((b.m[o:o + n].double() - m).abs() <= tm).all() and ((b.v[o:o + n].double() - v).abs() <= rv * v + 1e-37).all()
        else:
            end, blocks = o + -(-n // 256) * 256, slice(o // 256, o // 256 + -(-n // 256))
            top, tt = check_codes(b.m[o:end], m, tm, 127, 2, n)
            assert ((b.m_scale[blocks].double() - top).abs() <= tt).all()
            q = b.m[o:o + n]
            assert ((q == 0) | (q.sign() == m.sign()) | (m.abs() <= tm)).all()
            top, tt = check_codes(b.v[o:end], v, rv * v, 255, 4, n)
            assert ((b.v_scale[blocks].double() - top).abs() <= tt + 1e-37).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("types", [(F32, F32, None), (F32, BF16, BF16), (F32, F16, F16), (BF16, BF16, None), (F16, F16, BF16), (BF16, F32, None), (F16, F32, F16)],
                         ids=lambda t: "-".join(str(x).replace("torch.", "") for x in t))
@pytest.mark.parametrize("sizes", SIZES.values(), ids=SIZES.keys())
def test_step(sizes, types, bits, hip_ops):
    p, g, copy = types
    for shift in (0, 1):
        print(sizes, types, bits, shift, flush=True)
        b, buffers = make(hip_ops, sizes, p, g, copy, bits, seed=len(sizes) + shift, shift=shift)
        step_close(b, 7)
        norm = torch.zeros(1, device="cuda")
        step_close(b, 8, grad_scale=0.25, max_norm=0.3, norm=norm)      # clipped (or not, for the smallest lists)
        step_close(b, 9, max_norm=1e9, norm=norm)                         # not clipped
        for buf, s, n in buffers:
            assert (buf[:s] == 7).all() and (buf[s + n:] == 7).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_from_zero(bits, hip_ops):
    """The first steps from zero states, zero gradients among them: no moment, no update, no NaN."""
    b, _ = make(hip_ops, [300, 1000], bits=bits, zero=True, seed=3)
    b.entries[0][1][:256] = 0                     # a whole block without a gradient
    b.entries[1][1][5] = 0
    p0 = b.entries[0][0].clone()
    for t in (1, 2, 3):
        step_close(b, t)
    m, v = values(b)
    assert (m[:256] == 0).all() and (v[:256] == 0).all()
    keep = (1 - HYPER["lr"] * HYPER["weight_decay"]) ** 3
    assert ((b.entries[0][0][:256].double() - p0[:256].double() * keep).abs() <= 12 * U * p0[:256].abs()).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("h", [dict(beta1=0.0, beta2=0.0), dict(beta1=0.5, beta2=0.9, eps=0.1), dict(lr=0.0), dict(weight_decay=0.0), dict(beta1=0.99, beta2=0.9999)])
def test_hyper_parameters(h, bits, hip_ops):
    b, _ = make(hip_ops, [1000, 77], bits=bits, seed=4)
    for t in (1, 1000, 100000):
        step_close(b, t, h={**HYPER, **h})


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("h", [dict(beta1=0.0, beta2=0.0), dict(beta1=0.99, beta2=0.9999)])
def test_step_count_in_device_memory(h, bits, hip_ops):
    b, _ = make(hip_ops, [5000, 77], bits=bits, seed=4)
    h = {**HYPER, **h}
    for t in (1, 2, 100000):
        at = torch.tensor([t], dtype=torch.int64, device="cuda")
        step_close(b, t, h=h, call=lambda: b.step(at, **h))      # noqa: B023


def test_large_list(hip_ops):
    """More than 4096 chunks of 4096 elements and more than the cache holds: the other chunk size, and streamed requests."""
    for bits, sizes, g in ((32, [17000001, 255], BF16), (8, [17000001, 8000003], F32)):
        b, _ = make(hip_ops, sizes, g=g, copy=BF16, bits=bits, seed=12)
        step_close(b, 3)
        norm = torch.zeros(1, device="cuda")
        step_close(b, 4, max_norm=0.5, norm=norm)
        del b


@pytest.mark.parametrize("bits", [32, 8])
def test_far_magnitudes(bits, hip_ops):
    """Gradients whose squares leave fp32's range below: the norm is summed in 64 bits, second moments that underflow count as zero."""
    b, _ = make(hip_ops, [600], bits=bits, zero=True, spread=False)
    b.entries[0][1].mul_(1e-25)
    norm = torch.zeros(1, device="cuda")
    b.grad_norm(norm)
    want = float(b.entries[0][1].double().norm())
    assert want > 0 and abs(float(norm) - want) <= 4 * U * want
    b.step(1, **HYPER)
    assert b.entries[0][0].isfinite().all()
    b.entries[0][1].mul_(1e25).mul_(1e25)        # and above: the norm of 1e25s is a number, their squares are not
    b.grad_norm(norm, grad_scale=0.5)
    want = 0.5 * float(b.entries[0][1].double().norm())
    assert abs(float(norm) - want) <= 4 * U * want
    b.step(2, **HYPER, max_norm=1.0, norm=norm)
    assert b.entries[0][0].isfinite().all() and values(b)[1].isfinite().all()


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("bits", [32, 8])
def test_not_finite(bits, value, hip_ops):
    """With clipping, a gradient that is not finite leaves everything as it was; without, it stays in its element (32 bits) or its block
    (8 bits)."""
    b, _ = make(hip_ops, [1000, 300], bits=bits, copy=BF16, seed=5)
    b.entries[0][1][700] = value
    held = [t.clone() for t in (*b.state, *[t for e in b.entries for t in (e[0], e[3])])]
    norm = torch.zeros(1, device="cuda")
    b.step(3, **HYPER, max_norm=1.0, norm=norm)
    assert not norm.isfinite().any()
    assert all(torch.equal(x, y) for x, y in zip(held, (*b.state, *[t for e in b.entries for t in (e[0], e[3])])))
    b.step(3, **HYPER)
    p = b.entries[0][0]
    others = torch.ones(1000, dtype=torch.bool, device="cuda")
    others[700] = False
    assert p[700].isnan() and p[others].isfinite().all() and b.entries[1][0].isfinite().all()
    m, v = torch.empty(b.total, device="cuda"), torch.empty(b.total, device="cuda")
    b.moments(m, v)
    if bits == 32:
        assert not m[700].isfinite() and not v[700].isfinite() and m[:1000][others].isfinite().all() and v[:1000][others].isfinite().all()
    else:
        block = torch.zeros(b.total, dtype=torch.bool, device="cuda")
        block[512:768] = True
        assert m[block].isnan().all() and v[block].isnan().all() and m[~block].isfinite().all() and v[~block].isfinite().all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("bits", [32, 8])
def test_moments(bits, dtype, hip_ops):
    b, _ = make(hip_ops, [9000, 3], bits=bits, seed=6)
    mo, vo = torch.empty(b.total, dtype=dtype, device="cuda"), torch.empty(b.total, dtype=dtype, device="cuda")
    b.moments(mo, vo)
    for got, want in zip((mo, vo), values(b)):
        lim = (torch.finfo(dtype).eps / 2 + 8 * U) * want.abs() + (2.0 ** -25 if dtype == F16 else 1e-37)
        assert ((got.double() - want).abs() <= lim).all()
    only = torch.empty_like(vo)
    b.moments(None, only)
    assert torch.equal(only, vo)
    with pytest.raises(ValueError):
        b.moments(mo[:-1], None)
    with pytest.raises(ValueError):
        b.moments(mo, torch.empty(b.total, dtype=torch.float64, device="cuda"))


def test_empty_lists(hip_ops):
    norm = torch.full((1,), 3.0, device="cuda")
    for entries in ([], [(torch.empty(0, device="cuda"), torch.empty(0, device="cuda"), 1.0)]):
        for bits in (32, 8):
            b = hip_ops.make_adamw(entries, state_bits=bits)
            b.step(1, **HYPER)
            norm.fill_(3.0)
            b.step(1, **HYPER, max_norm=1.0, norm=norm)
            assert float(norm) == 0
            norm.fill_(3.0)
            b.grad_norm(norm)
            assert float(norm) == 0
            b.moments(torch.empty(0, device="cuda"), torch.empty(0, device="cuda"))


def test_call_refusals(hip_ops):
    b, _ = make(hip_ops, [100])
    n = torch.zeros(1, device="cuda")
    for bad in (dict(t=0), dict(t=1, lr=-1.0), dict(t=1, beta1=1.0)):
        with pytest.raises(Exception):
            b.step(**{"lr": 1e-3, **bad})
    for bad in (dict(max_norm=0.0), dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(norm=n), dict(max_norm=1.0, norm=n.double()), dict(max_norm=1.0, norm=n.cpu())):
        with pytest.raises(ValueError):
            b.step(1, 1e-3, **bad)
    for bad in (torch.ones(1, device="cuda"), torch.ones(1, dtype=torch.int64), torch.ones(2, dtype=torch.int64, device="cuda")):
        with pytest.raises(ValueError):
            b.step(bad, 1e-3)
    with pytest.raises(ValueError):
        b.grad_norm(None)
    p = b.entries[0][0].clone()
    torch.cuda.synchronize()
    assert torch.equal(p, b.entries[0][0])


@pytest.mark.parametrize("bits", [32, 8])
def test_adopted_state(bits, hip_ops):
    """Two batches over the same tensors, one handing its states to the other, continue as one."""
    b, _ = make(hip_ops, [900, 40], bits=bits, seed=7)
    twin = hip_ops.make_adamw([(p.clone(), g, d) for p, g, d, _ in b.entries], state_bits=bits, state=[s.clone() for s in b.state])
    b.step(2, **HYPER)
    twin.step(2, **HYPER)
    assert all(torch.equal(x, y) for x, y in zip(b.state, twin.state)) and all(torch.equal(e[0], f[0]) for e, f in zip(b.entries, twin.entries))


@pytest.mark.parametrize("bits", [32, 8])
def test_same_bits_every_run(bits, hip_ops):
    seen = []
    for _ in range(3):
        b, _ = make(hip_ops, [70001, 5, 4096], g=BF16, copy=BF16, bits=bits, seed=8)
        norm = torch.zeros(1, device="cuda")
        for t in (1, 2):
            b.step(t, **HYPER, max_norm=0.5, norm=norm)
        seen.append([t.clone() for t in (*b.state, norm, *[x for e in b.entries for x in (e[0], e[3])])])
    assert all(torch.equal(x, y) for other in seen[1:] for x, y in zip(seen[0], other))


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(bits, hip_ops):
    """Two batches' clipped steps in two graphs, their step counts in device memory, replayed side by side."""
    sets = []
    for k in range(2):
        b, _ = make(hip_ops, [5000 + k, 300], bits=bits, seed=9 + k)
        eager, _ = make(hip_ops, [5000 + k, 300], bits=bits, seed=9 + k)
        sets.append(dict(b=b, eager=eager, t=torch.zeros(1, dtype=torch.int64, device="cuda"), norm=torch.zeros(1, device="cuda"), stream=torch.cuda.Stream()))
    torch.cuda.synchronize()
    for s in sets:
        s["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s["graph"]):
            s["t"].add_(1)
            s["b"].step(s["t"], **HYPER, max_norm=0.5, norm=s["norm"])
    with pytest.raises(Exception):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            make(hip_ops, [10])
    torch.cuda.synchronize()
    for t in range(1, 5):
        for s in sets:
            for e in (*s["b"].entries, *s["eager"].entries):
                e[1].mul_(0.9)
        torch.cuda.synchronize()
        for s in sets:
            with torch.cuda.stream(s["stream"]):
                step = lambda: (s["graph"].replay(), torch.cuda.synchronize())      # noqa: E731,B023
                if t == 1:
                    step_close(s["b"], t, max_norm=0.5, norm=s["norm"], call=step)
                else:
                    s["graph"].replay()
        torch.cuda.synchronize()
        for s in sets:
            s["eager"].step(t, **HYPER, max_norm=0.5, norm=torch.zeros(1, device="cuda"))
            assert int(s["t"]) == t
    torch.cuda.synchronize()
    for s in sets:
        # the two bias corrections differ in the last digits only (8 u of the update), and each of the 4 steps rounds p on both sides,
        # 4 u of |p| each (its decay, sum and store): 4 * 2 * 4 u |p|, with |p| at its largest, and not an absolute 4 u
        for x, y in zip([e[0] for e in s["b"].entries], [e[0] for e in s["eager"].entries]):
            assert ((x - y).abs() <= 4 * (8 * U + (0 if bits == 32 else 0.05)) * HYPER["lr"] * 10 + 32 * U * y.abs()).all()


def test_another_stream_and_early_release(hip_ops):
    """A batch stepped on another stream than its own and dropped at once: its memory is not handed out before the step ends."""
    p, g = torch.zeros(1 << 22, device="cuda"), torch.ones(1 << 22, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    b = hip_ops.make_adamw([(p, g, 0.0)])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        b.step(1, 0.5, eps=0.0)
    del b
    junk = [torch.full((1 << 22,), float("nan"), device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    assert ((p + 0.5).abs() <= 8 * U).all() and len(junk) == 3


def test_past_32_bits(hip_ops):
    """A tensor of more than 2^31 elements: its far end is updated like any other."""
    n = (1 << 31) + 1000
    p, g = (torch.zeros(n, dtype=BF16, device="cuda") for _ in range(2))
    p[-2000:] = 1.0
    g[-2000:] = 0.5
    b = hip_ops.make_adamw([(p, g, 0.0)], state_bits=8)
    norm = torch.zeros(1, device="cuda")
    b.step(1, 0.25, eps=0.0, max_norm=1e6, norm=norm)
    assert abs(float(norm) - 0.5 * math.sqrt(2000)) < 1e-4
    assert (p[-2000:] == 0.75).all() and p[n - 2001].isnan()          # (0 / 0 without an epsilon, as the formula says)
    assert (b.m[n - 2000:n] == 127).all() and (b.v[n - 2000:n] == 255).all() and (b.m[:1000] == 0).all() and (b.m[n:] == 0).all()


def test_train_step_matches_the_oracle():
    """GanEngine.train_step with AdamW (clipped generator, 32-bit states): both networks' weights after one step against the same
    engine on the 64-bit backend, on the same random stream."""
    from downscaling.engine.hipops import HipOps
    from downscaling.engine.networks import DiscriminatorNet, GeneratorNet
    from downscaling.engine.trainer import AdamW, GanEngine, PhiloxSource
    from oracle.torch_backend import TorchOps
    from tests.helpers import randomize, rel_err, weights64
    hip_ops = HipOps("cuda:0")      # (one of its own: a train step picks the streams of its backend)
    B, T, S = 2, 1, 32
    g = torch.Generator().manual_seed(0)
    low, high = (torch.randn(B, T, S, S, c, generator=g, dtype=torch.float64) for c in (3, 2))
    out = []
    for ops, cv in ((hip_ops, lambda t: t.float().to(hip_ops.device)), (TorchOps(), lambda t: t)):
        gen, disc = GeneratorNet(ops, S, 3, 4, 2, T, feature_channels=32, seed=5), DiscriminatorNet(ops, S, S, 3, 2, T, feature_channels=8, seed=6)
        randomize(gen, 21), randomize(disc, 22)
        # (epsilon as the networks' own optimizers: the update stays a smooth function of the gradient where that is near zero)
        go, do = AdamW(1e-3, 0.5, 0.9, 0.1, weight_decay=0.05, global_clipnorm=0.5), AdamW(1e-3, 0.5, 0.9, 0.1, weight_decay=0.05)
        GanEngine(gen, disc, PhiloxSource(ops, seed=99), noise_std=0.1, n_critic=2).train_step(cv(low), cv(high), go, do)
        out.append((weights64(gen), weights64(disc), float(go.grad_norm)))
    (gw, dw, gn), (gr, dr, rn) = out
    assert abs(gn - rn) < 1e-4 * rn
    for got, want in ((gw, gr), (dw, dr)):
        assert max(rel_err(got[k], want[k]) for k in got) < 1e-4


@pytest.mark.parametrize("bits", [32, 8])
def test_norm_layer_trained(bits, hip_ops):
    """A run of the operators as they are used: norm -> linear map -> squared error, backward, clipped AdamW, several steps, against the
    same run in 64 bits.  epsilon = 0.1 makes the update a function of the gradient with slope <= lr / epsilon = 0.1; five steps of a
    gradient error of 1e-5 (relative to gradients below 0.5 after clipping) stay below 1e-5.  8-bit moments: each step's m is off by
    up to 2 * 0.5 / 127 of its block's largest, sqrt(v) by as little, so an update by 0.02 lr at most."""
    P, C, O, lr = 300, 200, 16, 1e-2
    gen = torch.Generator(device="cuda").manual_seed(11)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")      # noqa: E731
    x, y = 2 * r(P, C) + 1, r(P, O)
    w, gamma, beta = r(C, O) / C ** 0.5, torch.ones(C, device="cuda"), torch.zeros(C, device="cuda")
    ref = [t.double().clone().requires_grad_(True) for t in (w, gamma, beta)]
    opt = torch.optim.AdamW([dict(params=ref[:1], weight_decay=0.1), dict(params=ref[1:], weight_decay=0.0)], lr=lr, betas=(0.9, 0.99), eps=0.1)
    grads = [torch.zeros_like(t) for t in (w, gamma, beta)]
    b = hip_ops.make_adamw([(w, grads[0], 1.0), (gamma, grads[1], 0.0), (beta, grads[2], 0.0)], state_bits=bits)
    z, mr, dx, norm = torch.empty_like(x), torch.empty(P, 2, device="cuda"), torch.empty_like(x), torch.zeros(1, device="cuda")
    for t in range(1, 6):
        hip_ops.layernorm_fwd(x, gamma, beta, 1e-3, z, mr)
        d = (z @ w - y) * (2.0 / P)
        grads[0].copy_(z.t() @ d)
        grads[1].zero_(), grads[2].zero_()
        hip_ops.layernorm_bwd((d @ w.t()).contiguous(), x, mr, gamma, dx, grads[1], grads[2])
        b.step(t, lr, 0.9, 0.99, 0.1, 0.1, max_norm=0.5, norm=norm)
        opt.zero_grad()
        zz = torch.nn.functional.layer_norm(x.double(), (C,), ref[1], ref[2], 1e-3)
        ((zz @ ref[0] - y.double()) ** 2).sum().div(P).backward()
        total = torch.sqrt(sum((q.grad ** 2).sum() for q in ref))
        assert abs(float(norm) - float(total.detach())) < (1e-4 if bits == 32 else 0.02) * float(total.detach())
        for q in ref:
            q.grad.mul_(0.5 / total.clamp(min=0.5))
        opt.step()
    lim = 1e-5 if bits == 32 else 5 * 0.02 * lr
    for got, want in zip((w, gamma, beta), ref):
        assert float((got.double() - want.detach()).abs().max()) < lim
