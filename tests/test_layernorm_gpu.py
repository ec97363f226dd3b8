"""layernorm_fwd / layernorm_bwd (csrc/layernorm.hip) against the 64-bit definition.

Tolerances, derived: u = 2^-24 is half a step of fp32.  A thread adds at most `seq` terms one after another and the rest is a tree of at
most 16 levels, so a mean over the row is off by at most K u times the mean of the terms' magnitudes, K = seq + 16.  The centred value
x - mean therefore carries K u (|x - mean| + mean |x - mean|), rstd a relative (K + 8) u, and scaling, shifting and the centred value's own
rounding a few u of the terms that they add.  The first mean is off by K u |mean|; the mean of (x - mean) takes that out but for K u of it,
(K u)^2 |mean| — all there is in a row of equal values.  Both tensors round once more on store: finfo.eps / 2 of the value."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-3
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SHAPES = [(1, 1), (5, 2), (3, 7), (9, 8), (2, 9), (130, 16), (33, 100), (64, 64), (511, 40), (512, 2051), (700, 33), (3, 255), (4, 1024), (197, 1155), (5, 2048), (6, 4096),
          (1, 4097), (37, 5003), (2, 8192), (3, 16384), (2, 16385), (1, 70001)]


def chain(C):
    return 16 + max(8, C // 256) + 8


def rows(gen, P, C, dtype, pad=0, shift=0, scale=1.0, offset=0.0):
    """[P, C] values in a buffer with `pad` more columns, `shift` elements behind its start; the buffer's other elements hold 7."""
    buf = torch.full((P * (C + pad) + shift + 8,), 7.0, dtype=dtype, device="cuda")
    v = buf[shift:shift + P * (C + pad)].view(P, C + pad)[:, :C]
    v.copy_(torch.randn(P, C, generator=gen, device="cuda") * scale + offset)
    return v, buf


def forward_close(x, gamma, beta, z, mr, what=""):
    x64 = x.double()
    C = x.shape[1]
    mean = x64.mean(1, keepdim=True)
    d = x64 - mean
    rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
    g = torch.ones(C, device=x.device).double() if gamma is None else gamma.double()
    b = torch.zeros(C, device=x.device).double() if beta is None else beta.double()
    ref = d * rstd * g + b
    K = chain(C)
    spread = d.abs().mean(1, keepdim=True)
    tol = U * ((K * (d.abs() + spread + K * U * mean.abs()) * rstd + (K + 8) * (d * rstd).abs()) * g.abs() + 4 * (b.abs() + ref.abs())) + torch.finfo(z.dtype).eps / 2 * ref.abs() + 1e-30
    if z.dtype == F16:
        tol = tol + 2.0 ** -25                                                         # half of fp16's smallest step
    assert ((z.double() - ref).abs() <= tol).all(), (what, float(((z.double() - ref).abs() / tol).max()))
    if mr is not None:
        assert ((mr[:, :1].double() - mean).abs() <= U * (2 * mean.abs() + K * spread) + 1e-30).all(), what
        assert ((mr[:, 1:].double() - rstd).abs() <= (K + 8) * U * rstd).all(), what
    return ref


def backward_close(dz, x, mr, gamma, dx, dg, db, what="", dg0=0.0, db0=0.0):
    C, P = x.shape[1], x.shape[0]
    m, r = mr[:, :1].double(), mr[:, 1:].double()
    xh = (x.double() - m) * r
    g = dz.double()
    a = g if gamma is None else g * gamma.double()
    ref = r * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
    K = chain(C)
    # the terms' magnitudes; xh itself is within 3 u of (|x| + |mean|) rstd
    xa = xh.abs() + 0.5 * (x.double().abs() + m.abs()) * r
    terms = r * (a.abs() + a.abs().mean(1, keepdim=True) + xa * (a.abs() * xa).mean(1, keepdim=True))
    tol = (K + 8) * U * terms + torch.finfo(dx.dtype).eps / 2 * ref.abs() + (2.0 ** -25 if dx.dtype == F16 else 1e-30)
    assert ((dx.double() - ref).abs() <= tol).all(), (what, float(((dx.double() - ref).abs() / tol).max()))
    Kr = min(P, 128) + P // 128 + 24          # rows added one after another, then the partial sums' order
    for name, got, ref, mag, start in (("dgamma", dg, (g * xh).sum(0), (g.abs() * xa).sum(0), dg0), ("dbeta", db, g.sum(0), g.abs().sum(0), db0)):
        if got is not None:
            off = (got.double() - (ref + start)).abs()
            lim = Kr * U * (mag + abs(start)) + 1e-30
            assert (off <= lim).all(), (what, name, float((off / lim).max()))


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("P,C", SHAPES)
def test_forward_and_backward(P, C, dtype, hip_ops):
    gen = torch.Generator(device="cuda").manual_seed(P * 131 + C)
    for pad, shift in ((0, 0), (3, 1)):
        print(P, C, dtype, pad, shift, flush=True)
        x, _ = rows(gen, P, C, dtype, pad, shift, 1.5, 0.5)
        dz, _ = rows(gen, P, C, dtype, pad, shift)
        z, zb = rows(gen, P, C, dtype, pad, shift)
        dx, db_ = rows(gen, P, C, dtype, pad, shift)
        gamma, beta = 1 + 0.3 * torch.randn(C, generator=gen, device="cuda"), torch.randn(C, generator=gen, device="cuda")
        mr = torch.empty(P, 2, device="cuda")
        hip_ops.layernorm_fwd(x, gamma, beta, EPS, z, mr)
        forward_close(x, gamma, beta, z, mr)
        dg, db = torch.full((C,), 2.0, device="cuda"), torch.full((C,), -1.0, device="cuda")
        hip_ops.layernorm_bwd(dz, x, mr, gamma, dx, dg, db)
        backward_close(dz, x, mr, gamma, dx, dg, db, dg0=2.0, db0=-1.0)
        for view, buf in ((z, zb), (dx, db_)):           # nothing beside the rows was written
            mask = torch.ones_like(buf, dtype=torch.bool)
            mask[shift:shift + P * (C + pad)].view(P, C + pad)[:, :C] = False
            assert (buf[mask] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("P,C", [(37, 24), (5, 1155), (3, 4096), (2, 20011)])
def test_parameters_and_partial_gradients(P, C, dtype, hip_ops):
    """Parameters in the activations' type or left out, statistics not kept, one gradient of two or none, overwritten ones."""
    gen = torch.Generator(device="cuda").manual_seed(C)
    x, _ = rows(gen, P, C, dtype)
    dz, _ = rows(gen, P, C, dtype)
    gamma, beta = ((1 + 0.3 * torch.randn(C, generator=gen, device="cuda")).to(dtype) for _ in range(2))
    z, dx, mr = torch.empty_like(x), torch.empty_like(x), torch.empty(P, 2, device="cuda")
    for ga, be in ((gamma, beta), (None, beta), (gamma, None), (None, None)):
        hip_ops.layernorm_fwd(x, ga, be, EPS, z)
        forward_close(x, ga, be, z, None)
        hip_ops.layernorm_fwd(x, ga, be, EPS, z, mr)
        forward_close(x, ga, be, z, mr)
        for want in ((True, True), (True, False), (False, True), (False, False)):
            dg, db = (torch.full((C,), float("nan"), device="cuda") if w else None for w in want)
            hip_ops.layernorm_bwd(dz, x, mr, ga, dx, dg, db, accumulate=False)
            backward_close(dz, x, mr, ga, dx, dg, db)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("P,C", [(70, 16), (9, 1155), (3, 5003), (2, 30001)])
def test_in_place_and_broadcast(P, C, dtype, hip_ops):
    """z over x, dx over dz or x; every row one row of the input (stride 0); the two halves of a concatenation."""
    gen = torch.Generator(device="cuda").manual_seed(C + 1)
    x, _ = rows(gen, P, C, dtype)
    dz, _ = rows(gen, P, C, dtype)
    gamma, beta = 1 + 0.3 * torch.randn(C, generator=gen, device="cuda"), torch.randn(C, generator=gen, device="cuda")
    z, dx, mr, dg, db = torch.empty_like(x), torch.empty_like(x), torch.empty(P, 2, device="cuda"), torch.zeros(C, device="cuda"), torch.zeros(C, device="cuda")
    hip_ops.layernorm_fwd(x, gamma, beta, EPS, z, mr)
    hip_ops.layernorm_bwd(dz, x, mr, gamma, dx, dg, db)
    over = x.clone()
    hip_ops.layernorm_fwd(over, gamma, beta, EPS, over)
    assert torch.equal(over, z)
    for alias in ("dz", "x"):
        a, b = dz.clone(), x.clone()
        g2, b2 = torch.zeros(C, device="cuda"), torch.zeros(C, device="cuda")
        hip_ops.layernorm_bwd(a, b, mr, gamma, a if alias == "dz" else b, g2, b2)
        assert torch.equal(a if alias == "dz" else b, dx)
        backward_close(dz, x, mr, gamma, dx, g2, b2)      # (few rows: another order of the sums where dx is a tensor of its own)
    wide = x[:1].expand(P, C)
    hip_ops.layernorm_fwd(wide, gamma, beta, EPS, z, mr)
    forward_close(wide, gamma, beta, z, mr)
    hip_ops.layernorm_bwd(dz[:1].expand(P, C), wide, mr, gamma, dx, dg, db, accumulate=False)
    backward_close(dz[:1].expand(P, C), wide, mr, gamma, dx, dg, db)
    cat = torch.empty(P, 2 * C, dtype=dtype, device="cuda")
    cat[:, :C] = x
    hip_ops.layernorm_fwd(cat[:, :C], gamma, beta, EPS, cat[:, C:])
    assert torch.equal(cat[:, :C], x)
    forward_close(x, gamma, beta, cat[:, C:], None)


@pytest.mark.parametrize("C", [16, 1000, 4096, 20000])
def test_offsets_constants_and_empty(C, hip_ops):
    """Rows far from zero keep their digits, constant rows come out as beta, no rows at all."""
    gen = torch.Generator(device="cuda").manual_seed(C + 2)
    gamma, beta = 1 + 0.3 * torch.randn(C, generator=gen, device="cuda"), torch.randn(C, generator=gen, device="cuda")
    for offset in (1e4, -3e5):
        x, _ = rows(gen, 6, C, F32, scale=1.0, offset=offset)
        z, mr = torch.empty_like(x), torch.empty(6, 2, device="cuda")
        hip_ops.layernorm_fwd(x, gamma, beta, EPS, z, mr)
        forward_close(x, gamma, beta, z, mr, offset)
    x = torch.full((3, C), 0.1, device="cuda")
    z, mr = torch.empty_like(x), torch.empty(3, 2, device="cuda")
    hip_ops.layernorm_fwd(x, gamma, beta, EPS, z, mr)
    forward_close(x, gamma, beta, z, mr)
    e = torch.empty(0, C, device="cuda")
    hip_ops.layernorm_fwd(e, gamma, beta, EPS, torch.empty_like(e), torch.empty(0, 2, device="cuda"))
    dg, db = torch.full((C,), 3.0, device="cuda"), torch.full((C,), 3.0, device="cuda")
    hip_ops.layernorm_bwd(e, e.clone(), torch.empty(0, 2, device="cuda"), gamma, torch.empty_like(e), dg, db)
    assert (dg == 3).all() and (db == 3).all()
    hip_ops.layernorm_bwd(e, e.clone(), torch.empty(0, 2, device="cuda"), gamma, torch.empty_like(e), dg, db, accumulate=False)
    assert (dg == 0).all() and (db == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("C", [12, 1155, 4096, 17000])
def test_not_finite(C, dtype, hip_ops):
    """A NaN or an infinity makes its own row NaN (no value of it can be normalised) and reaches no other row."""
    gen = torch.Generator(device="cuda").manual_seed(C + 3)
    x, _ = rows(gen, 40, C, dtype)
    clean = x.clone()
    x[3, C - 1], x[17, 0], x[39, C // 2] = float("nan"), float("inf"), float("-inf")
    bad = torch.zeros(40, dtype=torch.bool, device="cuda")
    bad[[3, 17, 39]] = True
    z, zc, mr = torch.empty_like(x), torch.empty_like(x), torch.empty(40, 2, device="cuda")
    hip_ops.layernorm_fwd(x, None, None, EPS, z, mr)
    hip_ops.layernorm_fwd(clean, None, None, EPS, zc)
    assert z[bad].isnan().all() and torch.equal(z[~bad], zc[~bad])
    assert mr[bad, 1].isnan().all() and mr[~bad].isfinite().all()
    dz, _ = rows(gen, 40, C, dtype)
    hip_ops.layernorm_fwd(clean, None, None, EPS, zc, mr)
    dz2 = dz.clone()
    dz2[5, C - 1] = float("nan")
    dx, dx2, dg, db = torch.empty_like(x), torch.empty_like(x), torch.zeros(C, device="cuda"), torch.zeros(C, device="cuda")
    hip_ops.layernorm_bwd(dz, clean, mr, None, dx)
    hip_ops.layernorm_bwd(dz2, clean, mr, None, dx2, dg, db)
    assert dx2[5].isnan().all() and torch.equal(dx2[:5], dx[:5]) and torch.equal(dx2[6:], dx[6:])
    assert dg[C - 1].isnan() and db[C - 1].isnan() and dg[:C - 1].isfinite().all() and db[:C - 1].isfinite().all()


def test_far_rows(hip_ops):
    """Row offsets that pass 2^31 elements and 2^32 bytes."""
    ld, P, C = 1 << 30, 4, 1155
    buf = torch.empty(ld * (P - 1) + 2048, dtype=BF16, device="cuda")
    out = torch.empty_like(buf)
    view = lambda b: b.as_strided((P, C), (ld, 1))      # noqa: E731
    gen = torch.Generator(device="cuda").manual_seed(5)
    view(buf).copy_(torch.randn(P, C, generator=gen, device="cuda"))
    mr = torch.empty(P, 2, device="cuda")
    hip_ops.layernorm_fwd(view(buf), None, None, EPS, view(out), mr)
    forward_close(view(buf), None, None, view(out), mr)
    dz = torch.randn(P, C, generator=gen, device="cuda").to(BF16)
    dg, db = torch.zeros(C, device="cuda"), torch.zeros(C, device="cuda")
    hip_ops.layernorm_bwd(dz, view(buf), mr, None, view(out), dg, db)
    backward_close(dz, view(buf), mr, None, view(out), dg, db)


@pytest.mark.parametrize("P,C,dtype", [(70000, 1024, F32), (9000, 16384, BF16), (2200000, 32, F16), (17000, 4096, F32), (33000, 2048, BF16)])
def test_streamed_sizes(P, C, dtype, hip_ops):
    """Tensors that together pass the last-level cache take non-temporal requests."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    x, dz = ((torch.randn(P, C, generator=gen, device="cuda") + 0.5).to(dtype) for _ in range(2))
    gamma, beta = 1 + 0.3 * torch.randn(C, generator=gen, device="cuda"), torch.randn(C, generator=gen, device="cuda")
    z, dx, mr = torch.empty_like(x), torch.empty_like(x), torch.empty(P, 2, device="cuda")
    dg, db = torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
    hip_ops.layernorm_fwd(x, gamma, beta, EPS, z, mr)
    hip_ops.layernorm_bwd(dz, x, mr, gamma, dx, dg, db, accumulate=False)
    for a in range(0, P, 1 + P // 8):                # the rows are checked in pieces: their 64-bit copies are large
        r = slice(a, a + 1 + P // 8)
        forward_close(x[r], gamma, beta, z[r], mr[r])
        backward_close(dz[r], x[r], mr[r], gamma, dx[r], None, None)
    mag = torch.zeros(C, dtype=torch.float64, device="cuda")
    sums = torch.zeros(2, C, dtype=torch.float64, device="cuda")
    for a in range(0, P, 1 + P // 8):
        r = slice(a, a + 1 + P // 8)
        g, xh = dz[r].double(), (x[r].double() - mr[r, :1].double()) * mr[r, 1:].double()
        sums += torch.stack([(g * xh).sum(0), g.sum(0)])
        mag += (g.abs() * (1 + xh.abs() + 0.5 * (x[r].double().abs() + mr[r, :1].double().abs()) * mr[r, 1:].double())).sum(0)
    # a thread adds P / (workgroups x rows at a time) rows one after another, at most P / 128 of them here, the partial sums add 512 more
    lim = (P // 128 + 600) * U * mag
    assert ((dg.double() - sums[0]).abs() <= lim).all() and ((db.double() - sums[1]).abs() <= lim).all()


@pytest.mark.parametrize("P,C,dtype", [(5000, 16, F32), (900, 1155, F16), (1500, 4096, BF16), (40, 20000, BF16)])
def test_same_bits_every_run(P, C, dtype, hip_ops):
    gen = torch.Generator(device="cuda").manual_seed(6)
    x, _ = rows(gen, P, C, dtype)
    dz, _ = rows(gen, P, C, dtype)
    mr, dx = torch.empty(P, 2, device="cuda"), torch.empty_like(x)
    hip_ops.layernorm_fwd(x, None, None, EPS, torch.empty_like(x), mr)
    seen = []
    for _ in range(3):
        dg, db = torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
        hip_ops.layernorm_bwd(dz, x, mr, None, dx, dg, db, accumulate=False)
        seen.append((dg, db, dx.clone()))
    backward_close(dz, x, mr, None, dx, dg, db)
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))


def test_streams_and_graphs(hip_ops):
    """Calls side by side on two streams, and two captured graphs replayed side by side: no scratch is shared."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    sets = []
    for C, P in ((1155, 2000), (1155, 1900)):
        x, _ = rows(gen, P, C, BF16)
        dz, _ = rows(gen, P, C, BF16)
        mr = torch.empty(P, 2, device="cuda")
        hip_ops.layernorm_fwd(x, None, None, EPS, torch.empty_like(x), mr)
        dg, db = torch.zeros(C, device="cuda"), torch.zeros(C, device="cuda")
        hip_ops.layernorm_bwd(dz, x, mr, None, torch.empty_like(x), dg, db)
        sets.append(dict(x=x, dz=dz, mr=mr, want=(dg, db), dx=torch.empty_like(x), dg=torch.empty(C, device="cuda"), db=torch.empty(C, device="cuda"),
                         stream=torch.cuda.Stream()))

    def call(s):
        hip_ops.layernorm_bwd(s["dz"], s["x"], s["mr"], None, s["dx"], s["dg"], s["db"], accumulate=False)
    torch.cuda.synchronize()
    for _ in range(5):
        for s in sets:
            s["dg"].zero_()
        torch.cuda.synchronize()
        for s in sets:
            with torch.cuda.stream(s["stream"]):
                call(s)
        torch.cuda.synchronize()
        assert all(torch.equal(s["dg"], s["want"][0]) and torch.equal(s["db"], s["want"][1]) for s in sets)
    for s in sets:
        s["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(s["graph"]):
            call(s)
    for _ in range(4):
        for s in sets:
            s["dg"].zero_()
            s["db"].fill_(float("nan"))
        torch.cuda.synchronize()
        for s in sets:
            with torch.cuda.stream(s["stream"]):
                s["graph"].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(s["dg"], s["want"][0]) and torch.equal(s["db"], s["want"][1]) for s in sets)


def test_backward_against_differences(hip_ops):
    """The kernels' gradients against central differences of the 64-bit forward pass (difference error ~ h^2, kernels' ~ 1e-6)."""
    P, C = 12, 150
    gen = torch.Generator(device="cuda").manual_seed(8)
    x, gamma, beta, dz = (torch.randn(*s, generator=gen, device="cuda") for s in ((P, C), (C,), (C,), (P, C)))
    mr, dx, dg, db = torch.empty(P, 2, device="cuda"), torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(beta)
    hip_ops.layernorm_fwd(x, gamma, beta, EPS, torch.empty_like(x), mr)
    hip_ops.layernorm_bwd(dz, x, mr, gamma, dx, dg, db, accumulate=False)

    def loss(x, gamma, beta):
        d = x - x.mean(1, keepdim=True)
        return float(((d / torch.sqrt((d * d).mean(1, keepdim=True) + EPS) * gamma + beta) * dz.double()).sum())
    at, h = [x.double(), gamma.double(), beta.double()], 1e-4
    for which, grad in enumerate((dx, dg, db)):
        way = torch.randn(grad.shape, generator=gen, device="cuda").double()
        up, down = list(at), list(at)
        up[which], down[which] = at[which] + h * way, at[which] - h * way
        slope = (loss(*up) - loss(*down)) / (2 * h)
        assert abs(slope - float((grad.double() * way).sum())) < 1e-5 * float((grad.double() * way).abs().sum())
