"""layernorm_fwd / layernorm_bwd at the widths between the powers of two that one wave holds, where each width class takes kernels of its own
(fp32 up to 256, 512 and 1024 columns, 16-bit types up to 512 and 1024, whole rows or a last vector that reaches back), for few rows
(one backward launch) and for many (partial sums).  Tolerances: those of test_layernorm_gpu.py."""
import pytest
import torch

from tests.test_layernorm_gpu import BF16, EPS, F16, F32, backward_close, forward_close, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("C", [257, 264, 300, 511, 512, 513, 520, 700, 1000, 1016, 1023, 1024, 1025])
@pytest.mark.parametrize("P", [1, 37, 530, 2100])
def test_widths_of_one_wave(P, C, dtype, hip_ops):
    gen = torch.Generator(device="cuda").manual_seed(P * 31 + C)
    for pad, shift in ((0, 0), (5, 1)):
        print(P, C, dtype, pad, shift, flush=True)
        x, _ = rows(gen, P, C, dtype, pad, shift, 1.5, 0.5)
        dz, _ = rows(gen, P, C, dtype, pad, shift)
        z, zb = rows(gen, P, C, dtype, pad, shift)
        dx, db_ = rows(gen, P, C, dtype, pad, shift)
        gamma, beta = 1 + 0.3 * torch.randn(C, generator=gen, device="cuda"), torch.randn(C, generator=gen, device="cuda")
        mr = torch.empty(P, 2, device="cuda")
        hip_ops.layernorm_fwd(x, gamma, beta, EPS, z, mr)
        forward_close(x, gamma, beta, z, mr, (P, C))
        dg, db = torch.full((C,), 2.0, device="cuda"), torch.full((C,), -1.0, device="cuda")
        hip_ops.layernorm_bwd(dz, x, mr, gamma, dx, dg, db)
        backward_close(dz, x, mr, gamma, dx, dg, db, (P, C), dg0=2.0, db0=-1.0)
        over = dz.clone()                                # dx over dz: always by partial sums
        g2, b2 = torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
        hip_ops.layernorm_bwd(over, x, mr, gamma, over, g2, b2, accumulate=False)
        backward_close(dz, x, mr, gamma, over, g2, b2, (P, C, "over dz"))
        for view, buf in ((z, zb), (dx, db_)):           # nothing beside the rows was written
            mask = torch.ones_like(buf, dtype=torch.bool)
            mask[shift:shift + P * (C + pad)].view(P, C + pad)[:, :C] = False
            assert (buf[mask] == 7).all()


@pytest.mark.parametrize("dtype,C", [(F32, 512), (F32, 1024), (BF16, 512), (BF16, 1024), (F16, 256), (BF16, 3000), (F32, 900)])
def test_large_tensors_of_these_widths(dtype, C, hip_ops):
    """Past the last-level cache: whole rows are streamed, others are not; workgroups walk over many rows."""
    P = (280 << 20) // (2 * C * (4 if dtype is F32 else 2)) + 3
    gen = torch.Generator(device="cuda").manual_seed(C)
    x, dz = ((torch.randn(P, C, generator=gen, device="cuda") + 0.5).to(dtype) for _ in range(2))
    gamma, beta = 1 + 0.3 * torch.randn(C, generator=gen, device="cuda"), torch.randn(C, generator=gen, device="cuda")
    z, dx, mr = torch.empty_like(x), torch.empty_like(x), torch.empty(P, 2, device="cuda")
    dg, db = torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
    hip_ops.layernorm_fwd(x, gamma, beta, EPS, z, mr)
    hip_ops.layernorm_bwd(dz, x, mr, gamma, dx, dg, db, accumulate=False)
    sums, mag = torch.zeros(2, C, dtype=torch.float64, device="cuda"), torch.zeros(C, dtype=torch.float64, device="cuda")
    for a in range(0, P, 1 + P // 4):                # the rows are checked in pieces: their 64-bit copies are large
        r = slice(a, a + 1 + P // 4)
        forward_close(x[r], gamma, beta, z[r], mr[r])
        backward_close(dz[r], x[r], mr[r], gamma, dx[r], None, None)
        g, xh = dz[r].double(), (x[r].double() - mr[r, :1].double()) * mr[r, 1:].double()
        sums += torch.stack([(g * xh).sum(0), g.sum(0)])
        mag += (g.abs() * (1 + xh.abs() + 0.5 * (x[r].double().abs() + mr[r, :1].double().abs()) * mr[r, 1:].double())).sum(0)
    # at least 512 workgroups' waves share the rows: P / 512 one after another at most, then at most 1024 partial sums in sets
    lim = (P // 512 + 1100) * 2.0 ** -24 * mag
    assert ((dg.double() - sums[0]).abs() <= lim).all() and ((db.double() - sums[1]).abs() <= lim).all()
