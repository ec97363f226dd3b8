"""Moments of an AdamW batch read out into memory that they share with each other or with the states are refused: one of the two would be
lost, or the state.  No GPU: the addresses of the C entry's tests are never read."""
import pytest
import torch

from downscaling.engine import native

BASE = 1 << 20


def test_moments_refuse_shared_memory():
    lib, free = native.load(), 50 * BASE

    def moments(mo, vo, kind=0):
        return lib.wdg_adamw_moments(BASE, 2 * BASE, 3 * BASE, 4 * BASE, 4, mo, vo, kind, 0), lib.wdg_last_error()
    for mo, vo in ((free, free), (free, free + 4092), (free + 4, free), (BASE, 0), (0, BASE + 1020), (2 * BASE + 12, 0), (0, 3 * BASE), (4 * BASE - 4092, free), (free, 4 * BASE)):
        rc, why = moments(mo, vo)
        assert rc == -1 and b"overlap" in why, (hex(mo), hex(vo))
    rc, why = moments(free, free + 2046, 1)
    assert rc == -1 and b"overlap" in why


def test_moments_of_32_bits_refuse_shared_memory():
    from downscaling.engine.hipops import HipOps, _AdamWBatch
    o = object.__new__(HipOps)
    o.device, o.lib = torch.device("cpu"), native.load()
    b = object.__new__(_AdamWBatch)
    b.ops, b.state_bits, b.total, b.handle = o, 32, 256, None
    b.m, b.v = torch.ones(256), torch.full((256,), 2.0)
    b.state = (b.m, b.v)
    out, wide = torch.zeros(256), torch.zeros(300)
    for bad in ((out, out), (wide[:256], wide[10:266]), (b.v, None), (None, b.m)):
        with pytest.raises(ValueError, match="overlap"):
            b.moments(*bad)
    assert (b.m == 1).all() and (b.v == 2).all()
    b.moments(out, wide[:256])
    assert (out == 1).all() and (wide[:256] == 2).all()
    b.moments(b.m, b.v)                                            # each its own: nothing to do
    assert (b.m == 1).all() and (b.v == 2).all()
