"""What an AdamW batch refuses of the memory that its calls are given beside the list: a norm, a step count or scratch inside the list's own
tensors would be written while those are read, or read while those are written.  No GPU: the addresses are never read."""
import ctypes as C

import pytest

from downscaling.engine import native

BASE = 1 << 20


def batch(bits=32, shared=False):
    """Two tensors of 1000 and 300 elements at known places; `shared`: both read one gradient."""
    lib, h = native.load(), C.c_void_p()
    at = lambda k: BASE * k      # noqa: E731
    arr = (native.AdamWTensor * 2)(
        native.AdamWTensor(at(1), at(2), at(3), at(4), at(5), at(6), at(7), 1000, 0, 0, 1, 1.0),
        native.AdamWTensor(at(11), at(2) + 400 if shared else at(12), at(13), at(14), at(15), at(16), 0, 300, 0, 0, 0, 0.0))
    assert lib.wdg_adamw_create(C.byref(h), arr, 2, bits) == 0
    return lib, h


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("shared", [False, True])
def test_step_refuses_memory_of_the_list(bits, shared):
    lib, h = batch(bits, shared)
    free, size = 50 * BASE, int(lib.wdg_adamw_scratch_bytes())

    def step(norm=free, step_dev=0, scratch=2 * free):
        a = native.AdamWArgs(1e-3, .9, .999, 1e-8, .01, 1.0, 1.0, 1, step_dev, norm)
        return lib.wdg_adamw_step(h, C.byref(a), scratch, size, 0), lib.wdg_last_error()
    inside = [BASE, BASE + 3996, 2 * BASE + 400, 2 * BASE + 3996, 3 * BASE, 4 * BASE + 996, 7 * BASE + 1996, 11 * BASE + 1196, 14 * BASE, 14 * BASE + 296]
    if not shared:
        inside += [12 * BASE, 12 * BASE + 1196]
    if bits == 8:
        inside += [5 * BASE, 6 * BASE + 12, 15 * BASE + 4, 3 * BASE + 1020, 14 * BASE + 508]
    for p in inside:
        rc, why = step(norm=p)
        assert rc == -1 and b"norm" in why and b"overlap" in why, hex(p)
        rc, why = step(step_dev=p & ~7)
        assert rc == -1 and b"step count" in why, hex(p)
        rc, why = step(scratch=p & ~7)
        assert rc == -1 and b"scratch" in why, hex(p)
        assert lib.wdg_adamw_grad_norm(h, 1.0, p, 2 * free, size, 0) == -1 and b"overlap" in lib.wdg_last_error()
    rc, why = step(scratch=2 * BASE - size + 8)                    # reaches into the first gradient
    assert rc == -1 and b"scratch" in why
    rc, why = step(norm=2 * free + 8)                              # the norm inside the scratch
    assert rc == -1 and b"overlap" in why
    # beside the tensors nothing is wrong but that the table is not there yet
    for p in (BASE - 4, BASE + 4000, 2 * BASE + 4000, 11 * BASE + 1200, 7 * BASE + 2000, 8, free):
        rc, why = step(norm=p)
        assert rc == -1 and b"bind" in why, hex(p)
    assert b"bind" in step(step_dev=BASE + 4000)[1] and b"bind" in step(scratch=2 * BASE - size)[1]
    assert lib.wdg_adamw_destroy(h) == 0
