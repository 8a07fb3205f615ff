"""Arguments of edb200_rope_apply that go together: q and k, their outs, in the binding and in the library."""
import ctypes as C

import pytest
import torch


def test_k_needs_a_place(edb):
    r, a = edb.Rope([64]), torch.zeros(4, 2, 64)
    with pytest.raises(ValueError, match="k_out"):
        r.apply(None, a, a, a.clone())


def test_two_tensors_that_write_over_one_another(edb):
    """Both turned at once, in no order: an out that is the other's out or in would hold whichever came last, or be turned
    twice.  In place is each tensor's own."""
    r = edb.Rope([64])
    f = edb.lib().edb200_rope_apply
    strides = dict(in_token=256, in_head=64, out_token=256, out_head=64, heads=4)
    q = dict(strides, in_=4096, out=8192)
    for k in (dict(in_=16384, out=8192), dict(in_=8192, out=16384), dict(in_=16384, out=4096), dict(in_=4096, out=8192)):
        a, b = edb.RopeTensor(**q), edb.RopeTensor(**{**strides, **k})
        assert f(r.handle, C.byref(a), C.byref(b), edb.TYPE_F16, 64, 4, None, 0, None) == 1
        assert b"the other's" in edb.lib().edb200_last_error()


@pytest.mark.gpu
def test_one_source_and_two_places(edb, cuda):
    """The same tensor may be read twice; q and k side by side in one buffer may be turned in place."""
    r = edb.Rope([64])
    x = torch.randn(5, 2, 64, device="cuda")
    want, a, b = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    r.apply(None, x, want)
    r.apply(None, x, a, x, b)
    both = torch.cat((x, x), 1)
    r.apply(None, both[:, :2], both[:, :2], both[:, 2:], both[:, 2:])
    assert torch.equal(a, want) and torch.equal(b, want) and torch.equal(both, torch.cat((want, want), 1))
