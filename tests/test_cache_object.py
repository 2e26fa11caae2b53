"""A cache object keeps the tensors and sizes that it was made with (no GPU needed)."""
import pytest
import torch

from neko_amd import ops


@pytest.mark.parametrize("name", ["k", "v", "k_scale", "v_scale", "nseq", "heads", "cap", "hd", "block", "dtype", "other"])
def test_attributes_cannot_be_replaced(name):
    """The entry points are handed addresses and sizes that were taken when the cache was made: another tensor in an attribute would not be the one they
    use, and the old one's memory would be free for others."""
    c = ops.KV8Cache(2, 3, 128, 64, dtype=torch.int8, device="cpu")
    before = getattr(c, name, None)
    with pytest.raises(AttributeError):
        setattr(c, name, torch.zeros_like(before) if torch.is_tensor(before) else before)
    assert getattr(c, name, None) is before
    c.k.fill_(3)                                   # what the tensors hold may change
    assert int(c.k.sum()) == 3 * c.k.numel() and c._args[0] == c.k.data_ptr()


def test_copies_use_their_own_tensors():
    import copy
    c = ops.KV8Cache(2, 3, 128, 64, dtype=torch.int8, block=64, device="cpu")
    c.k.fill_(5)
    d = copy.deepcopy(c)
    assert d._args[:4] == (d.k.data_ptr(), d.v.data_ptr(), d.k_scale.data_ptr(), d.v_scale.data_ptr()) and d._args[4:] == c._args[4:]
    assert d._args[0] != c._args[0] and torch.equal(c.k, d.k) and d.block == 64
    assert copy.copy(c)._args == c._args
