"""Arguments past 32 bits: they mean what they say or are refused, never their low half."""
import pytest
import torch

from neko_amd import _lib, ops
from test_serving_refusals_cpu import DISTILL

BF16 = torch.bfloat16


def _wide(rows, cols, dtype=torch.float32):
    """A tensor of that shape without its memory (every row one and the same element)."""
    return torch.zeros(1, 1, dtype=dtype).expand(rows, cols)


@pytest.mark.parametrize("V", [(1 << 30) + 1, (1 << 31) + 8, (1 << 32) + 8])
def test_rows_too_long(V, monkeypatch):
    monkeypatch.setattr(ops, "_here", lambda t, name: 0)               # (the sizes are looked at before any memory is)
    with pytest.raises(AssertionError, match="logits a row"):
        ops.verify_draft(_wide(2, V)[None], torch.zeros(1, 1, dtype=torch.int64), temperature=0.0)
    with pytest.raises(AssertionError, match="columns"):
        ops.distill_topk(_Shape(1, V), V, V, None, None, torch.ones(1), target=torch.zeros(1, dtype=torch.int64), hard=1.0, loss_row=torch.zeros(1))
    if V < 1 << 31:
        assert _lib.load().neko_distill_topk(*{**DISTILL, "V": V, "Vpad": (V + 7) // 8 * 8, "ldz": V + 64, "ldd": V + 64}.values()) in (-1, -2)


class _Shape:
    """Looks like a float32 tensor of contiguous rows."""
    dtype = torch.float32

    def __init__(self, *shape):
        self.shape = shape

    def dim(self):
        return len(self.shape)

    def stride(self, i):
        return (self.shape[1], 1)[i]


@pytest.mark.gpu
def test_window_and_sinks_of_any_size():
    S, H, hd, cap, T = 1, 2, 64, 128, 3
    g = torch.Generator().manual_seed(0)
    x = torch.randn(S, cap, 3, H, hd, generator=g).to(BF16).cuda()
    cache = ops.KV8Cache(S, H, cap, hd)
    ops.kv8_append(cache, x[:, :, 1], x[:, :, 2], torch.zeros(1, dtype=torch.int32, device="cuda"))
    pos = torch.full((1,), 100, dtype=torch.int32, device="cuda")
    q = x[:, :T, 0]
    every = ops.attn_kv8(cache, q, pos)
    near = ops.attn_kv8(cache, q, pos, window=5)
    assert not torch.equal(every, near)
    for window in (103, cap, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 40 + 1):
        assert torch.equal(ops.attn_kv8(cache, q, pos, window=window), every), window
    for sinks in (103, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 33 + 1):
        assert float((ops.attn_kv8(cache, q, pos, window=5, sinks=sinks).float() - every.float()).abs().max()) <= 2.0 ** -7 * float(every.float().abs().max()), sinks
    for max_len in (2 ** 31, 2 ** 32 + 1, 2 ** 32 + 64):
        assert torch.equal(ops.attn_kv8(cache, q, pos, max_len=max_len), every)
