"""The 8-bit cache and the attention over it at the ends of the value range."""
import pytest
import torch

from serving_ref import RefCache

pytestmark = pytest.mark.gpu
E4, I8 = torch.float8_e4m3fn, torch.int8
BF16 = torch.bfloat16


def _dev_i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [E4, I8], ids=["e4m3", "int8"])
@pytest.mark.parametrize("T", [1, 3, 20])
@pytest.mark.parametrize("small,large", [(1e-30, 1e25), (1e-28, 1e38), (1e-20, 1e20), (1e-30, 1e15)])
def test_append_grid_grows_by_any_factor(T, small, large, dtype):
    """A block that holds tiny rows takes huge ones: on the new grid the older rows are what their codes round to there (nothing, mostly), by whatever
    power of two the grid grew -- factors below the smallest fp32 number among them."""
    from neko_amd import ops
    S, H, cap, hd, block, n0 = 2, 3, 64, 32, 32, 7
    g = torch.Generator().manual_seed(T)
    x = torch.randn(S, n0, 2, H, hd, generator=g).mul(small).to(BF16)
    y = torch.randn(S, T, 2, H, hd, generator=g).mul(large).to(BF16)
    cache = ops.KV8Cache(S, H, cap, hd, dtype=dtype, block=block)
    ref = RefCache(S, H, cap, hd, dtype, block)
    for rows, pos in ((x, 0), (y, n0)):
        d = rows.cuda()
        ops.kv8_append(cache, d[:, :, 0], d[:, :, 1], _dev_i([pos] * S))
        ref.append(rows[:, :, 0], rows[:, :, 1], [pos] * S, [rows.shape[1]] * S)
    k, v = ops.kv8_read(cache, _dev_i([n0 + T] * S), cap)
    rk, rv = ref.read([n0 + T] * S, cap)
    assert torch.equal(k.cpu().double(), rk) and torch.equal(v.cpu().double(), rv)
